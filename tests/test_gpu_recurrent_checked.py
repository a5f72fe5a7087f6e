"""Recurrent layers over state slots and log probabilities in the checked build (KRIKIL_CHECKED=1): clean calls set no bit
of the device status word; slots past the pool, offsets outside the rows and tokens outside the vocabulary are reported,
and left alone as in every build.  In a child process, since a process loads one build of the library."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import ctypes as C
import torch
from krikil_rs_b200 import kernels as K
from krikil_rs_b200._lib import lib, CHECKED, CHECK_POSITION, CHECK_TABLE, CHECK_TOKEN, OK

assert CHECKED and lib.krk_checked_build() == 1
dev = torch.device("cuda:0")

def status():
    torch.cuda.synchronize()
    b = C.c_uint32()
    assert lib.krk_check_status(C.byref(b), 1) == OK
    return b.value

def i32(v):
    return torch.tensor(v, device=dev, dtype=torch.int32)

for dtype in (torch.float32, torch.float16, torch.bfloat16):
    x, bc = torch.randn(9, 40, device=dev).to(dtype), torch.randn(9, 16, device=dev).to(dtype)
    w, a = torch.randn(40, 4, device=dev), -torch.rand(40, 16, device=dev)
    cs, hs = torch.zeros(4, 3, 40, device=dev, dtype=dtype), torch.zeros(4, 40, 16, device=dev)
    calls = (lambda cu, s, i: K.causal_conv(x, w, i32(cu), state=cs, slots=i32(s), init=i32(i)),
             lambda cu, s, i: K.selective_scan(x, x, a, bc, bc, i32(cu), state=hs, slots=i32(s), init=i32(i)))
    for call in calls:
        call([0, 4, 9], [3, -1], [-1, 2])
        assert status() == 0
        call([0, 4, 9], [3, 4], [-1, 2])
        assert status() == CHECK_TABLE
        call([0, 4, 9], [3, 2], [-1, 4])
        assert status() == CHECK_TABLE
        for cu in ([-1, 4, 9], [0, 4, 10], [0, 5, 4]):
            call(cu, [3, 2], [-1, -1])
            assert status() == CHECK_POSITION, cu
    for call in (lambda s: K.causal_conv_step(x[:2], w, cs, i32(s)),
                 lambda s: K.selective_step(x[:2], x[:2], a, bc[:2], bc[:2], hs, i32(s))):
        call([3, -1])
        assert status() == 0
        call([3, 4])
        assert status() == CHECK_TABLE
    K.token_logprobs(x, i32([39] * 8 + [-1]), 3)
    assert status() == 0
    K.token_logprobs(x, i32([39] * 8 + [40]), 3)
    assert status() == CHECK_TOKEN
print("checked ok")
'''


def test_checked_build_reports_what_is_not_there():
    env = dict(os.environ, KRIKIL_CHECKED="1", PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, env=env, cwd=ROOT, timeout=600)
    assert r.returncode == 0 and "checked ok" in r.stdout, r.stdout + r.stderr
