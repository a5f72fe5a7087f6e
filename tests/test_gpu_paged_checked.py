"""The paged cache's operators in the checked build (KRIKIL_CHECKED=1): clean calls set no bit of the device status
word; a length outside the table, a page outside the pool and a slot past it are reported, and skipped as in every
build.  In a child process, since a process loads one build of the library."""
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
from krikil_rs_b200._lib import lib, CHECKED, CHECK_POSITION, CHECK_TABLE, OK

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
    for page in (4, 16):
        n = 3 * page + 1
        kc, vc = (torch.randn(12, page, 2, 64, device=dev).to(dtype) for _ in range(2))
        q = torch.randn(2, 4, 64, device=dev).to(dtype)
        table = i32([[0, 1, 2, 3], [4, 5, 6, -1]])
        lens = i32([n, 3 * page])
        out = K.attn_decode_paged(q, kc, vc, table, lens)
        K.attn_decode_paged(q, kc, vc, table, lens, window=page + 1)
        assert status() == 0, (dtype, page)
        gone = i32([[-1, -1, 2, 3], [-1, 5, 6, -1]])  # pages before the window may be gone
        K.attn_decode_paged(q, kc, vc, gone, lens, window=page + 1)
        assert status() == 0, (dtype, page)
        K.attn_decode_paged(q, kc, vc, table, i32([n, 3 * page + 1]))
        assert status() == CHECK_TABLE, (dtype, page)
        got = K.attn_decode_paged(q, kc, vc, table, i32([n, -1]))
        assert status() == CHECK_POSITION and torch.equal(got[0], out[0]) and (got[1] == 0).all()
        K.attn_decode_paged(q, kc, vc, table, i32([4 * page + 1, 0]))
        assert status() == CHECK_POSITION
        kv = torch.randn(2, 2, 64, device=dev).to(dtype)
        K.rope_kv_append_paged(q, kv, kv, kc, vc, i32([-1, 12 * page - 1]), i32([0, 1]))
        assert status() == 0
        K.rope_kv_append_paged(q, kv, kv, kc, vc, i32([0, 12 * page]), i32([0, 1]))
        assert status() == CHECK_TABLE
print("checked ok")
'''


def test_checked_build_reports_bad_lengths_pages_and_slots():
    env = dict(os.environ, KRIKIL_CHECKED="1", PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "checked ok" in r.stdout, r.stdout + r.stderr


PLAN_CHILD = r'''
import ctypes as C
import torch
from krikil_rs_b200 import kernels as K
from krikil_rs_b200._lib import lib, CHECK_TABLE, OK

assert lib.krk_checked_build() == 1
dev = torch.device("cuda:0")

def status():
    torch.cuda.synchronize()
    b = C.c_uint32()
    assert lib.krk_check_status(C.byref(b), 1) == OK
    return b.value

def i32(v):
    return torch.tensor(v, device=dev, dtype=torch.int32)

for new in (3, 5000):  # in one block, and in two kernels
    pages = 2 * -(-new // 4) + 2
    table = torch.full((2, pages), 7, device=dev, dtype=torch.int32)
    free = torch.arange(pages, device=dev, dtype=torch.int32)
    lens, count = i32([0, 0]), i32([pages])
    out = K.kv_page_plan(i32([new, new]), lens, table, free, count, 4, 2 * new)
    assert out[5].item() == 0 and status() == 0
    free[pages - 1] = 2 ** 30 + 1  # * 4 is 4 in 32 bits
    out = K.kv_page_plan(i32([new, new]), lens, table, free, count, 4, 2 * new)
    assert out[5].item() == 0 and status() == CHECK_TABLE and (out[4][:3] == -1).all()
    held = i32([8, 4])
    table[:, :2] = i32([[-1, 3], [4, -1]])  # a page given back: skipped, and nothing amiss
    out = K.kv_page_release(torch.tensor([True, True], device=dev), held, table, free, i32([0]), 4)
    assert out[2].item() == 0 and out[1].item() == 2 and free[:2].tolist() == [3, 4] and status() == 0
print("checked ok")
'''


def test_checked_build_reports_planned_tokens_on_no_page():
    env = dict(os.environ, KRIKIL_CHECKED="1", PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", PLAN_CHILD], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "checked ok" in r.stdout, r.stdout + r.stderr
