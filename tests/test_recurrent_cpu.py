"""Refusals of the entry points of recurrent layers over state slots and of the log probabilities.  Arguments are
checked before a device is touched, so these run without a GPU: a refused call answers INVALID and names the fault, a
sound one gets as far as the missing device."""
import math

import pytest

torch = pytest.importorskip("torch")

from krikil_rs_b200 import _lib, kernels as K  # noqa: E402
from krikil_rs_b200._lib import lib  # noqa: E402

P = 4096  # a placeholder address, aligned to 16 bytes: never read
FAR = 1 << 40

SLOT = dict(state=P, stride=4096, num_slots=8, slots=P, init=P)
CONV = dict(x=P, x_st=64, weight=P, bias=P, out=FAR, o_st=64, type=0, **SLOT, cu=P, T=5, S=2, C=64, W=4, silu=1,
            stream=None)
CONV_STEP = dict(x=P, x_st=64, weight=P, bias=P, out=FAR, o_st=64, type=0, **SLOT, B=2, C=64, W=4, silu=1,
                 stream=None)
SCAN = dict(x=P, x_st=64, dt=P, dt_st=64, z=P, z_st=64, b=P, b_st=16, b_sg=16, c=P, c_st=16, c_sg=16, out=FAR, o_st=64,
            type=0, a=P, d=P, dt_bias=P, **SLOT, cu=P, T=5, S=2, D=64, N=16, G=1, max_len=0, work=None, work_floats=0,
            stream=None)
STEP = dict(x=P, x_st=64, dt=P, dt_st=64, z=P, z_st=64, b=P, b_st=16, b_sg=16, c=P, c_st=16, c_sg=16, out=FAR, o_st=64,
            type=0, a=P, d=P, dt_bias=P, **SLOT, B=2, D=64, N=16, G=1, stream=None)
LOGPROBS = dict(logits=P, ld=100, type=0, R=3, V=100, tokens=P, K=1, lp=P, entropy=P, top=5, ids=P, best=P, stream=None)


def refused(fn, base, what, value, word):
    args = dict(base)
    args.update(zip(what, value) if isinstance(what, tuple) else [(what, value)])
    assert list(args) == list(base)
    assert fn(*args.values()) == _lib.INVALID, (what, value)
    assert word in lib.krk_last_error().decode(), lib.krk_last_error()


POOL = [("num_slots", 0, "num_slots"), ("num_slots", -1, "num_slots"), ("stride", 100, "stride"), ("state", P + 2, "state")]
BARE = [("state", None, "need a state"), (("state", "slots", "init"), (None, None, None), "need a state")]
CONV_FAULTS = POOL + [("type", 3, "type"), ("type", -1, "type"), ("W", 1, "width"), ("W", 5, "width"), ("C", 0, "channels"),
                      ("C", 1 << 25, "channels"), ("weight", None, "weight"), ("weight", P + 2, "aligned"),
                      ("bias", P + 2, "aligned"), ("x", None, "x and out"), ("out", None, "x and out"),
                      ("x", P + 2, "aligned"), ("out", P + 2, "aligned"), ("o_st", 63, "overlap"),
                      ("out", P, "overlap x"), ("out", P + 4 * 32, "overlap x"),
                      (("x_st", "o_st", "out"), (100, 100, P + 4 * 63), "overlap x"),
                      (("x_st", "o_st", "out"), (100, 100, P + 4 * 137), "overlap x")]


@pytest.mark.parametrize("what,value,word", CONV_FAULTS + BARE + [("cu", None, "null"), ("T", -1, "rows"), ("S", -1, "rows")])
def test_conv_refuses(what, value, word):
    refused(lib.krk_k_causal_conv, CONV, what, value, word)


@pytest.mark.parametrize("what,value,word", CONV_FAULTS + [("state", None, "null"), ("B", -1, "rows")])
def test_conv_step_refuses(what, value, word):
    refused(lib.krk_k_causal_conv_step, CONV_STEP, what, value, word)


SCAN_FAULTS = POOL + [("type", 3, "type"), ("N", 0, "N must"), ("N", 257, "N must"), ("D", 0, "D must"), ("G", 0, "D must"),
                      ("G", 3, "D must"), ("D", 1 << 25, "D must"), ("a", None, "a must"), ("a", P + 1, "a must"),
                      ("d", P + 1, "aligned"), ("dt_bias", P + 1, "aligned"), ("z", P + 1, "aligned"),
                      ("o_st", 63, "overlap")] + [(n, None, "must be set") for n in ("x", "dt", "b", "c", "out")] + [
                          (n, P + 2, "aligned") for n in ("x", "dt", "b", "c", "out")]


@pytest.mark.parametrize("what,value,word", SCAN_FAULTS + BARE + [
    ("cu", None, "null"), ("T", -1, "rows"), ("S", -1, "rows"), ("max_len", -1, "max_len"), ("T", 5000, "work must"),
    (("T", "work", "work_floats"), (5000, P, 1000), "work must"), (("T", "work", "work_floats"), (5000, P + 4, 1 << 30), "work must")])
def test_scan_refuses(what, value, word):
    refused(lib.krk_k_selective_scan, SCAN, what, value, word)


@pytest.mark.parametrize("what,value,word", SCAN_FAULTS + [("state", None, "null"), ("B", -1, "rows")])
def test_step_refuses(what, value, word):
    refused(lib.krk_k_selective_step, STEP, what, value, word)


@pytest.mark.parametrize("what,value,word", [
    ("type", 3, "type"), ("R", -1, "R and K"), ("K", -1, "R and K"), ("V", 0, "V 1"), ("V", (1 << 30) + 1, "V 1"), ("top", -1, "top"),
    ("top", 33, "top"), (("top", "V"), (5, 4), "top"), ("logits", None, "logits"), ("logits", P + 2, "aligned"),
    ("tokens", None, "null"), ("lp", None, "null"), ("ids", None, "null"), ("best", None, "null")])
def test_logprobs_refuses(what, value, word):
    refused(lib.krk_k_token_logprobs, LOGPROBS, what, value, word)


def test_calls_of_nothing_are_fine():
    for fn, base, none in ((lib.krk_k_causal_conv, CONV, ("S", 0)), (lib.krk_k_causal_conv_step, CONV_STEP, ("B", 0)),
                           (lib.krk_k_selective_scan, SCAN, ("S", 0)), (lib.krk_k_selective_step, STEP, ("B", 0)),
                           (lib.krk_k_token_logprobs, LOGPROBS, ("R", 0))):
        assert fn(*dict(base, **dict([none])).values()) == _lib.OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="would read the placeholder addresses")
def test_sound_calls_reach_the_device():
    columns = dict(CONV, x_st=128, o_st=128, out=P + 4 * 64)  # two halves of one matrix
    for fn, args in ((lib.krk_k_causal_conv, CONV), (lib.krk_k_causal_conv, columns),
                     (lib.krk_k_causal_conv_step, CONV_STEP), (lib.krk_k_selective_scan, SCAN),
                     (lib.krk_k_selective_scan, dict(SCAN, z=None, d=None, dt_bias=None, state=None, stride=0, num_slots=0,
                                                     slots=None, init=None)),
                     (lib.krk_k_selective_step, STEP), (lib.krk_k_token_logprobs, LOGPROBS),
                     (lib.krk_k_token_logprobs, dict(LOGPROBS, entropy=None, top=0, ids=None, best=None))):
        assert fn(*args.values()) == _lib.CUDA, lib.krk_last_error()


def test_scan_scratch():
    """None for short requests; else room for every piece's states and step sums, whatever the requests' lengths."""
    floats = lib.krk_selective_scan_work_floats
    assert floats(320, 64, 16, 1, 0) == 0 and floats(321, 64, 16, 1, 0) > 0
    assert floats(100000, 64, 16, 1, 800) == 0 and floats(100000, 64, 16, 1, 100000) == floats(100000, 64, 16, 1, 0)
    assert floats(16384, 5120, 16, 1, 5000) == 0  # as many channels as the device has room for: a request is not split
    for args in ((0, 64, 16, 1, 0), (321, 64, 257, 1, 0), (321, 64, 16, 3, 0), (321, 64, 16, 1, -1), (321, 0, 16, 1, 0)):
        assert floats(*args) == 0


def test_wrappers_want_cuda_tensors():
    x, w, cu = torch.zeros(3, 8), torch.zeros(8, 4), torch.zeros(2, dtype=torch.int32)
    a, bc, state = torch.zeros(8, 4), torch.zeros(3, 4), torch.zeros(3, 8, 4)
    for call in (lambda: K.causal_conv(x, w, cu), lambda: K.causal_conv_step(x, w, torch.zeros(3, 3, 8)),
                 lambda: K.selective_scan(x, x, a, bc, bc, cu), lambda: K.selective_step(x, x, a, bc, bc, state),
                 lambda: K.token_logprobs(x)):
        with pytest.raises(ValueError, match="CUDA|cuda"):
            call()


# tensors far from one another, rows as long as they need be
APART = dict(x=FAR, dt=2 * FAR, z=3 * FAR, b=4 * FAR, c=5 * FAR, out=6 * FAR)
# out over others: a row or a part of one further, with other strides, over B or C or the second of their groups
OVER = [dict(out=FAR + 4 * 64), dict(out=FAR + 4 * 63), dict(out=FAR - 4), dict(x_st=65, out=FAR), dict(out=2 * FAR, dt_st=0),
        dict(out=3 * FAR + 4 * 63), dict(out=4 * FAR), dict(out=4 * FAR - 4 * 63), dict(out=5 * FAR + 4 * 15, c_st=64),
        dict(G=2, b_st=200, b_sg=100, o_st=200, out=4 * FAR + 4 * 90), dict(G=2, b_st=200, b_sg=100, o_st=200, out=4 * FAR + 4 * 37),
        dict(G=2, b_st=16, b_sg=-1000, out=4 * FAR - 4 * 1000), dict(z=FAR + 4 * 32, z_st=100, x_st=100, o_st=100, out=FAR)]
# and beside them: in place, columns of one matrix, the gap between two groups, other rows
BESIDE = [dict(out=FAR), dict(out=2 * FAR), dict(out=3 * FAR), dict(b=FAR + 4 * 64, c=FAR + 4 * 80, x_st=96, b_st=96, c_st=96, o_st=96, out=FAR),
          dict(G=2, b_st=200, b_sg=100, o_st=200, out=4 * FAR + 4 * 16), dict(G=2, b_st=200, b_sg=100, o_st=200, out=4 * FAR + 4 * 36),
          dict(G=2, b_st=200, b_sg=100, o_st=200, out=4 * FAR + 4 * 216),
          dict(x_st=128, o_st=128, out=FAR + 4 * 64), dict(z=None, z_st=0, out=3 * FAR), dict(x=FAR, dt=FAR, z=FAR, out=FAR)]


@pytest.mark.parametrize("name,rows", [("scan", "T"), ("step", "B")])
@pytest.mark.parametrize("how", OVER)
def test_scan_and_step_refuse_an_out_over_what_others_read(name, rows, how):
    fn, base = (lib.krk_k_selective_scan, SCAN) if name == "scan" else (lib.krk_k_selective_step, STEP)
    args = dict(base, **{rows: 5}, **APART)
    args.update(how)
    assert fn(*args.values()) == _lib.INVALID, lib.krk_last_error()
    assert "overlap" in lib.krk_last_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="would read the placeholder addresses")
@pytest.mark.parametrize("name,rows", [("scan", "T"), ("step", "B")])
@pytest.mark.parametrize("how", BESIDE)
def test_scan_and_step_take_an_out_in_place_or_beside(name, rows, how):
    fn, base = (lib.krk_k_selective_scan, SCAN) if name == "scan" else (lib.krk_k_selective_step, STEP)
    args = dict(base, **{rows: 5}, **APART)
    args.update(how)
    assert fn(*args.values()) == _lib.CUDA, lib.krk_last_error()
    one = dict(args, **{rows: 1}, x_st=7, dt_st=9, z_st=11)  # the stride of a single row does not matter
    assert fn(*one.values()) == _lib.CUDA, lib.krk_last_error()


class Tensor:
    """What the wrappers look at of a CUDA tensor, of any size."""

    def __init__(self, *shape, dtype=torch.float32, zeros=()):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cuda", 0)
        self.steps = [0 if i in zeros else math.prod(shape[i + 1:]) for i in range(len(shape))]

    def stride(self):
        return tuple(self.steps)

    def numel(self):
        return math.prod(self.shape)

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def data_ptr(self):
        return P

    def new_empty(self, *shape):
        return Tensor(*(shape[0] if isinstance(shape[0], (tuple, torch.Size)) else shape), dtype=self.dtype)


LONG = (1 << 32) + 2  # two of the low 32 bits


@pytest.mark.parametrize("what", ["conv rows", "conv channels", "conv width", "conv requests", "conv slots", "conv step rows", "scan rows",
                                  "scan requests", "scan slots", "scan states", "scan groups", "step rows", "step slots",
                                  "logprobs rows", "logprobs vocab", "logprobs asked", "scratch rows"])
def test_wrappers_refuse_sizes_past_31_bits(what, monkeypatch):
    """A size that the library's 32-bit arguments do not hold is not cut to its low bits."""

    class Lib:
        def __getattr__(self, name):
            if name == "krk_selective_scan_work_floats":
                return lambda *sizes: 0
            return lambda *args: pytest.fail(f"{name} was called")

    monkeypatch.setattr(K, "lib", Lib())
    monkeypatch.setattr(K, "_current_device", lambda: 0)
    monkeypatch.setattr(K, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(K.torch, "empty", lambda *shape, device=None, dtype=None: Tensor(*shape, dtype=dtype))
    n = {k: LONG if k == what.split()[-1] else v for k, v in dict(
        rows=2, channels=2, width=4, requests=1, slots=2, states=4, groups=1, vocab=9, asked=1).items()}
    ints = lambda *shape: Tensor(*shape, dtype=torch.int32)  # noqa: E731
    rows, ch = n["rows"], 2 * n["groups"] if n["groups"] > 1 else n["channels"]
    x, cu = Tensor(rows, ch), ints(n["requests"] + 1)
    bc, a = Tensor(rows, n["groups"], n["states"]), Tensor(ch, n["states"])
    conv = dict(weight=Tensor(ch, n["width"]), state=Tensor(n["slots"], n["width"] - 1, ch))
    state = Tensor(n["slots"], ch, n["states"])
    calls = {"conv": lambda: K.causal_conv(x, cu=cu, slots=ints(n["requests"]), **conv),
             "conv step": lambda: K.causal_conv_step(x, slots=ints(rows), **conv),
             "scan": lambda: K.selective_scan(x, x, a, bc, bc, cu, state=state, slots=ints(n["requests"])),
             "step": lambda: K.selective_step(x, x, a, bc, bc, state, slots=ints(rows)),
             "logprobs": lambda: K.token_logprobs(Tensor(rows, n["vocab"]), ints(rows, n["asked"])),
             "scratch": lambda: K.selective_scan_work_floats(rows, 2, 4)}
    with pytest.raises(ValueError, match="2\\^31|31 bits"):
        calls[what.rsplit(" ", 1)[0]]()
