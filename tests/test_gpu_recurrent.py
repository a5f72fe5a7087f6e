"""Recurrent layers over state slots (short causal convolution, selective state space scan, for packed requests and
single tokens) and token log probabilities against plain forms in 64 bits.

Tolerances follow each operation's rounding: half a step of 2^-24 for a float32 operation, 2^-22 for the exponential and
the reciprocal of the exponential unit, 2^-22 for expf and log1pf, and half a step of the result's type, carried through
the formulas by the oracle itself, which returns a bound beside each value."""
import ctypes as C
import itertools
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from krikil_rs_b200 import _lib, kernels as K, launch_count  # noqa: E402

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of float32
EX = 2.0 ** -22  # the exponential unit's, expf's and log1pf's error
F64 = torch.float64


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def close(got, want, bound, name=""):
    """|got - want| within the bound and half a step of got's type."""
    got, eps, tiny = got.to(F64), torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal
    same = (got == want) | (got.isnan() & want.isnan())  # infinities and NaN have to be where they are
    room = bound * (1 + eps) + eps * want.abs() + tiny
    bad = ~(same | ((got - want).abs() <= room))
    assert not bad.any(), (name, int(bad.sum()), got[bad][:5], want[bad][:5], room[bad][:5])


def silu64(y, e):
    """y * sigmoid(y) with the bound of what an error e of y and the exponential unit make of it."""
    s = torch.sigmoid(y)
    return y * s, 1.1 * e + (y * s).abs() * (2 * EX + 4 * U + 2 * U * y.abs())


def spans(cu, rows):
    cut = [min(max(v, 0), rows) for v in cu]
    return [(i, max(i, j)) for i, j in zip(cut[:-1], cut[1:])]


class Pool:
    """Slots as the calls take them: the oracle's books beside them."""

    def __init__(self, g, shape, dtype, requests, init="mixed", pad=()):
        n = 2 * requests + 3
        wide = normal(g, n, shape[0] * shape[1] + 8, dtype=dtype)
        self.state = wide[:, :shape[0] * shape[1]].unflatten(1, shape)  # slots apart by more than a state
        self.all, self.before = wide, wide.clone()
        order = torch.randperm(n, generator=g, device=DEV).tolist()
        self.slots = [-1 if s in pad else order[s] for s in range(requests)]
        self.init = {"same": None, "none": [-1] * requests,
                     "mixed": [[-1, order[s], order[requests + s], order[requests]][s % 4] for s in range(requests)]}[init]

    def args(self):
        return dict(state=self.state, slots=i32(self.slots), init=None if self.init is None else i32(self.init))

    def begun(self, s):
        i = self.slots[s] if self.init is None else self.init[s]
        old = self.before[:, :self.state.shape[1] * self.state.shape[2]].unflatten(1, self.state.shape[1:])
        return old[i].to(F64) if i >= 0 else torch.zeros_like(old[0], dtype=F64)

    def check(self, kept, bound=None):
        """kept: slot -> state; every other word is as it was."""
        want = self.before.to(F64)
        room = torch.zeros_like(want)
        size = self.state.shape[1] * self.state.shape[2]
        for slot, value in kept.items():
            want[slot, :size] = value.flatten()
            if bound is not None:
                room[slot, :size] = bound[slot].flatten()
        if bound is None:
            assert torch.equal(self.all.to(F64), want)
        else:
            untouched = torch.ones_like(want, dtype=torch.bool)
            for slot in kept:
                untouched[slot, :size] = False
            assert torch.equal(self.all[untouched], self.before[untouched])
            close(self.all, want, room, "state")


# ------------------------------------------------------------------ the convolution
def conv64(x, w, bias, old, silu):
    """One request: its outputs with their bounds, and the rows that it ends with."""
    width = w.shape[1]
    rows = torch.cat([old, x.to(F64)])
    n = x.shape[0]
    w = w.to(F64)
    y, size = bias.to(F64).expand(n, -1).clone(), bias.to(F64).abs().expand(n, -1).clone()
    for j in range(width):
        y += w[:, j] * rows[j:j + n]
        size += (w[:, j] * rows[j:j + n]).abs()
    e = (width + 1) * U * size
    return (*(silu64(y, e) if silu else (y, e)), rows[n:])


def run_conv(act, width, ch, lens, seed, init="mixed", pad=(), tail=0, silu=True, bias=True, strided=0, step=False):
    g, dtype = gen(seed), TYPES[act]
    rows = sum(lens) + tail
    x = normal(g, rows, ch + strided, dtype=dtype)[:, :ch]
    w, b = normal(g, ch, width), normal(g, ch) if bias else None
    pool = Pool(g, (width - 1, ch), dtype, len(lens), init, pad)
    out = torch.full((rows, ch + 2 * strided), 7.0, device=DEV, dtype=dtype)
    view = out[:, strided:strided + ch]
    cu = list(itertools.accumulate(lens, initial=0))
    if step:
        got = K.causal_conv_step(x, w, bias=b, silu=silu, out=view, **pool.args())
    else:
        got = K.causal_conv(x, w, i32(cu), bias=b, silu=silu, out=view, **pool.args())
    assert got is view
    want, bound, kept = torch.full((rows, ch), 7.0, device=DEV, dtype=F64), torch.zeros(rows, ch, device=DEV, dtype=F64), {}
    for s, (i, j) in enumerate(spans(cu, rows)):
        if pool.slots[s] >= 0:
            want[i:j], bound[i:j], kept[pool.slots[s]] = conv64(x[i:j], w, torch.zeros(ch, device=DEV) if b is None else b,
                                                                pool.begun(s), silu)
    close(view, want, bound, "out")
    assert (out[:, :strided] == 7).all() and (out[:, strided + ch:] == 7).all()
    pool.check(kept)


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("ch,strided", [(1, 0), (33, 3), (64, 8), (34, 2), (1472, 0), (520, 1)])
def test_conv_types_widths_and_channels(act, width, ch, strided):
    run_conv(act, width, ch, [5, 0, 1, 2, 17, 3, 40, 0], 3, strided=strided, tail=2)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [2] * 30, [1] * 67, [200], [7, 9, 8, 1, 0, 0, 23, 1, 1, 1, 8],
                                  [3] * 7 + [0] * 40 + [64, 1], [0] * 5 + [129]])
@pytest.mark.parametrize("init", ["same", "none", "mixed"])
def test_conv_lengths(act, lens, init):
    """Requests that begin and end at every place of the blocks' runs of rows, those that end before a window is full,
    and those without rows; states that are replaced where they are read."""
    run_conv(act, 4, 40, lens, 5, init=init, tail=len(lens) % 3)


def test_conv_long_runs():
    """Runs of more than the fewest rows a block takes."""
    run_conv("bf16", 4, 8192, [500, 3, 0, 1030, 61, 2, 700], 6)
    run_conv("f32", 3, 2051, [1500, 3, 0, 1030, 61, 2, 700], 6)


def test_conv_many_requests():
    """More requests than a warp looks at at once, or at once twice."""
    run_conv("f32", 4, 8, [(i * 7) % 3 for i in range(1500)], 7, init="same")


@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("rows,ch,width,pad", [(1, 1472, 4, ()), (5, 33, 4, (0, 3)), (64, 64, 3, (5,)), (3, 4096, 2, ())])
@pytest.mark.parametrize("init", ["same", "mixed"])
def test_conv_step(act, rows, ch, width, pad, init):
    run_conv(act, width, ch, [1] * rows, 8, init=init, pad=pad, step=True)


@pytest.mark.parametrize("act,rows,ch", [("bf16", 2501, 64), ("f32", 5003, 30), ("f16", 2400, 33)])
def test_conv_step_of_very_many_requests(act, rows, ch):
    """Blocks that take several turns, the last of them not whole."""
    run_conv(act, 4, ch, [1] * rows, 11, pad=(0, 7, rows - 1), step=True)


def test_conv_without_activation_bias_or_slots():
    run_conv("f16", 4, 48, [9, 4], 9, silu=False, bias=False)
    g = gen(1)
    x, w = normal(g, 6, 48), normal(g, 48, 4)
    got = K.causal_conv(x, w, i32([0, 2, 6]))
    zero, old = torch.zeros(48, device=DEV), torch.zeros(3, 48, device=DEV, dtype=F64)
    for i, j in ((0, 2), (2, 6)):
        y, e, _ = conv64(x[i:j], w, zero, old, True)
        close(got[i:j], y, e)
    state = normal(g, 3, 3, 48)
    before = state.to(F64)
    got = K.causal_conv_step(x[:2], w, state)  # request b in slot b
    for b in range(2):
        y, e, kept = conv64(x[b:b + 1], w, zero, before[b], True)
        close(got[b:b + 1], y, e)
        assert torch.equal(state[b].to(F64), kept)
    assert torch.equal(state[2].to(F64), before[2])


@pytest.mark.parametrize("lens", [[0] * 300 + [5], [5] + [0] * 300 + [70] + [0] * 33, [0] * 31 + [1] + [0] * 64 + [9] + [0],
                                  [3, 0, 0, 0, 200] + [0] * 40])
@pytest.mark.parametrize("init", ["same", "none", "mixed"])
def test_conv_many_requests_without_rows(lens, init):
    run_conv("f16", 4, 36, lens, 10, init=init, pad=(2, 3, len(lens) - 1), tail=1)


# ------------------------------------------------------------------ the scan
def scan64(x, dt, a, b, c, d, z, bias, h, e=0.0):
    """One request, row after row, from the state h (known within e): outputs, the last state, and bounds of what float32
    makes of them."""
    n, ch = x.shape
    share = ch // b.shape[1]
    x, dt, a = x.to(F64), dt.to(F64), a.to(F64)
    b, c = (t.to(F64).repeat_interleave(share, dim=1) for t in (b, c))
    v = dt + bias.to(F64)
    delta = torch.nn.functional.softplus(v, threshold=60.0)
    width_e = U * (dt.abs() + bias.to(F64).abs()) + 2 * EX  # of delta, relative: d log softplus(v) / dv <= 1
    e = e + torch.zeros_like(h)
    ys, es = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(n):
        rate = delta[t, :, None] * a
        decay = torch.exp(rate)
        decay_e = decay * (EX + rate.abs() * (width_e[t, :, None] + 4 * U)) + 2.0 ** -126
        put = (delta[t] * x[t])[:, None] * b[t]
        new = decay * h + put
        # (the exponential unit gives 0 for what is below 2^-126: a delta of less may be lost, with what it puts)
        lost = 2.0 ** -126 * (x[t].abs()[:, None] * b[t].abs())
        e = decay * e + decay_e * (h.abs() + e) + put.abs() * (width_e[t, :, None] + 3 * U) + lost + U * new.abs()
        e = torch.where(torch.isfinite(new), e, 0.0)
        h = new
        ys[t] = (h * c[t]).sum(1) + d.to(F64) * x[t]
        size = (h * c[t]).abs().sum(1) + (d.to(F64) * x[t]).abs()
        es[t] = (e * c[t].abs()).sum(1) + (h.shape[1] + 3) * U * size
    if z is not None:
        gate, ge = silu64(z.to(F64), torch.zeros_like(ys))
        ys, es = ys * gate, es * gate.abs() + ys.abs() * ge + U * (ys * gate).abs()
    return ys, es, h, e


def scan_inputs(g, act, rows, ch, n, groups, gate=True, wide=False, lead=3):
    dtype = TYPES[act]
    bc = normal(g, rows, lead + 2 * groups * n, dtype=dtype)
    x = normal(g, rows, ch + 5, dtype=dtype)[:, 5:] if wide else normal(g, rows, ch, dtype=dtype)
    return dict(x=x, dt=normal(g, rows, ch, dtype=dtype), a=-torch.exp(normal(g, ch, n)) * 3,
                b=bc[:, lead:lead + groups * n].unflatten(1, (groups, n)), c=bc[:, lead + groups * n:].unflatten(1, (groups, n)),
                d=normal(g, ch), z=normal(g, rows, 2 * ch, dtype=dtype)[:, ch:] if gate else None,
                dt_bias=normal(g, ch) - 3)


def scan_want(t, cu, pool, rows, fill):
    ch = t["x"].shape[1]
    want, bound = torch.full((rows, ch), fill, device=DEV, dtype=F64), torch.zeros(rows, ch, device=DEV, dtype=F64)
    kept, kept_e = {}, {}
    for s, (i, j) in enumerate(spans(cu, rows)):
        if pool.slots[s] < 0:
            continue
        y, e, h, he = scan64(t["x"][i:j], t["dt"][i:j], t["a"], t["b"][i:j], t["c"][i:j], t["d"],
                             None if t["z"] is None else t["z"][i:j], t["dt_bias"], pool.begun(s))
        want[i:j], bound[i:j], kept[pool.slots[s]], kept_e[pool.slots[s]] = y, e, h, he
    return want, bound, kept, kept_e


def run_scan(act, ch, n, groups, lens, seed, init="mixed", pad=(), tail=0, step=False, gate=True, wide=False, lead=3):
    g = gen(seed)
    rows = sum(lens) + tail
    t = scan_inputs(g, act, rows, ch, n, groups, gate, wide, lead)
    pool = Pool(g, (ch, n), torch.float32, len(lens), init, pad)
    out = torch.full((rows, ch), 7.0, device=DEV, dtype=TYPES[act])
    cu = list(itertools.accumulate(lens, initial=0))
    if step:
        got = K.selective_step(**t, out=out, **pool.args())
    else:
        got = K.selective_scan(**t, cu=i32(cu), out=out, **pool.args())
    assert got is out
    want, bound, kept, kept_e = scan_want(t, cu, pool, rows, 7.0)
    close(out, want, bound, "out")
    pool.check(kept, kept_e)


@pytest.mark.parametrize("n", [1, 4, 5, 8, 16, 17, 24, 32, 48, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("act", list(TYPES))
def test_scan_types_and_states(act, n):
    run_scan(act, 70, n, 1, [5, 0, 1, 33, 64, 2], 11, tail=2)


@pytest.mark.parametrize("n", [4, 8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("ch,groups,lens,gate", [(8, 1, [1, 17, 0, 16, 40], True), (72, 1, [33, 15, 2], False),
                                                 (400, 2, [9, 8, 7], True), (16, 2, [700, 5, 0, 461], True)])
def test_scan_of_aligned_inputs(act, n, ch, groups, lens, gate):
    """Rows of whole accesses, which come tile by tile: their ends, channels that end inside a block, requests in pieces."""
    run_scan(act, ch, n, groups, lens, 42, gate=gate, lead=8, tail=3)


@pytest.mark.parametrize("ch,groups,wide", [(1, 1, False), (6, 3, True), (130, 2, True), (1216, 1, False), (512, 4, True)])
@pytest.mark.parametrize("act", list(TYPES))
def test_scan_channels_and_groups(act, ch, groups, wide):
    run_scan(act, ch, 16, groups, [40, 3, 31], 12, wide=wide)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0], [31], [32], [33], [300], [1] * 40, [2, 0, 0, 65, 1, 0]])
@pytest.mark.parametrize("init", ["same", "none", "mixed"])
def test_scan_lengths(lens, init):
    run_scan("f32", 40, 16, 1, lens, 13, init=init, tail=len(lens) % 3)
    run_scan("bf16", 40, 16, 1, lens, 13, init=init, pad=(1,), gate=False)


@pytest.mark.parametrize("ch,n", [(96, 16), (48, 64), (2, 16)])
def test_scan_long_prompts(ch, n):
    run_scan("f32", ch, n, 1, [2500, 600], 14)
    run_scan("f16", ch, n, 1, [4001], 14)


@pytest.mark.parametrize("n", [3, 8, 16, 24, 64, 128, 130])
@pytest.mark.parametrize("init", ["same", "none", "mixed"])
def test_scan_long_prompts_among_others(n, init):
    """Requests that are walked in pieces, of every rest, beside those that are not; states replaced where they are read."""
    run_scan("f32", 10, n, 2, [449, 3, 0, 513, 448, 512, 64, 575, 0, 900], 19, init=init, pad=(3,), tail=5)


def test_scan_of_long_prompts_among_very_many():
    """More requests than a block has threads, some of them walked in pieces."""
    run_scan("bf16", 6, 4, 1, [(i * 7) % 4 for i in range(700)] + [1000, 3, 0, 1111] + [1] * 300, 41, init="mixed", pad=(5, 702))


def test_scan_is_repeatable_and_the_bound_only_sizes_it():
    g = gen(28)
    t = scan_inputs(g, "f32", 3000, 40, 16, 1)
    cu = i32([0, 2000, 2000, 2100, 2999])
    pool = type("P", (), {"slots": [0, 1, 2, 3], "begun": lambda self, s: torch.zeros(40, 16, device=DEV, dtype=F64)})()
    want, bound, *_ = scan_want(t, [0, 2000, 2000, 2100, 2999], pool, 3000, 0.0)
    for max_len in (0, 2000, 2001, 2999, 10 ** 6, 300):  # the last: too small, and not split
        work = torch.full((K.selective_scan_work_floats(3000, 40, 16, 1, max_len) + 4,), math.nan, device=DEV)
        out = K.selective_scan(**t, cu=cu, max_len=max_len, work=work)
        assert torch.equal(out[:2999], K.selective_scan(**t, cu=cu, max_len=max_len)[:2999])
        assert work[-4:].isnan().all()
        close(out[:2999], want[:2999], bound[:2999])
    with pytest.raises(_lib.KrikilError, match="work"):
        K.selective_scan(**t, cu=cu, work=torch.empty(1000, device=DEV))
    with pytest.raises(ValueError, match="work"):
        K.selective_scan(**t, cu=cu, work=torch.empty(1 << 20, device=DEV, dtype=torch.float16))


@pytest.mark.parametrize("cu", [[0, 3000, 0, 3000, 0, 3000], [0, 3000, 10, 2999, 1, 2], [-7, 5000, -7, 5000]])
def test_scan_of_long_requests_that_overlap_stays_in_bounds(cu):
    """Offsets that do not ascend can name more pieces than there is scratch for."""
    t = scan_inputs(gen(29), "f32", 3000, 40, 16, 1)
    floats = K.selective_scan_work_floats(3000, 40, 16)
    work = torch.full((floats + 100000,), 7.0, device=DEV)
    out = K.selective_scan(**t, cu=i32(cu), work=work[:floats])
    assert out.shape == (3000, 40) and (work[floats:] == 7).all()


def scan_want_of_many(t, lens, pool, rows, fill):
    """scan_want of many short requests: those of one length are walked as one request of all their channels."""
    ch, groups = t["x"].shape[1], t["b"].shape[1]
    want, bound = torch.full((rows, ch), fill, device=DEV, dtype=F64), torch.zeros(rows, ch, device=DEV, dtype=F64)
    kept, kept_e, starts = {}, {}, list(itertools.accumulate(lens, initial=0))
    for length in sorted(set(lens)):
        same = [s for s, k in enumerate(lens) if k == length and pool.slots[s] >= 0]
        at = torch.tensor([[starts[s] + i for s in same] for i in range(length)], device=DEV).long().view(length, len(same))
        flat = lambda v: v[at].flatten(1)  # noqa: E731
        group = lambda v: v[at].flatten(1, 2)  # noqa: E731
        often = lambda v: v.repeat(len(same), *[1] * (v.dim() - 1))  # noqa: E731
        y, e, h, he = scan64(flat(t["x"]), flat(t["dt"]), often(t["a"]), group(t["b"]), group(t["c"]), often(t["d"]),
                             flat(t["z"]), often(t["dt_bias"]), torch.cat([pool.begun(s) for s in same]))
        want[at], bound[at] = y.view(length, len(same), ch), e.view(length, len(same), ch)
        for i, s in enumerate(same):
            kept[pool.slots[s]], kept_e[pool.slots[s]] = h[i * ch:(i + 1) * ch], he[i * ch:(i + 1) * ch]
    return want, bound, kept, kept_e


@pytest.mark.parametrize("n", [4, 5, 8, 12, 16, 17, 24, 32, 50, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("requests,ch,groups,wide,lead", [(200, 40, 1, True, 3), (161, 48, 1, False, 8), (90, 80, 2, False, 8)])
def test_scan_of_many_short_requests(act, n, requests, ch, groups, wide, lead):
    """More blocks than multiprocessors and no request that may be split, as a server's prompts are: whole lanes of states,
    and the requests' order with and without a place for each in a block."""
    assert requests * groups > torch.cuda.get_device_properties(DEV).multi_processor_count
    assert K.selective_scan_work_floats(5 * requests, ch, n, groups, 9) == 0
    g, lens = gen(49), [(i * 7) % 10 for i in range(requests)]
    rows = sum(lens) + 2
    t = scan_inputs(g, act, rows, ch, n, groups, wide=wide, lead=lead)
    pool = Pool(g, (ch, n), torch.float32, requests, "mixed", (3, 77, requests - 1))
    out = torch.full((rows, ch), 7.0, device=DEV, dtype=TYPES[act])
    K.selective_scan(**t, cu=i32(list(itertools.accumulate(lens, initial=0))), out=out, max_len=9, **pool.args())
    want, bound, kept, kept_e = scan_want_of_many(t, lens, pool, rows, 7.0)
    close(out, want, bound, "out")
    pool.check(kept, kept_e)


@pytest.mark.parametrize("cu", [[0, 360, 10, 370], [0, 576, 0, 576], [0, 330, 100, 430, 200, 530, 576]])
@pytest.mark.parametrize("requests", [0, 200])
@pytest.mark.parametrize("init", ["same", "mixed"])
def test_scan_of_long_requests_that_overlap_takes_nothing_from_scratch(cu, requests, init):
    """Offsets that step back can name more requests in pieces than ascending ones: a slot holds its request's own state
    or what it held, and scratch of NaN reaches neither slots nor outputs."""
    g, rows, ch, n = gen(48), 576, 64, 16
    cu = cu + [cu[-1]] * (requests - len(cu))  # (the rest have no rows)
    t, pool = scan_inputs(g, "f32", rows, ch, n, 1), Pool(g, (ch, n), torch.float32, len(cu) - 1, init)
    out = torch.full((rows, ch), 7.0, device=DEV)
    work = torch.full((K.selective_scan_work_floats(rows, ch, n),), math.nan, device=DEV)
    assert work.numel() > 0
    K.selective_scan(**t, cu=i32(cu), out=out, work=work, **pool.args())
    assert not out.isnan().any()
    _, _, kept, kept_e = scan_want(t, cu, pool, rows, 7.0)
    for slot in list(kept):
        if torch.equal(pool.all[slot], pool.before[slot]):
            del kept[slot], kept_e[slot]
    assert pool.slots[0] in kept
    pool.check(kept, kept_e)


@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 16, 17, 24, 32, 64, 100, 128, 256])
@pytest.mark.parametrize("act", list(TYPES))
def test_step_types_and_states(act, n):
    run_scan(act, 70, n, 2, [1] * 9, 15, pad=(2, 8), step=True)


@pytest.mark.parametrize("n", [4, 8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("rows,ch,groups", [(1, 24, 1), (9, 70, 2), (1800, 96, 1)])
def test_step_of_aligned_inputs(act, n, rows, ch, groups):
    """States, B and C in whole groups of four, by one and by two requests a thread."""
    run_scan(act, ch, n, groups, [1] * (rows if n <= 32 else min(rows, 9)), 43, pad=(2, 8), step=True, lead=8, gate=n != 64)


@pytest.mark.parametrize("act,rows,ch,n,lead", [("bf16", 4003, 96, 32, 8), ("f32", 3001, 70, 48, 3)])
def test_step_of_very_many_requests(act, rows, ch, n, lead):
    """Blocks that take several turns, the last of them not whole."""
    run_scan(act, ch, n, 1, [1] * rows, 46, pad=(0, 7, rows - 1), step=True, lead=lead)


@pytest.mark.parametrize("rows,ch,groups,init", [(1, 1216, 1, "same"), (300, 24, 1, "mixed"), (3, 5120, 4, "none"),
                                                 (5, 1, 1, "mixed"), (2, 77, 7, "same")])
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_step_channels_and_groups(act, rows, ch, groups, init):
    run_scan(act, ch, 16, groups, [1] * rows, 16, init=init, step=True, gate=ch != 77, wide=ch == 24)


@pytest.mark.parametrize("step", [False, True])
def test_scan_steps_of_any_width(step):
    """Step widths from those that underflow to those past softplus's line, and decays of none and of all."""
    g = gen(17)
    rows, ch, n = 12, 64, 16
    t = scan_inputs(g, "f32", rows, ch, n, 1)
    t["dt"] = torch.linspace(-120.0, 90.0, rows * ch, device=DEV).view(ch, rows).T.contiguous()
    t["dt_bias"] = torch.zeros(ch, device=DEV)
    t["a"][::3] = 0.0
    t["a"][1::3] *= 1e4
    pool = Pool(g, (ch, n), torch.float32, rows if step else 1)
    cu = list(range(rows + 1)) if step else [0, rows]
    out = K.selective_step(**t, **pool.args()) if step else K.selective_scan(**t, cu=i32(cu), **pool.args())
    want, bound, kept, kept_e = scan_want(t, cu, pool, rows, 0.0)
    close(out, want, bound, "out")
    pool.check(kept, kept_e)


@pytest.mark.parametrize("n,rows", [(16, 40), (20, 40), (3, 40), (5, 40), (17, 40), (50, 40), (16, 900), (23, 900)])
def test_scan_infinite_inputs_stay_in_their_channels(n, rows):
    """An infinite x makes its channel infinite from its row on, and no other value."""
    g = gen(18)
    t = scan_inputs(g, "f32", rows, 24, n, 1, gate=False)
    t["b"], t["c"] = t["b"].abs() + 0.1, t["c"].abs() + 0.1
    t["a"] = -torch.exp(normal(g, 24, n)) * 0.01
    t["d"] = t["d"].abs() + 0.1
    t["x"][20, 5] = math.inf
    out = K.selective_scan(**t, cu=i32([0, rows]))
    want, bound, *_ = scan_want(t, [0, rows], type("P", (), {"slots": [0], "begun": lambda self, s: torch.zeros(
        24, n, device=DEV, dtype=F64)})(), rows, 0.0)
    assert (out[20:, 5] == math.inf).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[20:, 5] = False
    close(out[keep], want[keep], bound[keep])


# ------------------------------------------------------------------ both
@pytest.mark.parametrize("act", list(TYPES))
def test_padding_is_not_read_and_bad_slots_are_left_alone(act):
    g, dtype = gen(20), TYPES[act]
    ch, n, lens = 24, 16, [3, 2, 4, 1]
    cu = list(itertools.accumulate(lens, initial=0))
    rows = 14
    x = normal(g, rows, ch, dtype=dtype)
    x[10:] = math.nan  # rows of no request
    x[3:5] = math.nan  # rows of padding
    w = normal(g, ch, 4)
    for slots, init, live in (([2, -1, 0, 1], [-1, 3, 4, -9], [0, 2, 3]), ([2, 5, 0, 1], [-1, 3, 4, -1], [0, 2, 3]),
                              ([2, 3, 0, 1 << 30], [-1, 5, -1, -1], [0, 2])):
        # slot 4 of five may be continued from, 5 is past the pool; init 5 is, too
        state = normal(g, 5, 3, ch, dtype=dtype)
        before = state.clone()
        out = torch.full((rows, ch), 7.0, device=DEV, dtype=dtype)
        K.causal_conv(x, w, i32(cu), state=state, slots=i32(slots), init=i32(init), out=out)
        hs = normal(g, 5, ch, n)
        hs_before = hs.clone()
        t = scan_inputs(g, act, rows, ch, n, 1)
        t["x"] = x
        y = torch.full((rows, ch), 7.0, device=DEV, dtype=dtype)
        K.selective_scan(**t, cu=i32(cu), state=hs, slots=i32(slots), init=i32(init), out=y)
        touched = []
        for s, (i, j) in enumerate(spans(cu, rows)):
            if s not in live:
                assert (out[i:j] == 7).all() and (y[i:j] == 7).all()
                continue
            touched.append(slots[s])
            zero = torch.zeros(ch, device=DEV)
            old = before[init[s]].to(F64) if init[s] >= 0 else torch.zeros(3, ch, device=DEV, dtype=F64)
            want, e, kept = conv64(x[i:j], w, zero, old, True)
            close(out[i:j], want, e)
            assert torch.equal(state[slots[s]].to(F64), kept)
            assert torch.isfinite(y[i:j]).all()
        rest = [k for k in range(5) if k not in touched]
        assert torch.equal(state[rest], before[rest]) and torch.equal(hs[rest], hs_before[rest])
        assert (out[10:] == 7).all() and (y[10:] == 7).all()


@pytest.mark.parametrize("cu", [[-3, 4, 9], [0, 5, 400], [0, 6, 2], [9, 9, 9], [20, 30, 40], [-5, -4, -3], [5, 3, 1]])
def test_offsets_outside_the_rows(cu):
    """Offsets are cut to the rows that there are, and a request that ends before it begins has none."""
    g = gen(21)
    ch, n, rows = 40, 16, 9
    x, w = normal(g, rows, ch), normal(g, ch, 4)
    pool, out = Pool(g, (3, ch), torch.float32, 2, "same"), torch.full((rows, ch), 7.0, device=DEV)
    K.causal_conv(x, w, i32(cu), out=out, **pool.args())
    t = scan_inputs(g, "f32", rows, ch, n, 1)
    hp, y = Pool(g, (ch, n), torch.float32, 2, "same"), torch.full((rows, ch), 7.0, device=DEV)
    K.selective_scan(**t, cu=i32(cu), out=y, **hp.args())
    if cu[0] > cu[1] or cu[1] > cu[2]:  # in bounds is all that is promised to offsets that do not ascend
        return
    want, kept = torch.full((rows, ch), 7.0, device=DEV, dtype=F64), {}
    bound = torch.zeros_like(want)
    for s, (i, j) in enumerate(spans(cu, rows)):
        want[i:j], bound[i:j], kept[pool.slots[s]] = conv64(x[i:j], w, torch.zeros(ch, device=DEV), pool.begun(s), True)
    close(out, want, bound)
    pool.check(kept)
    want, bound, kept, kept_e = scan_want(t, cu, hp, rows, 7.0)
    close(y, want, bound)
    hp.check(kept, kept_e)


@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("cut", [1, 3, 4, 37])
def test_prompts_in_pieces_and_tokens_meet_the_whole(act, cut):
    """A prompt at once, and in two pieces and then token by token through its slots: the convolution's rows and states
    bit for bit, the scan's state within its bounds."""
    g, dtype = gen(22), TYPES[act]
    ch, n, rows = 72, 16, 45
    t = scan_inputs(g, act, rows, ch, n, 2)
    w, bias = normal(g, ch, 4), normal(g, ch)
    raw = t["x"]
    whole = K.causal_conv(raw, w, i32([0, rows]), bias=bias, state=(cs := torch.zeros(1, 3, ch, device=DEV, dtype=dtype)))
    t["x"] = whole
    y = K.selective_scan(**t, cu=i32([0, rows]), state=(hs := torch.zeros(1, ch, n, device=DEV)))
    conv, hidden = normal(g, 3, 3, ch, dtype=dtype), normal(g, 3, ch, n)
    slot, got, got_y = i32([2]), [], []

    def piece(i, j, init):
        p = {k: v[i:j] if k in ("x", "dt", "b", "c", "z") else v for k, v in t.items()}
        if j - i == 1 and i > cut:
            c = K.causal_conv_step(raw[i:j], w, conv, slot, bias=bias)
            p["x"] = c
            return c, K.selective_step(**p, state=hidden, slots=slot)
        c = K.causal_conv(raw[i:j], w, i32([0, j - i]), bias=bias, state=conv, slots=slot, init=init)
        p["x"] = c
        return c, K.selective_scan(**p, cu=i32([0, j - i]), state=hidden, slots=slot, init=init)

    ends = [0, cut, cut + 2] + list(range(cut + 3, rows + 1))
    for i, j in zip(ends[:-1], ends[1:]):
        c, o = piece(i, j, i32([-1]) if i == 0 else None)
        got.append(c)
        got_y.append(o)
    assert torch.equal(torch.cat(got), whole) and torch.equal(conv[2], cs[0])
    pool = type("P", (), {"slots": [0], "begun": lambda self, s: torch.zeros(ch, n, device=DEV, dtype=F64)})()
    want, bound, kept, kept_e = scan_want(t, [0, rows], pool, rows, 0.0)
    for out, h in ((y, hs[0]), (torch.cat(got_y), hidden[2])):
        close(out, want, bound)
        close(h, kept[0], kept_e[0])


@pytest.mark.parametrize("which", ["x", "dt", "z"])
@pytest.mark.parametrize("step", [False, True])
def test_scan_in_place(which, step):
    g = gen(23)
    t = scan_inputs(g, "bf16", 70, 100, 16, 1)
    state = normal(g, 70, 100, 16)
    call = (lambda **o: K.selective_step(**t, state=state.clone(), **o)) if step else (
        lambda **o: K.selective_scan(**t, cu=i32([0, 33, 70]), state=state.clone(), **o))
    want = call()
    got = call(out=t[which])
    assert got is t[which] and torch.equal(got, want)


def test_calls_replayed_from_a_graph_on_another_stream():
    """One graph of a serving step -- prompts, then a token of each -- over new offsets, slots and inputs."""
    g = gen(24)
    ch, n, rows, S = 64, 16, 50, 4
    cu, slots, init = i32([0] * (S + 1)), i32([-1] * S), i32([-1] * S)
    t = scan_inputs(g, "bf16", rows, ch, n, 1)
    w, conv, hidden = normal(g, ch, 4), normal(g, 9, 3, ch, dtype=torch.bfloat16), normal(g, 9, ch, n)
    logits, ids = normal(g, S, 500), i32([1, 2, 3, 4])
    raw = t["x"].clone()

    def step():
        p = dict(t)
        c1 = K.causal_conv(raw, w, cu, state=conv, slots=slots, init=init, out=t["x"])
        y1 = K.selective_scan(**p, cu=cu, state=hidden, slots=slots, init=init)
        p = {k: v[:S] if k in ("dt", "b", "c", "z") else v for k, v in t.items()}
        p["x"] = K.causal_conv_step(raw[-S:], w, conv, slots)
        return c1, y1, p["x"], K.selective_step(**p, state=hidden, slots=slots), *K.token_logprobs(logits, ids, top=3)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = step()
    torch.cuda.current_stream().wait_stream(stream)
    for lens, where in (([10, 0, 39, 1], [4, 2, 0, 8]), ([1, 1, 1, 1], [1, -1, 3, 5]), ([0, 20, 0, 30], [6, 7, -1, 0])):
        cu.copy_(i32(list(itertools.accumulate(lens, initial=0))))
        slots.copy_(i32(where))
        init.copy_(i32([where[0], -1, where[2], -1]))
        for name in ("dt", "z"):
            t[name].copy_(normal(g, *t[name].shape, dtype=torch.bfloat16))
        raw.copy_(normal(g, rows, ch, dtype=torch.bfloat16))
        logits.copy_(normal(g, S, 500))
        before = conv.clone(), hidden.clone()
        for c in captured[:4]:
            c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [c.clone() for c in captured]
        after = conv.clone(), hidden.clone()
        conv.copy_(before[0])
        hidden.copy_(before[1])
        eager = step()
        live = torch.tensor([s >= 0 for s in where], device=DEV)
        for k, (p, q) in enumerate(zip(replayed, eager)):
            if k < 2:  # rows of no request and of padding hold what their buffers held
                for s, (i, j) in enumerate(spans(cu.tolist(), rows)):
                    assert where[s] < 0 or torch.equal(p[i:j], q[i:j])
            elif k < 4:
                assert torch.equal(p[live], q[live])
            else:
                assert torch.equal(p, q)
        assert torch.equal(after[0], conv) and torch.equal(after[1], hidden)


@pytest.mark.parametrize("act", list(TYPES))
def test_views_off_the_grid(act):
    """Weights, decays, states and inputs that begin one element beside an aligned place give what their copies give: the
    same operations in the same order, bit for bit."""
    g, dtype = gen(47), TYPES[act]

    def beside(t):  # a copy one element into its memory, rows as far apart as a row and three
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, device=DEV, dtype=t.dtype)
        view = wide[..., 1:1 + t.shape[-1]]
        view.copy_(t)
        return view

    def shifted(t):  # dense, one element beside
        flat = torch.zeros(t.numel() + 1, device=DEV, dtype=t.dtype)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def pool(t):  # slots dense, apart, beside
        wide = torch.zeros(t.shape[0], t[0].numel() + 3, device=DEV, dtype=t.dtype)
        view = wide[:, 1:1 + t[0].numel()].unflatten(1, t.shape[1:])
        view.copy_(t)
        return view

    ch, rows, cu = 64, 70, i32([0, 33, 33, 70])
    x = normal(g, rows, ch, dtype=dtype)
    for width in (2, 3, 4):
        w, bias, state = normal(g, ch, width), normal(g, ch), normal(g, rows, width - 1, ch, dtype=dtype)
        for step in (False, True):
            s, p = state.clone(), pool(state)
            call = (lambda x, w, bias, s: K.causal_conv_step(x, w, s, bias=bias)) if step else (
                lambda x, w, bias, s: K.causal_conv(x, w, cu, bias=bias, state=s))
            assert torch.equal(call(x, w, bias, s), call(beside(x), shifted(w), shifted(bias), p)) and torch.equal(s, p)
            assert torch.equal(call(x, shifted(w), bias, state.clone()), call(x, w, bias, state.clone()))
    for n in (4, 16, 32):
        t = {k: v.contiguous() for k, v in scan_inputs(g, act, rows, ch, n, 1).items()}
        state = normal(g, rows, ch, n)
        off = {k: shifted(v) if k in ("a", "d", "dt_bias") else beside(v) for k, v in t.items()}
        for step in (False, True):
            s, p = state.clone(), pool(state)
            call = (lambda t, s: K.selective_step(**t, state=s)) if step else (lambda t, s: K.selective_scan(**t, cu=cu, state=s))
            assert torch.equal(call(t, s), call(off, p)) and torch.equal(s, p)


def test_offsets_past_32_bits():
    g = gen(25)
    far, ch, n = (1 << 31) // 2 + 64, 24, 16
    room = torch.zeros(2 * far + 64, device=DEV, dtype=torch.bfloat16)
    x = room.as_strided((3, ch), (far, 1))
    x.copy_(normal(g, 3, ch, dtype=torch.bfloat16))
    w, near = normal(g, ch, 4), x.clone().contiguous()
    assert torch.equal(K.causal_conv(x, w, i32([0, 3])), K.causal_conv(near, w, i32([0, 3])))
    t = scan_inputs(g, "bf16", 3, ch, n, 1)
    want = K.selective_scan(**dict(t, x=near), cu=i32([0, 3]))
    assert torch.equal(K.selective_scan(**dict(t, x=x), cu=i32([0, 3])), want)
    out = room.as_strided((3, ch), (far, 1), 32)
    K.selective_scan(**t, cu=i32([0, 3]), out=out)
    assert torch.equal(out, K.selective_scan(**t, cu=i32([0, 3])))
    K.token_logprobs(x)  # rows far apart
    for p, q in zip(K.token_logprobs(x, top=4), K.token_logprobs(near, top=4)):
        assert p is q or torch.equal(p, q)
    del room, x, out
    pool = torch.zeros(3, (1 << 30) + 4096, device=DEV)  # 13 GB of slots
    state = pool[:, :ch * n].unflatten(1, (ch, n))
    state.copy_(normal(g, 3, ch, n))
    small = state.clone()
    p = K.selective_step(**t, state=state, slots=i32([2, 0, 1]))
    assert torch.equal(p, K.selective_step(**t, state=small, slots=i32([2, 0, 1]))) and torch.equal(state, small)
    p = K.selective_scan(**t, cu=i32([0, 1, 1, 3]), state=state, slots=i32([2, 0, 1]), init=i32([1, 2, -1]))
    q = K.selective_scan(**t, cu=i32([0, 1, 1, 3]), state=small, slots=i32([2, 0, 1]), init=i32([1, 2, -1]))
    assert torch.equal(p, q)


def test_two_streams_at_once():
    """Calls on two streams that continue from the same slots, each with its own slots, scratch and outputs."""
    g = gen(44)
    t = scan_inputs(g, "bf16", 1500, 64, 16, 1, lead=8)
    w, x = normal(g, 64, 4), normal(g, 1500, 64, dtype=torch.bfloat16)
    cs, hs = normal(g, 9, 3, 64, dtype=torch.bfloat16), normal(g, 9, 64, 16)
    cu, init, logits = i32([0, 900, 1500]), i32([8, 7]), normal(g, 2, 140000)
    slots = [i32([0, 1]), i32([2, 3])]

    def calls(i):
        return (K.causal_conv(x, w, cu, state=cs, slots=slots[i], init=init),
                K.selective_scan(**t, cu=cu, state=hs, slots=slots[i], init=init), *K.token_logprobs(logits, None, 5)[1:])

    want = calls(0)
    states = cs[:2].clone(), hs[:2].clone()
    streams = [torch.cuda.Stream() for _ in slots]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls(i))
    torch.cuda.synchronize()
    for i in range(2):
        for call in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(call, want))
        assert torch.equal(cs[slots[i].long()], states[0]) and torch.equal(hs[slots[i].long()], states[1])


def test_calls_run_with_their_tensors_device_current(monkeypatch):
    """With another device current, every library call -- the size of the scratch, too -- is made with the tensors'
    device current, and the other device is current again behind it.  (The other device is pretended: what the wrappers
    ask and set is stood in for.)"""
    current, seen = [0], []

    class Device:
        def __init__(self, dev):
            self.index = dev.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, current[0]))
                return getattr(lib, name)(*args)
            return call

    lib = K.lib
    g = gen(45)
    t = scan_inputs(g, "f32", 600, 32, 16, 1)
    w, cs, hs = normal(g, 32, 4), normal(g, 600, 3, 32), normal(g, 600, 32, 16)

    def calls():
        return [K.causal_conv(t["x"], w, i32([0, 600])), K.causal_conv_step(t["x"], w, cs.clone()),
                K.selective_scan(**t, cu=i32([0, 600])), K.selective_step(**t, state=hs.clone()),
                *K.token_logprobs(t["x"], i32([3] * 600), 4)]

    here = calls()
    monkeypatch.setattr(K, "lib", Lib())
    monkeypatch.setattr(K, "_current_device", lambda: current[0])
    monkeypatch.setattr(K.torch.cuda, "device", Device)
    current[0] = 1
    there = calls()
    assert all(torch.equal(p, q) for p, q in zip(here, there))
    assert len(seen) == 6 and all(dev == 0 for _, dev in seen) and current[0] == 1, seen


def test_every_call_launches_its_own_kernels():
    g = gen(26)
    t = scan_inputs(g, "f32", 4, 32, 16, 1)
    w = normal(g, 32, 4)
    for call in (lambda: K.causal_conv(t["x"], w, i32([0, 4])),
                 lambda: K.causal_conv_step(t["x"], w, torch.zeros(4, 3, 32, device=DEV)),
                 lambda: K.selective_scan(**t, cu=i32([0, 4])),
                 lambda: K.selective_step(**t, state=torch.zeros(4, 32, 16, device=DEV)),
                 lambda: K.token_logprobs(t["x"])):
        before = launch_count()
        call()
        assert launch_count() >= before + 1


def test_calls_of_no_rows():
    e = torch.empty(0, 24, device=DEV)
    w, a = torch.zeros(24, 4, device=DEV), torch.zeros(24, 16, device=DEV)
    bc = torch.empty(0, 16, device=DEV)
    state, hs = torch.ones(2, 3, 24, device=DEV), torch.ones(2, 24, 16, device=DEV)
    assert K.causal_conv(e, w, i32([0])).shape == (0, 24)
    assert K.causal_conv_step(e, w, state).shape == (0, 24)
    assert K.selective_scan(e, e, a, bc, bc, i32([0])).shape == (0, 24)
    assert K.selective_step(e, e, a, bc, bc, hs).shape == (0, 24)
    # requests without rows leave what they continue from
    K.causal_conv(e, w, i32([0, 0, 0]), state=state, init=i32([-1, 1]))
    K.selective_scan(e, e, a, bc, bc, i32([0, 0, 0]), state=hs, init=i32([-1, 1]))
    assert (state[0] == 0).all() and (state[1] == 1).all() and (hs[0] == 0).all() and (hs[1] == 1).all()
    lp, entropy, ids, best = K.token_logprobs(torch.empty(0, 9, device=DEV), torch.empty(0, 2, device=DEV, dtype=torch.int32), 3)
    assert lp.shape == (0, 2) and entropy.shape == (0,) and ids.shape == best.shape == (0, 3)


def test_wrappers_refuse_what_does_not_belong_together():
    g = gen(27)
    t = scan_inputs(g, "f32", 4, 32, 16, 1)
    w, cu, state, hs = normal(g, 32, 4), i32([0, 4]), torch.zeros(2, 3, 32, device=DEV), torch.zeros(2, 32, 16, device=DEV)
    x = t["x"]
    conv = lambda **k: K.causal_conv(**dict(dict(x=x, weight=w, cu=cu), **k))  # noqa: E731
    scan = lambda **k: K.selective_scan(**dict(dict(t, cu=cu), **k))  # noqa: E731
    for call, word in (
            (lambda: conv(x=x.double()), "x"), (lambda: conv(x=x.T), "x|weight"), (lambda: conv(weight=w[:31]), "weight"),
            (lambda: conv(weight=w.half()), "weight"), (lambda: conv(weight=w.T.contiguous().T), "weight"),
            (lambda: conv(cu=cu.long()), "cu"), (lambda: conv(cu=cu[:0]), "cu"), (lambda: conv(cu=cu.cpu()), "cu"),
            (lambda: conv(bias=w), "bias"), (lambda: conv(slots=i32([0])), "state"), (lambda: conv(init=i32([0])), "state"),
            (lambda: conv(state=state.half()), "state"), (lambda: conv(state=state[:, :2]), "state"),
            (lambda: conv(state=state.transpose(1, 2).contiguous().transpose(1, 2)), "state"),
            (lambda: conv(state=state, slots=i32([0, 1])), "slots"), (lambda: conv(state=state, init=i32([0, 1])), "init"),
            (lambda: conv(out=x.half()), "out"), (lambda: conv(out=x[:3]), "out"),
            (lambda: K.causal_conv(x, w, i32([0, 1, 2, 4]), state=state), "slot"),
            (lambda: K.causal_conv_step(x, w, state), "slot"),
            (lambda: scan(dt=x.half()), "dt"), (lambda: scan(z=x[:, :31]), "z"), (lambda: scan(a=t["a"][:31]), "a"),
            (lambda: scan(b=t["b"][:, :, :15]), "b"), (lambda: scan(c=t["c"].half()), "c"),
            (lambda: scan(b=torch.zeros(4, 3, 16, device=DEV), c=torch.zeros(4, 3, 16, device=DEV)), "groups"),
            (lambda: scan(b=torch.zeros(4, 2, 16, device=DEV)), "groups"), (lambda: scan(d=w), "d"),
            (lambda: scan(dt_bias=t["d"].half()), "dt_bias"), (lambda: scan(state=hs.half()), "state"),
            (lambda: scan(state=state), "state"),
            (lambda: K.token_logprobs(x, i32([1, 2])), "tokens"), (lambda: K.token_logprobs(x, cu.long()), "tokens"),
            (lambda: K.token_logprobs(x.T), "logits"), (lambda: K.token_logprobs(x, top=-1), "top"),
            (lambda: K.token_logprobs(x, top=1 << 40), "top")):
        with pytest.raises(ValueError, match=word):
            call()
    for call in (lambda: conv(weight=normal(g, 32, 5)), lambda: conv(out=x), lambda: K.token_logprobs(x, top=33),
                 lambda: K.token_logprobs(torch.zeros(1, 100, device=DEV), top=33),
                 lambda: scan(b=torch.zeros(4, 300, device=DEV), c=torch.zeros(4, 300, device=DEV), a=torch.zeros(32, 300, device=DEV)),
                 lambda: scan(out=torch.zeros(1, 32, device=DEV).expand(4, 32))):
        with pytest.raises(_lib.KrikilError) as err:
            call()
        assert err.value.status == _lib.INVALID


# ------------------------------------------------------------------ log probabilities
def check_logprobs(logits, tokens, top, special=False):
    lp, entropy, ids, best = K.token_logprobs(logits, tokens, top)
    x = logits.to(F64)
    rows, vocab = x.shape
    m = x.amax(1, keepdim=True)
    u = torch.where(torch.isneginf(x), -math.inf, x - m)
    p = torch.exp(u)
    s = p.sum(1, keepdim=True)
    empty = torch.isneginf(m)
    logs = torch.log(s)
    lp64 = torch.where(empty, -math.inf, u - logs)
    pu = torch.where(p > 0, p * u.abs(), 0.0)
    mean_u = pu.sum(1, keepdim=True) / s
    # the sum: its terms' exponentials, their arguments' roundings, and a chain of additions a thread
    chain = (math.ceil(vocab / 256) + 16) * U
    sum_e = EX + 3 * U * mean_u + chain
    h64 = torch.where(empty, 0.0, logs + mean_u)[:, 0]
    if tokens is not None:
        ask = tokens.long().view(rows, -1)
        want = torch.gather(lp64, 1, ask.clamp(0, vocab - 1))
        want = torch.where(ask >= vocab, -math.inf, torch.where(ask < 0, 0.0, want))
        du = torch.gather(u, 1, ask.clamp(0, vocab - 1)).abs()
        room = torch.where(torch.isfinite(want), sum_e + U * (du + 4 * logs.abs() + want.abs()), 0.0)
        close(lp.view(rows, -1), want, room, "lp")
    close(entropy, h64, torch.where(empty[:, 0], 0.0, (sum_e * (1 + 2 * mean_u) + 4 * U * (logs.abs() + mean_u))[:, 0]
                                    + EX * mean_u[:, 0] + 2.0 ** -120 * vocab), "entropy")
    # the order, on whole numbers
    f = torch.where(logits.isnan(), -math.inf, logits.float()) + 0.0
    bits = f.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 31 - torch.arange(vocab, device=DEV)
    order = torch.argsort(key, dim=1, descending=True, stable=True)[:, :top]
    assert torch.equal(ids.long(), order)
    want = torch.gather(lp64, 1, order)
    du = torch.gather(u, 1, order).abs()
    room = torch.where(torch.isfinite(want), sum_e + U * (du + 4 * logs.abs() + want.abs()), 0.0)
    close(best, want, room, "best")


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 7, 7), (2, 63, 5), (300, 64, 32), (1024, 2048, 5),
                                            (3, 2049, 20), (17, 5003, 32), (2, 50001, 1), (1, 131072, 20), (4, 131073, 31),
                                            (1, 262144, 0), (700, 300, 3), (160, 9001, 20)])
@pytest.mark.parametrize("act", list(TYPES))
def test_logprobs_sizes(act, rows, vocab, top):
    g = gen(30)
    logits = (3 * normal(g, rows, vocab + 3)).to(TYPES[act])[:, 1:vocab + 1]
    tokens = torch.randint(-1, vocab, (rows, 3), generator=g, device=DEV, dtype=torch.int32)
    check_logprobs(logits, tokens, top)
    check_logprobs(logits.contiguous(), tokens[:, 0].contiguous(), min(top, 2))


@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("vocab", [40, 2048, 30011])
def test_logprobs_orders_and_ties(act, vocab):
    """Rising, falling, equal and few different logits; the best ones side by side, at the ends, or in one thread's way."""
    g, dtype = gen(31), TYPES[act]
    base = torch.linspace(-9, 9, vocab, device=DEV)
    rows = [base, base.flip(0), torch.zeros(vocab, device=DEV), torch.randint(0, 3, (vocab,), generator=g, device=DEV).float(),
            torch.cat([torch.zeros(vocab - 30, device=DEV), torch.ones(30, device=DEV)]),
            torch.cat([torch.ones(30, device=DEV), torch.zeros(vocab - 30, device=DEV)]),
            torch.where(torch.arange(vocab, device=DEV) % 256 == 3, 5.0, base), torch.where(
                torch.arange(vocab, device=DEV) % 2048 < 8, 20 + base, base), -0.0 * base.sign(),
            torch.where(torch.arange(vocab, device=DEV) % 2048 < 4, 20 - base, base)]
    check_logprobs(torch.stack(rows).to(dtype), i32([0] * len(rows)), min(vocab, 20))
    check_logprobs(torch.stack(rows).to(dtype), i32([vocab - 1] * len(rows)), 1)
    check_logprobs(torch.stack(rows).to(dtype), None, min(vocab, 32))


@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("vocab", [50, 2048, 10007])
def test_logprobs_masks_infinities_and_nan(act, vocab):
    g, dtype = gen(32), TYPES[act]
    lowest = torch.finfo(dtype).min
    x = (2 * normal(g, 9, vocab)).to(dtype)
    x[0] = -math.inf  # nothing is left
    x[1] = lowest  # as lowest values mask everything: all alike
    x[2, ::2] = -math.inf
    x[3, 1:] = lowest
    x[4, :-1] = -math.inf  # one is left
    x[5, 3] = torch.finfo(dtype).max
    x[6, :vocab // 2] = -math.inf
    x[7] = torch.where(torch.arange(vocab, device=DEV) % 3 == 0, lowest, -math.inf).to(dtype)
    tokens = i32([[1, vocab - 1, -1]] * 9)
    check_logprobs(x, tokens, 6)
    # NaN and infinity: NaN everywhere but where nothing was asked, the order of what can be ordered
    y = x[6:].clone()
    y[0, 5], y[1, vocab - 2], y[2, 7] = math.nan, math.inf, math.nan
    y[2, 9] = math.inf
    lp, entropy, ids, best = K.token_logprobs(y, i32([[4, vocab - 1, -1]] * 3), 4)
    assert lp[:, :2].isnan().all() and (lp[:, 2] == 0).all() and entropy.isnan().all() and best.isnan().all()
    f = torch.where(y.isnan(), -math.inf, y.float())
    assert torch.equal(ids.long(), torch.sort(f, dim=1, descending=True, stable=True).indices[:, :4])


@pytest.mark.parametrize("act", list(TYPES))
def test_logprobs_of_large_logits(act):
    g = gen(33)
    big = 3e38 if act != "f16" else 6e4
    x = (normal(g, 4, 777) * big / 5).clamp(-big, big).to(TYPES[act])
    x[1] = x[1].abs() / 2 + big / 2
    x[2] = -x[1]
    check_logprobs(x, i32([0, 1, 2, 776]), 5)


@pytest.mark.parametrize("act", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 131072), (5, 70001), (300, 40000)])
def test_logprobs_replayed_from_a_graph(act, rows, vocab):
    """Rows shared by the blocks of clusters and rows of one block each, over new logits."""
    g, x, tokens = gen(36), torch.zeros(rows, vocab, device=DEV, dtype=TYPES[act]), i32([0] * rows)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = K.token_logprobs(x, tokens, 9)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(2):
        x.copy_((2 * normal(g, rows, vocab)).to(x.dtype))
        tokens.copy_(torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32))
        graph.replay()
        for p, q in zip(captured, K.token_logprobs(x, tokens, 9)):
            assert torch.equal(p, q)


def test_logprobs_of_tokens_outside_the_vocabulary():
    x = normal(gen(34), 2, 100)
    lp = K.token_logprobs(x, i32([[100, -1, 2 ** 31 - 1, -2 ** 31], [99, 0, 101, 5]]))[0]
    assert lp[0].tolist() == [-math.inf, 0.0, -math.inf, 0.0] and lp[1, 2] == -math.inf
    assert torch.isfinite(lp[1, [0, 1, 3]]).all()


def test_logprobs_of_broadcast_rows_and_repeats():
    x = normal(gen(35), 1, 5000).expand(300, 5000)
    tokens = torch.arange(300, device=DEV, dtype=torch.int32)
    check_logprobs(x, tokens, 20)
    a, b = K.token_logprobs(x, tokens, 20), K.token_logprobs(x.contiguous(), tokens, 20)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert (a[1] == a[1][0]).all() and (a[3] == a[3][0]).all()


# ------------------------------------------------------------------ together
def test_scoring_prompts_and_serving_tokens():
    """Two layers of a small recurrent model over slots: prompts of different lengths scored at once, then a token of
    each; requests come, end and give their slots to others.  Each operator is held to 64-bit books of every request's
    rows and states, which go on from call to call and take what the operators before it made of the request."""
    g = gen(40)
    vocab, dim, ch, n, rank = 97, 24, 40, 16, 5
    embed, head = 0.5 * normal(g, vocab, dim), 0.3 * normal(g, dim, vocab)
    layers = [dict(into=0.3 * normal(g, dim, 2 * ch), conv=normal(g, ch, 4), bias=0.1 * normal(g, ch),
                   low=0.3 * normal(g, ch, rank + 2 * n), up=0.3 * normal(g, rank, ch), dt_bias=normal(g, ch) - 3,
                   a=-torch.exp(normal(g, ch, n)), d=normal(g, ch), back=0.2 * normal(g, ch, dim),
                   cs=normal(g, 5, 3, ch), hs=normal(g, 5, ch, n), books={}) for _ in range(2)]
    begun = (torch.zeros(3, ch, device=DEV, dtype=F64), torch.zeros(ch, n, device=DEV, dtype=F64), 0.0)

    def serve(tokens, cu, slots, fresh):
        """Logits of packed requests (cu: their offsets) or of one token each (cu None)."""
        x, at = embed[tokens.long()], dict(slots=i32(slots))
        if fresh:
            at["init"] = i32([-1] * len(slots))
        for p in layers:
            both = x @ p["into"]
            raw, z = both[:, :ch], both[:, ch:]
            conv = dict(weight=p["conv"], bias=p["bias"], state=p["cs"], **at)
            u = K.causal_conv_step(raw, **conv) if cu is None else K.causal_conv(raw, cu=i32(cu), **conv)
            low = u @ p["low"]
            t = dict(x=u, dt=low[:, :rank] @ p["up"], a=p["a"], b=low[:, rank:rank + n], c=low[:, rank + n:], d=p["d"], z=z,
                     dt_bias=p["dt_bias"], state=p["hs"], **at)
            y = K.selective_step(**t) if cu is None else K.selective_scan(cu=i32(cu), **t)
            for s, (i, j) in enumerate(spans(cu or list(range(len(slots) + 1)), len(tokens))):
                if slots[s] < 0:
                    continue
                rows, h, e = begun if fresh else p["books"][slots[s]]
                want, bound, rows = conv64(raw[i:j], p["conv"], p["bias"], rows, True)
                close(u[i:j], want, bound)
                want, bound, h, e = scan64(u[i:j], t["dt"][i:j], p["a"], t["b"][i:j, None], t["c"][i:j, None], p["d"], z[i:j],
                                           p["dt_bias"], h, e)
                close(y[i:j], want, bound)
                close(p["hs"][slots[s]], h, e)
                assert torch.equal(p["cs"][slots[s]].to(F64), rows)
                p["books"][slots[s]] = rows, h, e
            x = x + y @ p["back"]
        return x @ head

    texts = {}
    for lens, slots in (([7, 1, 30], [3, 0, 2]), ([12, 45], [1, 3])):  # slot 3 is given on
        tokens = torch.randint(0, vocab, (sum(lens),), generator=g, device=DEV, dtype=torch.int32)
        cu = list(itertools.accumulate(lens, initial=0))
        logits = serve(tokens, cu, slots, True)
        follows = torch.cat([tokens[1:], tokens[:1]])
        follows[torch.tensor(cu[1:], device=DEV) - 1] = -1  # nothing follows a text's last token yet
        check_logprobs(logits, follows, 3)
        ids = K.token_logprobs(logits, top=1)[2]
        for s, (i, j) in enumerate(spans(cu, len(tokens))):
            texts[slots[s]] = torch.cat([tokens[i:j], ids[j - 1]])
        for _ in range(4):
            live = list(texts)
            tokens = torch.cat([texts[slot][-1:] for slot in live] + [i32([0])])  # and one row of padding
            logits = serve(tokens, None, live + [-1], False)[:len(live)]
            check_logprobs(logits, tokens[:-1].contiguous(), 2)
            ids = K.token_logprobs(logits, top=1)[2]
            for k, slot in enumerate(live):
                texts[slot] = torch.cat([texts[slot], ids[k]])
