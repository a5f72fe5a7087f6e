"""The paged key-value cache on the GPU, against plain 64-bit implementations.

Tolerances count roundings.  With u = 2^-24 (half a step of float32) and h the
output type's half step (finfo.eps / 2):

append: cos and sin of a reduced angle are off by at most 3u (the fraction of a
turn rounded to 32 bits, times 2 pi) + 4u (two units in the last place) + 8u
(two roundings to 64 bits of 2^31 / (2 pi) turns) + 6u (the same in the reference
here); each product and the sum round once more: 24u (|a| + |b|), and h |result|
when it is stored.

attention: a score, a sum of dh products, is off by at most s = 2 (dh + 8) u
scale sum_d |q_d k_d| (2 for accumulators that may round towards zero); every
weight by 2 s + 16u relative, the two sums of n weights by 2 n u each; so the
result by (2 s + 2 (n + 32) u) max |v| and h |result|, and the logarithm by s +
2 (n + 32) u + 2u |lse|.  Exact tests (whole-number values under equal weights)
hold the long sums."""
import math
import os
import re
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from krikil_rs_b200 import KrikilError, kernels as K, launch_count  # noqa: E402
from krikil_rs_b200._lib import (PAGES_BAD_LENGTH, PAGES_EXHAUSTED, PAGES_OVERFLOW, PAGES_ROW_FULL,  # noqa: E402
                                 PAGES_ROWS)

DEV = torch.device("cuda:0")
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
IDS = ["f32", "f32-f16", "f32-bf16", "f16", "bf16"]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def i32(values):
    return torch.tensor(values, device=DEV, dtype=torch.int32)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Pool:
    """Requests of the given lengths on random pages; every cell that no request holds is NaN, unused
    table entries are far outside the pool."""

    def __init__(self, lens, hkv, dh, page, cache, seed, spare=3, layout="pthd", pad=0, fill=None):
        g = gen(seed)
        self.lens_h, self.page = list(lens), page
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        width = max(1, max(need))
        order = torch.randperm(self.pages, generator=g, device=DEV).tolist()
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [2 ** 30] * (width - n))
            at += n
        self.table, self.lens = i32(rows), i32(lens)
        full = torch.full((2, self.pages, page, hkv, dh + pad), float("nan"), device=DEV, dtype=cache)
        if layout == "phtd":
            full = torch.full((2, self.pages, hkv, page, dh + pad), float("nan"), device=DEV, dtype=cache)
            full = full.transpose(2, 3)
        self.kc, self.vc = full[0][..., :dh], full[1][..., :dh]
        self.k, self.v = [], []  # per request [n, hkv, dh], as stored
        for b, n in enumerate(lens):
            if fill is None:
                k = torch.randn(n, hkv, dh, generator=g, device=DEV).to(cache)
                v = torch.randn(n, hkv, dh, generator=g, device=DEV).to(cache)
            else:
                k, v = fill(n, hkv, dh, g)
                k, v = k.to(cache), v.to(cache)
            self.k.append(k)
            self.v.append(v)
            if n:
                j = torch.arange(n, device=DEV)
                where = self.table[b, j // page].long(), j % page
                self.kc[where], self.vc[where] = k, v


def attn_reference(pool, q, scale, window=0, keep=None):
    """out, lse and their tolerances in 64 bits, request by request."""
    b, hq, dh = q.shape
    out = torch.zeros(b, hq, dh, device=DEV, dtype=torch.float64)
    lse = torch.full((b, hq), -math.inf, device=DEV, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(pool.lens_h):
        first = max(0, n - window) if window else 0
        js = [j for j in range(first, n) if keep is None or keep(i, j)]
        if not js:
            continue
        k, v = pool.k[i][js].double(), pool.v[i][js].double()
        hkv = k.shape[1]
        share = hq // hkv
        qi = q[i].double().reshape(hkv, share, dh)
        x = torch.einsum("hgd,jhd->hgj", qi, k) * scale
        size = torch.einsum("hgd,jhd->hgj", qi.abs(), k.abs()).amax(-1) * abs(scale)
        p = torch.softmax(x, -1)
        out[i] = torch.einsum("hgj,jhd->hgd", p, v).reshape(hq, dh)
        lse[i] = torch.logsumexp(x, -1).reshape(hq)
        s = 2 * (dh + 8) * U * size
        n = len(js)
        top = v.abs().amax((0, 2))[:, None]
        tol[i] = (((2 * s + 2 * (n + 32) * U) * top).reshape(hq, 1) + half_step(q.dtype) * out[i].abs()
                  + torch.finfo(q.dtype).tiny)
        ltol[i] = (s + 2 * (n + 32) * U).reshape(hq) + 2 * U * lse[i].abs()
    return out, lse, tol, ltol


def check_attn(pool, q, window=0, scale=None, keep=None, **kw):
    sc = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out, lse = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, scale=scale, window=window,
                                   return_lse=True, **kw)
    ref, rl, tol, ltol = attn_reference(pool, q, sc, window, keep)
    empty = rl == -math.inf
    assert torch.equal(lse[empty], torch.full_like(lse[empty], -math.inf))
    assert torch.equal(out[empty], torch.zeros_like(out[empty]))
    bad = (out.double() - ref).abs() > tol
    assert not bad.any() and not out.isnan().any(), ((out.double() - ref).abs() / tol).nan_to_num(math.inf).max().item()
    off = (lse.double() - rl).abs()[~empty]
    assert (off <= ltol[~empty]).all(), (off / ltol[~empty]).max().item()
    return out, lse


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page", [(8, 8, 76, 16), (8, 8, 64, 8), (32, 8, 128, 64), (4, 4, 4, 1),
                                            (7, 1, 80, 32), (12, 4, 96, 4), (16, 2, 256, 16), (33, 1, 192, 2),
                                            (40, 2, 36, 128), (9, 1, 200, 16), (3, 3, 252, 2)])
def test_attention_types_heads_and_lengths(act, cache, hq, hkv, dh, page):
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 255, 300]
    pool = Pool(lens, hkv, dh, page, cache, seed=dh + page)
    q = torch.randn(len(lens), hq, dh, generator=gen(5), device=DEV).to(act)
    check_attn(pool, q)
    check_attn(pool, q, window=40)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page,lens", [
    (8, 8, 64, 16, [5000, 1, 0, 777]), (32, 8, 128, 16, [4097]), (4, 1, 76, 32, [1] * 300 + [9000]),
    (16, 2, 256, 1, [2500, 3]), (2, 2, 128, 4096, [10000]), (64, 1, 64, 8, [3001, 2999])])
@pytest.mark.parametrize("window", [0, 1, 1029])
def test_equal_weights_of_whole_numbers_are_exact(act, cache, hq, hkv, dh, page, lens, window):
    """With q = 0 every weight is 1 and the values' sums, whole numbers below 2^24, are exact in any
    order: a key that is left out, read twice or read from another page shows.  The quotient is off by
    the reciprocal's and the product's rounding (2u each, with room for an approximate reciprocal of
    one unit more) and by the store."""
    def fill(n, h, d, g):
        return (torch.randn(n, h, d, generator=g, device=DEV),
                torch.randint(-8, 9, (n, h, d), generator=g, device=DEV).float())
    pool = Pool(lens, hkv, dh, page, cache, seed=len(lens) + dh, fill=fill)
    q = torch.zeros(len(lens), hq, dh, device=DEV, dtype=act)
    out, lse = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, window=window, return_lse=True)
    for i, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        seen = pool.v[i][first:].double().sum(0).repeat_interleave(hq // hkv, 0) / max(1, n - first)
        tol = (8 * U + half_step(act)) * seen.abs() + torch.finfo(act).tiny
        assert ((out[i].double() - seen).abs() <= tol).all(), (i, n)
        want = math.log(n - first) if n else -math.inf
        assert torch.allclose(lse[i].double(), torch.full_like(lse[i].double(), want), rtol=8 * U, atol=8 * U)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("layout,pad,hq,hkv,dh", [("pthd", 0, 8, 4, 76), ("phtd", 0, 8, 4, 76), ("pthd", 4, 8, 4, 76),
                                                  ("phtd", 4, 6, 2, 64), ("phtd", 0, 32, 8, 128),
                                                  ("pthd", 52, 4, 1, 12), ("phtd", 8, 16, 2, 128)])
def test_attention_layouts_and_strides(act, cache, layout, pad, hq, hkv, dh):
    lens = [37, 0, 200, 129, 64]
    pool = Pool(lens, hkv, dh, 16, cache, seed=3, layout=layout, pad=pad)
    packed = torch.randn(len(lens), (hq + 2 * hkv) * dh + 4, generator=gen(6), device=DEV).to(act)
    q = packed[:, 4:4 + hq * dh].unflatten(1, (hq, dh))
    whole = torch.full((len(lens) + 2, hq + 3, dh + 12), 7.0, device=DEV, dtype=act)
    out = whole[1:-1, 1:hq + 1, 4:4 + dh]
    got, lse = check_attn(pool, q, out=out)
    assert got.data_ptr() == out.data_ptr()
    inside = torch.zeros_like(whole, dtype=torch.bool)
    inside[1:-1, 1:hq + 1, 4:4 + dh] = True
    assert (whole[~inside] == 7.0).all()  # nothing around the rows is written
    same, _ = check_attn(pool, q.contiguous())
    assert torch.equal(same, out)  # where rows lie does not change them


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_table_rows_may_be_strided(act, cache):
    pool = Pool([50, 3, 90], 2, 64, 8, cache, seed=9)
    q = torch.randn(3, 4, 64, generator=gen(1), device=DEV).to(act)
    a = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens)
    wide = torch.full((3, pool.table.shape[1] + 5), -9, device=DEV, dtype=torch.int32)
    wide[:, :pool.table.shape[1]] = pool.table
    assert torch.equal(a, K.attn_decode_paged(q, pool.kc, pool.vc, wide[:, :pool.table.shape[1]], pool.lens))


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_large_scores_and_scales(act, cache):
    """Scores in the thousands (one key takes all the weight), a negative scale, a scale of 0."""
    pool = Pool([1, 70, 400], 2, 64, 16, cache, seed=4)
    q = (100 * torch.randn(3, 6, 64, generator=gen(2), device=DEV)).to(act)
    for scale in (1.0, -1.0, 1e-3, 0.0):
        check_attn(pool, q, scale=scale)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_small_and_uneven_queries(act, cache):
    """Queries whose elements differ a thousandfold, large ones and tiny ones, under a scale that brings the scores
    back to one: parts of q that a shorter type would drop count."""
    pool = Pool([130, 17], 2, 64, 16, cache, seed=14)
    q = torch.randn(2, 4, 64, generator=gen(3), device=DEV)
    q[:, :, 1::2] *= 1e-3
    for size, scale in ((1.0, None), (2.0 ** -12, 512.0), (2.0 ** 10, 2.0 ** -13)):
        check_attn(pool, (q * size).to(act), scale=scale)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_one_dominant_key_and_a_long_faint_tail(act, cache):
    """One key of weight 1 and thousands near 2^-20: together they matter, each is faint."""
    n, dh = 6000, 64
    def fill(n, h, d, g):
        k = torch.zeros(n, h, d, device=DEV)
        k[:, :, 0] = -14.0
        k[n // 3, :, 0] = 0.0
        return k, torch.randn(n, h, d, generator=g, device=DEV)
    pool = Pool([n, 40], 1, dh, 16, cache, seed=8, fill=fill)
    q = torch.zeros(2, 8, dh, device=DEV, dtype=act)
    q[:, :, 0] = 1.0
    check_attn(pool, q, scale=1.0)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("dh,pad", [(64, 0), (64, 4), (76, 0), (76, 4), (120, 12)])
def test_infinities_and_nan_stay_where_they_are(act, cache, dh, pad):
    """A NaN key reaches its own request and cache head alone; a key of score -inf gets weight 0, and a row
    of nothing but -inf scores gives zeros; an infinite value of a visible key leaves its own column not finite
    (infinite or, where the product of a weight's parts is undefined, NaN) and nothing else."""
    def make(seed):
        return Pool([64, 90, 33, 5], 2, dh, 16, cache, seed=seed, pad=pad)
    pool = make(7)
    q = torch.rand(4, 4, dh, generator=gen(4), device=DEV).to(act) + 0.5
    clean, _ = check_attn(pool, q)
    def at(b, j):
        return int(pool.table[b, j // 16]), j % 16
    pool.kc[at(1, 40)][0] = float("nan")
    out = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens)
    assert out[1, :2].isnan().all()
    others = torch.ones(4, 4, dtype=torch.bool, device=DEV)
    others[1, :2] = False
    assert torch.equal(out[others], clean[others])
    pool = make(7)
    pool.kc[at(2, 10)][1] = -float("inf")
    out, lse = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, return_lse=True)
    pool.k[2][10, 1] = -1e4  # a weight of 0 in 32 bits
    ref, rl, tol, ltol = attn_reference(pool, q, 1 / math.sqrt(dh))
    # sum |q k| of the key that was moved away has no part in the others' rounding
    assert ((out.double() - ref).abs() <= tol).all() and not lse.isnan().any()
    pool = make(7)
    for j in range(5):
        pool.kc[at(3, j)][:] = -float("inf")
    out, lse = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, return_lse=True)
    assert (out[3] == 0).all() and (lse[3] == -math.inf).all()
    assert torch.equal(out[:3], clean[:3])
    pool = make(7)
    pool.vc[at(0, 3)][0, 5] = float("inf")
    out = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens)
    assert not out[0, :2, 5].isfinite().any()
    out[0, :2, 5] = clean[0, :2, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("dh,pad,page", [(64, 4, 16), (76, 0, 16), (76, 0, 4), (76, 4, 16), (12, 0, 16), (128, 4, 32),
                                         (252, 0, 16), (256, 4, 16)])
def test_nan_in_the_neighbouring_heads(act, cache, dh, pad, page):
    """Three cache heads of which the outer ones are NaN throughout: the one between, whose rows may begin and end
    within the same 16 bytes, is what it was."""
    pool = Pool([70, 9, 0, 33], 3, dh, page, cache, seed=6, pad=pad)
    q = torch.randn(4, 6, dh, generator=gen(4), device=DEV).to(act)
    clean, lse = check_attn(pool, q)
    for c in (pool.kc, pool.vc):
        c[:, :, 0] = float("nan")
        c[:, :, 2] = float("nan")
    out, got = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, return_lse=True)
    assert torch.equal(out[:, 2:4], clean[:, 2:4]) and torch.equal(got[:, 2:4], lse[:, 2:4])
    assert out[:2, [0, 1, 4, 5]].isnan().all()


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("page", [4, 16, 64])
def test_pages_outside_the_pool_are_left_out(act, cache, page):
    lens = [130, 64, 200]
    pool = Pool(lens, 2, 64, page, cache, seed=2)
    q = torch.randn(3, 4, 64, generator=gen(8), device=DEV).to(act)
    lost = {(0, 1): -1, (0, 64 // page): pool.pages, (1, 0): 2 ** 31 - 1, (2, 128 // page): -2 ** 31}
    for (b, i), bad in lost.items():
        pool.table[b, i] = bad
    check_attn(pool, q, keep=lambda b, j: (b, j // page) not in lost)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("page,window", [(4, 30), (16, 1), (16, 50), (64, 200), (2, 333)])
def test_what_lies_before_the_window_does_not_matter(act, cache, page, window):
    """Cells before the window hold NaN, and whole pages before it are gone from the table."""
    lens = [5, 64, 65, 400, 1500, 0]
    pool = Pool(lens, 2, 76, page, cache, seed=page)
    q = torch.randn(len(lens), 6, 76, generator=gen(9), device=DEV).to(act)
    want, lse = check_attn(pool, q, window=window)
    for b, n in enumerate(lens):
        for j in range(max(0, n - window)):
            if j // page == max(0, n - window) // page:  # the page on which the window begins
                at = int(pool.table[b, j // page]), j % page
                pool.kc[at] = float("nan")
                pool.vc[at] = float("nan")
        pool.table[b, :max(0, n - window) // page] = -1
    got, got_lse = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, window=window, return_lse=True)
    assert torch.equal(got, want) and torch.equal(got_lse, lse)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_lengths_outside_the_table(act, cache):
    """Longer than width * page_size: cut there; negative: empty."""
    pool = Pool([64, 64, 64], 2, 64, 16, cache, seed=2)
    q = torch.randn(3, 4, 64, generator=gen(8), device=DEV).to(act)
    want = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens)
    got = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, i32([65, 2 ** 31 - 1, -5]))
    assert torch.equal(got[:2], want[:2]) and (got[2] == 0).all()


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_attention_is_repeatable_and_the_bound_only_sizes_it(act, cache):
    pool = Pool([900, 0, 3000, 12], 2, 128, 16, cache, seed=12)
    q = torch.randn(4, 8, 128, generator=gen(3), device=DEV).to(act)
    first, _ = check_attn(pool, q)
    work = torch.full((K.attn_paged_work_floats(4, 8, 2, 128, 3008) + 8,), float("nan"), device=DEV)
    for _ in range(3):
        again = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, work=work)
        assert torch.equal(first, again)
    for bound in (1, 100, 3000, 2 ** 31 - 1):  # even a bound that is too small
        check_attn(pool, q, max_len=bound, work=work)


def test_scratch_that_is_too_small_is_refused():
    pool = Pool([64000], 2, 64, 16, F32, seed=2)
    q = torch.randn(1, 4, 64, device=DEV)
    need = K.attn_paged_work_floats(1, 4, 2, 64, 64000)
    assert need
    for work in (torch.empty(need - 1, device=DEV), torch.empty(need + 1, device=DEV)[1:]):
        with pytest.raises(KrikilError, match="work"):
            K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, work=work)
    K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, work=torch.empty(need, device=DEV))


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("b,hq,dh,page,longest,window", [
    (10, 32, 64, 16, 8192, 0), (10, 17, 128, 64, 5000, 0), (7, 48, 64, 8, 6000, 0), (4, 71, 80, 32, 12000, 0),
    (5, 64, 76, 16, 9000, 0), (10, 24, 64, 4, 9000, 5000)])
def test_many_heads_on_one_cache_head(act, cache, b, hq, dh, page, longest, window):
    """17 and more query heads a cache head, at bounds where the number of pieces, which differs from type to type,
    decides between clusters and shares: whichever a type takes has its scratch."""
    lens = [longest, 0, 1, longest // 2] + [longest - 17 * i for i in range(b - 4)]
    pool = Pool(lens, 1, dh, page, cache, seed=hq)
    assert K.attn_paged_work_floats(b, hq, 1, dh, pool.table.shape[1] * page, window) > 0
    check_attn(pool, torch.randn(b, hq, dh, generator=gen(hq), device=DEV).to(act), window=window)


@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)])
def test_attention_replayed_from_a_graph_on_another_stream(act, cache):
    """A captured call follows the lengths, table and queries that it finds at replay, beside eager calls of the
    same tensors with their own scratch."""
    lens = [10, 0, 700, 64]
    pool = Pool([800] * 4, 2, 64, 16, cache, seed=21)
    q = torch.randn(4, 8, 64, generator=gen(3), device=DEV).to(act)
    now = i32(lens)
    s = torch.cuda.Stream()
    out, work = torch.empty_like(q), torch.empty(K.attn_paged_work_floats(4, 8, 2, 64, 800), device=DEV)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, now, out=out, work=work, max_len=800)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, now, out=out, work=work, max_len=800)
    for step, lens in enumerate(([10, 0, 700, 64], [0, 0, 0, 0], [800, 800, 800, 800], [1, 2, 3, 799])):
        now.copy_(i32(lens))
        q.copy_(torch.randn(4, 8, 64, generator=gen(step), device=DEV).to(act))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        eager = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, now, max_len=800)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        pool.lens_h = lens
        ref, _, tol, _ = attn_reference(pool, q, 1 / 8)
        assert ((out.double() - ref).abs() <= tol).all()


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements a cache, of which the last and first pages are used."""
    hkv, dh, page = 8, 128, 16
    pages = 2 ** 31 // (hkv * dh * page) + 40
    if torch.cuda.mem_get_info()[0] < 5 * pages * page * hkv * dh:
        pytest.skip("not enough memory")
    kc = torch.empty(pages, page, hkv, dh, device=DEV, dtype=BF16)
    vc = torch.empty_like(kc)
    n = 100
    rows = [[pages - 1 - i for i in range(7)], [0, pages - 9, 1, pages - 10, 2, pages - 11, 3]]
    table, lens = i32(rows), i32([0, 0])
    k = torch.randn(2 * n, hkv, dh, generator=gen(1), device=DEV).to(BF16)
    v = torch.randn(2 * n, hkv, dh, generator=gen(2), device=DEV).to(BF16)
    slots = i32([rows[b][j // page] * page + j % page for b in range(2) for j in range(n)])
    K.rope_kv_append_paged(None, k, v, kc, vc, slots, torch.zeros_like(slots))  # position 0 turns nothing
    q = torch.randn(2, 32, dh, generator=gen(3), device=DEV).to(BF16)
    pool = Pool.__new__(Pool)
    pool.kc, pool.vc, pool.table, pool.lens_h, pool.lens = kc, vc, table, [n, n], i32([n, n])
    pool.k, pool.v = [k[:n], k[n:]], [v[:n], v[n:]]
    check_attn(pool, q)


# ------------------------------------------------------------------ RoPE + append
def rotated(x, positions, rot, theta=10000.0):
    """The rotation in 64 bits, and its tolerance before the store."""
    x = x.double()
    half = rot // 2
    if half == 0:
        return x, torch.zeros_like(x)
    rate = theta ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / rot)
    turn = positions.double()[:, None] * rate
    c, s = torch.cos(turn)[:, None], torch.sin(turn)[:, None]
    a, b = x[..., :half], x[..., half:rot]
    t = 24 * U * (a.abs() + b.abs())
    return (torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1),
            torch.cat([t, t, torch.zeros_like(x[..., rot:])], -1))


def close(got, ref, tol):
    off = (got.double() - ref).abs()
    lim = tol + half_step(got.dtype) * (ref.abs() + tol) + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert (off <= lim).all(), (off - lim).max().item()


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("t,hq,hkv,dh,rot,page,far", [
    (1, 8, 8, 76, 76, 16, 2048), (37, 32, 8, 128, 128, 16, 10 ** 6), (300, 4, 1, 64, 32, 1, 2 ** 31 - 1),
    (65, 7, 7, 80, 40, 8, 32768), (5, 2, 2, 256, 256, 256, 10 ** 6), (129, 1, 1, 4, 2, 4, 100),
    (40, 6, 2, 96, 0, 16, 1000), (1111, 12, 4, 192, 190, 32, 5000), (33, 3, 1, 4, 4, 8, 100), (70, 5, 5, 12, 12, 16, 999),
    (21, 2, 1, 252, 252, 16, 4000), (300, 9, 3, 36, 36, 32, 70000), (50, 4, 2, 76, 38, 16, 2048)])
def test_append_types_heads_and_positions(act, cache, t, hq, hkv, dh, rot, page, far):
    g = gen(t + dh)
    pages = -(-t // page) + 2
    packed = torch.randn(t, (hq + 2 * hkv) * dh, generator=g, device=DEV).to(act)
    q, k, v = (x.unflatten(1, (-1, dh)) for x in packed.split([hq * dh, hkv * dh, hkv * dh], 1))
    before = packed.clone()
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:t].int()
    positions = torch.randint(0, far, (t,), generator=g, device=DEV, dtype=torch.int64).int()
    kc = torch.full((pages, page, hkv, dh), 9.0, device=DEV, dtype=cache)
    vc = torch.full_like(kc, -9.0)
    got = K.rope_kv_append_paged(q, k, v, kc, vc, slots, positions, rot_dim=rot)
    assert torch.equal(packed, before)
    close(got, *rotated(q, positions, rot))
    ref, tol = rotated(k, positions, rot)
    close(kc.view(-1, hkv, dh)[slots.long()], ref, tol)
    assert torch.equal(vc.view(-1, hkv, dh)[slots.long()], v.to(cache))
    rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    rest[slots.long()] = False
    assert (kc.view(-1, hkv, dh)[rest] == 9.0).all() and (vc.view(-1, hkv, dh)[rest] == -9.0).all()
    # in place: the same values
    K.rope_kv_append_paged(q, k, v, kc, vc, slots, positions, rot_dim=rot, q_out=q)
    assert torch.equal(q, got) and torch.equal(packed[:, hq * dh:], before[:, hq * dh:])


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("pad,dh,layout", [(0, 76, "phtd"), (4, 76, "pthd"), (12, 64, "phtd"), (8, 128, "phtd")])
def test_append_layouts_padding_and_bad_slots(act, cache, pad, dh, layout):
    """Rows behind the last sequence (slot -1) and slots outside the pool write nothing, NaN in them included;
    cells between the heads of a padded layout are left alone."""
    t, hq, hkv, page, pages = 23, 6, 3, 8, 5
    shape = (pages, page, hkv, dh + pad) if layout == "pthd" else (pages, hkv, page, dh + pad)
    raw = torch.full((2,) + shape, 5.0, device=DEV, dtype=cache)
    view = raw if layout == "pthd" else raw.transpose(2, 3)
    kc, vc = view[0][..., :dh], view[1][..., :dh]
    g = gen(77)
    q = torch.randn(t, hq, dh + 4, generator=g, device=DEV).to(act)[..., :dh]
    k = torch.randn(hkv, t, dh, generator=g, device=DEV).to(act).transpose(0, 1)
    v = torch.randn(t, hkv, dh + 8, generator=g, device=DEV).to(act)[..., 8:]
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:t].int()
    skip = [3, 4, 11, 20, 21, 22]
    for i, s in zip(skip, (-1, pages * page, 2 ** 31 - 1, -1, -2 ** 31, -1)):
        slots[i] = s
    q[skip[-1]] = float("nan")
    k[skip[-1]] = float("nan")
    positions = torch.randint(0, 999, (t,), generator=g, device=DEV, dtype=torch.int32)
    positions[skip[0]] = -7
    q_out = torch.full((t, hq, dh), 3.0, device=DEV, dtype=act)
    K.rope_kv_append_paged(q, k, v, kc, vc, slots, positions, theta=500000.0, q_out=q_out)
    keep = [i for i in range(t) if i not in skip]
    assert (q_out[skip] == 3.0).all()
    close(q_out[keep], *rotated(q[keep], positions[keep], dh, 500000.0))
    p, o = slots[keep].long() // page, slots[keep].long() % page
    close(kc[p, o], *rotated(k[keep], positions[keep], dh, 500000.0))
    assert torch.equal(vc[p, o], v[keep].to(cache))
    kc[p, o], vc[p, o] = 5.0, 5.0
    assert (raw == 5.0).all()


@pytest.mark.parametrize("act,cache,t,hq,hkv,dh", [
    (F16, F16, 30000, 1, 1, 256), (BF16, BF16, 30011, 1, 1, 256), (F32, F32, 9001, 2, 1, 256), (F32, BF16, 40003, 0, 1, 64),
    (BF16, BF16, 700, 128, 16, 128), (F32, F16, 601, 71, 71, 76), (F16, F16, 333, 40, 8, 192)])
def test_append_long_runs_of_rows_and_many_heads(act, cache, t, hq, hkv, dh):
    """Few heads, so that a block takes several rows side by side in long runs, and more heads than a block's threads
    take at once."""
    g = gen(t)
    page, pages = 64, -(-t // 64)
    q = torch.randn(t, hq, dh, generator=g, device=DEV).to(act) if hq else None
    k, v = (torch.randn(t, hkv, dh, generator=g, device=DEV).to(act) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:t].int()
    slots[::17] = -1
    positions = torch.randint(0, 10 ** 6, (t,), generator=g, device=DEV, dtype=torch.int32)
    kc, vc = (torch.full((pages, page, hkv, dh), 9.0, device=DEV, dtype=cache) for _ in range(2))
    keep = slots >= 0
    out = torch.full((t, hq, dh), 3.0, device=DEV, dtype=act) if hq else None
    assert K.rope_kv_append_paged(q, k, v, kc, vc, slots, positions, q_out=out) is out
    if hq:
        close(out[keep], *rotated(q[keep], positions[keep], dh))
        assert (out[~keep] == 3.0).all()
    at = slots[keep].long()
    close(kc.view(-1, hkv, dh)[at], *rotated(k[keep], positions[keep], dh))
    assert torch.equal(vc.view(-1, hkv, dh)[at], v[keep].to(cache))
    kc.view(-1, hkv, dh)[at] = 9.0
    assert (kc == 9.0).all()


def test_append_stores_the_nearest_values():
    """float32 values into 16-bit caches: the values' own rounding (to even at ties, overflow to infinity), the
    last of what fits; NaN and infinities stay."""
    x = torch.tensor([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 65504.0, 65519.9, 65520.0, 3.4e38, float("inf"),
                      -float("inf"), float("nan"), 2.0 ** -24, 2.0 ** -25, 2.0 ** -26, -0.0, 2.0 ** -140, 1e-8, 3.0],
                     device=DEV)
    for cache in (F16, BF16):
        k = x.reshape(1, 1, 16)
        kc, vc = (torch.zeros(1, 1, 1, 16, device=DEV, dtype=cache) for _ in range(2))
        K.rope_kv_append_paged(None, k, k, kc, vc, i32([0]), i32([5]), rot_dim=0)
        for c in (kc, vc):
            assert torch.equal(c.view(-1).view(torch.int16)[x == x], x.to(cache).view(torch.int16)[x == x])
            assert c.view(-1)[8].isnan()


# ------------------------------------------------------------------ pages
class Books:
    """The same bookkeeping in plain Python."""

    def __init__(self, batch, width, num_pages, page, seed):
        rng = np.random.default_rng(seed)
        self.page, self.width = page, width
        self.free = [int(x) for x in rng.permutation(num_pages)]
        self.num_pages = num_pages
        self.lens = [0] * batch
        self.rows = [[] for _ in range(batch)]

    def fits(self, new, rows):
        need, st = 0, 0
        for b, n in enumerate(new):
            want = -(-(self.lens[b] + n) // self.page)
            st |= PAGES_ROW_FULL if want > self.width else 0
            need += want - len(self.rows[b])
        return st | (PAGES_EXHAUSTED if need > len(self.free) else 0) | (PAGES_ROWS if sum(new) > rows else 0)

    def plan(self, new):
        positions, slots = [], []
        for b, n in enumerate(new):
            while len(self.rows[b]) < -(-(self.lens[b] + n) // self.page):
                self.rows[b].append(self.free.pop())
            for i in range(self.lens[b], self.lens[b] + n):
                positions.append(i)
                slots.append(self.rows[b][i // self.page] * self.page + i % self.page)
            self.lens[b] += n
        return positions, slots

    def release(self, done):
        for b, d in enumerate(done):
            if d:
                self.free += self.rows[b]
                self.rows[b], self.lens[b] = [], 0


def device_books(books, batch):
    free = torch.full((books.num_pages,), -1, device=DEV, dtype=torch.int32)
    free[:len(books.free)] = i32(books.free)
    return {"lens": torch.zeros(batch, device=DEV, dtype=torch.int32), "free": free,
            "count": i32([len(books.free)]),
            "table": torch.full((batch, books.width), -1, device=DEV, dtype=torch.int32)}


def same_books(d, books):
    assert d["lens"].tolist() == books.lens and d["count"].item() == len(books.free)
    assert d["free"][:len(books.free)].tolist() == books.free
    table = d["table"].tolist()
    for b, row in enumerate(books.rows):
        assert table[b][:len(row)] == row


@pytest.mark.parametrize("batch,width,num_pages,page,most,rows", [
    (1, 4, 4, 16, 30, 64), (3, 8, 20, 1, 5, 20), (61, 33, 900, 64, 300, 20000), (1024, 5, 3000, 16, 3, 2048),
    (2500, 3, 7000, 8, 2, 6000), (5, 600, 2500, 16, 6000, 40000), (70, 20, 1000, 4, 40, 4096)])
def test_planned_steps_match_plain_books(batch, width, num_pages, page, most, rows):
    """Steps of random new tokens and releases, in place: pages, slots, positions and lengths as in plain Python,
    and steps that do not fit leave everything as it was."""
    rng = np.random.default_rng(batch)
    books = Books(batch, width, num_pages, page, seed=batch)
    d = device_books(books, batch)
    refusals = 0
    for step in range(14):
        if step % 3 == 2:
            done = rng.random(batch) < 0.4
            K.kv_page_release(torch.tensor(done, device=DEV), d["lens"], d["table"], d["free"], d["count"], page,
                              lens_out=d["lens"], free_count_out=d["count"])
            books.release(done)
            same_books(d, books)
        new = rng.integers(0, most + 1, batch)
        if step % 4 == 0:
            new[rng.random(batch) < 0.7] = 0
        new = [int(x) for x in new]
        want = books.fits(new, rows)
        before = d["table"].clone()
        _, _, cu, positions, slots, status = K.kv_page_plan(i32(new), d["lens"], d["table"], d["free"], d["count"],
                                                            page, rows, lens_out=d["lens"],
                                                            free_count_out=d["count"])
        assert status.item() == want
        if want:
            refusals += 1
            assert torch.equal(d["table"], before) and not cu.any() and (slots == -1).all() and not positions.any()
        else:
            p, s = books.plan(new)
            assert cu.tolist() == [0] + np.cumsum(new).tolist()
            assert positions[:len(p)].tolist() == p and not positions[len(p):].any()
            assert slots[:len(s)].tolist() == s and (slots[len(s):] == -1).all()
        same_books(d, books)
    assert refusals < 14


def test_page_requests_that_do_not_fit():
    d = dict(lens=i32([3, 0]), table=i32([[4, 5], [6, 7]]), free=i32([0, 1, 2, 3]), count=i32([2]))

    def plan(new, rows=64, **kw):
        a = dict(d, **kw)
        out = K.kv_page_plan(i32(new), a["lens"], a["table"], a["free"], a["count"], 4, rows)
        return out[5].item(), out

    assert plan([1, 4])[0] == 0
    st, out = plan([2, 8])
    assert st == PAGES_EXHAUSTED and out[0].tolist() == [3, 0] and out[1].item() == 2
    assert plan([6, 0])[0] == PAGES_ROW_FULL
    assert plan([1, 4], rows=4)[0] == PAGES_ROWS and plan([1, 4], rows=5)[0] == 0
    assert plan([0, 0], rows=0)[0] == 0
    assert plan([-1, 1])[0] == PAGES_BAD_LENGTH and plan([1, 1], lens=i32([-3, 0]))[0] & PAGES_BAD_LENGTH
    assert plan([0, 0], count=i32([5]))[0] == PAGES_BAD_LENGTH and plan([0, 0], count=i32([-1]))[0] & PAGES_BAD_LENGTH
    big = 2 ** 31 - 1
    assert plan([big, big])[0] == PAGES_ROW_FULL | PAGES_ROWS | PAGES_EXHAUSTED
    assert d["table"].tolist() == [[4, 1], [0, 7]] or d["table"].tolist() == [[4, 5], [1, 7]]

    def release(done, lens, count):
        free = d["free"].clone()
        out = K.kv_page_release(torch.tensor(done, device=DEV), i32(lens), d["table"], free, i32([count]), 4)
        return out[2].item(), out[0].tolist(), out[1].item(), free.tolist()

    assert release([True, False], [3, 8], 2) == (0, [0, 8], 3, [0, 1, 4, 3])
    assert release([True, True], [3, 8], 2) == (PAGES_OVERFLOW, [3, 8], 2, [0, 1, 2, 3])
    assert release([True, False], [9, 8], 0)[0] == PAGES_BAD_LENGTH  # more than its row holds
    assert release([True, False], [-1, 8], 0)[0] == PAGES_BAD_LENGTH
    assert release([False, False], [-1, 99], 0) == (0, [-1, 99], 0, [0, 1, 2, 3])
    assert release([False, False], [1, 1], 5)[0] & PAGES_BAD_LENGTH


def test_large_plans_replayed_from_a_graph():
    """Steps of thousands of tokens and releases of thousands of pages, which take two kernels each, updating the
    lengths and the count in place, captured once and replayed."""
    batch, width, page, rows = 40, 400, 16, 50000
    rng = np.random.default_rng(2)
    books = Books(batch, width, 9000, page, seed=3)
    d = device_books(books, batch)
    new_d, done_d = torch.zeros(batch, device=DEV, dtype=torch.int32), torch.zeros(batch, device=DEV, dtype=torch.bool)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        released = K.kv_page_release(done_d, d["lens"], d["table"], d["free"], d["count"], page, lens_out=d["lens"],
                                     free_count_out=d["count"])
        planned = K.kv_page_plan(new_d, d["lens"], d["table"], d["free"], d["count"], page, rows,
                                 lens_out=d["lens"], free_count_out=d["count"])
    for step in range(6):
        done = rng.random(batch) < 0.3
        books.release(done)
        new = [int(x) for x in rng.integers(0, 1200, batch)]
        want = books.fits(new, rows)
        new_d.copy_(i32(new))
        done_d.copy_(torch.tensor(done, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert released[2].item() == 0 and planned[5].item() == want
        p, sl = books.plan(new) if not want else ([], [])
        assert planned[3][:len(p)].tolist() == p and planned[4][:len(p)].tolist() == sl
        assert (planned[4][len(p):] == -1).all() and not planned[3][len(p):].any()
        assert planned[2].tolist() == [0] + (np.cumsum(new).tolist() if not want else [0] * batch)
        same_books(d, books)


# ------------------------------------------------------------------ together
def test_two_streams_at_once():
    """Calls on two streams that share the pages, each with its own scratch and outputs, in both ways that work is
    divided."""
    for lens in ([700, 64, 1], [40000, 3, 9000]):
        pool = Pool(lens, 2, 64, 16, BF16, seed=31)
        qs = [torch.randn(3, 8, 64, generator=gen(i), device=DEV).to(BF16) for i in range(2)]
        want = [K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens) for q in qs]
        streams = [torch.cuda.Stream() for _ in qs]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(20):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(K.attn_decode_paged(qs[i], pool.kc, pool.vc, pool.table, pool.lens))
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page", [(8, 8, 76, 16), (8, 2, 128, 8)])
def test_serving_steps_of_requests_that_come_and_go(act, cache, hq, hkv, dh, page):
    """A small server: two layers, six request rows, prompts admitted and finished at different times, one token
    a step for the rest, padded token rows.  Every decode step's attention is that of plain attention over each
    request's own keys and values, kept outside; the steps of single tokens run from one captured graph."""
    batch, width, rows, layers = 6, 12, 96, 2
    g = gen(100 + dh)
    rng = np.random.default_rng(dh)
    books = Books(batch, width, 50, page, seed=1)
    d = device_books(books, batch)
    pools = [[torch.full((50, page, hkv, dh), float("nan"), device=DEV, dtype=cache) for _ in range(2)]
             for _ in range(layers)]
    kept = [[[[], []] for _ in range(batch)] for _ in range(layers)]
    packed = torch.zeros(layers, rows, (hq + 2 * hkv) * dh, device=DEV, dtype=act)
    new_d, done_d = torch.zeros(batch, device=DEV, dtype=torch.int32), torch.zeros(batch, device=DEV, dtype=torch.bool)
    last = torch.zeros(batch, hq, dh, device=DEV, dtype=act)
    outs = [torch.zeros(batch, hq, dh, device=DEV, dtype=act) for _ in range(layers)]
    q_outs = [torch.zeros(rows, hq, dh, device=DEV, dtype=act) for _ in range(layers)]
    got = {}

    def step():
        K.kv_page_release(done_d, d["lens"], d["table"], d["free"], d["count"], page, lens_out=d["lens"],
                          free_count_out=d["count"])
        _, _, cu, positions, slots, status = K.kv_page_plan(new_d, d["lens"], d["table"], d["free"], d["count"],
                                                            page, rows, lens_out=d["lens"],
                                                            free_count_out=d["count"])
        for l in range(layers):
            q, k, v = (x.unflatten(1, (-1, dh)) for x in packed[l].split([hq * dh, hkv * dh, hkv * dh], 1))
            K.rope_kv_append_paged(q, k, v, *pools[l], slots, positions, q_out=q_outs[l])
            torch.index_select(q_outs[l], 0, (cu[1:] - 1).clamp_min(0), out=last)
            K.attn_decode_paged(last, *pools[l], d["table"], d["lens"], out=outs[l], max_len=width * page)
        got.update(status=status, cu=cu, positions=positions)

    graph = None
    for n in range(14):
        done = [books.lens[b] > 0 and rng.random() < 0.15 for b in range(batch)]
        books.release(done)
        new = [1 if books.lens[b] else (int(rng.integers(1, 30)) if n % 4 == 0 and rng.random() < 0.6 else 0)
               for b in range(batch)]
        if n > 8:
            new = [min(x, 1) for x in new]
        assert books.fits(new, rows) == 0
        positions, _ = books.plan(new)
        x = torch.randn(packed.shape, generator=g, device=DEV).to(act)
        packed.copy_(x)
        new_d.copy_(i32(new))
        done_d.copy_(torch.tensor(done, device=DEV))
        if n == 8:  # the rest runs from a graph
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            saved = {k: v.clone() for k, v in d.items()}
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                step()
            for k, v in saved.items():
                d[k].copy_(v)
        step() if graph is None else graph.replay()
        torch.cuda.synchronize()
        assert got["status"].item() == 0 and got["cu"].tolist() == [0] + np.cumsum(new).tolist()
        assert got["positions"][:len(positions)].tolist() == positions
        same_books(d, books)
        at = torch.tensor(positions, device=DEV)
        owner = [b for b in range(batch) for _ in range(new[b])]
        for l in range(layers):
            q, k, v = (y[:len(owner)].unflatten(1, (-1, dh)) for y in x[l].split([hq * dh, hkv * dh, hkv * dh], 1))
            if owner:
                kr, kt = rotated(k, at, dh)
                close(q_outs[l][:len(owner)], *rotated(q, at, dh))
            for b in range(batch):
                if done[b]:
                    kept[l][b] = [[], []]
            for r, b in enumerate(owner):  # what the cache holds, checked against the rotation as it is taken over
                j = len(kept[l][b][0])
                cell = (d["table"][b, j // page].long(), j % page)
                close(pools[l][0][cell], kr[r], kt[r])
                kept[l][b][0].append(pools[l][0][cell].clone())
                kept[l][b][1].append(v[r].to(cache))
            view = Pool.__new__(Pool)
            view.lens_h = books.lens
            view.k = [torch.stack(kept[l][b][0]) if kept[l][b][0] else None for b in range(batch)]
            view.v = [torch.stack(kept[l][b][1]) if kept[l][b][1] else None for b in range(batch)]
            queries = torch.stack([q_outs[l][max(0, int(c) - 1)] for c in np.cumsum(new)])
            ref, _, tol, _ = attn_reference(view, queries, 1 / math.sqrt(dh))
            assert ((outs[l].double() - ref).abs() <= tol).all()


def test_every_call_launches_its_own_kernels():
    n0 = launch_count()
    pool = Pool([40], 2, 64, 16, F32, seed=2)
    q = torch.randn(1, 4, 64, device=DEV)
    K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens)
    n1 = launch_count()
    K.rope_kv_append_paged(q, q[:, :2], q[:, :2], pool.kc, pool.vc, i32([0]), i32([0]))
    n2 = launch_count()
    K.kv_page_plan(i32([1]), pool.lens, pool.table, torch.arange(pool.pages, device=DEV, dtype=torch.int32), i32([1]),
                   16, 1)
    n3 = launch_count()
    assert n1 > n0 and n2 > n1 and n3 > n2
    K.rope_kv_append_paged(None, q[:0, :2], q[:0, :2], pool.kc, pool.vc, i32([]), i32([]))
    K.attn_decode_paged(q[:0], pool.kc, pool.vc, pool.table[:0], pool.lens[:0])
    assert launch_count() == n3  # empty steps launch nothing


def test_wrappers_refuse_what_does_not_belong_together():
    pool = Pool([40, 3], 2, 64, 16, F32, seed=2)
    q = torch.randn(2, 4, 64, device=DEV)
    kv = torch.randn(2, 2, 64, device=DEV)
    two = i32([0, 1])

    def attn(q=q, kc=pool.kc, vc=pool.vc, table=pool.table, lens=pool.lens, **kw):
        return K.attn_decode_paged(q, kc, vc, table, lens, **kw)

    for bad in (dict(q=q.double()), dict(q=q[0]), dict(q=q.transpose(1, 2)), dict(q=q.cpu()), dict(kc=pool.kc.half()),
                dict(vc=pool.vc[1:]), dict(table=pool.table.long()), dict(table=pool.table[:1]),
                dict(table=pool.table.t().contiguous().t()), dict(lens=pool.lens.long()), dict(lens=pool.lens[:1]),
                dict(lens=pool.lens.cpu()), dict(out=q[:1]), dict(out=q.half()), dict(work=q.half()),
                dict(q=q[..., :60])):
        with pytest.raises(ValueError):
            attn(**bad)
    with pytest.raises(KrikilError, match="16-bit q"):
        attn(q=q.half())
    with pytest.raises(KrikilError, match="multiple"):
        attn(q=q[:, :3])

    def append(q=q, k=kv, v=kv, kc=pool.kc, vc=pool.vc, slots=two, positions=two, **kw):
        return K.rope_kv_append_paged(q, k, v, kc, vc, slots, positions, **kw)

    for bad in (dict(k=kv[:, :1]), dict(v=kv[:1]), dict(slots=two[:1]), dict(positions=two.long()),
                dict(q=q.half()), dict(q_out=q.half()), dict(q=q[:1]), dict(v=kv.half()), dict(k=kv.cpu())):
        with pytest.raises(ValueError):
            append(**bad)
    with pytest.raises(KrikilError, match="rot_dim"):
        append(rot_dim=63)
    free, one = i32([0, 1]), i32([1])
    for bad in ((two.long(), pool.lens, pool.table, free, one), (two[:1], pool.lens, pool.table, free, one),
                (two, pool.lens, pool.table, free, two), (two, pool.lens[:1], pool.table, free, one),
                (two, pool.lens, pool.table[0], free, one), (two, pool.lens.cpu(), pool.table, free, one)):
        with pytest.raises(ValueError):
            K.kv_page_plan(*bad, 16, 4)
    with pytest.raises(ValueError, match="rows"):
        K.kv_page_plan(two, pool.lens, pool.table, free, one, 16, -1)
    with pytest.raises(ValueError):
        K.kv_page_release(two, *(pool.lens, pool.table, free, one), 16)


def test_wrappers_refuse_an_expanded_table():
    """One row for several requests (stride 0): refused by every call, before anything is read or written."""
    pool = Pool([40], 2, 64, 16, F32, seed=2)
    q = torch.randn(2, 4, 64, device=DEV)
    two, free, one = i32([40, 40]), i32([0, 1]), i32([1])
    shared = pool.table.expand(2, -1)
    with pytest.raises(ValueError, match="table"):
        K.attn_decode_paged(q, pool.kc, pool.vc, shared, two)
    with pytest.raises(ValueError, match="table"):
        K.kv_page_plan(i32([1, 1]), two, shared, free, one, 16, 4)
    with pytest.raises(ValueError, match="table"):
        K.kv_page_release(torch.tensor([True, False], device=DEV), two, shared, free, one, 16)
    out = K.attn_decode_paged(q, pool.kc, pool.vc, shared.contiguous(), two)
    alone = K.attn_decode_paged(q[:1], pool.kc, pool.vc, pool.table, pool.lens)
    assert torch.equal(out[:1], alone)


def test_calls_run_with_their_tensors_device_current(monkeypatch):
    """With another device current, every library call -- the size of the scratch, which depends on the device, too --
    is made with the tensors' device current, on that device's stream, and the other device is current again behind
    it.  (The other device is pretended: what the wrappers ask and set is stood in for.)"""
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
    pool = Pool([9000, 40], 2, 64, 16, BF16, seed=2)
    q = torch.randn(2, 4, 64, device=DEV).to(BF16)
    slots, new = i32([-1, 3]), i32([0, 0])
    free, count = i32(range(pool.pages)), i32([2])

    def calls():
        b = K.rope_kv_append_paged(q, q[:, :2], q[:, :2], pool.kc, pool.vc, slots, slots)[1]
        a = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, return_lse=True)
        c = K.kv_page_plan(new, pool.lens, pool.table, free, count, 16, 4)
        d = K.kv_page_release(new.bool(), pool.lens, pool.table, free, count, 16)
        return [*a, b, *c, *d]

    here = calls()
    monkeypatch.setattr(K, "lib", Lib())
    monkeypatch.setattr(K, "_current_device", lambda: current[0])
    monkeypatch.setattr(K.torch.cuda, "device", Device)
    current[0] = 1
    there = calls()
    assert all(torch.equal(x, y) for x, y in zip(here, there))
    assert len(seen) == 5 and all(dev == 0 for _, dev in seen) and current[0] == 1, seen


@pytest.mark.parametrize("far", [2 ** 32, -2 ** 32, 2 ** 31, -1])
def test_wrappers_refuse_numbers_past_31_bits(far):
    """A window of 2^32 + 5 is not one of 5."""
    pool = Pool([40], 2, 64, 16, F32, seed=2)
    q = torch.randn(1, 4, 64, device=DEV)
    free, one = i32([0, 1]), i32([1])
    with pytest.raises(ValueError, match="window"):
        K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, window=far + 5 * (far > 2))
    with pytest.raises(ValueError, match="max_len"):
        K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, max_len=far)
    with pytest.raises(ValueError, match="rot_dim"):
        K.rope_kv_append_paged(q, q[:, :2], q[:, :2], pool.kc, pool.vc, one, one, rot_dim=far + 64 * (far > 2))
    for size in (dict(page_size=far + 16 * (far > 2), rows=4), dict(page_size=16, rows=far)):
        with pytest.raises(ValueError, match="page_size" if size["rows"] == 4 else "rows"):
            K.kv_page_plan(one, pool.lens, pool.table, free, one, **size)
    with pytest.raises(ValueError, match="page_size"):
        K.kv_page_release(one.bool(), pool.lens, pool.table, free, one, far + 16 * (far > 2))
    wide = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, window=2 ** 31 - 1, max_len=2 ** 31 - 1)
    assert torch.equal(wide, K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens))


@pytest.mark.parametrize("page", [1, 4, 64, 65536])
@pytest.mark.parametrize("tokens", [3, 6000])
def test_planned_slots_of_pages_outside_the_pool(page, tokens):
    """Ids that are no pages, on the stack or in a row: copied as they are, and their tokens get slot -1, also where
    id * page_size leaves 32 bits and comes back to a slot of the pool."""
    per = -(-tokens // page)
    bad = [2 ** 32 // page % 2 ** 31 + 1, -1, 2 * per + 4, 2 ** 31 - 1, -2 ** 31]
    num_pages = 2 * per + 4
    free = list(range(num_pages))
    held = bad[::-1]  # a request that holds five pages, all of them gone, the last one with a token to spare
    table = i32([held + [7] * (per + 1), [7] * (per + 6)])
    for i, x in enumerate(bad):
        if num_pages - 1 - i >= 0:
            free[num_pages - 1 - i] = x
    new, lens = [tokens, tokens], [5 * page - (page > 1), 0]
    out = K.kv_page_plan(i32(new), i32(lens), table, i32(free), i32([num_pages]), page, 2 * tokens)
    assert out[5].item() == 0
    rows = [list(held), []]
    want = []
    for b in range(2):
        while len(rows[b]) < -(-(lens[b] + new[b]) // page):
            rows[b].append(free.pop())
        assert table[b, :len(rows[b])].tolist() == rows[b]
        at = [(j // page, j % page) for j in range(lens[b], lens[b] + new[b])]
        want += [rows[b][p] * page + o if 0 <= rows[b][p] < num_pages else -1 for p, o in at]
    assert out[4].tolist() == want and out[3].tolist() == [j for b in range(2) for j in range(lens[b], lens[b] + new[b])]


@pytest.mark.parametrize("batch,width,page,most", [(1, 6, 16, 96), (5, 40, 4, 160), (700, 5, 8, 40), (60, 300, 16, 4800),
                                                   (1500, 33, 1, 33), (3, 9000, 2, 18000), (2048, 2, 8, 16)])
@pytest.mark.parametrize("gone", [0.0, 0.001, 0.3, 1.0])
@pytest.mark.parametrize("full", [False, True])
def test_release_skips_entries_that_were_given_back(batch, width, page, most, gone, full):
    """Negative entries of finished rows are left out, the others keep their order.  Where all of a pool's pages come
    back (`full`), the entries with the negative ones are more than the stack holds; one page fewer, and nothing
    changes."""
    rng = np.random.default_rng(batch + width)
    lens = [int(x) for x in rng.integers(0, most + 1, batch)]
    done = rng.random(batch) < 0.7
    held = [-(-n // page) for n in lens]
    ids = iter(rng.permutation(sum(held) + 5).tolist())
    rows = [[next(ids) for _ in range(n)] for n in held]
    left = list(ids)
    for row in rows:
        for i in range(len(row)):
            if rng.random() < gone:
                left.append(row[i])
                row[i] = -1 if i % 2 else -2 ** 31
    num_pages = sum(held) + 5
    back = [x for row, d in zip(rows, done) if d for x in row if x >= 0]
    if full:  # the pages that stay with their requests are not of this pool
        num_pages = len(left) + len(back)
    free = left + [77] * (num_pages - len(left))
    table = i32([row + [5] * (width - len(row)) for row in rows])

    def release(free, lens_d, count):
        return K.kv_page_release(torch.tensor(done, device=DEV), lens_d, table, free, count, page, lens_out=lens_d,
                                 free_count_out=count)[2].item()

    stack, lens_d, count = i32(free), i32(lens), i32([len(left)])
    assert release(stack, lens_d, count) == 0
    assert lens_d.tolist() == [0 if d else n for n, d in zip(lens, done)]
    assert count.item() == len(left) + len(back)
    assert stack[:count.item()].tolist() == left + back
    if full and back:
        if num_pages > 1:
            short, lens_d, count = i32(free[:-1]), i32(lens), i32([min(len(left), num_pages - 1)])
            assert release(short, lens_d, count) == PAGES_OVERFLOW
            assert lens_d.tolist() == lens and short.tolist() == free[:-1] and count.item() == len(left)


@pytest.mark.parametrize("hq,hkv,dh,page,window", [(4, 2, 64, 4, 10), (8, 8, 76, 16, 40)])
def test_serving_with_pages_given_back_behind_a_window(hq, hkv, dh, page, window):
    """Requests of one token a step whose pages go back as the window leaves them behind: no page is ever held twice,
    and attention is that of plain attention over the window."""
    batch, width, num_pages = 5, 24, 40
    rng = np.random.default_rng(page)
    g = gen(page)
    kc, vc = (torch.full((num_pages, page, hkv, dh), float("nan"), device=DEV) for _ in range(2))
    d = dict(lens=i32([0] * batch), table=i32([[-1] * width] * batch), free=i32(list(range(num_pages))),
             count=i32([num_pages]))
    keys = [[[], []] for _ in range(batch)]
    for step in range(3 * width * page // 4):
        lens = d["lens"].tolist()
        done = [n >= width * page or (n > 0 and rng.random() < 0.01) for n in lens]
        kw = dict(lens_out=d["lens"], free_count_out=d["count"])
        status = K.kv_page_release(torch.tensor(done, device=DEV), d["lens"], d["table"], d["free"], d["count"], page,
                                   **kw)[2]
        new = [1 if n and not x else int(rng.integers(0, 2 * page)) for n, x in zip(lens, done)]
        plan = K.kv_page_plan(i32(new), d["lens"], d["table"], d["free"], d["count"], page, 16 * page, **kw)
        assert status.item() == 0 and plan[5].item() == 0
        rows = sum(new)
        q, k, v = (torch.randn(16 * page, h, dh, generator=g, device=DEV) for h in (hq, hkv, hkv))
        K.rope_kv_append_paged(q, k, v, kc, vc, plan[4], plan[3], rot_dim=0, q_out=q)
        owner = [b for b in range(batch) for _ in range(new[b])]
        for b in range(batch):
            if done[b]:
                keys[b] = [[], []]
        for r, b in enumerate(owner):
            keys[b][0].append(k[r])
            keys[b][1].append(v[r])
        view = Pool.__new__(Pool)
        view.lens_h = d["lens"].tolist()
        assert view.lens_h == [len(x[0]) for x in keys] and rows == len(owner)
        view.k = [torch.stack(x[0]) if x[0] else None for x in keys]
        view.v = [torch.stack(x[1]) if x[1] else None for x in keys]
        last = q[(plan[2][1:] - 1).clamp_min(0).long()]
        out = K.attn_decode_paged(last, kc, vc, d["table"], d["lens"], window=window)
        if step % 7 == 0:
            ref, _, tol, _ = attn_reference(view, last, 1 / math.sqrt(dh), window)
            assert ((out.double() - ref).abs() <= tol).all()
        # what the next token's window has left behind goes back
        table, free = d["table"].tolist(), d["free"][:d["count"].item()].tolist()
        for b, n in enumerate(view.lens_h):
            for i in range(max(0, n + 1 - window) // page):
                if table[b][i] >= 0:
                    free.append(table[b][i])
                    table[b][i] = -1
            assert all(x >= 0 for x in table[b][max(0, n + 1 - window) // page:-(-n // page)])
        here = [x for b, n in enumerate(view.lens_h) for x in table[b][:-(-n // page)] if x >= 0]
        assert sorted(here + free) == list(range(num_pages))
        d["table"].copy_(i32(table))
        d["free"][:len(free)] = i32(free)
        d["count"].fill_(len(free))


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page,lens", [
    (4, 4, 64, 16, [1, 40, 300, 0]), (8, 2, 76, 16, [17, 3, 129]), (16, 2, 128, 4, [64, 1000]), (17, 1, 96, 32, [333, 2]),
    (4, 2, 192, 16, [50, 50]), (2, 1, 256, 8, [31, 700]), (8, 1, 64, 64, [30000, 5, 70])])
def test_infinite_values_of_visible_keys(act, cache, hq, hkv, dh, page, lens):
    """An infinite value makes its column infinite, one of each sign NaN, whatever a weight's parts are (a weight of 1,
    which a 16-bit type holds exactly, included); nothing else changes."""
    def fill(n, h, d, g):
        return 0.1 * torch.randn(n, h, d, generator=g, device=DEV), torch.randn(n, h, d, generator=g, device=DEV)
    pool = Pool(lens, hkv, dh, page, cache, seed=hq, fill=fill)
    q = torch.randn(len(lens), hq, dh, generator=gen(4), device=DEV).to(act)
    clean, lse = check_attn(pool, q)
    inf = float("inf")
    want = clean.clone().float()
    share = hq // hkv
    for b, n in enumerate(lens):
        marks = [(0, 0, inf), (n - 1, 1, -inf), (n // 2, dh - 1, inf), (n // 3, dh // 2, -inf), (n // 2, dh // 2, -inf),
                 (0, 5, inf), (n - 1, 5, inf)]
        if n > 1:
            marks += [(0, 9, inf), (n - 1, 9, -inf)]
        for j, d, x in marks if n else []:
            h = (j + d) % hkv
            if d in (5, 9):  # both of one head
                h = d % hkv
            pool.vc[int(pool.table[b, j // page]), j % page, h, d] = x
            cells = want[b, h * share:(h + 1) * share, d]
            cells[:] = float("nan") if (cells == -x).any() else x
    out, got = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, return_lse=True)
    assert torch.equal(got, lse)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.float().nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh", [(1, 1, 64), (4, 2, 76), (16, 1, 128)])
@pytest.mark.parametrize("far", [10.0, 27.0, 35.0, 60.0])
def test_infinite_values_of_faint_keys(act, cache, hq, hkv, dh, far):
    """A weight of e^-far is not 0 in 32 bits, and times infinity is infinity."""
    def fill(n, h, d, g):
        k = torch.zeros(n, h, d, device=DEV)
        k[:, :, 0] = torch.arange(n, device=DEV)[:, None] % 2 * -far
        return k, torch.randn(n, h, d, generator=g, device=DEV)
    pool = Pool([2, 40], hkv, dh, 16, cache, seed=8, fill=fill)
    q = torch.zeros(2, hq, dh, device=DEV, dtype=act)
    q[:, :, 0] = 1.0
    want, _ = check_attn(pool, q, scale=1.0)
    for b, j, d, x in ((0, 1, 3, float("inf")), (1, 39, 2, -float("inf")), (1, 5, dh - 1, float("inf"))):
        pool.vc[int(pool.table[b, j // 16]), j % 16, :, d] = x
        want[b, :, d] = x
    assert torch.equal(K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, scale=1.0), want)


# ------------------------------------------------------------------ attention in shares
@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_scratch_of_nan_and_bounds_that_are_too_small(act, cache):
    """Long keys, which go through the scratch: what it held before does not matter, calls repeat bit for bit, and a
    bound below the lengths sizes the launch and nothing else."""
    lens = [40000, 0, 9000, 12]
    pool = Pool(lens, 2, 128, 16, cache, seed=12)
    q = torch.randn(4, 8, 128, generator=gen(3), device=DEV).to(act)
    need = K.attn_paged_work_floats(4, 8, 2, 128, 40000)
    assert need > 0
    first, first_lse = check_attn(pool, q)
    for fill in (float("nan"), float("inf"), -1.0):
        work = torch.full((need + 8,), fill, device=DEV)
        out, lse = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, work=work, return_lse=True)
        assert torch.equal(first, out) and torch.equal(first_lse, lse)
        assert not torch.equal(work[:need].nan_to_num(5.0), torch.full_like(work[:need], fill).nan_to_num(5.0))
        assert torch.equal(work[need:].nan_to_num(5.0), torch.full_like(work[need:], fill).nan_to_num(5.0))
    work = torch.full((need,), float("nan"), device=DEV)
    for bound in (1, 5000, 13000, 20000, 2 ** 31 - 1):
        if bound > 12500:
            assert K.attn_paged_work_floats(4, 8, 2, 128, min(bound, 40000)) > 0
        check_attn(pool, q, max_len=bound, work=work)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page", [(8, 2, 64, 16), (17, 1, 76, 64), (40, 1, 128, 4)])
def test_shares_replayed_from_a_graph(act, cache, hq, hkv, dh, page):
    """The captured pair of kernels follows the lengths, table and queries that it finds, whatever its scratch holds,
    beside eager calls that run at the same time with their own."""
    most = 30016
    pool = Pool([most] * 3, hkv, dh, page, cache, seed=21)
    q = torch.randn(3, hq, dh, generator=gen(3), device=DEV).to(act)
    now, s = i32([10, 0, 20000]), torch.cuda.Stream()
    need = K.attn_paged_work_floats(3, hq, hkv, dh, most)
    assert need > 0
    out, work = torch.empty_like(q), torch.empty(need, device=DEV)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, now, out=out, work=work)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, now, out=out, work=work)
    for step, lens in enumerate(([most, 0, 64], [0, 0, 0], [most] * 3, [1, 20000, 29999], [17, 16, 65])):
        now.copy_(i32(lens))
        q.copy_(torch.randn(3, hq, dh, generator=gen(step), device=DEV).to(act))
        work.fill_(float("nan"))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
        eager = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, now)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        view = Pool.__new__(Pool)
        view.lens_h, view.k, view.v = lens, [k[:n] for k, n in zip(pool.k, lens)], [v[:n] for v, n in zip(pool.v, lens)]
        ref, _, tol, _ = attn_reference(view, q, 1 / math.sqrt(dh))
        assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page,window", [(2, 2, 64, 16, 0), (8, 8, 76, 32, 0), (16, 8, 36, 16, 0),
                                                   (24, 2, 96, 64, 0), (32, 4, 128, 8, 0), (32, 8, 128, 16, 1500),
                                                   (6, 2, 252, 16, 0)])
def test_large_batches_take_neighbouring_heads_together(act, cache, hq, hkv, dh, page, window):
    """Batches with 8 units of 64 keys and more for each of 592 blocks when two heads of the cache go together: a
    block's warps then take two or four neighbouring ones.  Random values against 64 bits; then every weight 1 and
    values that are whole numbers, so that a key of another head or request shows, exactly."""
    batch = 600 // hkv + 60
    lens = [int(2000 * (i + 0.5) / batch) for i in np.random.default_rng(hq).permutation(batch)]
    lens[3] = lens[-1] = 0
    longest = -(-max(lens) // page) * page
    units = -(-(min(longest, window + 16) if window else longest) // 64)
    assert batch * hkv // 2 * units >= 8 * 592 and K.attn_paged_work_floats(batch, hq, hkv, dh, longest, window) > 0

    def fill(n, h, d, g):
        return (torch.randn(n, h, d, generator=g, device=DEV),
                torch.randint(-8, 9, (n, h, d), generator=g, device=DEV).float())
    pool = Pool(lens, hkv, dh, page, cache, seed=dh, fill=fill)
    q = torch.randn(batch, hq, dh, generator=gen(7), device=DEV).to(act)
    first, _ = check_attn(pool, q, window=window)
    again = K.attn_decode_paged(q, pool.kc, pool.vc, pool.table, pool.lens, window=window)
    assert torch.equal(first, again)
    out, lse = K.attn_decode_paged(torch.zeros_like(q), pool.kc, pool.vc, pool.table, pool.lens, window=window,
                                   return_lse=True)
    for i, n in enumerate(lens):
        seen = min(n, window) if window else n
        mean = pool.v[i][n - seen:].double().sum(0).repeat_interleave(hq // hkv, 0) / max(1, seen)
        tol = (8 * U + half_step(act)) * mean.abs() + torch.finfo(act).tiny
        assert ((out[i].double() - mean).abs() <= tol).all(), (i, n)
        want = math.log(seen) if seen else -math.inf
        assert torch.allclose(lse[i].double(), torch.full_like(lse[i].double(), want), rtol=8 * U, atol=8 * U)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("hq,hkv,dh,page,lens,window", [
    (33, 1, 64, 16, [30000, 0, 9000], 0), (40, 1, 76, 4, [16000, 16001], 0), (64, 1, 128, 32, [20000], 0),
    (66, 2, 80, 16, [14000, 1, 15000], 0), (71, 1, 192, 64, [13000], 0), (128, 1, 256, 16, [13000, 5], 0),
    (40, 1, 64, 16, [60000, 40], 20000)])
def test_many_query_heads_in_shares(act, cache, hq, hkv, dh, page, lens, window):
    """More query heads a cache head than a block takes at once, over keys that go through the scratch."""
    pool = Pool(lens, hkv, dh, page, cache, seed=hq)
    q = torch.randn(len(lens), hq, dh, generator=gen(hq), device=DEV).to(act)
    assert K.attn_paged_work_floats(len(lens), hq, hkv, dh, pool.table.shape[1] * page, window) > 0
    check_attn(pool, q, window=window)


@pytest.mark.parametrize("cache", [F32, F16, BF16])
@pytest.mark.parametrize("hq,dh", [(4, 64), (8, 76), (34, 128)])
@pytest.mark.parametrize("power", [-118, -100, 100, 114, 116, 118, 122])
def test_float32_queries_of_any_size(cache, hq, dh, power):
    """Queries far from 1 under a scale that brings the scores back: no part of them leaves its type."""
    pool = Pool([130, 17], 2, dh, 16, cache, seed=14)
    q = torch.randn(2, hq, dh, generator=gen(3), device=DEV) * 2.0 ** power
    check_attn(pool, q, scale=2.0 ** -power / math.sqrt(dh))


def test_the_serving_step_of_the_readme():
    """The step as README.md has it: requests without a new token first and last, then a step that does not fit."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "README.md"), encoding="utf-8") as f:
        code = next(x for x in re.findall(r"```python\n(.*?)```", f.read(), re.S) if "kv_page_plan" in x)
    hq, hkv, dh, page, batch = 4, 2, 64, 4, 4
    g = gen(1)
    layers = [SimpleNamespace(kc=torch.full((9, page, hkv, dh), float("nan"), device=DEV),
                              vc=torch.full((9, page, hkv, dh), float("nan"), device=DEV)) for _ in range(2)]
    names = dict(layers=layers, lens=i32([0] * batch), count=i32([9]), free_pages=i32(list(range(9))), page_size=page,
                 table=torch.full((batch, 8), -1, device=DEV, dtype=torch.int32), rows=batch, bound=32)
    kept = [[[[], []] for _ in range(batch)] for _ in layers]
    for step in range(12):
        new = [0, 1, int(step % 3 == 0), 0] if step < 10 else [0, 1, 1, 0]
        names["new_tokens"] = i32(new)
        for l in layers:
            l.q, l.k, l.v = (torch.randn(batch, h, dh, generator=g, device=DEV) for h in (hq, hkv, hkv))
        exec(code, names)
        for i, l in enumerate(layers):
            q = K.rope_kv_append_paged(l.q, l.k, l.v, l.kc.clone(), l.vc.clone(), names["slots"], names["positions"])
            owner = [b for b in range(batch) if new[b]]
            for r, b in enumerate(owner):
                j = names["lens"].tolist()[b] - 1
                cell = names["table"][b, j // page].long(), j % page
                kept[i][b][0].append(l.kc[cell].clone())
                kept[i][b][1].append(l.v[r])
            view = Pool.__new__(Pool)
            view.lens_h = [len(x[0]) for x in kept[i]]
            assert view.lens_h == names["lens"].tolist()
            view.k, view.v = ([torch.stack(x[c]) if x[c] else None for x in kept[i]] for c in (0, 1))
            mine = torch.zeros(batch, hq, dh, device=DEV)
            mine[owner] = q[:len(owner)]
            ref, _, tol, _ = attn_reference(view, mine, 1 / math.sqrt(dh))
            assert ((l.out.double() - ref).abs() <= tol)[owner].all()
    names["new_tokens"], before = i32([1, 1, 1, 2]), [l.kc.clone() for l in layers]  # five tokens in four rows
    with pytest.raises(MemoryError):
        exec(code, names)
    assert all(torch.equal(l.kc.nan_to_num(9.0), x.nan_to_num(9.0)) for l, x in zip(layers, before))


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
@pytest.mark.parametrize("batch,hq,hkv,dh,page", [(100003, 1, 1, 4, 1), (66000, 3, 3, 8, 2), (30011, 8, 4, 12, 4)])
def test_very_many_requests(act, cache, batch, hq, hkv, dh, page):
    """Tens of thousands of requests of 0 to 5 tokens, planned, appended and attended."""
    g = gen(batch)
    new = torch.randint(0, 6, (batch,), generator=g, device=DEV, dtype=torch.int32)
    tokens, width = int(new.sum()), -(-5 // page)
    need = int(((new + page - 1) // page).sum())
    free = torch.randperm(need + 3, generator=g, device=DEV).int()
    table = torch.full((batch, width), -1, device=DEV, dtype=torch.int32)
    lens, count, cu, positions, slots, status = K.kv_page_plan(new, torch.zeros_like(new), table, free, i32([need + 3]),
                                                               page, tokens + 5)
    assert status.item() == 0 and count.item() == 3 and torch.equal(lens, new)
    assert torch.equal(cu[1:].long(), torch.cumsum(new.long(), 0)) and (slots[tokens:] == -1).all()
    row = torch.repeat_interleave(torch.arange(batch, device=DEV), new.long())
    at = torch.arange(tokens, device=DEV) - cu[row].long()
    assert torch.equal(positions[:tokens].long(), at)
    page_of = table[row, at // page].long()
    assert torch.equal(slots[:tokens].long(), page_of * page + at % page)
    held = page_of[at % page == 0]
    assert held.unique().numel() == need  # no page twice
    kc, vc = (torch.full((need + 3, page, hkv, dh), float("nan"), device=DEV, dtype=cache) for _ in range(2))
    k = torch.randn(tokens + 5, hkv, dh, generator=g, device=DEV).to(act)
    v = torch.randint(-8, 9, (tokens + 5, hkv, dh), generator=g, device=DEV).to(act)
    K.rope_kv_append_paged(None, k, v, kc, vc, slots, positions, rot_dim=0)
    assert torch.equal(kc[page_of, at % page], k[:tokens].to(cache))
    out, lse = K.attn_decode_paged(torch.zeros(batch, hq, dh, device=DEV, dtype=act), kc, vc, table, lens,
                                   return_lse=True)
    total = torch.zeros(batch, hkv, dh, device=DEV, dtype=torch.float64).index_add_(0, row, v[:tokens].double())
    mean = (total / new.clamp_min(1)[:, None, None]).repeat_interleave(hq // hkv, 1)
    assert ((out.double() - mean).abs() <= (8 * U + half_step(act)) * mean.abs() + torch.finfo(act).tiny).all()
    want = torch.log(new.double())[:, None].expand(-1, hq)
    assert torch.equal(lse == -math.inf, want == -math.inf)
    assert (lse.double() - want).abs()[new > 0].max() <= 16 * U
    done = torch.rand(batch, generator=g, device=DEV) < 0.5
    after, left, status = K.kv_page_release(done, lens, table, free, count, page)
    assert status.item() == 0 and torch.equal(after, torch.where(done, 0, new))
    back = table[row, at // page][(at % page == 0) & done[row]]
    assert left.item() == 3 + back.numel() and torch.equal(free[3:left.item()], back)


@pytest.mark.parametrize("act,cache", TYPES, ids=IDS)
def test_one_query_and_one_cache_for_all(act, cache):
    """Inputs that are read only may be broadcast: one query row expanded over requests and heads, values that are the
    keys themselves."""
    pool = Pool([33, 0, 200], 2, 64, 16, cache, seed=3)
    one = torch.randn(1, 1, 64, generator=gen(1), device=DEV).to(act)
    pool.vc, pool.v = pool.kc, pool.k
    a, _ = check_attn(pool, one.expand(3, 8, 64))
    b, _ = check_attn(pool, one.expand(3, 8, 64).contiguous())
    assert torch.equal(a, b)
    kv = one.expand(5, 2, 64)
    kc, vc = torch.zeros(2, 4, 2, 64, device=DEV, dtype=cache), torch.zeros(2, 4, 2, 64, device=DEV, dtype=cache)
    K.rope_kv_append_paged(None, kv, kv, kc, vc, i32([0, 1, 2, 7, -1]), i32([0] * 5))
    for c in (kc, vc):
        cells = c.view(8, 2, 64)
        assert torch.equal(cells[[0, 1, 2, 7]], one.to(cache).expand(4, 2, 64)) and not cells[3:7].any()
