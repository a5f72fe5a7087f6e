"""Per-kernel entry points of the C ABI on torch CUDA tensors.

torch only provides device memory and the current stream here; every op is one
of this library's sm_100a kernels (krk_k_* in include/krikil_cuda.h).
"""
from __future__ import annotations

import itertools
from typing import Optional

import torch

from ._lib import TYPE_BF16, TYPE_F16, TYPE_F32, check, lib


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _f32(*ts):
    for t in ts:
        if t is None:
            continue
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
            raise ValueError("expected contiguous float32 CUDA tensors")


def rmsnorm_rows(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    _f32(x, w)
    y = torch.empty_like(x)
    check(lib.krk_k_rmsnorm_rows(x.data_ptr(), w.data_ptr(), eps, x.shape[0], x.shape[1], y.data_ptr(), _stream()))
    return y


def rmsnorm_fm(x_t: torch.Tensor, w: torch.Tensor, eps: float, m: Optional[int] = None) -> torch.Tensor:
    """x_t: feature-major [K, ld]; normalises columns 0..m-1."""
    _f32(x_t, w)
    k, ld = x_t.shape
    out = torch.zeros_like(x_t)
    check(lib.krk_k_rmsnorm_fm(x_t.data_ptr(), ld, w.data_ptr(), eps, k, m or ld, out.data_ptr(), ld, _stream()))
    return out


def gated_rmsnorm_residual(x, z, res, w, eps: float, y=None) -> torch.Tensor:
    _f32(x, z, res, w, y)
    if y is None:
        y = torch.empty_like(x)
    check(lib.krk_k_gated_rmsnorm_residual(x.data_ptr(), z.data_ptr(), res.data_ptr(), w.data_ptr(), eps,
                                           x.shape[0], x.shape[1], y.data_ptr(), _stream()))
    return y


def gemm(a_t: torch.Tensor, w_t: torch.Tensor, epilogue: int = 0, out_fm: bool = False,
         c: Optional[torch.Tensor] = None, tile_rows: int = 0) -> torch.Tensor:
    """C = A . W^T with a_t = A^T [K, M] and w_t = W^T [K, N]; tile_rows 0/16/32/64."""
    _f32(a_t, w_t, c)
    k, m = a_t.shape
    k2, n = w_t.shape
    assert k == k2
    if c is None:
        c = torch.empty((n, m) if out_fm else (m, n), device=a_t.device, dtype=torch.float32)
    check(lib.krk_k_gemm_tiled(a_t.data_ptr(), m, w_t.data_ptr(), n, c.data_ptr(), c.shape[1], m, n, k, epilogue,
                               int(out_fm), tile_rows, _stream()))
    return c


def embed(tok: torch.Tensor, wte: torch.Tensor, ld: Optional[int] = None) -> torch.Tensor:
    _f32(wte)
    vocab, k = wte.shape
    m = tok.numel()
    out = torch.zeros((k, ld or m), device=wte.device, dtype=torch.float32)
    check(lib.krk_k_embed(tok.data_ptr(), wte.data_ptr(), vocab, k, m, out.data_ptr(), out.shape[1], _stream()))
    return out


def pointwise(op: int, x: torch.Tensor) -> torch.Tensor:
    _f32(x)
    y = torch.empty_like(x)
    check(lib.krk_k_pointwise(op, x.data_ptr(), y.data_ptr(), x.numel(), _stream()))
    return y


def conv_ssd_step(x, bm, cm, dt, conv_state, conv_w, conv_b, ssm, dt_bias, a_neg, dsk, y=None) -> torch.Tensor:
    """x [B,H*P], bm/cm [B,N], dt [B,H]; conv_state [B,H*P,3] and ssm [B,H,P,N]
    updated in place; returns y [B,H*P]."""
    _f32(x, bm, cm, dt, conv_state, conv_w, conv_b, ssm, dt_bias, a_neg, dsk, y)
    b, h, p, n = ssm.shape
    if y is None:
        y = torch.empty((b, h * p), device=x.device, dtype=torch.float32)
    check(lib.krk_k_conv_ssd_step(x.data_ptr(), bm.data_ptr(), cm.data_ptr(), dt.data_ptr(), conv_state.data_ptr(),
                                  conv_w.data_ptr(), conv_b.data_ptr(), ssm.data_ptr(), dt_bias.data_ptr(),
                                  a_neg.data_ptr(), dsk.data_ptr(), y.data_ptr(), b, h, p, n, _stream()))
    return y


def conv_ssd_scan(x, bm, cm, dt, conv_state, conv_w, conv_b, ssm, dt_bias, a_neg, dsk, y=None) -> torch.Tensor:
    """x [B,T,H*P], bm/cm [B,T,N], dt [B,T,H]; states updated in place; y [B,T,H*P]."""
    _f32(x, bm, cm, dt, conv_state, conv_w, conv_b, ssm, dt_bias, a_neg, dsk, y)
    b, h, p, n = ssm.shape
    t = x.shape[1]
    if y is None:
        y = torch.empty((b, t, h * p), device=x.device, dtype=torch.float32)
    check(lib.krk_k_conv_ssd_scan(x.data_ptr(), bm.data_ptr(), cm.data_ptr(), dt.data_ptr(), conv_state.data_ptr(),
                                  conv_w.data_ptr(), conv_b.data_ptr(), ssm.data_ptr(), dt_bias.data_ptr(),
                                  a_neg.data_ptr(), dsk.data_ptr(), y.data_ptr(), b, t, h, p, n, _stream()))
    return y


def attn_work_floats(b: int, h: int, dh: int, ctx: int, split: int = 0) -> int:
    return int(lib.krk_attn_work_floats(b, h, dh, ctx, split))


def wait_probe(src16, status, polls: int, copy: bool) -> None:
    """krk_k_wait_probe: the bounded copy wait with (copy) or without its copy;
    bit 0 of status (int32, device) is set when the wait runs out."""
    check(lib.krk_k_wait_probe(src16.data_ptr() if src16 is not None else None, polls, int(copy),
                               status.data_ptr(), _stream()))


def rope_kv_attn_decode(q, k, v, kc, vc, pos, split: int = 0, theta: float = 10000.0, work=None, out=None):
    """q,k,v [B,H,dh]; kc,vc [B,H,ctx,dh] (updated at pos); pos int32 [B].
    split 0: the cluster kernel (no scratch); split > 0: splits of that many
    keys merged through `work` (allocated here when not given)."""
    _f32(q, k, v, kc, vc, work, out)
    b, h, dh = q.shape
    ctx = kc.shape[2]
    if out is None:
        out = torch.empty_like(q)
    if work is None:
        work = torch.empty(max(1, attn_work_floats(b, h, dh, ctx, split)), device=q.device, dtype=torch.float32)
    check(lib.krk_k_rope_kv_attn_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                                        pos.data_ptr(), out.data_ptr(), work.data_ptr(), b, h, dh, ctx, split, theta,
                                        _stream()))
    return out


def gemm_sgemm_order(a_t: torch.Tensor, w_t: torch.Tensor) -> torch.Tensor:
    """C = A . W^T (a_t = A^T [K, M], w_t = W^T [K, N]) summed in the order of
    matrixmultiply's sgemm (the reference's prefill GEMM)."""
    _f32(a_t, w_t)
    k, m = a_t.shape
    k2, n = w_t.shape
    assert k == k2
    c = torch.empty((m, n), device=a_t.device, dtype=torch.float32)
    check(lib.krk_k_gemm_sgemm_order(a_t.data_ptr(), m, w_t.data_ptr(), n, c.data_ptr(), n, m, n, k, _stream()))
    return c


def attn_prefill_rows(kmax: int, dh: int) -> int:
    return int(lib.krk_k_attn_prefill_rows(kmax, dh))


def rope_kv_attn_prefill(qkv, kc, vc, lens, start, H: int, dh: int, theta: float = 10000.0,
                         cache_layout: str = "model"):
    """Packed prefill rows of len(lens) sequences: qkv [rows, 3*H*dh] (q rotated
    in place), sequence s starting at position start[s] of its cache.  Caches:
    "model" [S, ctx, H*dh] (the model's layout) or "bhtd" [S, H, ctx, dh].
    Builds the row-block table as the model does and returns out [rows, H*dh]."""
    _f32(qkv, kc, vc)
    lens = [int(x) for x in lens]
    start = [int(x) for x in start]
    S, rows = len(lens), sum(lens)
    if cache_layout == "model":
        ctx = kc.shape[1]
        c_sb, c_sh, c_st = ctx * H * dh, dh, H * dh
    else:
        ctx = kc.shape[2]
        c_sb, c_sh, c_st = H * ctx * dh, ctx * dh, dh
    kmax = max(s0 + n for s0, n in zip(start, lens))
    rpb = attn_prefill_rows(kmax, dh)
    blocks = [(s, r0) for s in range(S) for r0 in range(0, lens[s], rpb)]
    dev = qkv.device
    cu = torch.tensor([0] + list(itertools.accumulate(lens)), dtype=torch.int32, device=dev)
    st = torch.tensor(start, dtype=torch.int32, device=dev)
    blk = torch.tensor(blocks, dtype=torch.int32, device=dev).reshape(-1)
    out = torch.zeros((rows, H * dh), device=dev, dtype=torch.float32)
    check(lib.krk_k_rope_kv_attn_prefill(qkv.data_ptr(), qkv.shape[1], kc.data_ptr(), vc.data_ptr(), c_sb, c_sh,
                                         c_st, cu.data_ptr(), st.data_ptr(), S, rows, H, dh, theta, blk.data_ptr(),
                                         len(blocks), rpb, kmax, out.data_ptr(), H * dh, 1, _stream()))
    return out


def greedy(logits: torch.Tensor, seen: Optional[torch.Tensor] = None, penalty: float = 1.0) -> torch.Tensor:
    _f32(logits)
    b, v = logits.shape
    tok = torch.empty(b, device=logits.device, dtype=torch.int32)
    check(lib.krk_k_greedy(logits.data_ptr(), v, v, b, seen.data_ptr() if seen is not None else None, penalty,
                           tok.data_ptr(), _stream()))
    return tok


# ------------------------------------------------------ paged key-value cache
# The wrappers' checks are a large part of a small call's time: each tensor's
# type, device, shape and strides are read once, and small outputs come from one
# allocation.
_TYPES = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = torch.cuda.current_device


def _elsewhere(dev, fn, *args) -> int:
    """fn(*args, stream) on dev's current stream with dev current, when another device is."""
    with torch.cuda.device(dev):
        return fn(*args, _raw_stream(dev.index))


def _number(x, name) -> None:
    """Refuses what does not fit the 31 bits that the library takes (more would be cut off on the way)."""
    if x >> 31:
        raise ValueError(f"{name} must lie between 0 and 2^31 - 1")


def _cuda_device(t):
    if not t.is_cuda:
        raise ValueError("expected CUDA tensors")
    return t.device


def _not_elems(name, dims, dev):
    return ValueError(f"{name}: expected a float32, float16 or bfloat16 tensor of {dims} dimensions on {dev} whose "
                      "last dimension is dense")


def _elems3(t, dev, name):
    """(type, shape, strides) of a float tensor [., ., dh] whose last dimension is dense."""
    kind, shape, strides = _TYPES.get(t.dtype), t.shape, t.stride()
    if kind is None or len(shape) != 3 or (strides[2] != 1 and shape[2] > 1) or t.device != dev:
        raise _not_elems(name, 3, dev)
    return kind, shape, strides


def _ints(t, n, dev, name) -> int:
    """The address of a dense int32 tensor of n elements."""
    if t.dtype != torch.int32 or t.numel() != n or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {n} elements on {dev}")
    return t.data_ptr()


def _table(t, dev):
    """(rows, width, row stride) of a page table."""
    shape, strides = t.shape, t.stride()
    if t.dtype != torch.int32 or len(shape) != 2 or (strides[1] != 1 and shape[1] > 1) or t.device != dev:
        raise ValueError(f"table: expected an int32 [requests, pages] tensor on {dev} with dense rows")
    rows, width = shape
    ld = strides[0]
    if ld < width:  # the stride of a single row does not matter
        if rows > 1:
            raise ValueError("table: rows that overlap (an expanded row?) must be copied out first")
        ld = width
    return rows, width, ld


def _pool(kc, vc, dev):
    """(type, shape, strides) of the two caches."""
    kind, shape, strides = _TYPES.get(kc.dtype), kc.shape, kc.stride()
    if kind is None or len(shape) != 4 or (strides[3] != 1 and shape[3] > 1) or kc.device != dev:
        raise _not_elems("kc", 4, dev)
    if vc.dtype != kc.dtype or vc.shape != shape or vc.stride() != strides or vc.device != dev:
        raise ValueError("kc and vc: expected the same type, device, shape and strides")
    return kind, shape, strides


def kv_page_plan(new_tokens, lens, table, free_pages, free_count, page_size: int, rows: int, lens_out=None,
                 free_count_out=None):
    """Plans a step of new_tokens[b] tokens on top of lens[b] (int32 [B]): takes
    the pages that requests lack from the top of the stack free_pages
    [num_pages] (free_count int32 [1]) into table [B, width], in place.  Returns
    (lens_out, free_count_out, cu [B+1], positions [rows], slots [rows], status
    [1]): the lengths after the step, what is left on the stack, the packed
    offsets of each request's tokens, and each packed token's position and cache
    slot (-1 behind the last one).  status is 0, or PAGES_* bits of what does
    not fit, in which case nothing was taken.  lens_out and free_count_out may be
    the inputs; they and the others are new tensors when not given."""
    dev = _cuda_device(table)
    b, width, ld = _table(table, dev)
    new_at, lens_at = _ints(new_tokens, b, dev, "new_tokens"), _ints(lens, b, dev, "lens")
    pages = free_pages.numel()
    free_at, count_at = _ints(free_pages, pages, dev, "free_pages"), _ints(free_count, 1, dev, "free_count")
    _number(rows, "rows")
    _number(page_size, "page_size")
    padded = -rows % 4 + rows
    buf = lens.new_empty(2 * padded + 2 * b + 3)
    positions, _, slots, _, cu, lens_new, count_new, status = buf.unsafe_split_with_sizes(
        (rows, padded - rows, rows, padded - rows, b + 1, b, 1, 1))
    at = buf.data_ptr()
    cu_at = at + 8 * padded
    if lens_out is None:
        lens_out, lens_out_at = lens_new, cu_at + 4 * b + 4
    else:
        lens_out_at = _ints(lens_out, b, dev, "lens_out")
    if free_count_out is None:
        free_count_out, count_out_at = count_new, cu_at + 8 * b + 4
    else:
        count_out_at = _ints(free_count_out, 1, dev, "free_count_out")
    args = (new_at, lens_at, table.data_ptr(), ld, b, width, free_at, count_at, pages, page_size, lens_out_at,
            count_out_at, cu_at, at, at + 4 * padded, rows, cu_at + 8 * b + 8)
    index = dev.index
    if index == _current_device():
        rc = lib.krk_k_kv_page_plan(*args, _raw_stream(index))
    else:
        rc = _elsewhere(dev, lib.krk_k_kv_page_plan, *args)
    if rc:
        check(rc)
    return lens_out, free_count_out, cu, positions, slots, status


def kv_page_release(done, lens, table, free_pages, free_count, page_size: int, lens_out=None, free_count_out=None):
    """Puts the pages of the requests whose done flag (bool or uint8 [B]) is set
    back on the stack free_pages, in place, and their lengths to 0.  Negative
    entries of their rows are skipped: set those of pages that were given back
    before (behind a window) to -1.  Returns (lens_out, free_count_out, status)."""
    dev = _cuda_device(table)
    b, width, ld = _table(table, dev)
    if done.dtype not in (torch.bool, torch.uint8) or done.numel() != b or done.device != dev or not done.is_contiguous():
        raise ValueError(f"done: expected a contiguous bool or uint8 tensor of {b} elements on {dev}")
    _number(page_size, "page_size")
    lens_at, pages = _ints(lens, b, dev, "lens"), free_pages.numel()
    free_at, count_at = _ints(free_pages, pages, dev, "free_pages"), _ints(free_count, 1, dev, "free_count")
    buf = lens.new_empty(b + 2)
    lens_new, count_new, status = buf.unsafe_split_with_sizes((b, 1, 1))
    at = buf.data_ptr()
    if lens_out is None:
        lens_out, lens_out_at = lens_new, at
    else:
        lens_out_at = _ints(lens_out, b, dev, "lens_out")
    if free_count_out is None:
        free_count_out, count_out_at = count_new, at + 4 * b
    else:
        count_out_at = _ints(free_count_out, 1, dev, "free_count_out")
    args = (done.data_ptr(), lens_at, table.data_ptr(), ld, b, width, free_at, count_at, pages, page_size, lens_out_at,
            count_out_at, at + 4 * b + 4)
    index = dev.index
    if index == _current_device():
        rc = lib.krk_k_kv_page_release(*args, _raw_stream(index))
    else:
        rc = _elsewhere(dev, lib.krk_k_kv_page_release, *args)
    if rc:
        check(rc)
    return lens_out, free_count_out, status


def rope_kv_append_paged(q, k, v, kc, vc, slots, positions, theta: float = 10000.0, rot_dim: Optional[int] = None,
                         q_out=None):
    """Rotates q [T, Hq, dh] and k [T, Hkv, dh] by their positions (int32 [T];
    rotate-half on the first rot_dim elements, all by default) and writes k and
    v to the slots (int32 [T], -1: padding) of the pages kc, vc [pages,
    page_size, Hkv, dh]; no two rows may have the same slot.  Strided views are fine as long as dh is dense.
    Returns the rotated q (q_out, which may be q; padding rows of a given q_out
    are left as they were).  q may be None."""
    dev = _cuda_device(k)
    ctype, (pages, page_size, hkv, dh), (c_sp, c_st, c_sh, _) = _pool(kc, vc, dev)
    kind, shape, (k_st, k_sh, _) = _elems3(k, dev, "k")
    vkind, vshape, (v_st, v_sh, _) = _elems3(v, dev, "v")
    t = shape[0]
    if shape[1] != hkv or shape[2] != dh or vshape != shape or vkind != kind:
        raise ValueError(f"expected k and v of [T, {hkv}, {dh}] and one type")
    hq = q_at = q_st = q_sh = o_at = o_st = o_sh = 0
    if q is not None:
        qkind, qshape, (q_st, q_sh, _) = _elems3(q, dev, "q")
        hq = qshape[1]
        if qshape[0] != t or qshape[2] != dh or qkind != kind:
            raise ValueError(f"expected q of [T, heads, {dh}] and k's type")
        if q_out is None:
            q_out, o_st, o_sh = q.new_empty(t, hq, dh), hq * dh, dh
        else:
            okind, oshape, (o_st, o_sh, _) = _elems3(q_out, dev, "q_out")
            if oshape != qshape or okind != kind:
                raise ValueError("q_out: expected q's shape and type")
        q_at, o_at = q.data_ptr(), q_out.data_ptr()
    rot_dim = dh if rot_dim is None else rot_dim
    _number(rot_dim, "rot_dim")
    args = (q_at, q_st, q_sh, k.data_ptr(), k_st, k_sh, v.data_ptr(), v_st, v_sh, kind, o_at, o_st, o_sh,
            kc.data_ptr(), vc.data_ptr(), c_sp, c_st, c_sh, ctype, _ints(slots, t, dev, "slots"),
            _ints(positions, t, dev, "positions"), t, hq, hkv, dh, rot_dim, pages, page_size,
            theta)
    index = dev.index
    if index == _current_device():
        rc = lib.krk_k_rope_kv_append_paged(*args, _raw_stream(index))
    else:
        rc = _elsewhere(dev, lib.krk_k_rope_kv_append_paged, *args)
    if rc:
        check(rc)
    return q_out


def attn_paged_work_floats(b: int, hq: int, hkv: int, dh: int, max_len: int, window: int = 0) -> int:
    return int(lib.krk_attn_paged_work_floats(b, hq, hkv, dh, max_len, window))


def attn_decode_paged(q, kc, vc, table, lens, scale: Optional[float] = None, window: int = 0, max_len: int = 0,
                      out=None, work=None, return_lse: bool = False):
    """Attention of one token a request, q [B, Hq, dh], over the lens[b] (int32
    [B]) tokens in its pages table[b] of kc, vc [pages, page_size, Hkv, dh], the
    last `window` of them if that is not 0.  scale defaults to 1/sqrt(dh);
    max_len, a bound of the lengths, only sizes the launch (0: what a table row
    holds).  `work` is scratch of attn_paged_work_floats floats (allocated here
    when not given).  Returns out [B, Hq, dh], or (out, lse)."""
    dev = _cuda_device(q)
    index = dev.index
    if index != _current_device():  # the scratch is sized for the current device
        with torch.cuda.device(dev):
            return attn_decode_paged(q, kc, vc, table, lens, scale, window, max_len, out, work, return_lse)
    ctype, (pages, page_size, hkv, dh), (c_sp, c_st, c_sh, _) = _pool(kc, vc, dev)
    kind, shape, (q_sb, q_sh, _) = _elems3(q, dev, "q")
    b, hq, qdh = shape
    rows, width, ld = _table(table, dev)
    if qdh != dh or rows != b:
        raise ValueError(f"expected q of [B, heads, {dh}] and a table of B rows")
    if out is None:
        out, o_sb, o_sh = q.new_empty(b, hq, dh), hq * dh, dh
    else:
        okind, oshape, (o_sb, o_sh, _) = _elems3(out, dev, "out")
        if oshape != shape or okind != kind:
            raise ValueError("out: expected q's shape and type")
    _number(window, "window")
    _number(max_len, "max_len")
    lse, lse_at = None, None
    if return_lse:
        lse = torch.empty(b, hq, device=dev, dtype=torch.float32)
        lse_at = lse.data_ptr()
    if work is None:
        cap = width * page_size
        need = lib.krk_attn_paged_work_floats(b, hq, hkv, dh, max_len if 0 < max_len < cap else cap, window)
        work_at = None
        if need:
            work = torch.empty(need, device=dev, dtype=torch.float32)
            work_at = work.data_ptr()
    else:
        if work.dtype != torch.float32 or work.device != dev or not work.is_contiguous():
            raise ValueError(f"work: expected a contiguous float32 tensor on {dev}")
        need, work_at = work.numel(), work.data_ptr()
    args = (q.data_ptr(), q_sb, q_sh, kind, kc.data_ptr(), vc.data_ptr(), c_sp, c_st, c_sh, ctype, table.data_ptr(),
            ld, width, pages, page_size, _ints(lens, b, dev, "lens"), b, hq, hkv, dh,
            dh ** -0.5 if scale is None else scale, window, max_len, out.data_ptr(), o_sb, o_sh, lse_at, work_at,
            need)
    rc = lib.krk_k_attn_decode_paged(*args, _raw_stream(index))
    if rc:
        check(rc)
    return (out, lse) if return_lse else out


# ------------------------------------------- recurrent layers over state slots
# (checked in few steps, as above: what x is, and that the others are like it)
def _like(t, dtype, shape, index, name):
    """(address, row stride) of a tensor of this type, shape [rows, width] and device whose last dimension is dense."""
    st = t.stride()
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index or (st[1] != 1 and shape[1] > 1):
        raise ValueError(f"{name}: expected {list(shape)} of {dtype} on cuda:{index} whose last dimension is dense")
    return t.data_ptr(), st[0]


def _rows2(t, name):
    """(type, shape, device index) of a float CUDA tensor [rows, width]."""
    kind, shape, index = _TYPES.get(t.dtype), t.shape, t.get_device()
    if index < 0:
        raise ValueError("expected CUDA tensors")
    if kind is None or len(shape) != 2:
        raise _not_elems(name, 2, t.device)
    return kind, shape, index


def _weights(t, shape, index, name):
    """The address of a dense float32 tensor of this shape (None: None)."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous float32 tensor of {tuple(shape)} on cuda:{index}")
    return t.data_ptr()


def _indexes(t, n, index, name):
    """The address of a dense int32 tensor of n elements (None: None)."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.numel() != n or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {n} elements on cuda:{index}")
    return t.data_ptr()


def _slot_args(state, rows, width, dtype, slots, init, requests, index):
    """The pool's address, slot stride and size, and the addresses of slots and init."""
    if state is None:
        if slots is not None or init is not None:
            raise ValueError("slots and init need a state")
        return None, 0, 0, None, None
    shape, strides = state.shape, state.stride()
    if state.dtype is not dtype or state.get_device() != index or len(shape) != 3 or shape[1] != rows or (
            shape[2] != width) or (width > 1 and strides[2] != 1) or (rows > 1 and strides[1] != width):
        raise ValueError(f"state: expected {dtype} [slots, {rows}, {width}] on cuda:{index} with dense slots")
    _number(shape[0], "the number of slots")
    if slots is None and shape[0] < requests:
        raise ValueError(f"state: expected a slot for each of {requests} requests, or their slots")
    return (state.data_ptr(), strides[0], shape[0], _indexes(slots, requests, index, "slots"),
            _indexes(init, requests, index, "init"))


def _requests(cu, index):
    """(address, number of requests) of packed requests' offsets."""
    n = cu.numel()
    if n < 1:
        raise ValueError("cu: expected the requests' offsets, one more than there are requests")
    _number(n - 1, "the number of requests")
    return _indexes(cu, n, index, "cu"), n - 1


def _call(index, fn, args) -> None:
    """fn(*args, stream) on the device's current stream with the device current."""
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        rc = _elsewhere(torch.device("cuda", index), fn, *args)
    if rc:
        check(rc)


def _conv_args(x, weight, bias, state, slots, init, out, requests):
    kind, shape, index = _rows2(x, "x")
    dtype, (rows, ch), w = x.dtype, shape, weight.shape
    x_at, x_st = _like(x, dtype, shape, index, "x")
    if len(w) != 2 or w[0] != ch:
        raise ValueError(f"weight: expected [{ch}, width]")
    _number(rows | ch | w[1], "the sizes of x and weight")
    if out is None:
        out = x.new_empty(shape)
    out_at, o_st = _like(out, dtype, shape, index, "out")
    return index, out, (x_at, x_st, _weights(weight, w, index, "weight"), _weights(bias, (ch,), index, "bias"), out_at,
                        o_st, kind, *_slot_args(state, w[1] - 1, ch, dtype, slots, init,
                                                rows if requests is None else requests, index)), rows, ch, w[1]


def causal_conv(x, weight, cu, bias=None, state=None, slots=None, init=None, silu: bool = True, out=None):
    """Causal depthwise convolution of packed requests: x [T, C], weight [C, W]
    (W 2 to 4) and bias [C] float32, then x * sigmoid(x) unless silu is False.
    Request s owns rows cu[s] .. cu[s+1]-1 (cu int32 [S+1]); its last W-1 rows go
    to slot slots[s] (int32 [S]; -1: padding, left alone; None: slot s) of state
    [slots, W-1, C] of x's type, and those before it come from slot init[s] (-1:
    it begins; None: the same slot).  Without a state every request begins.
    Returns out [T, C], whose rows of no request are left as they were."""
    cu_at, requests = _requests(cu, x.get_device())
    index, out, args, rows, ch, width = _conv_args(x, weight, bias, state, slots, init, out, requests)
    _call(index, lib.krk_k_causal_conv, (*args, cu_at, rows, requests, ch, width, 1 if silu else 0))
    return out


def causal_conv_step(x, weight, state, slots=None, bias=None, init=None, silu: bool = True, out=None):
    """causal_conv of one token a request: row b of x [B, C] is request b's."""
    index, out, args, rows, ch, width = _conv_args(x, weight, bias, state, slots, init, out, None)
    _call(index, lib.krk_k_causal_conv_step, (*args, rows, ch, width, 1 if silu else 0))
    return out


def _groups(t, dtype, rows, n, index, name):
    """(address, row stride, group stride, groups) of B or C."""
    shape, st = t.shape, t.stride()
    groups = shape[1] if len(shape) == 3 else 1
    if t.dtype is not dtype or t.get_device() != index or len(shape) not in (2, 3) or shape[0] != rows or (
            shape[-1] != n) or (st[-1] != 1 and n > 1):
        raise ValueError(f"{name}: expected [{rows}, {n}] or [{rows}, groups, {n}] of {dtype} on cuda:{index} whose last "
                         "dimension is dense")
    return t.data_ptr(), st[0], st[1] if len(shape) == 3 else n, groups


def _scan_args(x, dt, a, b, c, d, z, dt_bias, state, slots, init, out, requests):
    kind, shape, index = _rows2(x, "x")
    dtype, (rows, ch), decay = x.dtype, shape, a.shape
    if len(decay) != 2 or decay[0] != ch:
        raise ValueError(f"a: expected [{ch}, states]")
    n = decay[1]
    b_at, b_st, b_sg, groups = _groups(b, dtype, rows, n, index, "b")
    c_at, c_st, c_sg, c_groups = _groups(c, dtype, rows, n, index, "c")
    if c_groups != groups or not groups or ch % groups:
        raise ValueError(f"b and c: expected as many groups, dividing {ch} channels")
    _number(rows | ch | n, "the sizes of x and a")
    x_at, x_st = _like(x, dtype, shape, index, "x")
    dt_at, dt_st = _like(dt, dtype, shape, index, "dt")
    z_at, z_st = (None, 0) if z is None else _like(z, dtype, shape, index, "z")
    if out is None:
        out = x.new_empty(shape)
    out_at, o_st = _like(out, dtype, shape, index, "out")
    return index, out, (x_at, x_st, dt_at, dt_st, z_at, z_st, b_at, b_st, b_sg, c_at, c_st, c_sg, out_at, o_st, kind,
                        _weights(a, decay, index, "a"), _weights(d, (ch,), index, "d"),
                        _weights(dt_bias, (ch,), index, "dt_bias"),
                        *_slot_args(state, ch, n, torch.float32, slots, init, rows if requests is None else requests,
                                    index)), (ch, n, groups), rows


def selective_scan_work_floats(rows: int, channels: int, states: int, groups: int = 1, max_len: int = 0) -> int:
    sizes = rows, channels, states, groups, max_len
    if max(sizes) >> 31 > 0 or min(sizes) >> 31 < -1:  # (no scratch for negative ones)
        raise ValueError("sizes must lie below 2^31")
    return int(lib.krk_selective_scan_work_floats(*sizes))


def selective_scan(x, dt, a, b, c, cu, d=None, z=None, dt_bias=None, state=None, slots=None, init=None, out=None,
                   max_len: int = 0, work=None):
    """Selective state space scan of packed requests: x, dt and the gate z [T, D],
    b and c [T, N] or [T, G, N] of one type; the decay a [D, N] (negative), the
    skip d [D] and dt_bias [D] float32.  With delta = softplus(dt + dt_bias), h =
    exp(delta a) h + delta x b and out = (h . c + d x) * z * sigmoid(z).  Requests
    and slots as for causal_conv; state is float32 [slots, D, N].  max_len, a
    bound of the requests' rows (0: T), only sizes the launch; `work` is scratch
    of selective_scan_work_floats floats (allocated here when not given).  Returns
    out [T, D], which may be x, dt or z and shares no other memory with the
    inputs, and whose rows of no request are left as they were."""
    index = x.get_device()
    if index >= 0 and index != _current_device():  # the scratch is sized for the current device
        with torch.cuda.device(torch.device("cuda", index)):
            return selective_scan(x, dt, a, b, c, cu, d, z, dt_bias, state, slots, init, out, max_len, work)
    cu_at, requests = _requests(cu, index)
    index, out, args, sizes, rows = _scan_args(x, dt, a, b, c, d, z, dt_bias, state, slots, init, out, requests)
    _number(max_len, "max_len")
    if work is None:
        need, work_at = lib.krk_selective_scan_work_floats(rows, *sizes, max_len), None
        if need:
            work = torch.empty(need, device=x.device, dtype=torch.float32)
            work_at = work.data_ptr()
    else:
        if work.dtype != torch.float32 or work.get_device() != index or not work.is_contiguous():
            raise ValueError(f"work: expected a contiguous float32 tensor on cuda:{index}")
        need, work_at = work.numel(), work.data_ptr()
    rc = lib.krk_k_selective_scan(*args, cu_at, rows, requests, *sizes, max_len, work_at, need, _raw_stream(index))
    if rc:
        check(rc)
    return out


def selective_step(x, dt, a, b, c, state, slots=None, d=None, z=None, dt_bias=None, init=None, out=None):
    """selective_scan of one token a request: row t of x [B, D] is request t's."""
    index, out, args, sizes, rows = _scan_args(x, dt, a, b, c, d, z, dt_bias, state, slots, init, out, None)
    _call(index, lib.krk_k_selective_step, (*args, rows, *sizes))
    return out


def token_logprobs(logits, tokens=None, top: int = 0):
    """Log probabilities under softmax of each row of logits [R, V]: of tokens
    (int32 [R] or [R, K]; negative: none asked, 0), the entropy [R], and the ids
    and log probabilities [R, top] of the largest logits (at most 32), the lower
    id first among equal ones.  Returns (logprobs like tokens, or None; entropy;
    top_ids; top_logprobs), float32 and int32."""
    kind, shape, index = _rows2(logits, "logits")
    at, ld = _like(logits, logits.dtype, shape, index, "logits")
    rows, vocab = shape
    _number(top, "top")
    _number(rows | vocab, "the sizes of logits")
    lp, asked, lp_at, tokens_at = None, 0, None, None
    if tokens is not None:
        like = tokens.shape
        if len(like) not in (1, 2) or like[0] != rows:
            raise ValueError(f"tokens: expected [{rows}] or [{rows}, tokens]")
        asked = 1 if len(like) == 1 else like[1]
        _number(asked, "the tokens of a row")
        tokens_at = _indexes(tokens, rows * asked, index, "tokens")
    entropy = torch.empty(rows, device=logits.device, dtype=torch.float32)
    if tokens is not None:
        lp = entropy.new_empty(like)
        lp_at = lp.data_ptr()
    best = entropy.new_empty(rows, top)
    ids = torch.empty(rows, top, device=logits.device, dtype=torch.int32) if tokens is None else tokens.new_empty(rows, top)
    _call(index, lib.krk_k_token_logprobs, (at, ld, kind, rows, vocab, tokens_at, asked, lp_at, entropy.data_ptr(), top,
                                            ids.data_ptr(), best.data_ptr()))
    return lp, entropy, ids, best
