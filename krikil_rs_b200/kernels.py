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
