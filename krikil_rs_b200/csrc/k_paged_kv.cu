// Paged key-value cache: page planning and release on the device, and RoPE +
// append through a slot map.
#include <math.h>

#include "elem.cuh"
#include "kernels.h"
#include "paged.h"

namespace krk {
namespace {

constexpr int PLAN_THREADS = 1024;

// Exclusive prefix sums of one value pair a thread over the block, and the
// totals.  scratch: 2 * 33 values.
KRK_DEV void block_scan2(long long a, long long b, long long& ea, long long& eb, long long& ta, long long& tb,
                         long long* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    long long ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long xa = __shfl_up_sync(0xffffffffu, ia, o), xb = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) {
            ia += xa;
            ib += xb;
        }
    }
    __syncthreads();
    if (lane == 31) {
        scratch[warp] = ia;
        scratch[33 + warp] = ib;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        long long sa = 0, sb = 0;
        for (int w = 0; w < nw; ++w) {
            const long long xa = scratch[w], xb = scratch[33 + w];
            scratch[w] = sa;
            scratch[33 + w] = sb;
            sa += xa;
            sb += xb;
        }
        scratch[32] = sa;
        scratch[65] = sb;
    }
    __syncthreads();
    ea = scratch[warp] + ia - a;
    eb = scratch[33 + warp] + ib - b;
    ta = scratch[32];
    tb = scratch[65];
}

// One block.  Two passes over the requests: the first adds up what they need
// and decides whether the step fits, the second writes it.
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(PagePlanArgs a) {
    __shared__ long long scratch[66];
    __shared__ int bad;
    const int tid = threadIdx.x, P = 1 << a.page_shift;
    if (tid == 0) bad = 0;
    __syncthreads();
    const int count = *a.free_count;
    long long tokens = 0, pages = 0;
    int err = 0;
    if (count < 0 || count > a.num_pages) err |= PAGES_BAD_LENGTH;
    for (int b = tid; b < a.B; b += PLAN_THREADS) {
        const long long len = a.lens[b], add = a.new_tokens[b];
        if (len < 0 || add < 0) {
            err |= PAGES_BAD_LENGTH;
            continue;
        }
        const long long have = (len + P - 1) >> a.page_shift, want = (len + add + P - 1) >> a.page_shift;
        if (want > a.width) err |= PAGES_ROW_FULL;
        tokens += add;
        pages += want - have;
    }
    long long e0, e1, total_tokens, total_pages;
    block_scan2(tokens, pages, e0, e1, total_tokens, total_pages, scratch);
    if (total_tokens > a.rows) err |= PAGES_ROWS;
    if (total_pages > count) err |= PAGES_EXHAUSTED;
    if (err) atomicOr(&bad, err);
    __syncthreads();
    err = bad;
    __syncthreads();
    if (tid == 0) {
        *a.status = err;
        a.cu_new[0] = 0;
    }
    if (err) {
        for (int b = tid; b < a.B; b += PLAN_THREADS) {
            a.lens_out[b] = a.lens[b];
            a.cu_new[b + 1] = 0;
        }
        for (int r = tid; r < a.rows; r += PLAN_THREADS) {
            a.slots[r] = -1;
            a.positions[r] = 0;
        }
        if (tid == 0) *a.free_count_out = count;
        return;
    }
    long long base_t = 0, base_p = 0;
    for (int b0 = 0; b0 < a.B; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        const long long len = b < a.B ? a.lens[b] : 0, add = b < a.B ? a.new_tokens[b] : 0;
        const long long have = (len + P - 1) >> a.page_shift, want = (len + add + P - 1) >> a.page_shift;
        long long t0, p0, tt, tp;
        block_scan2(add, want - have, t0, p0, tt, tp, scratch);
        t0 += base_t;
        p0 += base_p;
        if (b < a.B) {
            int32_t* row = a.table + b * a.table_ld;
            for (long long i = have; i < want; ++i) row[i] = a.free_pages[count - 1 - (p0 + i - have)];
            for (long long i = 0; i < add; ++i) {
                const int pos = (int)(len + i);
                a.positions[t0 + i] = pos;
                a.slots[t0 + i] = (row[pos >> a.page_shift] << a.page_shift) + (pos & (P - 1));
            }
            a.lens_out[b] = (int)(len + add);
            a.cu_new[b + 1] = (int)(t0 + add);
        }
        base_t += tt;
        base_p += tp;
    }
    for (int r = (int)base_t + tid; r < a.rows; r += PLAN_THREADS) {
        a.slots[r] = -1;
        a.positions[r] = 0;
    }
    if (tid == 0) *a.free_count_out = (int)(count - base_p);
}

__global__ void __launch_bounds__(PLAN_THREADS) page_release_kernel(PageReleaseArgs a) {
    __shared__ long long scratch[66];
    __shared__ int bad;
    const int tid = threadIdx.x, P = 1 << a.page_shift;
    if (tid == 0) bad = 0;
    __syncthreads();
    const int count = *a.free_count;
    long long pages = 0;
    int err = 0;
    if (count < 0 || count > a.num_pages) err |= PAGES_BAD_LENGTH;
    for (int b = tid; b < a.B; b += PLAN_THREADS) {
        if (!a.done[b]) continue;
        const long long len = a.lens[b], held = (len + P - 1) >> a.page_shift;
        if (len < 0 || held > a.width) err |= PAGES_BAD_LENGTH;
        else pages += held;
    }
    long long e0, e1, total, unused;
    block_scan2(pages, 0, e0, e1, total, unused, scratch);
    if (count + total > a.num_pages) err |= PAGES_OVERFLOW;
    if (err) atomicOr(&bad, err);
    __syncthreads();
    err = bad;
    __syncthreads();
    if (tid == 0) *a.status = err;
    if (err) {
        for (int b = tid; b < a.B; b += PLAN_THREADS) a.lens_out[b] = a.lens[b];
        if (tid == 0) *a.free_count_out = count;
        return;
    }
    long long base = 0;
    for (int b0 = 0; b0 < a.B; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        const bool done = b < a.B && a.done[b];
        const int len = b < a.B ? a.lens[b] : 0;
        const long long held = done ? ((long long)len + P - 1) >> a.page_shift : 0;
        long long p0, x, tp, y;
        block_scan2(held, 0, p0, x, tp, y, scratch);
        p0 += base;
        if (b < a.B) {
            for (long long i = 0; i < held; ++i) a.free_pages[count + p0 + i] = a.table[b * a.table_ld + i];
            a.lens_out[b] = done ? 0 : len;
        }
        base += tp;
    }
    if (tid == 0) *a.free_count_out = (int)(count + base);
}

// One thread per pair (or unrotated element) of a row's head.
template <typename T, typename C>
__global__ void __launch_bounds__(256) rope_append_kernel(RopeAppendArgs a) {
    const int half = a.rot / 2, per_head = a.dh - half, heads = a.Hq + 2 * a.Hkv;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)a.T * heads * per_head) return;
    const int u = (int)(i % per_head), h = (int)(i / per_head % heads);
    const long long t = i / per_head / heads;
    const int slot = a.slots[t];
    if (slot < 0) return;
    if (slot >= a.num_slots) {
        check_fail(CHK_TABLE);
        return;
    }
    const int lo = u < half ? u : u + half, hi = u < half ? u + half : lo;
    const long long cell = (slot >> a.page_shift) * a.c_sp + (slot & ((1 << a.page_shift) - 1)) * a.c_st;
    if (h >= a.Hq + a.Hkv) {
        const int hv = h - a.Hq - a.Hkv;
        const T* src = (const T*)a.v + t * a.v_st + hv * a.v_sh;
        C* dst = (C*)a.vc + cell + hv * a.c_sh;
        dst[lo] = from_f32<C>(to_f32(src[lo]));
        if (hi != lo) dst[hi] = from_f32<C>(to_f32(src[hi]));
        return;
    }
    const bool is_q = h < a.Hq;
    const T* src = is_q ? (const T*)a.q + t * a.q_st + h * a.q_sh : (const T*)a.k + t * a.k_st + (h - a.Hq) * a.k_sh;
    float x = to_f32(src[lo]), y = to_f32(src[hi]);
    if (u < half) {
        const double turns = (double)a.positions[t] * a.turns.f[u];
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        const float x0 = x, y0 = y;
        x = x0 * cs - y0 * sn;
        y = y0 * cs + x0 * sn;
    }
    if (is_q) {
        T* dst = (T*)a.q_out + t * a.qo_st + h * a.qo_sh;
        dst[lo] = from_f32<T>(x);
        if (hi != lo) dst[hi] = from_f32<T>(y);
    } else {
        C* dst = (C*)a.kc + cell + (h - a.Hq) * a.c_sh;
        dst[lo] = from_f32<C>(x);
        if (hi != lo) dst[hi] = from_f32<C>(y);
    }
}

template <typename T, typename C>
cudaError_t launch_append(const RopeAppendArgs& a, cudaStream_t s) {
    const long long n = (long long)a.T * (a.Hq + 2 * a.Hkv) * (a.dh - a.rot / 2);
    rope_append_kernel<T, C><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    add_launches(1);
    return cudaGetLastError();
}

}  // namespace

cudaError_t kv_page_plan(const PagePlanArgs& a, cudaStream_t s) {
    page_plan_kernel<<<1, PLAN_THREADS, 0, s>>>(a);
    add_launches(1);
    return cudaGetLastError();
}

cudaError_t kv_page_release(const PageReleaseArgs& a, cudaStream_t s) {
    page_release_kernel<<<1, PLAN_THREADS, 0, s>>>(a);
    add_launches(1);
    return cudaGetLastError();
}

// Powers of r = theta^(-2/rot) by repeated products in extended precision:
// 128 roundings of 2^-64 leave the 64-bit rates exact to their last place.
RopeTurns rope_turns(int rot_dim, double theta) {
    RopeTurns r{};
    if (rot_dim <= 0) return r;
    const long double step = powl((long double)theta, -2.0L / rot_dim);
    long double f = 0.5L / acosl(-1.0L);
    for (int i = 0; i < rot_dim / 2 && i < ROPE_PAGED_PAIRS; ++i, f *= step) r.f[i] = (double)f;
    return r;
}

cudaError_t rope_kv_append_paged(const RopeAppendArgs& a, int act, int cache, cudaStream_t s) {
    if (act == ELEM_F32 && cache == ELEM_F32) return launch_append<float, float>(a, s);
    if (act == ELEM_F32 && cache == ELEM_F16) return launch_append<float, __half>(a, s);
    if (act == ELEM_F32 && cache == ELEM_BF16) return launch_append<float, __nv_bfloat16>(a, s);
    if (act == ELEM_F16 && cache == ELEM_F16) return launch_append<__half, __half>(a, s);
    if (act == ELEM_BF16 && cache == ELEM_BF16) return launch_append<__nv_bfloat16, __nv_bfloat16>(a, s);
    return cudaErrorInvalidValue;
}

}  // namespace krk
