// Decode attention of one new token a request over a paged key-value cache.
#include "elem.cuh"
#include "kernels.h"
#include "paged.h"

namespace krk {
namespace {

constexpr int PA_THREADS = 128;
constexpr int PA_MAX_DH = 256;

// One block per (request, query head): its warps take every fourth key with a
// running maximum and sum each, and are merged through shared memory.
template <typename T, typename C>
__global__ void __launch_bounds__(PA_THREADS) paged_attn_kernel(PagedAttnArgs a) {
    __shared__ float so[4][PA_MAX_DH];
    __shared__ float sm[4], sl[4];
    const int b = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int hk = h / (a.Hq / a.Hkv), n4 = a.dh / 4;
    const long long cap = (long long)a.width << a.page_shift;
    long long len = a.lens[b];
    if (len < 0 || len > cap) {
        if (threadIdx.x == 0) check_fail(CHK_POSITION);
        len = len < 0 ? 0 : cap;
    }
    const long long first = a.window > 0 && len > a.window ? len - a.window : 0;
    const T* q = (const T*)a.q + b * a.q_sb + h * a.q_sh;
    float4 qv[2], acc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = lane + 32 * i;
        qv[i] = c < n4 ? load4(q + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = -INFINITY, l = 0.f;
    for (long long j = first + warp; j < len; j += 4) {
        const int page = a.table[b * a.table_ld + (j >> a.page_shift)];
        if ((unsigned)page >= (unsigned)a.num_pages) {
            check_fail(CHK_TABLE);
            continue;
        }
        const long long at = page * a.c_sp + (j & ((1 << a.page_shift) - 1)) * a.c_st + hk * a.c_sh;
        float s = 0.f;
        float4 vv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = lane + 32 * i;
            vv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < n4) {
                const float4 k = load4((const C*)a.kc + at + 4 * c);
                s = fmaf(k.x, qv[i].x, fmaf(k.y, qv[i].y, fmaf(k.z, qv[i].z, fmaf(k.w, qv[i].w, s))));
                vv[i] = load4((const C*)a.vc + at + 4 * c);
            }
        }
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s);
        const float f = m == -INFINITY ? 0.f : expf(m - mn), p = mn == -INFINITY ? 0.f : expf(s - mn);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            acc[i].x = fmaf(p, vv[i].x, acc[i].x * f);
            acc[i].y = fmaf(p, vv[i].y, acc[i].y * f);
            acc[i].z = fmaf(p, vv[i].z, acc[i].z * f);
            acc[i].w = fmaf(p, vv[i].w, acc[i].w * f);
        }
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 32 * i < n4) *reinterpret_cast<float4*>(&so[warp][4 * (lane + 32 * i)]) = acc[i];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float w[4], total = 0.f;
    for (int i = 0; i < 4; ++i) {
        w[i] = sm[i] == -INFINITY ? 0.f : expf(sm[i] - top);
        total += w[i] * sl[i];
    }
    const float inv = total > 0.f ? 1.0f / total : total;
    T* out = (T*)a.out + b * a.o_sb + h * a.o_sh;
    for (int d = threadIdx.x; d < a.dh; d += PA_THREADS) {
        float o = 0.f;
        for (int i = 0; i < 4; ++i) o = fmaf(w[i], so[i][d], o);
        out[d] = from_f32<T>(o * inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[(long long)b * a.Hq + h] = top + logf(total);
}

template <typename T, typename C>
cudaError_t launch_attn(const PagedAttnArgs& a, cudaStream_t s) {
    paged_attn_kernel<T, C><<<dim3(a.B, a.Hq), PA_THREADS, 0, s>>>(a);
    add_launches(1);
    return cudaGetLastError();
}

}  // namespace

size_t attn_paged_work_floats(int, int, int) { return 0; }

cudaError_t attn_decode_paged(const PagedAttnArgs& a, int act, int cache, cudaStream_t s) {
    if (act == ELEM_F32 && cache == ELEM_F32) return launch_attn<float, float>(a, s);
    if (act == ELEM_F32 && cache == ELEM_F16) return launch_attn<float, __half>(a, s);
    if (act == ELEM_F32 && cache == ELEM_BF16) return launch_attn<float, __nv_bfloat16>(a, s);
    if (act == ELEM_F16 && cache == ELEM_F16) return launch_attn<__half, __half>(a, s);
    if (act == ELEM_BF16 && cache == ELEM_BF16) return launch_attn<__nv_bfloat16, __nv_bfloat16>(a, s);
    return cudaErrorInvalidValue;
}

}  // namespace krk
