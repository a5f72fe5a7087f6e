// The selective scan's choices, and its step for single tokens:
//   h[n] = exp(delta A[d][n]) h[n] + delta x B[n],   y = (sum_n h[n] C[n] + D x) silu(z).
#include "kernels.h"
#include "paged.h"
#include "recurrent.cuh"

namespace krk {

cudaError_t selective_scan_f32(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s);
cudaError_t selective_scan_f16(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s);
cudaError_t selective_scan_bf16(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s);

namespace {

// ---------------------------------------------------------------- single tokens
// Bound by memory: a request's states are read and written once.  A lane has Q
// times four of a channel's states, and a thread R requests' of them at once,
// for which it reads the channel's decays once.
constexpr int STEP_THREADS = 256;

KRK_DEV float4 load_four(const float* p, int n, int N, bool wide) {
    if (wide) return *reinterpret_cast<const float4*>(p + n);
    return make_float4(n < N ? p[n] : 0.0f, n + 1 < N ? p[n + 1] : 0.0f, n + 2 < N ? p[n + 2] : 0.0f,
                       n + 3 < N ? p[n + 3] : 0.0f);
}
template <typename T>
KRK_DEV float4 load_four(const T* p, int n, int N, bool wide) {
    if (wide) return load4(p + n);
    return make_float4(n < N ? to_f32(p[n]) : 0.0f, n + 1 < N ? to_f32(p[n + 1]) : 0.0f,
                       n + 2 < N ? to_f32(p[n + 2]) : 0.0f, n + 3 < N ? to_f32(p[n + 3]) : 0.0f);
}

// WIDE: whole groups of four states, aligned (states and decays; wide_bc: B and C).
template <typename T, bool WIDE, int Q, int R>
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(ScanArgs a, int lane_bits, int side, bool wide_bc) {
    const int t0 = blockIdx.x / side * R, i = (blockIdx.x - blockIdx.x / side * side) * STEP_THREADS + threadIdx.x;
    const int lanes = 1 << lane_bits, lane = i & (lanes - 1), d = min(i >> lane_bits, a.D - 1);
    const bool open = (i >> lane_bits) < a.D;
    const int64_t row = (int64_t)d * a.N;
    int to[R], from[R];
    bool live[R];
    float4 h[R][Q];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        live[r] = t0 + r < a.T && request_slots(a.slot, t0 + r, to[r], from[r]) && open;
        const float* old = (const float*)a.slot.state + from[r] * a.slot.stride + row;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int n = 4 * (q * lanes + lane);
            h[r][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live[r] && from[r] >= 0 && n < a.N) h[r][q] = load_four(old, n, a.N, WIDE);
        }
    }
    float4 rate[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int n = 4 * (q * lanes + lane);
        const float4 v = n < a.N ? load_four(a.a + row, n, a.N, WIDE) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        rate[q] = make_float4(scan_rate(v.x), scan_rate(v.y), scan_rate(v.z), scan_rate(v.w));
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, skip = a.d ? a.d[d] : 0.0f;
    const int g = a.G == 1 ? 0 : d / (a.D / a.G);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int t = t0 + r;
        float sum = 0.0f, x = 0.0f;
        if (live[r]) {
            x = to_f32(((const T*)a.x)[t * a.x_st + d]);
            const float delta = step_width(to_f32(((const T*)a.dt)[t * a.dt_st + d]) + bias), put = delta * x;
            const T* b = (const T*)a.b + t * a.b_st + g * a.b_sg;
            const T* c = (const T*)a.c + t * a.c_st + g * a.c_sg;
            float* kept = (float*)a.slot.state + to[r] * a.slot.stride + row;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int n = 4 * (q * lanes + lane);
                if (n >= a.N) continue;
                const float4 b4 = load_four(b, n, a.N, WIDE && wide_bc), c4 = load_four(c, n, a.N, WIDE && wide_bc);
                float4 v = h[r][q];
                v.x = fmaf(fast_exp2(delta * rate[q].x), v.x, put * b4.x);
                v.y = fmaf(fast_exp2(delta * rate[q].y), v.y, put * b4.y);
                v.z = fmaf(fast_exp2(delta * rate[q].z), v.z, put * b4.z);
                v.w = fmaf(fast_exp2(delta * rate[q].w), v.w, put * b4.w);
                if (WIDE) {
                    *reinterpret_cast<float4*>(kept + n) = v;
                    sum = fmaf(v.x, c4.x, fmaf(v.y, c4.y, fmaf(v.z, c4.z, fmaf(v.w, c4.w, sum))));
                } else {
                    kept[n] = v.x;
                    sum = fmaf(v.x, c4.x, sum);
                    if (n + 1 < a.N) kept[n + 1] = v.y, sum = fmaf(v.y, c4.y, sum);
                    if (n + 2 < a.N) kept[n + 2] = v.z, sum = fmaf(v.z, c4.z, sum);
                    if (n + 3 < a.N) kept[n + 3] = v.w, sum = fmaf(v.w, c4.w, sum);
                }
            }
        }
        for (int o = lanes / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (live[r] && lane == 0) {
            const float gate = a.z ? fast_silu(to_f32(((const T*)a.z)[t * a.z_st + d])) : 1.0f;
            ((T*)a.out)[t * a.o_st + d] = from_f32<T>(fmaf(skip, x, sum) * gate);
        }
    }
}

template <typename T, bool WIDE, int Q, int R>
cudaError_t launch_step(const ScanArgs& a, int lane_bits, cudaStream_t s) {
    const int64_t side = (((int64_t)a.D << lane_bits) + STEP_THREADS - 1) / STEP_THREADS;
    const int64_t blocks = side * ((a.T + (int64_t)R - 1) / R);
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    const int64_t rows = a.T > 1, groups = a.G > 1;
    const bool wide_bc = fits(a.b, rows * a.b_st, 4 * sizeof(T), sizeof(T)) && fits(a.c, rows * a.c_st, 4 * sizeof(T), sizeof(T)) &&
                         groups * a.b_sg % 4 == 0 && groups * a.c_sg % 4 == 0;
    step_kernel<T, WIDE, Q, R><<<(unsigned)blocks, STEP_THREADS, 0, s>>>(a, lane_bits, (int)side, wide_bc);
    add_launches(1);
    return cudaGetLastError();
}

template <typename T, bool WIDE, int Q>
cudaError_t step_rows(const ScanArgs& a, int lane_bits, cudaStream_t s) {
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    // several requests a thread once that leaves every multiprocessor a full set of threads
    const bool many = ((int64_t)a.D << lane_bits) * a.T >= (int64_t)sms * 2048 * 4;
    return many ? launch_step<T, WIDE, Q, 4>(a, lane_bits, s) : launch_step<T, WIDE, Q, 1>(a, lane_bits, s);
}

template <typename T>
cudaError_t step_type(const ScanArgs& a, cudaStream_t s) {
    int bits = 0;
    while (bits < 5 && 4 << bits < a.N) ++bits;
    const bool wide = a.N % 4 == 0 && fits(a.slot.state, a.slot.num_slots > 1 ? a.slot.stride : 0, 16, 4) && fits(a.a, 0, 16, 4);
    if (a.N > 128) return wide ? step_rows<T, true, 2>(a, bits, s) : step_rows<T, false, 2>(a, bits, s);
    return wide ? step_rows<T, true, 1>(a, bits, s) : step_rows<T, false, 1>(a, bits, s);
}

}  // namespace

// A piece is the rows that leave the device one wave of blocks over all rows.
ScanPlan scan_plan(int T, int S, int D, int N, int G, int max_len) {
    int sms = paged_sm_count();
    if (sms <= 0) sms = 148;
    int lanes = 1;
    while (SCAN_LANE * lanes < N) lanes *= 2;
    const int ch = SCAN_THREADS / lanes;
    const int64_t side = (int64_t)((D / G + ch - 1) / ch) * G, slots = (int64_t)sms * SCAN_BLOCKS;
    const int64_t pieces = slots / side > 1 ? slots / side : 1;
    int64_t rows = (T + pieces - 1) / pieces;
    rows = rows < SCAN_PIECE ? SCAN_PIECE : (rows + 3) / 4 * 4;
    const int bound = max_len > 0 && max_len < T ? max_len : T;
    return {bound > SCAN_ALONE * rows ? (int)rows : 0, side * S <= sms};
}
size_t scan_work_floats(int T, int D, int N, int G, int max_len) {
    const int rows = scan_plan(T, 1, D, N, G, max_len).rows;
    return rows > 0 ? (size_t)scan_split_room(T, rows) * D * (N + 1) : 0;
}

cudaError_t selective_scan(const ScanArgs& a, int type, int max_len, float* work, cudaStream_t s) {
    const ScanPlan plan = scan_plan(a.T, a.S, a.D, a.N, a.G, max_len);
    return type == ELEM_F32 ? selective_scan_f32(a, work, plan, s)
                            : type == ELEM_F16 ? selective_scan_f16(a, work, plan, s) : selective_scan_bf16(a, work, plan, s);
}
cudaError_t selective_step(const ScanArgs& a, int type, cudaStream_t s) {
    return type == ELEM_F32 ? step_type<float>(a, s)
                            : type == ELEM_F16 ? step_type<__half>(a, s) : step_type<__nv_bfloat16>(a, s);
}

}  // namespace krk
