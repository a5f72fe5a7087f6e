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
// times four of a channel's states, and a thread `turns` times R requests' of
// them, for which it reads the channel's decays once.  253 requests x 5120
// bfloat16 channels of 16 states (177 MB): 36 us, 74% of the measured copy rate;
// about 150 instructions for a lane's eight states and what the channel's step
// and gate take leave half of the issue slots free, and the rest is waiting.
constexpr float kLog2e = 1.44269504088896341f;
constexpr int STEP_THREADS = 128;

// States n .. n + 3 (some there): WIDE, all of them and aligned.
template <bool WIDE, typename T>
KRK_DEV float4 load_four(const T* p, int n, int N) {
    if (WIDE) return load4(p + n);
    return make_float4(to_f32(p[n]), to_f32(p[min(n + 1, N - 1)]), to_f32(p[min(n + 2, N - 1)]), to_f32(p[min(n + 3, N - 1)]));
}

// The form of a call: states and decays in whole and aligned groups of four, B and
// C, too, and as many states as the lanes hold.
enum StepForm { STEP_ANY, STEP_WIDE, STEP_WIDE_BC, STEP_WHOLE };

// Everything that the rows need is loaded before the first of them is
// computed, whether they need it or not -- the last states again in the place of
// those that are not there: where branches meet, a thread waits for the loads
// that were in them.
template <typename T, StepForm FORM, int Q, int R>
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(ScanArgs a, int lane_bits, int turns, int side) {
    constexpr bool WIDE = FORM != STEP_ANY, WIDE_BC = FORM >= STEP_WIDE_BC;
    const int group = blockIdx.x / side, i = (blockIdx.x - group * side) * STEP_THREADS + threadIdx.x;
    const int lanes = 1 << lane_bits, lane = i & (lanes - 1), d = min(i >> lane_bits, a.D - 1);
    const bool open = (i >> lane_bits) < a.D;
    const int64_t row = (int64_t)d * a.N;
    const int g = a.G == 1 ? 0 : d / (a.D / a.G);
    const T* zp = a.z ? (const T*)a.z : (const T*)a.x;  // (unused when there is none)
    const int64_t z_st = a.z ? a.z_st : a.x_st;
    int at[Q];    // the first of a group's states, or of the last group's
    bool there[Q];
    float4 rate[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int n = 4 * (q * lanes + lane);
        there[q] = FORM == STEP_WHOLE || n < a.N;
        at[q] = there[q] ? n : (a.N - 1) / 4 * 4;
        rate[q] = load_four<WIDE>(a.a + row, at[q], a.N);
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, skip = a.d ? a.d[d] : 0.0f;
    const int64_t share = (int64_t)turns * R;
    for (int64_t turn = group * share; turn < min((group + 1) * share, (int64_t)a.T); turn += R) {
        const int t0 = (int)turn;
        int to[R], from[R];
        load_slots(a.slot, t0, a.T, to, from);
        float4 h[R][Q], b[R][Q], c[R][Q];
        T x[R], dt[R], z[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int t = min(t0 + r, a.T - 1);
            const T* bt = (const T*)a.b + t * a.b_st + g * a.b_sg;
            const T* ct = (const T*)a.c + t * a.c_st + g * a.c_sg;
            x[r] = ((const T*)a.x)[t * a.x_st + d];
            dt[r] = ((const T*)a.dt)[t * a.dt_st + d];
            z[r] = zp[t * z_st + d];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                b[r][q] = load_four<WIDE_BC>(bt, at[q], a.N);
                c[r][q] = load_four<WIDE_BC>(ct, at[q], a.N);
            }
        }
        bool live[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            live[r] = t0 + r < a.T && valid_slots(a.slot, to[r], from[r]);
            const bool begun = live[r] && from[r] >= 0;
            const float* old = (const float*)a.slot.state + (begun ? from[r] * a.slot.stride : 0) + row;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                h[r][q] = load_four<WIDE>(old, at[q], a.N);
                if (!begun) h[r][q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float xv = to_f32(x[r]), delta = step_width(to_f32(dt[r]) + bias), put = delta * xv;
            const float2 step2 = make_float2(delta * kLog2e, delta * kLog2e), put2 = make_float2(put, put);
            float* kept = (float*)a.slot.state + (live[r] ? to[r] * a.slot.stride : 0) + row;
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const int n = at[q];
                float2 lo = make_float2(h[r][q].x, h[r][q].y), hi = make_float2(h[r][q].z, h[r][q].w);
                const float2 e = __fmul2_rn(step2, make_float2(rate[q].x, rate[q].y));
                const float2 f = __fmul2_rn(step2, make_float2(rate[q].z, rate[q].w));
                lo = __ffma2_rn(make_float2(fast_exp2(e.x), fast_exp2(e.y)), lo,
                                __fmul2_rn(put2, make_float2(b[r][q].x, b[r][q].y)));
                hi = __ffma2_rn(make_float2(fast_exp2(f.x), fast_exp2(f.y)), hi,
                                __fmul2_rn(put2, make_float2(b[r][q].z, b[r][q].w)));
                float2 part;
                if (WIDE) {
                    part = __fmul2_rn(lo, make_float2(c[r][q].x, c[r][q].y));
                    part = __ffma2_rn(hi, make_float2(c[r][q].z, c[r][q].w), part);
                } else {  // an infinite x makes no NaN of states that are not there
                    part = make_float2(lo.x * c[r][q].x, n + 1 < a.N ? lo.y * c[r][q].y : 0.0f);
                    if (n + 2 < a.N) part.x = fmaf(hi.x, c[r][q].z, part.x);
                    if (n + 3 < a.N) part.y = fmaf(hi.y, c[r][q].w, part.y);
                }
                if (!there[q]) continue;
                sum = __fadd2_rn(sum, part);
                if (!live[r] || !open) continue;
                if (WIDE) {
                    *reinterpret_cast<float4*>(kept + n) = make_float4(lo.x, lo.y, hi.x, hi.y);
                } else {
                    kept[n] = lo.x;
                    if (n + 1 < a.N) kept[n + 1] = lo.y;
                    if (n + 2 < a.N) kept[n + 2] = hi.x;
                    if (n + 3 < a.N) kept[n + 3] = hi.y;
                }
            }
            float y = sum.x + sum.y;
            for (int o = lanes / 2; o > 0; o /= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
            if (live[r] && open && lane == 0) {
                const float gate = a.z ? fast_silu(to_f32(z[r])) : 1.0f;
                ((T*)a.out)[(t0 + r) * a.o_st + d] = from_f32<T>(fmaf(skip, xv, y) * gate);
            }
        }
    }
}

template <typename T, StepForm FORM, int Q, int R>
cudaError_t launch_step(const ScanArgs& a, int lane_bits, int64_t side, int turns, cudaStream_t s) {
    const int64_t blocks = side * ((a.T + (int64_t)R * turns - 1) / ((int64_t)R * turns));
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    step_kernel<T, FORM, Q, R><<<(unsigned)blocks, STEP_THREADS, 0, s>>>(a, lane_bits, turns, (int)side);
    add_launches(1);
    return cudaGetLastError();
}

template <typename T, StepForm FORM, int Q>
cudaError_t step_rows(const ScanArgs& a, int lane_bits, cudaStream_t s) {
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    const int64_t side = (((int64_t)a.D << lane_bits) + STEP_THREADS - 1) / STEP_THREADS, units = side * a.T;
    // two requests a thread at once when that leaves every multiprocessor a full set of threads
    if (units < (int64_t)sms * 2048 * 2 / STEP_THREADS) return launch_step<T, FORM, Q, 1>(a, lane_bits, side, 1, s);
    // and up to four times, with the channels' decays loaded once, while there are two waves of blocks, six a
    // multiprocessor: 253 requests x 5120 channels, 36.1 us by four times, 38.5 by one, 41.8 by eight (six are what the
    // registers of whole groups of eight states leave room for, 80 a thread; of other forms three to nine)
    const int64_t turns = units / 2 / (12LL * sms);
    return launch_step<T, FORM, Q, 2>(a, lane_bits, side, turns < 1 ? 1 : turns > 4 ? 4 : (int)turns, s);
}

template <typename T, int Q>
cudaError_t step_wide(const ScanArgs& a, int lane_bits, cudaStream_t s) {
    const int64_t rows = a.T > 1, groups = a.G > 1;
    const bool wide = a.N % 4 == 0 && fits(a.slot.state, a.slot.num_slots > 1 ? a.slot.stride : 0, 16, 4) && fits(a.a, 0, 16, 4);
    const bool wide_bc = fits(a.b, rows * a.b_st, 4 * sizeof(T), sizeof(T)) && fits(a.c, rows * a.c_st, 4 * sizeof(T), sizeof(T)) &&
                         groups * a.b_sg % 4 == 0 && groups * a.c_sg % 4 == 0;
    if (!wide) return step_rows<T, STEP_ANY, Q>(a, lane_bits, s);
    if (!wide_bc) return step_rows<T, STEP_WIDE, Q>(a, lane_bits, s);
    return a.N == 4 * Q << lane_bits ? step_rows<T, STEP_WHOLE, Q>(a, lane_bits, s) : step_rows<T, STEP_WIDE_BC, Q>(a, lane_bits, s);
}

template <typename T>
cudaError_t step_type(const ScanArgs& a, cudaStream_t s) {
    int bits = 0;  // lanes of eight states
    while (bits < 5 && 8 << bits < a.N) ++bits;
    return a.N <= 4 ? step_wide<T, 1>(a, 0, s) : step_wide<T, 2>(a, bits, s);
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
