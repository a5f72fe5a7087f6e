// Selective state space scan over packed requests and its step for single
// tokens, with the requests' states in a pool of slots.  With delta =
// softplus(dt + bias), channel d's N states and output are
//   h[n] = exp(delta A[d][n]) h[n] + delta x B[n],   y = (sum_n h[n] C[n] + D x) silu(z).
#include "kernels.h"
#include "paged.h"
#include "recurrent.cuh"

namespace krk {
namespace {

constexpr float kLog2e = 1.44269504088896341f;

// log1p keeps the small steps that large negative arguments make.
KRK_DEV float step_width(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

// ---------------------------------------------------------------- the prompts
// The recurrence is walked row by row: its work is one exponential a state and
// row, which no other order makes fewer of.  K lanes share a channel, each with
// SPT states in registers, so that a block of 128 threads walks 128 / K
// channels of one request; a tile of rows is staged in shared memory, its step
// widths computed once, and the next tile's inputs are on their way meanwhile.
constexpr int SCAN_THREADS = 128;

template <int K, int SPT>
struct ScanShape {
    static constexpr int CH = SCAN_THREADS / K, NP = K * SPT;
    static constexpr int ROWS = NP <= 32 ? 32 : 1024 / NP;  // a tile's
    static constexpr int E = (ROWS * CH + SCAN_THREADS - 1) / SCAN_THREADS;  // elements a thread stages of x, dt, z
    static constexpr int F = ROWS * NP / SCAN_THREADS;      // and of B and of C
};

// Sums v[0..R) over K lanes: the lane whose low bits are r ends with row r's.
// The first steps halve the rows a lane still adds, the rest add one value.
template <int R, int K>
KRK_DEV float sum_rows(float (&v)[R], int lane) {
    int off = K / 2;
#pragma unroll
    for (int n = R / 2; n > 0; n /= 2, off /= 2) {
        const bool upper = lane & off;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float mine = upper ? v[i + n] : v[i], theirs = upper ? v[i] : v[i + n];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, theirs, off);
        }
    }
    for (; off > 0; off /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    return v[0];
}

template <typename T, int K, int SPT, bool PADDED>
__global__ void __launch_bounds__(SCAN_THREADS) scan_kernel(ScanArgs a, int side) {
    using Sh = ScanShape<K, SPT>;
    constexpr int CH = Sh::CH, NP = Sh::NP, ROWS = Sh::ROWS, E = Sh::E, F = Sh::F;
    constexpr int R = K < 8 ? K : ROWS < 8 ? ROWS : 8;  // rows whose sums over the lanes are formed together
    __shared__ float2 s_step[ROWS][CH];                 // delta, delta x
    __shared__ float s_y[ROWS][CH];
    __shared__ __align__(16) float s_b[ROWS][NP], s_c[ROWS][NP];

    const int tid = threadIdx.x, lane = tid % K, per = a.D / a.G;
    const int req = blockIdx.x / side, cb = blockIdx.x - req * side, sides = side / a.G;
    const int g = cb / sides, ch0 = (cb - g * sides) * CH;  // within the group
    const int live = min(CH, per - ch0), d0 = g * per + ch0, ch = tid / K;
    const Span span = request_rows(a.cu, req, a.T);
    int to, from;
    if (!request_slots(a.slot, req, to, from)) return;

    float h[SPT], rate[SPT];
#pragma unroll
    for (int j = 0; j < SPT; ++j) {
        const int n = lane * SPT + j;
        const bool in = ch < live && (!PADDED || n < a.N);
        const int64_t at = (int64_t)(d0 + ch) * a.N + n;
        rate[j] = in ? a.a[at] * kLog2e : 0.0f;
        h[j] = in && from >= 0 ? ((const float*)a.slot.state)[from * a.slot.stride + at] : 0.0f;
    }

    // Element e of this thread is row (e * 128 + tid) / CH of the tile and channel tid % CH.
    const int mine = tid % CH, row0 = tid / CH;
    constexpr int STEP = SCAN_THREADS / CH;
    const bool open = mine < live;
    const float bias = open && a.dt_bias ? a.dt_bias[d0 + mine] : 0.0f, skip = open && a.d ? a.d[d0 + mine] : 0.0f;
    T xr[E], dtr[E], zr[E], br[F], cr[F];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int r = row0 + e * STEP, t = t0 + r;
            const bool in = open && r < ROWS && t < span.end;
            xr[e] = in ? ((const T*)a.x)[t * a.x_st + d0 + mine] : from_f32<T>(0.0f);
            dtr[e] = in ? ((const T*)a.dt)[t * a.dt_st + d0 + mine] : from_f32<T>(0.0f);
            zr[e] = in && a.z ? ((const T*)a.z)[t * a.z_st + d0 + mine] : from_f32<T>(0.0f);
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int i = f * SCAN_THREADS + tid, t = t0 + i / NP, n = i % NP;
            const bool in = t < span.end && n < a.N;
            br[f] = in ? ((const T*)a.b)[t * a.b_st + g * a.b_sg + n] : from_f32<T>(0.0f);
            cr[f] = in ? ((const T*)a.c)[t * a.c_st + g * a.c_sg + n] : from_f32<T>(0.0f);
        }
    };

    if (span.begin < span.end) fetch(span.begin);
    for (int t0 = span.begin; t0 < span.end; t0 += ROWS) {
        float dx[E], gate[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int r = row0 + e * STEP;
            const float x = to_f32(xr[e]);
            // rows behind the last one step by nothing: the states stay
            const float delta = t0 + r < span.end ? step_width(to_f32(dtr[e]) + bias) : 0.0f;
            if (r < ROWS) s_step[r][mine] = make_float2(delta, delta * x);
            dx[e] = skip * x;
            gate[e] = a.z ? fast_silu(to_f32(zr[e])) : 1.0f;
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int i = f * SCAN_THREADS + tid;
            s_b[i / NP][i % NP] = to_f32(br[f]);
            s_c[i / NP][i % NP] = to_f32(cr[f]);
        }
        __syncthreads();
        if (t0 + ROWS < span.end) fetch(t0 + ROWS);

        for (int r0 = 0; r0 < ROWS; r0 += R) {
            float y[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float2 st = s_step[r0 + i][ch];
                const float* b = s_b[r0 + i] + lane * SPT;
                const float* c = s_c[r0 + i] + lane * SPT;
                y[i] = 0.0f;
#pragma unroll
                for (int j = 0; j < SPT; ++j) {
                    h[j] = fmaf(fast_exp2(st.x * rate[j]), h[j], st.y * b[j]);
                    if (!PADDED || lane * SPT + j < a.N) y[i] = fmaf(h[j], c[j], y[i]);
                }
            }
            const float sum = sum_rows<R, K>(y, lane);
            // the lanes' bits from the highest: the row; lanes that differ in the others hold the same
            const int r = r0 + lane / (K / R);
            if (lane % (K / R) == 0) s_y[r][ch] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int r = row0 + e * STEP, t = t0 + r;
            if (open && r < ROWS && t < span.end)
                ((T*)a.out)[t * a.o_st + d0 + mine] = from_f32<T>((s_y[r][mine] + dx[e]) * gate[e]);
        }
    }

    if (to < 0) return;
#pragma unroll
    for (int j = 0; j < SPT; ++j) {
        const int n = lane * SPT + j;
        if (ch < live && (!PADDED || n < a.N))
            ((float*)a.slot.state)[to * a.slot.stride + (int64_t)(d0 + ch) * a.N + n] = h[j];
    }
}

// ---------------------------------------------------------------- single tokens
// Bound by memory: a request's states are read and written once.
constexpr int STEP_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(ScanArgs a, int lanes, int side) {
    const int t = blockIdx.x / side, i = (blockIdx.x - t * side) * STEP_THREADS + threadIdx.x;
    const int d = i / lanes, lane = i - d * lanes;
    int to, from;
    const bool live = request_slots(a.slot, t, to, from) && d < a.D;
    float x = 0.0f, sum = 0.0f;
    if (live) {
        const int g = d / (a.D / a.G);
        x = to_f32(((const T*)a.x)[t * a.x_st + d]);
        const float dt = to_f32(((const T*)a.dt)[t * a.dt_st + d]) + (a.dt_bias ? a.dt_bias[d] : 0.0f);
        const float delta = step_width(dt);
        const T* b = (const T*)a.b + t * a.b_st + g * a.b_sg;
        const T* c = (const T*)a.c + t * a.c_st + g * a.c_sg;
        const float* old = (const float*)a.slot.state + from * a.slot.stride + (int64_t)d * a.N;
        float* kept = (float*)a.slot.state + to * a.slot.stride + (int64_t)d * a.N;
        for (int n = lane; n < a.N; n += lanes) {
            float h = from >= 0 ? old[n] : 0.0f;
            h = fmaf(fast_exp2(delta * (a.a[(int64_t)d * a.N + n] * kLog2e)), h, delta * x * to_f32(b[n]));
            kept[n] = h;
            sum = fmaf(h, to_f32(c[n]), sum);
        }
    }
    for (int o = lanes / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (live && lane == 0) {
        const float y = sum + (a.d ? a.d[d] : 0.0f) * x;
        const float gate = a.z ? fast_silu(to_f32(((const T*)a.z)[t * a.z_st + d])) : 1.0f;
        ((T*)a.out)[t * a.o_st + d] = from_f32<T>(y * gate);
    }
}

template <typename T, int K, int SPT, bool PADDED>
cudaError_t launch_scan(const ScanArgs& a, cudaStream_t s) {
    using Sh = ScanShape<K, SPT>;
    const int per = a.D / a.G, side = (per + Sh::CH - 1) / Sh::CH * a.G;
    if ((int64_t)side * a.S > INT32_MAX) return cudaErrorInvalidValue;
    scan_kernel<T, K, SPT, PADDED><<<side * a.S, SCAN_THREADS, 0, s>>>(a, side);
    add_launches(1);
    return cudaGetLastError();
}

template <typename T, int K, int SPT>
cudaError_t scan_padded(const ScanArgs& a, cudaStream_t s) {
    return a.N == K * SPT ? launch_scan<T, K, SPT, false>(a, s) : launch_scan<T, K, SPT, true>(a, s);
}

template <typename T>
cudaError_t scan_type(const ScanArgs& a, cudaStream_t s) {
    if (a.N <= 4) return scan_padded<T, 4, 1>(a, s);
    if (a.N <= 8) return scan_padded<T, 4, 2>(a, s);
    if (a.N <= 16) return scan_padded<T, 8, 2>(a, s);
    if (a.N <= 32) return scan_padded<T, 8, 4>(a, s);
    if (a.N <= 64) return scan_padded<T, 16, 4>(a, s);
    if (a.N <= 128) return scan_padded<T, 32, 4>(a, s);
    return scan_padded<T, 32, 8>(a, s);
}

template <typename T>
cudaError_t step_type(const ScanArgs& a, cudaStream_t s) {
    int lanes = 1;
    while (lanes < 32 && lanes < a.N) lanes *= 2;
    const int64_t side = ((int64_t)a.D * lanes + STEP_THREADS - 1) / STEP_THREADS;
    if (side * a.T > INT32_MAX) return cudaErrorInvalidValue;
    step_kernel<T><<<(unsigned)(side * a.T), STEP_THREADS, 0, s>>>(a, lanes, (int)side);
    add_launches(1);
    return cudaGetLastError();
}

}  // namespace

cudaError_t selective_scan(const ScanArgs& a, int type, cudaStream_t s) {
    return type == ELEM_F32 ? scan_type<float>(a, s)
                            : type == ELEM_F16 ? scan_type<__half>(a, s) : scan_type<__nv_bfloat16>(a, s);
}
cudaError_t selective_step(const ScanArgs& a, int type, cudaStream_t s) {
    return type == ELEM_F32 ? step_type<float>(a, s)
                            : type == ELEM_F16 ? step_type<__half>(a, s) : step_type<__nv_bfloat16>(a, s);
}

}  // namespace krk
