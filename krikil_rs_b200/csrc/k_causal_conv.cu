// Short causal depthwise convolution over packed requests and over single
// tokens, with the rows before a request in a pool of state slots:
//   y[t] = act(bias + sum_j w[j] x[t - (W-1) + j]).
// Bound by memory: each element of x is read once from HBM (the W-1 rows that
// runs share come from L2) and each of y written once.  A thread takes a run of
// rows of its channels, so that a row's element is loaded once for the W outputs
// that it is in; the exponential unit (two a value for SiLU) is busy two thirds of
// that time.  64 prompts of 16,352 rows x 8192 bfloat16 channels (541 MB): 96 us,
// 86% of the measured copy rate; 38 us for 4080 rows x 4001 channels, whose rows
// allow two bytes an access (1.7 TB/s).
#include "kernels.h"
#include "paged.h"
#include "recurrent.cuh"

namespace krk {
namespace {

constexpr int CONV_THREADS = 128;
constexpr int CONV_GROUP = 4;  // rows that are computed together
constexpr int CONV_AHEAD = 8;   // rows on their way to a thread

// A thread's copy of V elements into its place in shared memory; none for those of two bytes, which are loaded.
template <int BYTES>
KRK_DEV void copy_ahead(void* smem, const void* gmem) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(smem)), "l"(gmem), "n"(BYTES) : "memory");
}

// One thread: V channels, their taps and bias; in pairs, a lone channel in the first half.
template <typename T, int W, int V>
struct ConvColumn {
    static constexpr int P = pairs_of<V>;
    const ConvArgs& a;
    int c;
    float2 w[W][P], bias[P];

    KRK_DEV ConvColumn(const ConvArgs& args, int channel) : a(args), c(channel) {
        __align__(16) float flat[V * W];
        const float* from = a.w + (int64_t)c * W;
        if (V * W % 4 == 0 && a.aligned) {
#pragma unroll
            for (int i = 0; i < V * W / 4; ++i) reinterpret_cast<float4*>(flat)[i] = reinterpret_cast<const float4*>(from)[i];
        } else {
#pragma unroll
            for (int i = 0; i < V * W; ++i) flat[i] = from[i];
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            constexpr int next = V > 1;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = make_float2(flat[2 * i * W + j], flat[(2 * i + next) * W + j]);
            bias[i] = a.bias ? make_float2(a.bias[c + 2 * i], a.bias[c + 2 * i + next]) : make_float2(0.0f, 0.0f);
        }
    }
    KRK_DEV const T* row(int t) const { return (const T*)a.x + t * a.x_st + c; }
    KRK_DEV T* kept(int slot, int k) const { return (T*)a.slot.state + slot * a.slot.stride + (int64_t)k * a.C + c; }
    // Row t of a request whose rows begin at `begin`: a packed row, or one of the W-1 before them.
    KRK_DEV Pack<T, V> tap(int t, int begin, int from) const {
        if (t >= begin) return load_pack<T, V>(row(t));
        if (from >= 0) return load_pack<T, V>(kept(from, W - 1 + t - begin));
        Pack<T, V> zero;
#pragma unroll
        for (int i = 0; i < V; ++i) zero.v[i] = from_f32<T>(0.0f);
        return zero;
    }
    // One row's output, from the rows before it (the latest last) and itself.
    KRK_DEV Pack<T, V> convolve(const float2 (&win)[W - 1][P], const float2 (&x)[P]) const {
        float2 y[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            y[i] = bias[i];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) y[i] = __ffma2_rn(w[j][i], win[j][i], y[i]);
            y[i] = __ffma2_rn(w[W - 1][i], x[i], y[i]);
            if (a.silu) y[i] = fast_silu(y[i]);
        }
        return pack<T, V>(y);
    }
    // Rows [i, j) of a request that begins at `begin`, CONV_AHEAD rows on their way to the thread's own places of `ring`
    // (so many, of all threads, keep the memory busy; in registers there is room for a quarter of them).
    KRK_DEV void run(int i, int j, int begin, int from, Pack<T, V> (*ring)[CONV_THREADS]) const {
        if (i >= j) return;
        constexpr int BYTES = V * sizeof(T);
        const T* in = row(i);
        T* out = (T*)a.out + i * a.o_st + c;
        const int left = j - i;
        const auto fetch = [&](int u) {
            if (u < left) {
                Pack<T, V>* place = &ring[u % CONV_AHEAD][threadIdx.x];
                if constexpr (BYTES >= 4)
                    copy_ahead<BYTES>(place, in);
                else
                    *place = load_pack<T, V>(in);
            }
            in += a.x_st;
        };
        for (int u = 0; u < CONV_AHEAD; u += CONV_GROUP) {
#pragma unroll
            for (int k = 0; k < CONV_GROUP; ++k) fetch(u + k);
            cp_async_commit();
        }
        float2 win[W - 1][P];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) unpack(tap(i - (W - 1) + k, begin, from), win[k]);
        for (int u = 0; u < left; u += CONV_GROUP) {
            cp_async_wait<CONV_AHEAD / CONV_GROUP - 1>();
            Pack<T, V> now[CONV_GROUP];
#pragma unroll
            for (int k = 0; k < CONV_GROUP; ++k) now[k] = ring[(u + k) % CONV_AHEAD][threadIdx.x];
#pragma unroll
            for (int k = 0; k < CONV_GROUP; ++k) fetch(u + CONV_AHEAD + k);
            cp_async_commit();
#pragma unroll
            for (int k = 0; k < CONV_GROUP; ++k) {
                float2 x[P];
                unpack(now[k], x);
                const Pack<T, V> y = convolve(win, x);
                if (u + k < left) store_pack<T, V>(out, y);
                out += a.o_st;
#pragma unroll
                for (int v = 0; v < P; ++v) {
#pragma unroll
                    for (int q = 0; q + 1 < W - 1; ++q) win[q][v] = win[q + 1][v];
                    win[W - 2][v] = x[v];
                }
            }
        }
    }
    // The W-1 rows that the request ends with, into its slot (which may be the one that they are read from).
    KRK_DEV void keep(const Span& span, int to, int from) const {
        if (to < 0) return;
        Pack<T, V> last[W - 1];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) last[k] = tap(span.end - (W - 1) + k, span.begin, from);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) store_pack<T, V>(kept(to, k), last[k]);
    }
};

// The number of requests that begin before row r (their beginnings ascend): a
// warp looks at 32 of them at a time.
KRK_DEV int requests_before(const int32_t* cu, int S, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = S;  // the answer lies in [lo, lo + n]
    while (n > 0) {
        const int step = (n + 31) / 32, i = lo + (lane + 1) * step - 1;
        const bool before = i < lo + n && cu[i] < r;
        const int k = __popc(__ballot_sync(0xffffffffu, before));
        const int end = lo + n;
        lo += k * step;
        n = min(step - 1, end - lo);
    }
    return lo;
}

// A block takes `rows` packed rows of CONV_THREADS * V channels, and the
// requests that begin there: it keeps their states, and computes their first
// W-1 rows even past its own, so that whatever reads a request's old state is
// the thread that writes the new one.  Requests without rows, of which there may
// be any number in one place, are left to blocks of their own, 32 for each.
template <typename T, int W, int V>
__global__ void __launch_bounds__(CONV_THREADS) conv_kernel(ConvArgs a, int rows, int chunks, int side) {
    __shared__ Pack<T, V> ring[CONV_AHEAD][CONV_THREADS];
    const int chunk = blockIdx.x / side, c = ((blockIdx.x - chunk * side) * CONV_THREADS + threadIdx.x) * V;
    const bool open = c < a.C;
    const ConvColumn<T, W, V> col(a, open ? c : 0);
    int to, from;
    if (chunk >= chunks) {
        const int s0 = (chunk - chunks) * 32, s = s0 + (threadIdx.x & 31);
        bool idle = false;
        if (s < a.S) {
            const Span span = request_rows(a.cu, s, a.T);
            idle = span.begin == span.end && request_slots(a.slot, s, to, from) && to >= 0 && to != from;
        }
        for (unsigned left = __ballot_sync(0xffffffffu, idle); left; left &= left - 1) {
            const int i = s0 + __ffs(left) - 1;
            if (open && request_slots(a.slot, i, to, from)) col.keep({0, 0}, to, from);
        }
        return;
    }
    const int r0 = chunk * rows;
    const bool last = chunk == chunks - 1;
    const int r1 = last ? a.T : r0 + rows;
    int s = chunk == 0 ? 0 : requests_before(a.cu, a.S, r0);
    if (s > 0) {
        const Span span = request_rows(a.cu, s - 1, a.T);
        if (open && span.end > r0 && request_slots(a.slot, s - 1, to, from))
            col.run(max(r0, min(span.begin + W - 1, span.end)), min(span.end, r1), span.begin, from, ring);
    }
    while (s < a.S) {
        const Span span = request_rows(a.cu, s, a.T);
        if (!last && span.begin >= r1) break;
        if (span.begin == span.end) {  // on to the one that has this place's row
            s = max(s + 1, requests_before(a.cu + 1, a.S, span.begin + 1));
            continue;
        }
        if (open && request_slots(a.slot, s, to, from)) {
            col.run(span.begin, min(span.end, max(r1, span.begin + W - 1)), span.begin, from, ring);
            col.keep(span, to, from);
        }
        ++s;
    }
}

// One row a request: a thread takes `turns` times R of them, with the same taps.
template <typename T, int W, int V, int R>
__global__ void __launch_bounds__(CONV_THREADS) conv_step_kernel(ConvArgs a, int turns, int side) {
    const int group = blockIdx.x / side, c = ((blockIdx.x - group * side) * CONV_THREADS + threadIdx.x) * V;
    if (c >= a.C) return;
    const ConvColumn<T, W, V> col(a, c);
    const int64_t share = (int64_t)turns * R;
    for (int64_t t = group * share; t < min((group + 1) * share, (int64_t)a.T); t += R) {
        const int t0 = (int)t;
        int to[R], from[R];
        load_slots(a.slot, t0, a.T, to, from);
        bool live[R];
        Pack<T, V> rows[R][W];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            live[r] = t0 + r < a.T && valid_slots(a.slot, to[r], from[r]);
            rows[r][W - 1] = load_pack<T, V>(col.row(min(t0 + r, a.T - 1)));
            const bool begun = live[r] && from[r] >= 0;  // (any slot's rows if not: in a branch each load is waited for)
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                rows[r][k] = load_pack<T, V>(col.kept(begun ? from[r] : 0, k));
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (!begun) rows[r][k].v[v] = from_f32<T>(0.0f);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (!live[r]) continue;
            float2 win[W - 1][pairs_of<V>], x[pairs_of<V>];
#pragma unroll
            for (int k = 0; k < W - 1; ++k) unpack(rows[r][k], win[k]);
            unpack(rows[r][W - 1], x);
            store_pack<T, V>((T*)a.out + (t0 + r) * a.o_st + c, col.convolve(win, x));
#pragma unroll
            for (int k = 0; k < W - 1; ++k) store_pack<T, V>(col.kept(to[r], k), rows[r][k + 1]);
        }
    }
}

template <typename T, int W, int V>
cudaError_t launch_conv(const ConvArgs& a, cudaStream_t s) {
    const int side = (a.C + CONV_THREADS * V - 1) / (CONV_THREADS * V);
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    if (!a.cu) {
        // two requests a thread at once when that leaves every multiprocessor a full set of threads, then so many times
        // that there are seven blocks a multiprocessor, which load the taps once (509 requests x 8192 bfloat16 channels:
        // 16 us by four times, 18.6 by one; that form's 62 registers leave room for eight blocks, those of fewer taps or
        // channels a thread for more, which no measurement has set apart)
        const int64_t units = (int64_t)a.T * side;
        if (units > INT32_MAX) return cudaErrorInvalidValue;
        if (units >= (int64_t)sms * 2048 / CONV_THREADS) {
            const int turns = (int)((units / 2 + 7 * sms - 1) / (7 * sms));
            conv_step_kernel<T, W, V, 2><<<(unsigned)((a.T + 2LL * turns - 1) / (2 * turns) * side), CONV_THREADS, 0, s>>>(
                a, turns, side);
        } else {
            conv_step_kernel<T, W, V, 1><<<(unsigned)units, CONV_THREADS, 0, s>>>(a, 1, side);
        }
    } else {
        const int64_t share = (int64_t)a.T * side / (sms * 16);
        const int rows = share < 8 ? 8 : share > 64 ? 64 : (int)share;
        const int64_t chunks = a.T > 0 ? (a.T + (int64_t)rows - 1) / rows : 1;
        const int64_t blocks = (chunks + (a.slot.state ? (a.S + 31LL) / 32 : 0)) * side;
        if (blocks > INT32_MAX) return cudaErrorInvalidValue;
        conv_kernel<T, W, V><<<(unsigned)blocks, CONV_THREADS, 0, s>>>(a, rows, (int)chunks, side);
    }
    add_launches(1);
    return cudaGetLastError();
}

// Whether rows are accessed V channels at a time.
template <typename T>
bool conv_fits(const ConvArgs& a, int V) {
    const size_t bytes = V * sizeof(T);
    return a.C % V == 0 && fits(a.x, a.T > 1 ? a.x_st : 0, bytes, sizeof(T)) &&
           fits(a.out, a.T > 1 ? a.o_st : 0, bytes, sizeof(T)) &&
           fits(a.slot.state, a.slot.num_slots > 1 ? a.slot.stride : 0, bytes, sizeof(T));
}

// Eight bytes a thread: with sixteen its taps and window leave too few threads a multiprocessor (98 and 121 us for
// 16,352 rows of 8192 bfloat16 channels).
template <typename T, int W>
cudaError_t conv_width(ConvArgs a, cudaStream_t s) {
    a.aligned = fits(a.w, 0, 16, 4);
    constexpr int V = 8 / sizeof(T);
    if (conv_fits<T>(a, V)) return launch_conv<T, W, V>(a, s);
    if (V > 2 && conv_fits<T>(a, 2)) return launch_conv<T, W, 2>(a, s);
    return launch_conv<T, W, 1>(a, s);
}

template <typename T>
cudaError_t conv_type(const ConvArgs& a, int W, cudaStream_t s) {
    return W == 2 ? conv_width<T, 2>(a, s) : W == 3 ? conv_width<T, 3>(a, s) : conv_width<T, 4>(a, s);
}

}  // namespace

cudaError_t causal_conv(const ConvArgs& a, int W, int type, cudaStream_t s) {
    return type == ELEM_F32 ? conv_type<float>(a, W, s)
                            : type == ELEM_F16 ? conv_type<__half>(a, W, s) : conv_type<__nv_bfloat16>(a, W, s);
}

}  // namespace krk
