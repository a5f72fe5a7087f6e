// Log probabilities of given tokens, the entropy and the best alternatives of
// each row of logits: with m the row's maximum and s = sum e^(x - m),
//   lp(i) = (x_i - m) - log s,   H = log s - sum e^(x - m) (x - m) / s.
//
// One pass over the row, 16 bytes an access: each thread keeps the running
// maximum of its own logits with the two sums relative to it, and where that
// maximum is.  Bound by memory for 32 bits; for 16 bits the exponential unit (one
// a logit, 16 a clock and multiprocessor) is close behind.
//
// The alternatives cost the pass nothing: of the threads' maxima the top-th
// largest is a bound that no alternative lies below, and only the threads whose
// maximum reaches it can hold one, as many as there are alternatives.  Their
// logits are read again, and of the few that reach the bound each one's rank is
// its place.  Few rows are shared by the blocks of a cluster, whose sums and
// lists its first block joins.
//
// Measured: float32, 1024 x 50001, 36 us (5.6 TB/s, 85% of the copy rate);
// bfloat16, 4096 x 50001, 82 us (5.0 TB/s; issue slots 75% busy, the exponential
// unit 62%); float32, one row of 131,072 with 20 alternatives, 8.5 us in 16 blocks;
// bfloat16, 4096 x 32768 with 20 alternatives, 80 us, 54 without them; 8192 x 2048
// with five, 32 us, 15 without them.
#include <cooperative_groups.h>

#include "kernels.h"
#include "paged.h"
#include "recurrent.cuh"

namespace krk {
namespace {

namespace cg = cooperative_groups;

constexpr int LP_SHORT = 1024;  // accesses of a row that a small block takes in any case
constexpr int LP_LIST = 32;     // entries of a sorted list, LOGPROBS_MAX_TOP of them used
constexpr int LP_ROOM = 1024;   // logits that reach the bound; for more (the best ones all in few threads' ways) see below
constexpr int LP_AHEAD = 4;     // accesses on their way
// Threads a multiprocessor that registers are left for: all of them in 32 bits, and 40 registers each in 16 (82 us for
// 4096 x 50001; 87 with 56 registers, 136 with 32, which spill).  Blocks of two warps reach 1024, by their shared memory
// (12.8 KB, so that 16 of them fit).
template <typename T>
constexpr int LP_RESIDENT = sizeof(T) == 4 ? 2048 : 1536;
constexpr float kLog2e = 1.44269504088896341f, kLowest = -3.402823466e38f;
using Key = unsigned long long;

// The order of the alternatives as whole numbers: larger logits first, of equal
// ones the lower index; NaN counts as -inf and -0 as 0.  Never 0.
KRK_DEV Key order_key(float x, int i) {
    x = x == x ? x + 0.0f : -INFINITY;
    const unsigned u = __float_as_uint(x);
    return (Key)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - (unsigned)i);
}
KRK_DEV int key_index(Key k) { return (int)(0xffffffffu - (unsigned)k); }
KRK_DEV Key later(Key a, Key b) { return a < b ? a : b; }
KRK_DEV Key sooner(Key a, Key b) { return a > b ? a : b; }

// sum e^(x - ref) and sum e^(x - ref) (x - ref) over some logits with maximum m; ref = max(m, lowest).
struct Sums {
    float m, s, e;
};
KRK_DEV float ref_of(float m) { return fmaxf(m, kLowest); }
// Of a warp's, relative to their common maximum.
KRK_DEV Sums warp_join(const Sums& a) {
    const float m = warp_max(a.m), d = fmaxf(ref_of(a.m) - ref_of(m), -1000.0f), f = fast_exp2(d * kLog2e);
    // (what lies 1000 below adds nothing)
    return {m, warp_sum(a.s * f), warp_sum(f * fmaf(a.s, d, a.e))};
}
// (x - m) - log s; a row that its mask leaves empty gives every token -inf.
KRK_DEV float log_prob(float x, const Sums& a) { return a.s == 0.0f ? -INFINITY : (x - ref_of(a.m)) - logf(a.s); }

// Sorts a warp's keys, one a lane, the first the largest.
KRK_DEV Key sort_step(Key k, int lane, int size, int o) {
    const Key other = __shfl_xor_sync(0xffffffffu, k, o);
    const bool first = ((lane & o) == 0) == ((lane & size) == 0);
    return first ? sooner(k, other) : later(k, other);
}
KRK_DEV Key warp_sort(Key k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int o = size / 2; o > 0; o /= 2) k = sort_step(k, lane, size, o);
    return k;
}
// The 32 largest of two sorted lists, sorted.
KRK_DEV Key warp_merge(const Key* a, const Key* b, int lane) {
    Key k = sooner(a[lane], b[31 - lane]);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) k = sort_step(k, lane, 32, o);
    return k;
}
// Merges n (a power of two) sorted lists into the first.  All WARPS warps take part.
template <int WARPS, typename L>
KRK_DEV void merge_lists(L lists, int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int half = n / 2; half > 0; half /= 2) {
        for (int i = warp; i < half; i += WARPS) {
            const Key k = warp_merge(lists(i), lists(i + half), lane);
            __syncwarp();
            lists(i)[lane] = k;
        }
        __syncthreads();
    }
}

template <typename T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    using Vec = Pack<T, VEC>;
    const T* x;      // logits [0, V)
    int V, lead;     // vector k holds logits k * VEC - lead ..
    KRK_DEV Row(const LogprobArgs& a, int row) : x((const T*)a.logits + row * a.ld), V(a.V) {
        lead = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    }
    KRK_DEV int vectors() const { return (int)(((int64_t)lead + V + VEC - 1) / VEC); }
    KRK_DEV int first(int k) const { return k * VEC - lead; }
    KRK_DEV bool whole(int k) const { return first(k) >= 0 && first(k) <= V - VEC; }
    KRK_DEV Vec load(int k) const { return load_pack<T, VEC>(x + first(k)); }
    // Any vector; NaN-free -inf where there is no logit.
    KRK_DEV void floats(int k, float (&v)[VEC]) const {
        if (whole(k)) {
            const Vec p = load(k);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = to_f32(p.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int i = first(k) + j;
                v[j] = i >= 0 && i < V ? to_f32(x[i]) : -INFINITY;
            }
        }
    }
    KRK_DEV bool has(int k, int j) const { return first(k) + j >= 0 && first(k) + j < V; }
};

// A thread's sums over its vectors, in two halves, and the first vector that holds its maximum (-1: none yet).
template <int VEC>
struct Running {
    float m = -INFINITY;
    float2 s = {0.0f, 0.0f}, e = {0.0f, 0.0f};
    int best = -1;
    // A larger maximum, or the first one; NaN counts as -inf.
    KRK_DEV void raise(float top, int k) {
        top = top == top ? top : -INFINITY;
        if (top <= m && best >= 0) return;
        const float d = fmaxf(ref_of(m) - ref_of(top), -1000.0f), f = fast_exp2(d * kLog2e);
        e = make_float2(f * fmaf(s.x, d, e.x), f * fmaf(s.y, d, e.y));
        s = make_float2(s.x * f, s.y * f);
        m = top;
        best = k;
    }
    KRK_DEV void add(const float (&x)[VEC], int k) {
        float top = x[0];
#pragma unroll
        for (int j = 1; j < VEC; ++j) top = fmaxf(top, x[j]);
        if (!(top <= m) || best < 0) raise(top, k);
        const float r = ref_of(m);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 u = __fadd2_rn(make_float2(x[j], x[j + 1]), make_float2(-r, -r));
            const float2 t = __fmul2_rn(u, make_float2(kLog2e, kLog2e));
            const float2 p = make_float2(fast_exp2(t.x), fast_exp2(t.y));
            s = __fadd2_rn(s, p);
            e = __ffma2_rn(p, make_float2(fmaxf(u.x, -1000.0f), fmaxf(u.y, -1000.0f)), e);  // 0 times -inf is 0 here
        }
    }
};

template <int WARPS>
struct Shared {
    Sums part[WARPS], all;
    Key list[WARPS][LP_LIST];   // sorted lists; in the end the first is the block's
    Key near[LP_ROOM];             // logits that reach the bound
    Key gathered[16][LP_LIST];     // a cluster's lists
    int count;
};

// The largest of a warp's keys: of their high halves, then of the low ones that go with it.
KRK_DEV Key warp_first(Key k) {
    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32));
    const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32) == high ? (unsigned)k : 0u);
    return (Key)high << 32 | low;
}

// The block's `top` first keys into sh.list[0], sorted, 0 behind them.  `best`: the thread's first key.
template <typename T, int WARPS>
KRK_DEV void best_keys(const Row<T>& row, int k0, int k1, int top, Key best, Shared<WARPS>& sh) {
    constexpr int VEC = Row<T>::VEC, THREADS = 32 * WARPS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (top == 1) {
        best = warp_first(best);
        sh.list[warp][lane] = lane == 0 ? best : 0;
        __syncthreads();
        if (warp == 0) {
            best = warp_first(lane < WARPS ? sh.list[lane][0] : 0);
            if (lane == 0) sh.list[0][0] = best;
        }
        __syncthreads();
        return;
    }
    sh.list[warp][lane] = warp_sort(best, lane);
    if (tid == 0) sh.count = 0;
    __syncthreads();
    merge_lists<WARPS>([&](int i) { return sh.list[i]; }, WARPS);
    // The top-th thread's first key (0: there are not so many threads with logits) is one that `top` keys reach, so
    // that those that do are the first ones; they are in the ways of the threads that the list names.
    const Key bound = sh.list[0][top - 1];
    const unsigned high = (unsigned)(bound >> 32);
    const float bound_value = bound == 0 ? -INFINITY : __uint_as_float(high & 0x80000000u ? high & 0x7fffffffu : ~high);
    const int ways = (k1 - k0 + THREADS - 1) / THREADS;
    for (int i = tid; i < top * ways; i += THREADS) {
        const int which = i / ways;
        const Key first = sh.list[0][which];
        const int k = k0 + ((key_index(first) + row.lead) / VEC - k0) % THREADS + (i - which * ways) * THREADS;
        if (first == 0 || k >= k1) continue;
        float v[VEC];
        row.floats(k, v);
        float near = v[0];
#pragma unroll
        for (int q = 1; q < VEC; ++q) near = fmaxf(near, v[q]);
        if (near < bound_value) continue;  // (NaN counts as -inf, and only that bound takes it)
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
            if (v[q] < bound_value) continue;
            const Key key = order_key(v[q], row.first(k) + q);
            if (key >= bound && row.has(k, q)) {
                const int at = atomicAdd(&sh.count, 1);  // (in any order: ranks tell)
                if (at < LP_ROOM) sh.near[at] = key;
            }
        }
    }
    __syncthreads();
    const int n = sh.count;
    if (tid < LP_LIST) sh.list[0][tid] = 0;
    __syncthreads();
    if (n <= LP_ROOM) {
        for (int i = tid; i < n; i += THREADS) {
            const Key key = sh.near[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += sh.near[j] > key;
            if (rank < top) sh.list[0][rank] = key;
        }
        __syncthreads();
        return;
    }
    // More than there is room for: one after the other, a pass each.
    Key before = ~0ull;
    for (int i = 0; i < top; ++i) {
        Key next = 0;
        for (int k = k0 + tid; k < k1; k += THREADS) {
            float v[VEC];
            row.floats(k, v);
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                const Key key = order_key(v[q], row.first(k) + q);
                if (key < before && row.has(k, q)) next = sooner(next, key);
            }
        }
        next = warp_first(next);
        if (lane == 0) sh.near[warp] = next;
        __syncthreads();
        next = sh.near[0];
        for (int w = 1; w < WARPS; ++w) next = sooner(next, sh.near[w]);
        __syncthreads();
        if (tid == 0) sh.list[0][i] = next;
        if (next == 0) break;
        before = next;
    }
    __syncthreads();
}

// One block a row, or the `parts` blocks of a cluster.
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, LP_RESIDENT<T> / (32 * WARPS)) logprobs_kernel(LogprobArgs a, int part_bits) {
    constexpr int VEC = Row<T>::VEC, THREADS = 32 * WARPS;
    __shared__ Shared<WARPS> sh;
    const int parts = 1 << part_bits, r = blockIdx.x >> part_bits, part = blockIdx.x & (parts - 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Row<T> row(a, r);
    const int64_t n = row.vectors();
    const int k0 = (int)(n * part >> part_bits), k1 = (int)(n * (part + 1) >> part_bits);

    Running<VEC> run;
    // (a thread's vectors are THREADS apart, the row's ends among them, which may not be whole)
    const int w0 = row.whole(k0) ? k0 : k0 + 1, w1 = k1 > w0 && !row.whole(k1 - 1) ? k1 - 1 : k1;
    int k = k0 + tid;
    if (k < w0) {
        float v[VEC];
        row.floats(k, v);
        run.add(v, k);
        k += THREADS;
    }
    const auto take = [&](const typename Row<T>::Vec& p, int at) {
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = to_f32(p.v[j]);
        run.add(v, at);
    };
    typename Row<T>::Vec p[LP_AHEAD];
    for (; k + (LP_AHEAD - 1) * THREADS < w1; k += LP_AHEAD * THREADS) {
#pragma unroll
        for (int i = 0; i < LP_AHEAD; ++i) p[i] = row.load(k + i * THREADS);
#pragma unroll
        for (int i = 0; i < LP_AHEAD; ++i) take(p[i], k + i * THREADS);
    }
    if (w0 < w1) {  // (the last one again where there are no more: in a branch each load would be waited for)
#pragma unroll
        for (int i = 0; i < LP_AHEAD - 1; ++i) p[i] = row.load(min(k + i * THREADS, w1 - 1));
#pragma unroll
        for (int i = 0; i < LP_AHEAD - 1; ++i)
            if (k + i * THREADS < w1) take(p[i], k + i * THREADS);
    }
    if (w1 < k1 && (w1 - k0) % THREADS == tid) {
        float v[VEC];
        row.floats(w1, v);
        run.add(v, w1);
    }

    Sums sums = warp_join({run.m, run.s.x + run.s.y, run.e.x + run.e.y});
    if (lane == 0) sh.part[warp] = sums;
    if (a.top > 0) {
        Key best = 0;
        if (run.best >= 0) {  // the first of the vector's logits that is the maximum
            float v[VEC];
            row.floats(run.best, v);
            int at = VEC;
#pragma unroll
            for (int j = VEC - 1; j >= 0; --j)
                if ((v[j] == run.m || run.m == -INFINITY) && row.has(run.best, j)) at = j;
            best = order_key(run.m, row.first(run.best) + at);
        }
        best_keys<T, WARPS>(row, k0, k1, a.top, best, sh);
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        sums = warp_join(lane < WARPS ? sh.part[lane] : Sums{-INFINITY, 0.0f, 0.0f});
        if (lane == 0) sh.all = sums;
    }
    if (parts > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (part == 0) {
            if (a.top > 0) {
                for (int i = warp; i < parts; i += WARPS)
                    sh.gathered[i][lane] = cluster.map_shared_rank(&sh, i)->list[0][lane];
                __syncthreads();
                merge_lists<WARPS>([&](int i) { return sh.gathered[i]; }, parts);
                if (warp == 0) sh.list[0][lane] = sh.gathered[0][lane];
            }
            if (warp == 0) {
                sums = warp_join(lane < parts ? cluster.map_shared_rank(&sh, lane)->all : Sums{-INFINITY, 0.0f, 0.0f});
            }
        }
        cluster.sync();  // the others' memory is theirs until here
        if (part > 0) return;
        if (warp == 0 && lane == 0) sh.all = sums;
    }
    __syncthreads();
    sums = sh.all;
    if (a.entropy && tid == 0) a.entropy[r] = sums.s == 0.0f ? 0.0f : logf(sums.s) - sums.e / sums.s;
    for (int i = tid; i < a.K; i += THREADS) {
        const int id = a.tokens[(int64_t)r * a.K + i];
        if (id >= a.V) check_fail(CHK_TOKEN);
        a.lp[(int64_t)r * a.K + i] = id < 0 ? 0.0f : id >= a.V ? -INFINITY : log_prob(to_f32(row.x[id]), sums);
    }
    if (tid < a.top) {
        const int id = key_index(sh.list[0][tid]);
        a.top_ids[(int64_t)r * a.top + tid] = id;
        a.top_lp[(int64_t)r * a.top + tid] = log_prob(to_f32(row.x[id]), sums);
    }
}

template <typename T, int WARPS>
cudaError_t launch(const LogprobArgs& a, int part_bits, cudaStream_t s) {
    const int parts = 1 << part_bits;
    if ((int64_t)a.R * parts > INT32_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.R * parts));
    cfg.blockDim = dim3(32 * WARPS);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1;
    if (parts > 8) {
        const cudaError_t e = cudaFuncSetAttribute(logprobs_kernel<T, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    const cudaError_t e = cudaLaunchKernelEx(&cfg, logprobs_kernel<T, WARPS>, a, part_bits);
    if (e == cudaSuccess) add_launches(1);
    return e;
}

template <typename T>
cudaError_t logprobs_type(const LogprobArgs& a, cudaStream_t s) {
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    const int64_t vectors = (int64_t)a.V * sizeof(T) / 16;
    // A row's end costs each warp about 500 instructions, as much as ten accesses: small blocks for short rows, and for
    // 16 bits, where instructions are short, when there are rows for all multiprocessors (bfloat16, 4096 x 32768 with
    // 20 alternatives: 84 us with four warps, 90 with eight, 153 with two; float32, 1024 x 50001: 47, 36 and 51).
    if (vectors <= LP_SHORT) return launch<T, 2>(a, 0, s);
    if (sizeof(T) == 2 && a.R >= 4 * sms) return launch<T, 4>(a, 0, s);
    // A cluster for each of few rows: up to a block a multiprocessor while a thread has two accesses, up to five while it
    // has sixteen (float32, 148 x 262144: 58 us in one block a row, 31 in four, 36 in eight; bfloat16, 64 x 131072 with 20
    // alternatives: 13.6 in two, 12.8 in four, 15.5 in eight).
    int bits = 0;
    while (bits < 4) {
        const int64_t blocks = (int64_t)a.R << (bits + 1), accesses = vectors / (8 * 32) >> (bits + 1);
        if (blocks > 5 * sms || accesses < (blocks <= sms ? 2 : 16)) break;
        ++bits;
    }
    return launch<T, 8>(a, bits, s);
}

}  // namespace

cudaError_t token_logprobs(const LogprobArgs& a, int type, cudaStream_t s) {
    return type == ELEM_F32 ? logprobs_type<float>(a, s)
                            : type == ELEM_F16 ? logprobs_type<__half>(a, s) : logprobs_type<__nv_bfloat16>(a, s);
}

}  // namespace krk
