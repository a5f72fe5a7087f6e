// Paged key-value cache: page planning and release on the device, and RoPE +
// append through a slot map.
#include <math.h>

#include "elem.cuh"
#include "kernels.h"
#include "paged.h"

namespace krk {
namespace {

// ---------------------------------------------------------------- the pages
// Planning is two prefix sums over the requests -- of their new tokens and of
// the pages that they lack -- and then independent writes: one entry a page and
// a position and a slot a token, found by bisecting a chunk's prefix sums.
// Every block scans all requests itself (a few KB from L2), so blocks need
// nothing of each other.  A small step, bound by latency, is one block's work.
// A large one is dealt to the whole device by a kernel that writes only what no
// block reads, and a second kernel of one block, which scans while the first
// one writes, then updates what both have read: the lengths and the count may
// be updated in place.  (249,880 prompt tokens: 438 us in one block, 19 us in a
// cluster of eight, whose stores bound it, 5.9 us so.)
constexpr int PLAN_THREADS = 1024, PLAN_WARPS = PLAN_THREADS / 32, PLAN_MIN_THREADS = 128;
constexpr int PLAN_ONE_BLOCK = 4096;  // writes up to which one block does all (61 requests' 7800 tokens: 8.3 us, 5.8 us
                                      // in two kernels; 1024 requests' 4096: 7.7 and 9.4 us)
enum PlanMode { PLAN_ALL, PLAN_FILL, PLAN_COMMIT };

struct PlanScratch {
    long long warp[2][PLAN_WARPS + 1];
    int bad;
    // of a chunk's requests: tokens and pages before them, what they hold, their pages so far
    int tokens[PLAN_THREADS], pages[PLAN_THREADS], len[PLAN_THREADS], have[PLAN_THREADS];
};

// Sums of two values a thread over the block.
KRK_DEV void block_sum2(long long& x, long long& y, PlanScratch& sc) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    if (lane == 0) {
        sc.warp[0][warp] = x;
        sc.warp[1][warp] = y;
    }
    __syncthreads();
    const bool in = lane < (int)(blockDim.x >> 5);
    x = in ? sc.warp[0][lane] : 0;
    y = in ? sc.warp[1][lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    __syncthreads();
}

// The sum of the threads before this one, and all threads' in total.  Two
// counts below 2^31 fit one value: no carry crosses the halves.
KRK_DEV long long block_scan(long long x, long long& total, PlanScratch& sc) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long upto = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) sc.warp[0][warp] = upto;
    __syncthreads();
    long long w = lane < (int)(blockDim.x >> 5) ? sc.warp[0][lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    __syncthreads();
    return upto - x + (warp ? before : 0);
}

// The last i < n with first[i] <= x (first[0] <= x).
KRK_DEV int bisect(const int* first, int n, int x) {
    int lo = 0;
    while (n > 1) {
        const int half = n >> 1;
        if (first[lo + half] <= x) {
            lo += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return lo;
}

KRK_DEV long long pages_for(long long tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

// Rows [r0, r1) of positions and slots get those that `at` gives, four at a time.
template <typename F>
KRK_DEV void write_rows(const PagePlanArgs& a, int r0, int r1, int thread, int threads, F at) {
    const bool wide = ((reinterpret_cast<uintptr_t>(a.positions) | reinterpret_cast<uintptr_t>(a.slots)) & 15) == 0;
    for (long long q = (r0 >> 2) + thread; q * 4 < r1; q += threads) {
        const int r = (int)(q * 4), lo = max(r, r0), hi = (int)min((long long)r + 4, (long long)r1);
        int pos[4], slot[4];
        at(lo, hi, r, pos, slot);
        if (wide && lo == r && hi == r + 4) {
            *reinterpret_cast<int4*>(a.positions + r) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            *reinterpret_cast<int4*>(a.slots + r) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r + i >= lo && r + i < hi) {
                    a.positions[r + i] = pos[i];
                    a.slots[r + i] = slot[i];
                }
        }
    }
}

template <int MODE>
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const __grid_constant__ PagePlanArgs a) {
    __shared__ PlanScratch sc;
    const int tid = threadIdx.x, nt = blockDim.x, shift = a.page_shift, low = (1 << shift) - 1;
    const int thread = blockIdx.x * nt + tid, threads = gridDim.x * nt;
    if (MODE == PLAN_FILL) pdl_trigger();
    if (tid == 0) sc.bad = 0;
    const int count = *a.free_count;
    // what the step needs, and whether it fits
    long long tokens = 0, pages = 0;
    int err = count < 0 || count > a.num_pages ? PAGES_BAD_LENGTH : 0;
    for (int b = tid; b < a.B; b += nt) {
        const long long len = a.lens[b], add = a.new_tokens[b];
        if (len < 0 || add < 0) {
            err |= PAGES_BAD_LENGTH;
            continue;
        }
        const long long want = pages_for(len + add, shift);
        if (want > a.width) err |= PAGES_ROW_FULL;
        tokens += add;
        pages += want - pages_for(len, shift);
    }
    block_sum2(tokens, pages, sc);
    if (tokens > a.rows) err |= PAGES_ROWS;
    if (pages > count) err |= PAGES_EXHAUSTED;
    if (err) atomicOr(&sc.bad, err);
    __syncthreads();
    err = sc.bad;
    if (MODE == PLAN_COMMIT) pdl_wait();  // the other kernel has read what is written here
    auto padding = [](int, int, int, int* pos, int* slot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pos[i] = 0;
            slot[i] = -1;
        }
    };
    int base_t = 0, base_p = 0;
    for (int b0 = 0; b0 < a.B; b0 += nt) {
        const int b = b0 + tid, n = min(nt, a.B - b0);
        const int len = tid < n ? a.lens[b] : 0, add = tid < n && !err ? a.new_tokens[b] : 0;
        const int have = (int)pages_for(len, shift), lack = (int)pages_for((long long)len + add, shift) - have;
        long long total;
        const long long before = block_scan((long long)lack << 32 | (unsigned)add, total, sc);
        sc.tokens[tid] = (int)before;
        sc.pages[tid] = (int)(before >> 32);
        sc.len[tid] = len;
        sc.have[tid] = have;
        const int tt = (int)total, tp = (int)(total >> 32);
        __syncthreads();
        if (MODE != PLAN_FILL && tid < n) {
            a.lens_out[b] = len + add;
            a.cu_new[b + 1] = base_t + (int)before + add;
        }
        if (MODE != PLAN_COMMIT) {
            for (int j = thread; j < tp; j += threads) {
                const int i = bisect(sc.pages, n, j);
                a.table[(b0 + i) * a.table_ld + sc.have[i] + j - sc.pages[i]] = a.free_pages[count - 1 - base_p - j];
            }
            write_rows(a, base_t, base_t + tt, thread, threads, [&](int lo, int hi, int r, int* pos, int* slot) {
                int i = bisect(sc.tokens, n, lo - base_t);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = r + k - base_t;
                    if (r + k < lo || r + k >= hi) continue;
                    while (i + 1 < n && sc.tokens[i + 1] <= at) ++i;
                    pos[k] = sc.len[i] + at - sc.tokens[i];
                    const int p = pos[k] >> shift;
                    const int page = p < sc.have[i]
                                         ? a.table[(b0 + i) * a.table_ld + p]
                                         : a.free_pages[count - 1 - base_p - (sc.pages[i] + p - sc.have[i])];
                    const bool in = (unsigned)page < (unsigned)a.num_pages;  // (another's slots may wrap into the pool)
                    if (!in) check_fail(CHK_TABLE);
                    slot[k] = in ? (page << shift) + (pos[k] & low) : -1;
                }
            });
        }
        base_t += tt;
        base_p += tp;
        __syncthreads();
    }
    if (MODE != PLAN_COMMIT) write_rows(a, base_t, a.rows, thread, threads, padding);
    if (MODE != PLAN_FILL && tid == 0) {
        *a.status = err;
        a.cu_new[0] = 0;
        *a.free_count_out = count - base_p;
    }
}

// Puts entries 0 .. n - 1, which `id` gives, on the stack in their order, without the negative ones; returns how many.
// `id` may read them from the stack itself, where they lie in the same order from the first one on.
template <typename F>
KRK_DEV int push_pages(int32_t* stack, int n, PlanScratch& sc, F id) {
    const int tid = threadIdx.x, nt = blockDim.x;
    int kept = 0;
    for (int j0 = 0; j0 < n; j0 += nt) {
        const bool mine = tid < n - j0;
        const int page = mine ? id(j0 + tid) : -1;
        if (__syncthreads_and(page >= 0 || !mine)) {
            if (mine) stack[kept + tid] = page;
            kept += min(nt, n - j0);
        } else {
            long long total;
            const int before = (int)block_scan(page >= 0, total, sc);
            if (page >= 0) stack[kept + before] = page;
            kept += (int)total;
        }
    }
    return kept;
}

// Negative entries of a row are pages that the caller has given back already.  The rule is that there are none: the
// entries are written as they are, and one block closes the gaps behind them if there are any.  The kernel that fills
// leaves word of gaps in the status, which the commit writes in any case (were the word there by chance, nothing would
// be found to close).  Only when the entries would not fit with the negative ones does one block count them first.
constexpr int PAGES_GAPS = INT32_MIN;

template <int MODE>
__global__ void __launch_bounds__(PLAN_THREADS) page_release_kernel(const __grid_constant__ PageReleaseArgs a) {
    __shared__ PlanScratch sc;
    const int tid = threadIdx.x, nt = blockDim.x, shift = a.page_shift;
    const int thread = blockIdx.x * nt + tid, threads = gridDim.x * nt;
    if (MODE == PLAN_FILL) pdl_trigger();
    if (tid == 0) sc.bad = 0;
    const int count = *a.free_count;
    long long pages = 0, unused = 0;
    int err = count < 0 || count > a.num_pages ? PAGES_BAD_LENGTH : 0;
    for (int b = tid; b < a.B; b += nt) {
        if (!a.done[b]) continue;
        const long long len = a.lens[b], held = pages_for(len, shift);
        if (len < 0 || held > a.width)
            err |= PAGES_BAD_LENGTH;
        else
            pages += held;
    }
    block_sum2(pages, unused, sc);
    if (pages > INT32_MAX) err |= PAGES_OVERFLOW;
    const bool fits = count + pages <= a.num_pages;
    if (err) atomicOr(&sc.bad, err);
    __syncthreads();
    err = sc.bad;
    if (err && !fits) err |= PAGES_OVERFLOW;
    if (MODE == PLAN_FILL && (err || !fits)) return;
    if (MODE == PLAN_COMMIT) pdl_wait();  // the other kernel has read what is written here
    // The requests, a chunk of them at a time: use(b0, n, len, gone, total) with this thread's request and the entries of
    // all that are gone, of which entry(b0, n, j) is one.
    auto walk = [&](auto use) {
        for (int b0 = 0; b0 < a.B; b0 += nt) {
            const int b = b0 + tid, n = min(nt, a.B - b0);
            const int len = tid < n ? a.lens[b] : 0;
            const bool gone = !err && tid < n && a.done[b];
            long long total;
            const int before = (int)block_scan(gone ? pages_for(len, shift) : 0, total, sc);
            sc.pages[tid] = before;
            __syncthreads();
            use(b0, n, len, gone, (int)total);
            __syncthreads();
        }
    };
    auto entry = [&](int b0, int n, int j) {
        const int i = bisect(sc.pages, n, j);
        return a.table[(b0 + i) * a.table_ld + j - sc.pages[i]];
    };
    if (MODE != PLAN_FILL && !err && !fits) {
        long long real = 0;
        walk([&](int b0, int n, int, bool, int total) {
            for (int j = tid; j < total; j += nt) real += entry(b0, n, j) >= 0;
        });
        block_sum2(real, unused, sc);
        if (count + real > a.num_pages) err = PAGES_OVERFLOW;
    }
    int32_t* stack = a.free_pages + count;
    int kept = 0;
    bool gaps = false;
    walk([&](int b0, int n, int len, bool gone, int total) {
        if (MODE != PLAN_FILL && tid < n) a.lens_out[b0 + tid] = gone ? 0 : len;
        if (MODE != PLAN_FILL && !fits) {
            kept += push_pages(stack + kept, total, sc, [&](int j) { return entry(b0, n, j); });
            return;
        }
        if (MODE != PLAN_COMMIT)
            for (int j = thread; j < total; j += threads) {
                const int page = entry(b0, n, j);
                stack[kept + j] = page;
                gaps |= page < 0;
            }
        kept += total;
    });
    if (MODE == PLAN_FILL) {
        if (gaps) *a.status = PAGES_GAPS;
        return;
    }
    if (MODE == PLAN_ALL) gaps = __syncthreads_or(gaps);
    if (MODE == PLAN_COMMIT) gaps = fits && __ldcg(a.status) == PAGES_GAPS;
    if (gaps) kept = push_pages(stack, kept, sc, [&](int j) { return stack[j]; });
    __syncthreads();  // the word has been read
    if (tid == 0) {
        *a.status = err;
        *a.free_count_out = count + kept;
    }
}

// One block for `writes` entries, or fill and commit.
template <typename Args>
cudaError_t launch_plan(void (*all)(Args), void (*fill)(Args), void (*commit)(Args), const Args& a, long long writes,
                        cudaStream_t s) {
    int nt = PLAN_MIN_THREADS;
    while (nt < PLAN_THREADS && nt < a.B) nt *= 2;
    if (writes <= PLAN_ONE_BLOCK) {
        all<<<1, writes > nt ? PLAN_THREADS : nt, 0, s>>>(a);
        add_launches(1);
        return cudaGetLastError();
    }
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    // four entries a thread, in one wave at most
    const long long blocks = (writes + 4LL * nt - 1) / (4LL * nt), wave = (long long)sms * (2048 / nt);
    fill<<<(unsigned)(blocks < wave ? blocks : wave), nt, 0, s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    add_launches(1);
    PdlScope pdl(true);
    e = launch_pdl(commit, dim3(1), dim3(nt), 0, s, a);
    if (e == cudaSuccess) add_launches(1);
    return e;
}

// ---------------------------------------------------------------- RoPE + append
// Every input is read and every output written once, W elements (16 bytes) at
// a time: HBM bounds it.  A unit is W pairs (i, i + rot/2) of a query or key
// head, or 2 W neighbours that are not rotated; a thread keeps one unit and takes
// it in two heads at once.  Where half a head is an odd number of half units (76 =
// 2 x 38 of four), units are RAGGED: the second parts are taken in two pieces, and
// the last unit is half of one.  One wave of blocks takes equal runs of rows and
// loads the next row before it stores the present one.  The rows' cos and sin
// are computed eight rows at a time, once a pair for all heads: the turns,
// position times rate, are reduced to a fraction in 64 bits.
constexpr int APPEND_THREADS = 256, APPEND_HEADS = 2, APPEND_BATCH = 8, APPEND_SIDE = 8, APPEND_BLOCKS = 3;

template <int BYTES>
struct Raw;
template <>
struct Raw<16> { using type = uint4; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<2> { using type = uint16_t; };

template <typename T, int W>
union Vec {
    typename Raw<sizeof(T) * W>::type raw;
    typename Raw<W == 1 ? sizeof(T) : sizeof(T) * W / 2>::type part[2];
    T e[W];
    uint32_t w[sizeof(T) * W / 4 ? sizeof(T) * W / 4 : 1];
    KRK_DEV Vec() {}
};
template <typename T, int W>
KRK_DEV void load_vec(Vec<T, W>& v, const T* p) {
    v.raw = *reinterpret_cast<const typename Raw<sizeof(T) * W>::type*>(p);
}
// The same from half the alignment, the second part only if `whole`.
template <typename T, int W>
KRK_DEV void load_parts(Vec<T, W>& v, const T* p, bool whole) {
    using R = typename Raw<W == 1 ? sizeof(T) : sizeof(T) * W / 2>::type;
    v.part[0] = reinterpret_cast<const R*>(p)[0];
    if (whole) v.part[1] = reinterpret_cast<const R*>(p)[1];
}
template <typename T, int W>
KRK_DEV void store_vec(T* p, const Vec<T, W>& v) {
    *reinterpret_cast<typename Raw<sizeof(T) * W>::type*>(p) = v.raw;
}
KRK_DEV void to_f32x2(float& x, float& y, uint32_t u, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    x = f.x;
    y = f.y;
}
KRK_DEV void to_f32x2(float& x, float& y, uint32_t u, __nv_bfloat16) {
    x = __uint_as_float(u << 16);
    y = __uint_as_float(u & 0xffff0000u);
}
KRK_DEV uint32_t from_f32x2(float x, float y, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
KRK_DEV uint32_t from_f32x2(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T, int W>
KRK_DEV void widen(float (&x)[W], const Vec<T, W>& v) {
    if constexpr (sizeof(T) == 2 && W > 1) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) to_f32x2(x[2 * i], x[2 * i + 1], v.w[i], T());
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] = to_f32(v.e[i]);
    }
}
template <typename T, int W>
KRK_DEV void put(T* p, const float (&x)[W]) {
    Vec<T, W> v;
    if constexpr (sizeof(T) == 2 && W > 1) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) v.w[i] = from_f32x2(x[2 * i], x[2 * i + 1], T());
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v.e[i] = from_f32<T>(x[i]);
    }
    store_vec<T, W>(p, v);
}

template <typename T, int W>
KRK_DEV void put_parts(T* p, const float (&x)[W], bool whole) {
    if constexpr (W > 1) {
        float a[W / 2], b[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            a[i] = x[i];
            b[i] = x[W / 2 + i];
        }
        put<T, W / 2>(p, a);
        if (whole) put<T, W / 2>(p + W / 2, b);
    }
}

// How a block divides its rows: `side` rows at once, `lanes` threads of each
// unit taking a row's heads; `depth` times.
struct AppendShape {
    int side, lanes, depth;
};

template <typename T, typename C, int W, bool RAGGED>
__global__ void __launch_bounds__(APPEND_THREADS, APPEND_BLOCKS)
    rope_append_kernel(const __grid_constant__ RopeAppendArgs a, const AppendShape sh) {
    extern __shared__ __align__(16) float turned[];  // [row of the batch][cos, sin][rot / 2]
    const int half = a.rot / 2, units = RAGGED ? (half + W / 2) / W : a.dh / (2 * W);
    const int rot_units = RAGGED ? units : half / W, heads = a.Hq + 2 * a.Hkv;
    const int r = threadIdx.x / (sh.lanes * units), in_row = threadIdx.x - r * sh.lanes * units;
    const int lane = in_row / units, unit = in_row - lane * units;
    const long long t0 = (long long)blockIdx.x * sh.side * sh.depth;
    const long long t1 = min(t0 + sh.side * sh.depth, (long long)a.T);
    // where the unit's two parts lie in a rotated head and in a value head
    const bool turns = unit < rot_units, whole = !RAGGED || unit < units - 1;
    const int at = turns ? unit * W : a.rot + (unit - rot_units) * 2 * W, next = at + (turns ? half : W);
    Vec<T, W> lo[APPEND_HEADS], hi[APPEND_HEADS];
    int slot = -1;
    auto load = [&](long long t, int h0) {
#pragma unroll
        for (int i = 0; i < APPEND_HEADS; ++i) {
            const int h = h0 + i * sh.lanes;
            if (t >= t1 || h >= heads) continue;
            if (h < a.Hq + a.Hkv) {
                const T* p = h < a.Hq ? (const T*)a.q + t * a.q_st + h * a.q_sh
                                      : (const T*)a.k + t * a.k_st + (h - a.Hq) * a.k_sh;
                load_vec<T, W>(lo[i], p + at);
                if (RAGGED)
                    load_parts<T, W>(hi[i], p + next, whole);
                else
                    load_vec<T, W>(hi[i], p + next);
            } else {
                const T* p = (const T*)a.v + t * a.v_st + (h - a.Hq - a.Hkv) * a.v_sh + unit * 2 * W;
                load_vec<T, W>(lo[i], p);
                if (whole) load_vec<T, W>(hi[i], p + W);
            }
        }
    };
    load(t0 + r, lane);
    if (t0 + r < t1) slot = a.slots[t0 + r];
    for (int d = 0; d < sh.depth; ++d) {
        const int in_batch = d % APPEND_BATCH;
        if (in_batch == 0) {
            if (d > 0) __syncthreads();  // the batch before has been read
            const long long first = t0 + (long long)d * sh.side;
            const int rows = (int)min((long long)sh.side * APPEND_BATCH, t1 - first);
            for (int i = threadIdx.x; i < rows * half; i += blockDim.x) {
                const int row = i / half, j = i - row * half;
                const double x = (double)a.positions[first + row] * a.turns.f[j];
                float sn, cs;
                sincospif(2.0f * (float)(x - rint(x)), &sn, &cs);
                turned[row * a.rot + j] = cs;
                turned[row * a.rot + half + j] = sn;
            }
            __syncthreads();
        }
        const long long t = t0 + (long long)d * sh.side + r, tn = t + sh.side;
        int now = slot;
        if (t >= t1 || now >= a.num_slots) {
            if (t < t1) check_fail(CHK_TABLE);
            now = -1;
        }
        if (tn < t1 && d + 1 < sh.depth) slot = a.slots[tn];
        const float* cs = turned + (in_batch * sh.side + r) * a.rot + (turns ? unit * W : 0);
        const long long cell = (now >> a.page_shift) * a.c_sp + (now & ((1 << a.page_shift) - 1)) * a.c_st;
        for (int h0 = lane; h0 < heads;) {
            Vec<T, W> lo_now[APPEND_HEADS], hi_now[APPEND_HEADS];
#pragma unroll
            for (int i = 0; i < APPEND_HEADS; ++i) {
                lo_now[i] = lo[i];
                hi_now[i] = hi[i];
            }
            const int h1 = h0 + APPEND_HEADS * sh.lanes;
            if (h1 < heads)
                load(t, h1);
            else if (d + 1 < sh.depth)
                load(tn, lane);
            if (now >= 0) {
#pragma unroll
                for (int i = 0; i < APPEND_HEADS; ++i) {
                    const int h = h0 + i * sh.lanes;
                    if (h >= heads) continue;
                    float x[W], y[W];
                    widen<T, W>(x, lo_now[i]);
                    widen<T, W>(y, hi_now[i]);
                    if (h >= a.Hq + a.Hkv) {
                        C* p = (C*)a.vc + cell + (h - a.Hq - a.Hkv) * a.c_sh + unit * 2 * W;
                        put<C, W>(p, x);
                        if (whole) put<C, W>(p + W, y);
                        continue;
                    }
                    if (turns) {
#pragma unroll
                        for (int j = 0; j < W; ++j) {
                            if (j >= W / 2 && !whole) break;
                            const float x0 = x[j], y0 = y[j], c = cs[j], s = cs[half + j];
                            x[j] = fmaf(x0, c, -(y0 * s));
                            y[j] = fmaf(y0, c, x0 * s);
                        }
                    }
                    if (h < a.Hq) {
                        T* p = (T*)a.q_out + t * a.qo_st + h * a.qo_sh;
                        if (RAGGED && !whole)
                            put_parts<T, W>(p + at, x, false);
                        else
                            put<T, W>(p + at, x);
                        if (RAGGED)
                            put_parts<T, W>(p + next, y, whole);
                        else
                            put<T, W>(p + next, y);
                    } else {
                        C* p = (C*)a.kc + cell + (h - a.Hq) * a.c_sh;
                        if (RAGGED && !whole)
                            put_parts<C, W>(p + at, x, false);
                        else
                            put<C, W>(p + at, x);
                        if (RAGGED)
                            put_parts<C, W>(p + next, y, whole);
                        else
                            put<C, W>(p + next, y);
                    }
                }
            }
            h0 = h1;
        }
    }
}

template <typename T, typename C, int W, bool RAGGED = false>
cudaError_t launch_append_w(const RopeAppendArgs& a, cudaStream_t s) {
    const int units = RAGGED ? (a.rot / 2 + W / 2) / W : a.dh / (2 * W), heads = a.Hq + 2 * a.Hkv;
    AppendShape sh{1, (heads + APPEND_HEADS - 1) / APPEND_HEADS, 1};
    if (sh.lanes > APPEND_THREADS / units) sh.lanes = APPEND_THREADS / units;  // several rounds of heads
    sh.side = APPEND_THREADS / (sh.lanes * units);
    // (48 KB of cos and sin at most)
    while (sh.side > 1 && (size_t)sh.side * APPEND_BATCH * a.rot * sizeof(float) > 48 * 1024) --sh.side;
    if (sh.side > APPEND_SIDE) sh.side = APPEND_SIDE;
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    // One wave of blocks, each with its run of rows (16321 x 32/8 x 128 bf16: 69 us, 5.9 TB/s; 89 us with a block
    // a row, whose start is not hidden).
    const int threads = sh.side * sh.lanes * units;
    const long long wave = (long long)sms * (APPEND_BLOCKS * APPEND_THREADS / threads) * sh.side;
    sh.depth = (int)((a.T + wave - 1) / wave);
    const long long rows = (long long)sh.side * sh.depth, batch = sh.depth < APPEND_BATCH ? sh.depth : APPEND_BATCH;
    rope_append_kernel<T, C, W, RAGGED><<<(unsigned)((a.T + rows - 1) / rows), threads,
                                  (size_t)sh.side * batch * a.rot * sizeof(float), s>>>(a, sh);
    add_launches(1);
    return cudaGetLastError();
}

// The widest unit that divides the rotated half and what is left of a head.  An odd rotated half, as of heads of 76
// rotated by 38, goes one element at a time (16,384 x 8 x 76 f32: 80 us, 49 us rotated as a whole; bf16: 115 and 40 us;
// 1024 rows f32: 7.8 and 5.7 us).
template <typename T, typename C>
cudaError_t launch_append(const RopeAppendArgs& a, cudaStream_t s) {
    auto fits = [&](int w) { return a.rot / 2 % w == 0 && (a.dh - a.rot) % (2 * w) == 0 && a.dh % (2 * w) == 0; };
    if constexpr (sizeof(T) == 2) {
        auto wide = [](const void* p, int64_t x, int64_t y) {
            return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && x % 8 == 0 && y % 8 == 0;
        };
        if (fits(8) && wide(a.k, a.k_st, a.k_sh) && wide(a.v, a.v_st, a.v_sh) && wide(a.kc, a.c_sp, a.c_st) &&
            wide(a.vc, a.c_sh, 0) && (a.Hq == 0 || (wide(a.q, a.q_st, a.q_sh) && wide(a.q_out, a.qo_st, a.qo_sh))))
            return launch_append_w<T, C, 8>(a, s);
    }
    if (fits(4)) return launch_append_w<T, C, 4>(a, s);
    if (a.rot == a.dh && a.dh % 8 == 4) return launch_append_w<T, C, 4, true>(a, s);
    if (fits(2)) return launch_append_w<T, C, 2>(a, s);
    return launch_append_w<T, C, 1>(a, s);
}

}  // namespace

cudaError_t kv_page_plan(const PagePlanArgs& a, cudaStream_t s) {
    return launch_plan(page_plan_kernel<PLAN_ALL>, page_plan_kernel<PLAN_FILL>, page_plan_kernel<PLAN_COMMIT>, a,
                       a.rows, s);
}

cudaError_t kv_page_release(const PageReleaseArgs& a, cudaStream_t s) {
    return launch_plan(page_release_kernel<PLAN_ALL>, page_release_kernel<PLAN_FILL>,
                       page_release_kernel<PLAN_COMMIT>, a, (long long)a.B * a.width, s);
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
