// Decode attention over a paged key-value cache: the kernel's frame, shared by
// the float32 and the 16-bit engines (k_paged_attn_f32.cu, k_paged_attn_half.cu).
//
// One token a request reads every visible key and value once and computes 4 dh
// operations for each pair and query head, so for the up to some tens of heads
// that share a cache head the cache's bytes bound it.  The frame therefore
// divides bytes: the visible keys of every (request, cache head) are cut into
// units of 64, and the units of the whole batch -- whatever the requests'
// lengths -- are dealt to one resident wave of blocks in equal contiguous
// shares.  A block works off its share piece by piece (a piece lies within one
// request and one cache head, or up to four neighbours of it); its warps take
// tiles of keys in turn, each with a running maximum and sum, and are merged in
// shared memory at the piece's end.  A piece
// that covers all of its keys is written as the result; otherwise its sums go
// to the scratch, where attn_paged_join adds them up in the order of the
// blocks, so that results do not depend on timing.
#pragma once
#include <math.h>

#include "elem.cuh"
#include "kernels.h"
#include "paged.h"

namespace krk {

constexpr int PA_THREADS = 128, PA_WARPS = 4;
constexpr int PA_UNIT = 64;          // keys of one unit of work
constexpr int PA_WHOLE_UNITS = 4;    // up to this many units a block takes a whole (request, head)
constexpr int PA_MAX_BLOCKS = 592;   // blocks of a wave: four on each of 148 SMs
constexpr int PA_MAX_ROWS = 32;      // query heads of a piece, at most
constexpr int PA_SIDE_UNITS = 8;     // units a block from which on its warps take different cache heads
constexpr int PA_ALIGN = 16;         // a piece's first key is aligned down to the largest tile

// Scratch of a launch: two partial results a block -- slot 0 for a piece that
// does not start its keys, slot 1 for one that does -- and their owners.
struct PagedParts {
    float* acc;  // [blocks][2][rows][dh]
    float2* ml;  // [blocks][2][rows] running maximum (base 2) and sum
    int2* rec;   // [blocks] (request, heads) of slots 0 and 1, -1: none
};

// How a block's warps divide a piece: `side` neighbouring cache heads, `groups`
// sets of query heads of each, and the keys among the warps that are left.
struct PagedShape {
    int side, groups;
    int per_kv;   // pieces for the query heads of one cache head
    int rows;     // query heads of a piece
    int whole;    // blocks take whole (request, heads)
};

KRK_DEV int pa_len(const PagedAttnArgs& a, int b) {
    const int cap = (int)((long long)a.width << a.page_shift);
    const int n = a.lens[b];
    if (n < 0 || n > cap) check_fail(CHK_POSITION);
    return min(max(n, 0), cap);
}
KRK_DEV int pa_first(const PagedAttnArgs& a, int n) { return a.window > 0 && n > a.window ? n - a.window : 0; }
// Units of a request of n tokens; an empty one has a unit too, which writes its zeros.
KRK_DEV int pa_units(int n, int first) {
    const int keys = n - (first & ~(PA_ALIGN - 1));
    return max(1, (keys + PA_UNIT - 1) / PA_UNIT);
}

// The first unit of this block's share: its request and its place among the
// request's units over all heads; and the share's size.  All threads call it.
struct PagedShare {
    int b;
    long long at, size;
};
KRK_DEV PagedShare pa_share(const PagedAttnArgs& a, int pieces, PagedShare* out, long long* warp_sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (a.B + PA_THREADS - 1) / PA_THREADS;
    const int b0 = min(a.B, tid * each), b1 = min(a.B, b0 + each);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = pa_len(a, b);
        mine += (long long)pa_units(n, pa_first(a, n)) * pieces;
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < PA_WARPS; ++w) {
        if (w < warp) upto += warp_sums[w];
        total += warp_sums[w];
    }
    // no empty share lies between two that have work: the join counts on neighbours
    const long long shares = min(total, (long long)gridDim.x), mine_at = min((long long)blockIdx.x, shares);
    const long long s = total * mine_at / shares, e = total * min(mine_at + 1, shares) / shares;
    long long before = upto - mine;
    if (tid == 0 && s == e) *out = PagedShare{0, 0, 0};
    if (s < e && s >= before && s < upto) {
        int b = b0;
        for (;; ++b) {
            const int n = pa_len(a, b);
            const long long u = (long long)pa_units(n, pa_first(a, n)) * pieces;
            if (s < before + u) break;
            before += u;
        }
        *out = PagedShare{b, s - before, e - s};
    }
    __syncthreads();
    return *out;
}

// Where a tile's keys lie.  Tiles are aligned, so pages of 16 tokens or more
// hold a tile in one piece: off is its first key's offset and the others follow
// by c_st.  On smaller pages lane i holds the offset of key i (mod KT).
struct PagedTile {
    long long off;
    unsigned mask;  // the visible keys
};
template <int KT>
KRK_DEV int pa_page(const PagedAttnArgs& a, const int32_t* row, int key0, int k1) {
    const int key = a.page_shift >= 4 ? key0 : key0 + (threadIdx.x & (KT - 1));
    return key < k1 ? row[key >> a.page_shift] : -1;
}
template <int KT>
KRK_DEV PagedTile pa_tile(const PagedAttnArgs& a, int page, int key0, int first, int k1) {
    constexpr unsigned kAll = KT == 32 ? ~0u : (1u << KT) - 1;
    const int low = (1 << a.page_shift) - 1;
    const bool in = (unsigned)page < (unsigned)a.num_pages;
    PagedTile t;
    if (a.page_shift >= 4) {
        if (!in && key0 < k1) check_fail(CHK_TABLE);
        t.mask = in ? kAll : 0u;
        if (key0 < first) t.mask &= ~0u << min(first - key0, 31);
        if (key0 + KT > k1) t.mask &= key0 < k1 ? kAll >> (key0 + KT - k1) : 0u;
        t.off = page * a.c_sp + (key0 & low) * a.c_st;
    } else {
        const int key = key0 + (threadIdx.x & (KT - 1));
        if (!in && key >= first && key < k1) check_fail(CHK_TABLE);
        t.mask = __ballot_sync(0xffffffffu, in && key >= first && key < k1) & kAll;
        t.off = page * a.c_sp + (key & low) * a.c_st;
    }
    return t;
}
// The element offset of key `key` of the tile (a fixed key for each lane).
KRK_DEV long long pa_key(const PagedAttnArgs& a, const PagedTile& t, int key) {
    return a.page_shift >= 4 ? t.off + key * a.c_st : __shfl_sync(0xffffffffu, t.off, key);
}

// Barrier of the warps that share a group's queries.
KRK_DEV void pa_group_sync(int group, int warps) {
    if (warps > 1)
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
    else
        __syncwarp();
}

// Asynchronous copy of BYTES (16 or 8) to shared memory; zeros, and no access, when !take.
template <int BYTES>
KRK_DEV void pa_copy(uint32_t to, const void* from, bool take) {
    const int n = take ? BYTES : 0;
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
}

// E: an engine.  Its warp holds KT keys of a tile and HW query heads:
//   init(a, q, heads, qs)       loads a warp's queries (or prepares them in shared memory)
//   issue(base, tile, to)       starts the copies of a tile's keys or values to a ring slot
//   scores(qs, from)            q . k of the slot's keys
//   weigh(mask)                 softmax step over the visible keys of the tile
//   values(from)                weighted values into the accumulators
//   finish(obuf, m, l)          accumulators, maxima and sums of the warp to shared memory
// A warp's ring has SLOTS slots for keys and as many for values; a slot is
// filled again as soon as the warp has read it, with no barrier beyond the warp.
template <class E>
__global__ void __launch_bounds__(PA_THREADS, E::BLOCKS) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a,
                                                                           const PagedShape sh,
                                                                           const PagedParts parts) {
    using T = typename E::Act;
    using C = typename E::Cache;
    constexpr int KT = E::KT, HW = E::HW, LD = E::DC + 4, S = E::SLOTS, HALF = E::TILE_BYTES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sm[PA_WARPS][HW], sl[PA_WARPS][HW], sf[PA_WARPS][HW];
    __shared__ long long warp_sums[PA_WARPS];
    __shared__ PagedShare share_out;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.Hq / a.Hkv, pieces = a.Hkv / sh.side * sh.per_kv;
    // warp -> (keys, cache head, query heads)
    const int sets = sh.side * sh.groups, kwarps = PA_WARPS / sets, kwarp = warp / sets, set = warp % sets;
    unsigned char* ring = smem + (size_t)warp * 2 * S * HALF;
    unsigned char* qs = smem + (size_t)PA_WARPS * 2 * S * HALF + (size_t)set * E::Q_BYTES;
    const uint32_t ring_at = smem_addr(ring);

    PagedShare share;
    if (sh.whole) {
        share.b = blockIdx.x / pieces;
    } else {
        pdl_trigger();
        share = pa_share(a, pieces, &share_out, warp_sums);
    }
    int b = share.b, n = pa_len(a, b), first = pa_first(a, n), units = pa_units(n, first);
    if (sh.whole) {
        share.at = (long long)(blockIdx.x % pieces) * units;
        share.size = units;
    }
    int piece = (int)(share.at / units), unit = (int)(share.at % units);
    long long left = share.size;
    int2 rec = make_int2(-1, -1);

    while (left > 0) {
        const int take = (int)min((long long)(units - unit), left);
        const int hk0 = piece / sh.per_kv * sh.side, head0 = piece % sh.per_kv * sh.rows;  // head0: within G
        const int hk = hk0 + set / sh.groups, head = head0 + set % sh.groups * HW;
        const int base = first & ~(PA_ALIGN - 1);
        const int k0 = base + unit * PA_UNIT, k1 = min(n, base + (unit + take) * PA_UNIT);
        const int32_t* row = a.table + b * a.table_ld;
        const C* kc = (const C*)a.kc + hk * a.c_sh;
        const C* vc = (const C*)a.vc + hk * a.c_sh;

        E e;
        int key = k0 + kwarp * KT;
        const int step = kwarps * KT;
        // the first tiles' pages, then the queries while they are on their way
        int pages[S + 1];
#pragma unroll
        for (int i = 0; i <= S; ++i) pages[i] = pa_page<KT>(a, row, key + i * step, k1);
        e.init(a, (const T*)a.q + b * a.q_sb + ((long long)hk * G + head) * a.q_sh, min(HW, G - head), qs, lane, kwarp,
               kwarps);
        if (E::Q_BYTES) pa_group_sync(set, kwarps);
        if (key < k1) {
            unsigned mask[S + 1];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const PagedTile t = pa_tile<KT>(a, pages[i], key + i * step, first, k1);
                mask[i] = t.mask;
                if (key + i * step < k1) e.issue(a, kc, t, ring_at + i * HALF, lane);
                cp_async_commit();
                if (key + i * step < k1) e.issue(a, vc, t, ring_at + (S + i) * HALF, lane);
                cp_async_commit();
            }
            int page = pages[S];
            for (int slot = 0;; slot = slot + 1 == S ? 0 : slot + 1) {
                const int ahead = key + S * step;
                cp_async_wait<2 * S - 1>();
                __syncwarp();
                e.scores(qs, ring + slot * HALF, lane);
                __syncwarp();
                const PagedTile t = pa_tile<KT>(a, page, ahead, first, k1);
                mask[S] = t.mask;
                if (ahead < k1) e.issue(a, kc, t, ring_at + slot * HALF, lane);
                cp_async_commit();
                page = pa_page<KT>(a, row, ahead + step, k1);
                e.weigh(mask[0], lane);
                cp_async_wait<2 * S - 1>();
                __syncwarp();
                e.values(ring + (S + slot) * HALF, lane);
                key += step;
                if (key >= k1) break;
                __syncwarp();
                if (ahead < k1) e.issue(a, vc, t, ring_at + (S + slot) * HALF, lane);
                cp_async_commit();
#pragma unroll
                for (int i = 0; i < S; ++i) mask[i] = mask[i + 1];
            }
        }
        __syncwarp();  // the warp's sums go where its tiles were
        e.finish(reinterpret_cast<float*>(ring), sm[warp], sl[warp], lane);
        __syncthreads();
        // each query head's factors for its warps' sums
        const int rows = sh.side * sh.rows;
        if (tid < sets * HW) {
            const int w0 = tid / HW, h = tid % HW, in_g = w0 % sh.groups * HW + h;
            float top = -INFINITY, total = 0.f;
            for (int w = w0; w < PA_WARPS; w += sets) top = fmaxf(top, sm[w][h]);
            for (int w = w0; w < PA_WARPS; w += sets) {
                const float f = top == -INFINITY ? (sl[w][h] == 0.f ? 0.f : sl[w][h]) : exp2f(sm[w][h] - top);
                sf[w][h] = f;
                total = fmaf(f, sl[w][h], total);
            }
            if (in_g < sh.rows && head0 + in_g < G) {
                if (take == units) {
                    const float inv = total == 0.f ? 0.f : 1.0f / total;
                    for (int w = w0; w < PA_WARPS; w += sets) sf[w][h] *= inv;
                    if (a.lse)
                        a.lse[(long long)b * a.Hq + (long long)(hk0 + w0 / sh.groups) * G + head0 + in_g] =
                            (top + log2f(total * (1.0f / E::SCALE))) * 0.693147180559945309f;
                } else {
                    parts.ml[((long long)blockIdx.x * 2 + (unit == 0)) * rows + w0 / sh.groups * sh.rows + in_g] =
                        make_float2(top, total);
                }
            }
        }
        __syncthreads();
        const int n4 = a.dh / 4;
        for (int i = tid; i < rows * n4; i += PA_THREADS) {
            const int r = i / n4, d = (i - r * n4) * 4, s = r / sh.rows, in_g = r - s * sh.rows;
            if (head0 + in_g >= G) continue;
            const int w0 = s * sh.groups + in_g / HW, h = in_g % HW;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = w0; w < PA_WARPS; w += sets) {
                const float f = sf[w][h];
                const float4 x = *reinterpret_cast<const float4*>(smem + (size_t)w * 2 * S * HALF + (h * LD + d) * 4);
                o.x = fmaf(f, x.x, o.x);
                o.y = fmaf(f, x.y, o.y);
                o.z = fmaf(f, x.z, o.z);
                o.w = fmaf(f, x.w, o.w);
            }
            if (take == units)
                store4((T*)a.out + b * a.o_sb + ((long long)(hk0 + s) * G + head0 + in_g) * a.o_sh + d, o);
            else
                *reinterpret_cast<float4*>(
                    parts.acc + (((long long)blockIdx.x * 2 + (unit == 0)) * rows + r) * a.dh + d) = o;
        }
        if (take != units) (unit == 0 ? rec.y : rec.x) = b * pieces + piece;
        left -= take;
        if (left <= 0) break;
        unit = 0;
        if (++piece == pieces) {
            piece = 0;
            ++b;
            n = pa_len(a, b);
            first = pa_first(a, n);
            units = pa_units(n, first);
        }
        __syncthreads();  // the next piece's tiles go where this one's sums were
    }
    if (!sh.whole && tid == 0) parts.rec[blockIdx.x] = rec;
}

// Joins the partial results: block (c, r) looks whether block c of the
// attention began a piece's keys without finishing them, and if so adds up query
// head r of the piece over the blocks c, c + 1, ... that worked on it.
template <typename T>
__global__ void __launch_bounds__(PA_THREADS) paged_join_kernel(const PagedAttnArgs a, const PagedShape sh,
                                                               const PagedParts parts, int blocks, float scale) {
    __shared__ float weight[PA_MAX_BLOCKS + 1];
    __shared__ float red[2][PA_WARPS];
    __shared__ float4 sums[PA_THREADS];
    const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    pdl_wait();
    const int item = parts.rec[c].y;
    if (item < 0) return;
    const int G = a.Hq / a.Hkv, pieces = a.Hkv / sh.side * sh.per_kv, rows = sh.side * sh.rows;
    const int b = item / pieces, piece = item % pieces, in_g = piece % sh.per_kv * sh.rows + r % sh.rows;
    if (in_g >= G) return;
    const long long head = (long long)(piece / sh.per_kv * sh.side + r / sh.rows) * G + in_g;
    int count = 1;  // the blocks of an item are neighbours
    for (int i = c + 1; i < blocks; i += PA_THREADS)
        count += __syncthreads_count(i + tid < blocks && parts.rec[min(i + tid, blocks - 1)].x == item);
    // weights 2^(m - top) and the sum
    float top = -INFINITY, total = 0.f;
    auto ml = [&](int i) { return parts.ml[((long long)(c + i) * 2 + (i == 0)) * rows + r]; };
    for (int i = tid; i < count; i += PA_THREADS) top = fmaxf(top, ml(i).x);
    top = warp_max(top);
    if ((tid & 31) == 0) red[0][tid >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    for (int i = tid; i < count; i += PA_THREADS) {
        const float2 x = ml(i);
        const float f = top == -INFINITY ? (x.y == 0.f ? 0.f : x.y) : exp2f(x.x - top);
        weight[i] = f;
        total = fmaf(f, x.y, total);
    }
    total = warp_sum(total);
    if ((tid & 31) == 0) red[1][tid >> 5] = total;
    __syncthreads();
    total = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    // dh/4 threads a partial result, as many side by side as fit
    const int n4 = a.dh / 4, side = PA_THREADS / n4, d = (tid % n4) * 4, s0 = tid / n4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s0 < side) {
#pragma unroll 8
        for (int i = s0; i < count; i += side) {
            const float4 x = *reinterpret_cast<const float4*>(
                parts.acc + (((long long)(c + i) * 2 + (i == 0)) * rows + r) * a.dh + d);
            const float f = weight[i];
            o.x = fmaf(f, x.x, o.x);
            o.y = fmaf(f, x.y, o.y);
            o.z = fmaf(f, x.z, o.z);
            o.w = fmaf(f, x.w, o.w);
        }
    }
    sums[tid] = o;
    __syncthreads();
    if (s0 == 0) {
        for (int s = 1; s < side; ++s) {
            const float4 x = sums[s * n4 + tid];
            o.x += x.x;
            o.y += x.y;
            o.z += x.z;
            o.w += x.w;
        }
        o.x *= inv;
        o.y *= inv;
        o.z *= inv;
        o.w *= inv;
        store4((T*)a.out + b * a.o_sb + head * a.o_sh + d, o);
    }
    if (tid == 0 && a.lse)
        a.lse[(long long)b * a.Hq + head] = (top + log2f(total * (1.0f / scale))) * 0.693147180559945309f;
}

// Whether blocks take whole (request, heads): lengths up to `bound` are not worth a second kernel.
inline bool pa_whole(int bound) { return bound <= PA_WHOLE_UNITS * PA_UNIT; }

template <class E>
cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t s) {
    static DeviceOnce once;
    constexpr size_t kRing = (size_t)PA_WARPS * 2 * E::SLOTS * E::TILE_BYTES;
    static_assert(E::HW * (E::DC + 4) * 4 <= 2 * E::SLOTS * E::TILE_BYTES, "a warp's sums fit in its ring");
    const int G = a.Hq / a.Hkv, sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    cudaError_t e = once.set_smem((const void*)paged_attn_kernel<E>, kRing + PA_WARPS * E::Q_BYTES);
    if (e != cudaSuccess) return e;
    const int slots = sms * E::BLOCKS < PA_MAX_BLOCKS ? sms * E::BLOCKS : PA_MAX_BLOCKS;
    const int bound = a.window > 0 && a.window < a.max_len ? a.window + PA_ALIGN : a.max_len;
    const long long units = (bound + PA_UNIT - 1) / PA_UNIT;
    PagedShape sh{1, 1, 1, 0, 0};
    while (sh.groups < PA_WARPS && sh.groups * E::HW < G) sh.groups *= 2;
    sh.per_kv = (G + sh.groups * E::HW - 1) / (sh.groups * E::HW);
    sh.rows = G < sh.groups * E::HW ? G : sh.groups * E::HW;
    // With work for every block, warps take neighbouring cache heads of the same keys.
    while (sh.side * sh.groups < PA_WARPS && a.Hkv % (2 * sh.side) == 0 &&
           (long long)a.B * (a.Hkv / sh.side / 2) * sh.per_kv * units >= PA_SIDE_UNITS * (long long)slots)
        sh.side *= 2;
    const size_t smem = kRing + (size_t)sh.side * sh.groups * E::Q_BYTES;
    const long long items = (long long)a.B * (a.Hkv / sh.side) * sh.per_kv;
    if (pa_whole(a.max_len)) {
        sh.whole = 1;
        paged_attn_kernel<E><<<(unsigned)items, PA_THREADS, smem, s>>>(a, sh, PagedParts{});
        add_launches(1);
        return cudaGetLastError();
    }
    const int blocks = items * units < slots ? (int)(items * units) : slots, rows = sh.side * sh.rows;
    PagedParts parts;
    parts.acc = a.work;
    parts.ml = reinterpret_cast<float2*>(a.work + (size_t)PA_MAX_BLOCKS * 2 * rows * a.dh);
    parts.rec = reinterpret_cast<int2*>(parts.ml + (size_t)PA_MAX_BLOCKS * 2 * rows);
    paged_attn_kernel<E><<<blocks, PA_THREADS, smem, s>>>(a, sh, parts);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    add_launches(1);
    PdlScope pdl(true);
    e = launch_pdl(paged_join_kernel<typename E::Act>, dim3(blocks, rows), dim3(PA_THREADS), 0, s, a, sh, parts, blocks,
                   E::SCALE);
    if (e == cudaSuccess) add_launches(1);
    return e;
}

}  // namespace krk
