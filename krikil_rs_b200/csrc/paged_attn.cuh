// Decode attention over a paged key-value cache: the kernel's frame, shared by
// the float32 and the 16-bit engines (k_paged_attn_f32.cu, paged_attn_half.cuh).
//
// One token a request reads every visible key and value once and computes 4 dh
// operations for each pair and query head, so for the up to some tens of heads
// that share a cache head the cache's bytes bound it.  The frame therefore
// divides bytes, in one of two ways:
//
// Shares, for much work.  The visible keys of every (request, cache head) are
// cut into units of 64, and the units of the whole batch -- whatever the
// requests' lengths -- are dealt to one resident wave of blocks in equal
// contiguous shares.  A block works off its share piece by piece (a piece lies
// within one request and one cache head, or up to four neighbours of it).  A
// piece that covers all of its keys is written as the result; otherwise its sums
// go to the scratch, where paged_join_kernel adds them up in the order of the
// blocks.
//
// Clusters, where latency counts: 1, 2, 4 or 8 blocks of a thread-block cluster
// take equal parts of one piece and add up their sums through each other's shared
// memory.  One kernel, no scratch and no look at the other requests.  What bounds
// it is a chain of latencies: launch, length, page, first keys, about 1 us a tile
// of each warp, the merge (8 x 76 f32: 4.4 us of 32 keys, 7.6 us of 1000).
//
// Either way a block's warps take tiles of keys in turn, each with a running
// maximum and sum, and are merged in shared memory at the end; all orders are
// fixed, so that results do not depend on timing.
#pragma once
#include <math.h>

#include "elem.cuh"
#include "kernels.h"
#include "paged.h"

namespace krk {

constexpr int PA_THREADS = 128, PA_WARPS = 4;
constexpr int PA_UNIT = 64;          // keys of one unit of work
constexpr int PA_CLUSTER = 8;        // blocks of a cluster, at most
constexpr int PA_PART_UNITS = 2;     // units of a block down to which clusters grow
constexpr int PA_FULL_UNITS = 24;    // units of a block up to which clusters are used when they fill the device,
constexpr int PA_FEW_UNITS = 8;      // and when they do not
constexpr int PA_JOIN = 512;         // threads of a join's block, at most
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
    int rows;     // query heads of a piece of one cache head
    int extra;    // units that a piece counts for beyond its own when work is shared out
    int cluster;  // blocks that share a piece, 0: shares of the whole batch
};

// 2^x to about a unit in the last place, 0 below 2^-126.
KRK_DEV float pa_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// total * i / n, in 32 bits where they do.
KRK_DEV long long pa_part(long long total, long long i, long long n) {
    if (total < (1 << 21)) return (unsigned)total * (unsigned)i / (unsigned)n;  // i, n <= PA_MAX_BLOCKS
    return total * i / n;
}

// Beginning and ending a piece costs a block about as much as a few units of one
// cache head, so each piece counts for that much more: `extra` places come before
// its units'.  This is the first place of a block's share -- its request and its
// place in the request's pieces -- and the share's size.  All threads call it.
struct PagedShare {
    int b;
    long long at, size;
};
KRK_DEV PagedShare pa_share(const PagedAttnArgs& a, int pieces, int extra, PagedShare* out,
                            long long* warp_sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (a.B + PA_THREADS - 1) / PA_THREADS;
    const int b0 = min(a.B, tid * each), b1 = min(a.B, b0 + each);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = pa_len(a, b);
        mine += (long long)(pa_units(n, pa_first(a, n)) + extra) * pieces;
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
    const long long s = pa_part(total, mine_at, shares), e = pa_part(total, min(mine_at + 1, shares), shares);
    long long before = upto - mine;
    if (tid == 0 && s == e) *out = PagedShare{0, 0, 0};
    if (s < e && s >= before && s < upto) {
        int b = b0;
        for (;; ++b) {
            const int n = pa_len(a, b);
            const long long u = (long long)(pa_units(n, pa_first(a, n)) + extra) * pieces;
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
// (Entries past the request's last page are read, and not used.)
template <int KT>
KRK_DEV int pa_page(const PagedAttnArgs& a, const int32_t* row, int key0) {
    const int key = a.page_shift >= 4 ? key0 : key0 + (threadIdx.x & (KT - 1));
    return row[min(key >> a.page_shift, a.width - 1)];
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

KRK_DEV void pa_cluster_sync() {
    asm volatile("barrier.cluster.arrive;\nbarrier.cluster.wait;" ::: "memory");
}
// Shared memory of block `rank` of the cluster at this block's address `at`.
KRK_DEV uint32_t pa_peer(uint32_t at, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
KRK_DEV float4 pa_peer_load4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
}
KRK_DEV float2 pa_peer_load2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

// Barrier of the warps that share a group's queries.
KRK_DEV void pa_group_sync(int group, int warps) {
    if (warps > 1)
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
    else
        __syncwarp();
}

// Asynchronous copy of BYTES (16 or 8) to shared memory; zeros, and no access, when !take.  L1: rows that begin or end
// inside a sector find the half that a neighbouring head's warp has fetched in L1 (f32 64 x 8 x 76 of 4096 keys: 217 us,
// 237 us past L1).  It costs where rows are whole sectors (f32 heads of 80: 232 and 225 us), where several query heads
// slow a tile down (f32 8/2 heads of 76: 96 and 90 us) and for the shorter 16-bit rows (f32 queries on bf16 heads of 76:
// 232 and 161 us).
template <int BYTES, bool L1 = false>
KRK_DEV void pa_copy(uint32_t to, const void* from, bool take) {
    const int n = take ? BYTES : 0;
    if (BYTES == 16 && !L1)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;\n" ::"r"(to), "l"(from), "r"(n), "n"(BYTES)
                     : "memory");
}

// E: an engine.  Its warp holds KT keys of a tile and HW query heads:
//   init(a, q, k, v, heads, qs) loads a warp's queries (or prepares them in shared memory)
//   issue(base, tile, to)       starts the copies of a tile's keys or values to a ring slot
//   scores(qs, from)            q . k of the slot's keys
//   weigh(mask)                 softmax step over the visible keys of the tile
//   values<again>(from)         weighted values into the accumulators
//   spoilt()                    whether sums are NaN that may not be, and the tiles are to be taken again
//   finish(obuf, m, l)          accumulators, maxima and sums of the warp to shared memory
// A warp's ring has SLOTS slots for keys and as many for values; a slot is
// filled again as soon as the warp has read it, with no barrier beyond the warp.
// (The same tiles held in registers, loads issued as early: f32 1024 x 8 x 76 in
// 604 us, 271 us from a ring; bf16 128 x 32/8 x 128 in 435 us, 331 us.)

// One part of a head's sums, with maximum m and sum l, onto others; top: the largest maximum of all.
KRK_DEV void pa_add(float4& o, float& total, const float4& x, float m, float l, float top) {
    // (no visible key at all: weight 0, or NaN if the sum is)
    const float f = top == -INFINITY ? (l == 0.f ? 0.f : l) : pa_exp2(m - top);
    total = fmaf(f, l, total);
    o.x = fmaf(f, x.x, o.x);
    o.y = fmaf(f, x.y, o.y);
    o.z = fmaf(f, x.z, o.z);
    o.w = fmaf(f, x.w, o.w);
}
// Elements d .. d + 3 of a query head's result from its sums, and with the first of them its logarithm.
template <class E>
KRK_DEV void pa_result(const PagedAttnArgs& a, int b, long long head, int d, float4 o, float top, float total) {
    float inv;  // within a unit in the last place
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(total));
    if (total == 0.f) inv = 0.f;
    store4((typename E::Act*)a.out + b * a.o_sb + head * a.o_sh + d,
           make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (a.lse && d == 0)
        a.lse[(long long)b * a.Hq + head] = (top + log2f(total * (1.0f / E::SCALE))) * 0.693147180559945309f;
}

// Adds up the sums of a cluster's blocks, each block a part of the elements.
template <class E>
KRK_DEV void pa_join_cluster(const PagedAttnArgs& a, const PagedShape& sh, const unsigned char* smem,
                             const float2* sums, int b, int hk0, int head0, int rank) {
    constexpr int LD = E::DC + 4, HW = E::HW;
    const int G = a.Hq / a.Hkv, n4 = a.dh / 4, rows = sh.side * sh.rows;
    const uint32_t sums_at = smem_addr(sums), acc_at = smem_addr(smem);
    for (int i = rank * PA_THREADS + threadIdx.x; i < rows * n4; i += sh.cluster * PA_THREADS) {
        const int r = i / n4, d = (i - r * n4) * 4, s = r / sh.rows, in_g = r - s * sh.rows;
        if (head0 + in_g >= G) continue;
        const int w0 = s * sh.groups + in_g / HW, h = in_g % HW;
        const uint32_t ml_at = sums_at + (w0 * HW + h) * 8;
        const uint32_t at = acc_at + w0 * 2 * E::SLOTS * E::TILE_BYTES + (h * LD + d) * 4;
        float2 ml[PA_CLUSTER];
        float4 x[PA_CLUSTER];
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int c = 0; c < PA_CLUSTER; ++c) {
            ml[c] = make_float2(-INFINITY, 0.f);
            x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < sh.cluster) {
                ml[c] = pa_peer_load2(pa_peer(ml_at, c));
                x[c] = pa_peer_load4(pa_peer(at, c));
            }
        }
#pragma unroll
        for (int c = 0; c < PA_CLUSTER; ++c) top = fmaxf(top, ml[c].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < PA_CLUSTER; ++c) pa_add(o, total, x[c], ml[c].x, ml[c].y, top);
        pa_result<E>(a, b, (long long)(hk0 + s) * G + head0 + in_g, d, o, top, total);
    }
}

// A warp's tiles of a piece: the keys from `key` on, `step` apart, up to k1.  pages: of the first tiles; prepare: run
// while those are on their way.
template <class E, bool AGAIN, class F>
KRK_DEV void pa_tiles(E& e, const PagedAttnArgs& a, const int32_t* row, const typename E::Cache* kc,
                      const typename E::Cache* vc, unsigned char* ring, const unsigned char* qs,
                      const int (&pages)[E::SLOTS + 1], int key, int step, int first, int k1, int lane, F prepare) {
    constexpr int KT = E::KT, S = E::SLOTS, SLOT = E::TILE_BYTES;
    const uint32_t ring_at = smem_addr(ring);
    unsigned mask[S + 1];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        if (key + i * step < k1) {
            const PagedTile t = pa_tile<KT>(a, pages[i], key + i * step, first, k1);
            mask[i] = t.mask;
            e.issue(a, kc, t, ring_at + i * SLOT, lane);
            cp_async_commit();
            e.issue(a, vc, t, ring_at + (S + i) * SLOT, lane);
            cp_async_commit();
        } else {
            mask[i] = 0u;
            cp_async_commit();
            cp_async_commit();
        }
    }
    prepare();
    if (key >= k1) return;
    int page = pages[S];
    for (int slot = 0;; slot = slot + 1 == S ? 0 : slot + 1) {
        const int ahead = key + S * step;
        cp_async_wait<2 * S - 1>();
        __syncwarp();
        e.scores(qs, ring + slot * SLOT, lane);
        __syncwarp();
        const PagedTile t = pa_tile<KT>(a, page, ahead, first, k1);
        mask[S] = t.mask;
        if (ahead < k1) e.issue(a, kc, t, ring_at + slot * SLOT, lane);
        cp_async_commit();
        page = pa_page<KT>(a, row, ahead + step);
        e.weigh(mask[0], lane);
        cp_async_wait<2 * S - 1>();
        __syncwarp();
        e.template values<AGAIN>(ring + (S + slot) * SLOT, lane);
        key += step;
        if (key >= k1) break;
        __syncwarp();
        if (ahead < k1) e.issue(a, vc, t, ring_at + (S + slot) * SLOT, lane);
        cp_async_commit();
#pragma unroll
        for (int i = 0; i < S; ++i) mask[i] = mask[i + 1];
    }
}

// The same once more for a warp whose sums are NaN and may not be, up to its sums in shared memory.  A call by itself,
// since its registers would cost the loop that is always taken (16 query heads a cache head, bf16 64 x 128/8 x 128:
// 239 us; 264 us with the parts apart in every tile, 248 us with infinite values left to come out as NaN).
template <class E>
__device__ __noinline__ void pa_again(float c, const PagedAttnArgs& a, const int32_t* row, const typename E::Cache* kc,
                                      const typename E::Cache* vc, unsigned char* ring, const unsigned char* qs, int key,
                                      int step, int first, int k1, float* sm, float* sl) {
    const int lane = threadIdx.x & 31;
    E e;
    e.resume(a, kc, vc, c);
    int pages[E::SLOTS + 1];
#pragma unroll
    for (int i = 0; i <= E::SLOTS; ++i) pages[i] = pa_page<E::KT>(a, row, key + i * step);
    pa_tiles<E, true>(e, a, row, kc, vc, ring, qs, pages, key, step, first, k1, lane, [] {});
    __syncwarp();
    e.finish(reinterpret_cast<float*>(ring), sm, sl, lane);
}

template <class E>
__global__ void __launch_bounds__(PA_THREADS, E::BLOCKS) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a,
                                                                           const PagedShape sh,
                                                                           const PagedParts parts) {
    using T = typename E::Act;
    using C = typename E::Cache;
    constexpr int KT = E::KT, HW = E::HW, LD = E::DC + 4, S = E::SLOTS, SLOT = E::TILE_BYTES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sm[PA_WARPS][HW], sl[PA_WARPS][HW];
    __shared__ __align__(8) float2 sums[PA_MAX_ROWS];
    __shared__ long long warp_sums[PA_WARPS];
    __shared__ PagedShare share_out;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.Hq / a.Hkv, pieces = a.Hkv / sh.side * sh.per_kv;
    // warp -> (keys, cache head, query heads)
    const int sets = sh.side * sh.groups, kwarps = PA_WARPS / sets, kwarp = warp / sets, set = warp % sets;
    unsigned char* ring = smem + (size_t)warp * 2 * S * SLOT;
    unsigned char* qs = smem + (size_t)PA_WARPS * 2 * S * SLOT + (size_t)set * E::Q_BYTES;

    PagedShare share;
    int pages[S + 1];
    const int rank = sh.cluster > 1 ? blockIdx.x % sh.cluster : 0;
    // a block with one part of one piece from the first key on reads its first pages beside the request's length
    const bool early = sh.cluster == 1 && a.window == 0;
    if (early) {
#pragma unroll
        for (int i = 0; i <= S; ++i)
            pages[i] = pa_page<KT>(a, a.table + blockIdx.x / pieces * a.table_ld, (kwarp + i * kwarps) * KT);
    }
    if (sh.cluster) {
        share.b = blockIdx.x / sh.cluster / pieces;
    } else {
        pdl_trigger();
        share = pa_share(a, pieces, sh.extra, &share_out, warp_sums);
    }
    int b = share.b, n = pa_len(a, b), first = pa_first(a, n), units = pa_units(n, first);
    int piece, at = 0, unit, take;
    if (sh.cluster) {  // no unit for some blocks of a short request's cluster
        piece = blockIdx.x / sh.cluster % pieces;
        unit = (int)((long long)units * rank / sh.cluster);
        take = (int)((long long)units * (rank + 1) / sh.cluster) - unit;
        share.size = 1;
    } else {
        piece = (int)(share.at / (units + sh.extra));
        at = (int)(share.at % (units + sh.extra));
    }
    long long left = share.size;
    int2 rec = make_int2(-1, -1);

    while (left > 0) {
        if (!sh.cluster) {
            const int places = (int)min((long long)(units + sh.extra - at), left);
            unit = max(0, at - sh.extra);
            take = max(0, at + places - sh.extra) - unit;
            left -= places;
        }
        if (sh.cluster || take > 0) {
            const int hk0 = piece / sh.per_kv * sh.side, head0 = piece % sh.per_kv * sh.rows;  // head0: within G
            const int hk = hk0 + set / sh.groups, head = head0 + set % sh.groups * HW;
            const int base = first & ~(PA_ALIGN - 1);
            const int k0 = base + unit * PA_UNIT, k1 = min(n, base + (unit + take) * PA_UNIT);
            const int32_t* row = a.table + b * a.table_ld;
            const C* kc = (const C*)a.kc + hk * a.c_sh;
            const C* vc = (const C*)a.vc + hk * a.c_sh;

            E e;
            const int key = k0 + kwarp * KT;
            const int step = kwarps * KT;
            // the first tiles, and the queries while they are on their way
            if (!early) {
#pragma unroll
                for (int i = 0; i <= S; ++i) pages[i] = pa_page<KT>(a, row, key + i * step);
            }
            pa_tiles<E, false>(e, a, row, kc, vc, ring, qs, pages, key, step, first, k1, lane, [&] {
                e.init(a, (const T*)a.q + b * a.q_sb + ((long long)hk * G + head) * a.q_sh, kc, vc, min(HW, G - head),
                       qs, lane, kwarp, kwarps);
                if (E::Q_BYTES) pa_group_sync(set, kwarps);
            });
            __syncwarp();  // the warp's sums go where its tiles were
            if (E::PARTS && e.spoilt())
                pa_again<E>(e.c, a, row, kc, vc, ring, qs, key, step, first, k1, sm[warp], sl[warp]);
            else
                e.finish(reinterpret_cast<float*>(ring), sm[warp], sl[warp], lane);
            __syncthreads();
            // Each thread joins its four elements over the head's warps by itself: one barrier, and the warps' loads
            // side by side (with the factors computed once a head between two barriers, f32 1 x 8 x 76 of 96 keys
            // took 6.9 us instead of 5.8).
            const int rows = sh.side * sh.rows, n4 = a.dh / 4;
            for (int i = tid; i < rows * n4; i += PA_THREADS) {
                const int r = i / n4, d = (i - r * n4) * 4, s = r / sh.rows, in_g = r - s * sh.rows;
                if (head0 + in_g >= G) continue;
                const int w0 = s * sh.groups + in_g / HW, h = in_g % HW;
                float mw[PA_WARPS], lw[PA_WARPS];
                float4 x[PA_WARPS];
#pragma unroll
                for (int w = 0; w < PA_WARPS; ++w) {
                    const bool his = (w & (sets - 1)) == w0;
                    mw[w] = his ? sm[w][h] : -INFINITY;
                    lw[w] = his ? sl[w][h] : 0.f;
                    x[w] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (his) x[w] = *reinterpret_cast<const float4*>(smem + (size_t)w * 2 * S * SLOT + (h * LD + d) * 4);
                }
                const float top = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
                float total = 0.f;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < PA_WARPS; ++w) pa_add(o, total, x[w], mw[w], lw[w], top);
                const long long head = (long long)(hk0 + s) * G + head0 + in_g;
                if (sh.cluster > 1) {  // over the first of the warps' sums, which nobody else reads
                    *reinterpret_cast<float4*>(smem + (size_t)w0 * 2 * S * SLOT + (h * LD + d) * 4) = o;
                    if (d == 0) sums[w0 * HW + h] = make_float2(top, total);
                } else if (take == units) {
                    pa_result<E>(a, b, head, d, o, top, total);
                } else {
                    const long long at_row = ((long long)blockIdx.x * 2 + (unit == 0)) * rows + r;
                    *reinterpret_cast<float4*>(parts.acc + at_row * a.dh + d) = o;
                    if (d == 0) parts.ml[at_row] = make_float2(top, total);
                }
            }
            if (sh.cluster) {
                if (sh.cluster > 1) {
                    pa_cluster_sync();
                    pa_join_cluster<E>(a, sh, smem, sums, b, hk0, head0, rank);
                    pa_cluster_sync();  // the others may still read this block's sums
                }
                return;
            }
            if (take != units) (unit == 0 ? rec.y : rec.x) = b * pieces + piece;
            __syncthreads();  // the next piece's tiles go where this one's sums were
        }
        if (left <= 0) break;
        at = 0;
        if (++piece == pieces) {
            piece = 0;
            ++b;
            n = pa_len(a, b);
            first = pa_first(a, n);
            units = pa_units(n, first);
        }
    }
    if (tid == 0) parts.rec[blockIdx.x] = rec;
}

// Joins the partial results: block (c, r) looks whether block c of the
// attention began a piece's keys without finishing them, and if so adds up query
// head r of the piece over the blocks c, c + 1, ... that worked on it.  With few
// pieces (`by_piece`) block (i, r) looks for the block that began piece i instead.
template <typename T>
__global__ void __launch_bounds__(PA_JOIN) paged_join_kernel(const PagedAttnArgs a, const PagedShape sh,
                                                            const PagedParts parts, int blocks, int by_piece,
                                                            float scale) {
    __shared__ float weight[PA_MAX_BLOCKS + 1];
    __shared__ float red[2][32];
    __shared__ float4 sums[PA_JOIN];
    __shared__ int began;
    const int r = blockIdx.y, tid = threadIdx.x, threads = blockDim.x;
    int c = blockIdx.x, item = c;
    if (tid == 0) began = -1;
    if (by_piece) __syncthreads();
    pdl_wait();
    if (by_piece) {
        for (int i = tid; i < blocks; i += threads)
            if (parts.rec[i].y == item) began = i;  // one block at most
        __syncthreads();
        c = began;
        if (c < 0) return;
    } else {
        item = parts.rec[c].y;
        if (item < 0) return;
    }
    const int G = a.Hq / a.Hkv, pieces = a.Hkv / sh.side * sh.per_kv, rows = sh.side * sh.rows;
    const int b = item / pieces, piece = item % pieces, in_g = piece % sh.per_kv * sh.rows + r % sh.rows;
    if (in_g >= G) return;
    const long long head = (long long)(piece / sh.per_kv * sh.side + r / sh.rows) * G + in_g;
    int count = 1;  // the blocks of an item are neighbours
    for (int i = c + 1; i < blocks; i += threads) {
        const int here = __syncthreads_count(i + tid < blocks && parts.rec[min(i + tid, blocks - 1)].x == item);
        count += here;
        if (here < threads) break;
    }
    // weights 2^(m - top) and the sum
    float top = -INFINITY, total = 0.f;
    auto ml = [&](int i) { return parts.ml[((long long)(c + i) * 2 + (i == 0)) * rows + r]; };
    for (int i = tid; i < count; i += threads) top = fmaxf(top, ml(i).x);
    top = warp_max(top);
    if ((tid & 31) == 0) red[0][tid >> 5] = top;
    __syncthreads();
    for (int w = 0; w < threads / 32; ++w) top = fmaxf(top, red[0][w]);
    for (int i = tid; i < count; i += threads) {
        const float2 x = ml(i);
        const float f = top == -INFINITY ? (x.y == 0.f ? 0.f : x.y) : pa_exp2(x.x - top);
        weight[i] = f;
        total = fmaf(f, x.y, total);
    }
    total = warp_sum(total);
    if ((tid & 31) == 0) red[1][tid >> 5] = total;
    __syncthreads();
    total = 0.f;
    for (int w = 0; w < threads / 32; ++w) total += red[1][w];
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    // dh/4 threads a partial result, as many side by side as fit, eight loads of each on their way
    const int n4 = a.dh / 4, side = threads / n4, d = (tid % n4) * 4, s0 = tid / n4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s0 < side) {
        for (int i0 = s0; i0 < count; i0 += 8 * side) {
            float4 x[8];
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = i0 + j * side;
                f[j] = 0.f;
                x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < count) {
                    f[j] = weight[i];
                    x[j] = *reinterpret_cast<const float4*>(
                        parts.acc + (((long long)(c + i) * 2 + (i == 0)) * rows + r) * a.dh + d);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                o.x = fmaf(f[j], x[j].x, o.x);
                o.y = fmaf(f[j], x[j].y, o.y);
                o.z = fmaf(f[j], x[j].z, o.z);
                o.w = fmaf(f[j], x[j].w, o.w);
            }
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

// Blocks of a cluster for pieces of at most `bound` keys, 0: shares.  Clusters
// grow while their blocks have more than PA_PART_UNITS units and there are at most
// three a multiprocessor -- one wave, except for 16-bit heads of more than 128
// elements, of which two are resident (bf16 25 x 32/8 x 256 of 1500 keys, 400
// blocks: 63.5 us for 48 us of bytes); they are used for few units a block, since they
// last as long as the longest request.  (In clusters and in shares, bf16
// 32 x 32/8 x 128: 25.5 and 32.8 us of 1000 keys each, 18.7 and 20.3 of 1 .. 1000,
// 43.5 and 51.5 of 2000, 33.8 and 32.6 of 1 .. 2000; f32 on bf16 48 x 12/4 x 80, 31
// units a block: 48.9 and 53.7 us of 4000, 38.0 and 33.0 of 1 .. 4000.  When they
// cannot fill the device, bf16 1 x 32/8 x 128: 12.2 and 15.4 us of 4000 keys, 17.4
// and 16.9 of 8000.)
inline int pa_clusters(long long items, int bound, int sms) {
    const int units = (bound + PA_UNIT - 1) / PA_UNIT;
    if (items > 3LL * sms) return 0;
    int n = 1;
    while (n < PA_CLUSTER && units > PA_PART_UNITS * n && items * 2 * n <= 3LL * sms) n *= 2;
    return units <= (items * n >= sms ? PA_FULL_UNITS : PA_FEW_UNITS) * n ? n : 0;
}
inline int pa_bound(int max_len, int window) {  // of a piece's keys
    return window > 0 && window < max_len ? window + PA_ALIGN : max_len;
}
// How a launch divides its work, by its engine's query heads a warp.  The size of the scratch and the launch are both
// taken from here: the rule above is not monotone in the pieces, so that a size from another number of them may find
// clusters, which need no scratch, where the launch takes shares.
inline PagedShape pa_shape(int B, int Hq, int Hkv, int heads, int bound, int sms) {
    const int G = Hq / Hkv;
    PagedShape sh{1, 1, 1, 0, 0, 0};
    while (sh.groups < PA_WARPS && sh.groups * heads < G) sh.groups *= 2;
    sh.per_kv = (G + sh.groups * heads - 1) / (sh.groups * heads);
    sh.rows = G < sh.groups * heads ? G : sh.groups * heads;
    sh.cluster = pa_clusters((long long)B * Hkv * sh.per_kv, bound, sms);
    return sh;
}
inline size_t pa_scratch_floats(int rows, int dh) {  // of shares with pieces of `rows` query heads
    return (size_t)PA_MAX_BLOCKS * (2 * (size_t)rows * (dh + 2) + 2);
}
// Query heads a warp of the engines that may take a call of G heads a cache head: on float32 pages, on 16-bit pages,
// and on 16-bit pages with the parts of float32 queries packed.
inline int pa_heads_f32(int G) { return G == 1 ? 1 : G == 2 ? 2 : 4; }
constexpr int PA_HEADS_HALF = 8, PA_HEADS_PACKED = 4;

// E2: the engine with two slots a warp, for clusters, whose few blocks leave room for it (bf16 32 x 32/8 x 128 of 1000
// keys: 26.5 us, 29.7 us with one).
template <class E, class E2>
cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t s) {
    static_assert(E::HW * (E::DC + 4) * 4 <= 2 * E::SLOTS * E::TILE_BYTES, "a warp's sums fit in its ring");
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    const int bound = pa_bound(a.max_len, a.window);
    PagedShape sh = pa_shape(a.B, a.Hq, a.Hkv, E::HW, bound, sms);
    long long items = (long long)a.B * a.Hkv * sh.per_kv;
    if (sh.cluster) {
        static DeviceOnce once;
        constexpr size_t kRing = (size_t)PA_WARPS * 2 * E2::SLOTS * E2::TILE_BYTES;
        cudaError_t e = once.set_smem((const void*)paged_attn_kernel<E2>, kRing + PA_WARPS * E2::Q_BYTES);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(items * sh.cluster));
        cfg.blockDim = dim3(PA_THREADS);
        cfg.dynamicSmemBytes = kRing + (size_t)sh.groups * E2::Q_BYTES;
        cfg.stream = s;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = sh.cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = sh.cluster > 1;
        e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<E2>, a, sh, PagedParts{});
        if (e == cudaSuccess) add_launches(1);
        return e;
    }
    static DeviceOnce once;
    constexpr size_t kRing = (size_t)PA_WARPS * 2 * E::SLOTS * E::TILE_BYTES;
    cudaError_t e = once.set_smem((const void*)paged_attn_kernel<E>, kRing + PA_WARPS * E::Q_BYTES);
    if (e != cudaSuccess) return e;
    const int slots = sms * E::BLOCKS < PA_MAX_BLOCKS ? sms * E::BLOCKS : PA_MAX_BLOCKS;
    const long long units = (bound + PA_UNIT - 1) / PA_UNIT;
    // With work for every block, warps take neighbouring cache heads of the same keys: a token's heads lie side by
    // side, and rows of 304 bytes share sectors (f32 1024 x 8 x 76, 128 .. 384 keys: 245 us, 291 us with one head a
    // block; bf16 128 x 32/8 x 128 the same either way; from 2 units a block on instead of 8, bf16 8 x 32/8 x 128 of
    // 8000 keys takes 72 us instead of 54).
    while (sh.side * sh.groups < PA_WARPS && a.Hkv % (2 * sh.side) == 0 &&
           items / 2 * units >= PA_SIDE_UNITS * (long long)slots) {
        sh.side *= 2;
        items /= 2;
    }
    // (of 0, 2 and 6 for one head: bf16 32 x 32/8 x 128 of 1 .. 2000 keys 48, 35 and 38 us, of 2000 each 55, 55 and
    // 57 us; the same of 0, 1 and 2 for two, and more than 0 for four loses 2% where the keys are many)
    sh.extra = sh.side == 1 ? 2 : sh.side == 2 ? 1 : 0;
    int blocks = items * units < slots ? (int)(items * units) : slots;
    const int rows = sh.side * sh.rows;
    if (!a.work || a.work_floats < pa_scratch_floats(rows, a.dh)) return cudaErrorInvalidValue;
    // a whole number of shares a piece, if that costs few blocks: requests of one length are cut evenly (bf16
    // 64 x 32/8 x 128 of 4000 keys: 173 us, 178 us with 592 blocks)
    if (items <= blocks && blocks / items * items * 5 >= 4LL * blocks) blocks = (int)(blocks / items * items);
    PagedParts parts;
    parts.acc = a.work;
    parts.ml = reinterpret_cast<float2*>(a.work + (size_t)PA_MAX_BLOCKS * 2 * rows * a.dh);
    parts.rec = reinterpret_cast<int2*>(parts.ml + (size_t)PA_MAX_BLOCKS * 2 * rows);
    paged_attn_kernel<E>
        <<<blocks, PA_THREADS, kRing + (size_t)sh.side * sh.groups * E::Q_BYTES, s>>>(a, sh, parts);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    add_launches(1);
    PdlScope pdl(true);
    // by pieces, and in large blocks, for the joins of many parts (bf16 1 x 32/8 x 128 of 8000 keys, 74 parts: 16.7 us,
    // 20.1 us by blocks; f16 1 x 16/2 x 256 of 131071 keys, 148 parts: 58 us, 63 us in small blocks)
    const int by_piece = items * 16 <= blocks;
    e = launch_pdl(paged_join_kernel<typename E::Act>, dim3(by_piece ? (unsigned)items : blocks, rows),
                   dim3(by_piece ? PA_JOIN : PA_THREADS), 0, s, a, sh, parts, blocks, by_piece, E::SCALE);
    if (e == cudaSuccess) add_launches(1);
    return e;
}

}  // namespace krk
