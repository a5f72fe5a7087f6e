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
// request and head); its warps take tiles of keys in turn, each with a running
// maximum and sum, and are merged in shared memory at the piece's end.  A piece
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
constexpr int PA_MAX_HEADS = 32;     // query heads of a block, at most
constexpr int PA_SLOTS = 2;          // tiles of a warp's ring
constexpr int PA_ALIGN = 16;         // a piece's first key is aligned down to the largest tile

// Scratch of a launch: two partial results a block -- slot 0 for a piece that
// does not start its keys, slot 1 for one that does -- and their owners.
struct PagedParts {
    float* acc;  // [blocks][2][heads][dh]
    float2* ml;  // [blocks][2][heads] running maximum (base 2) and sum
    int2* rec;   // [blocks] (request, head) of slots 0 and 1, -1: none
    int heads;
};

struct PagedShape {
    int groups;   // warps that share a tile, each with its own query heads
    int per_kv;   // pieces side by side for the query heads of one cache head
    int whole;    // blocks take whole (request, head)s
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

// The row offset of this lane's key (key0 + lane % KT) of a tile, -1 when the
// key is not visible or its page is outside the pool.
template <int KT>
KRK_DEV int pa_page(const PagedAttnArgs& a, const int32_t* row, int key0, int k1) {
    const int key = key0 + (threadIdx.x & (KT - 1));
    return key < k1 ? row[key >> a.page_shift] : 0;
}
template <int KT>
KRK_DEV long long pa_offset(const PagedAttnArgs& a, int page, int key0, int first, int k1) {
    const int key = key0 + (threadIdx.x & (KT - 1));
    if (key < first || key >= k1) return -1;
    if ((unsigned)page >= (unsigned)a.num_pages) {
        check_fail(CHK_TABLE);
        return -1;
    }
    return page * a.c_sp + (key & ((1 << a.page_shift) - 1)) * a.c_st;
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
//   init(a, q, heads, qs)     loads a warp's queries (or prepares them in shared memory)
//   issue(k, v, off, to)      starts the copies of a tile, from the lanes' row offsets to its ring slot
//   scores(qs, from)          q . k of the slot's keys
//   weigh(mask)               softmax step over the visible keys of the tile
//   values(from)              weighted values into the accumulators
//   finish(obuf, m, l)        accumulators, maxima and sums of the warp to shared memory
// A lane copies exactly the 16-byte pieces that it reads itself, each load of a
// tile in 512 consecutive bytes of the warp's ring: no bank conflicts, no
// barrier, and two tiles a warp in flight without holding registers.
template <class E>
__global__ void __launch_bounds__(PA_THREADS, E::BLOCKS) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a,
                                                                           const PagedShape sh,
                                                                           const PagedParts parts) {
    using T = typename E::Act;
    using C = typename E::Cache;
    constexpr int KT = E::KT, HW = E::HW, LD = E::DC + 4;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float sm[PA_WARPS][HW], sl[PA_WARPS][HW], sf[PA_WARPS][HW];
    __shared__ long long warp_sums[PA_WARPS];
    __shared__ PagedShare share_out;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.Hq / a.Hkv, pieces = a.Hkv * sh.per_kv;
    const int kwarps = PA_WARPS / sh.groups, group = warp % sh.groups, kwarp = warp / sh.groups;
    unsigned char* ring = smem + (size_t)warp * PA_SLOTS * E::TILE_BYTES;
    unsigned char* qs = smem + PA_WARPS * PA_SLOTS * E::TILE_BYTES + (size_t)group * E::Q_BYTES;
    const uint32_t ring_at = smem_addr(ring) + lane * 16;

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
        const int hk = piece / sh.per_kv, head0 = (piece % sh.per_kv) * sh.groups * HW;  // within the cache head's G
        const int base = first & ~(PA_ALIGN - 1);
        const int k0 = base + unit * PA_UNIT, k1 = min(n, base + (unit + take) * PA_UNIT);
        const int32_t* row = a.table + b * a.table_ld;
        const C* kc = (const C*)a.kc + hk * a.c_sh;
        const C* vc = (const C*)a.vc + hk * a.c_sh;

        E e;
        const int mine = min(HW, G - head0 - group * HW);  // this warp's heads, maybe none
        const long long h0 = (long long)hk * G + head0 + group * HW;
        // the first tiles' pages, then the queries while they are on their way
        int key = k0 + kwarp * KT;
        const int step = kwarps * KT;
        const int page0 = pa_page<KT>(a, row, key, k1), page1 = pa_page<KT>(a, row, key + step, k1);
        int page = pa_page<KT>(a, row, key + 2 * step, k1);
        e.init(a, (const T*)a.q + b * a.q_sb + h0 * a.q_sh, mine, qs, lane, kwarp, kwarps);
        if (key < k1) {
            long long off = pa_offset<KT>(a, page0, key, first, k1);
            unsigned mask = __ballot_sync(0xffffffffu, off >= 0);
            e.issue(a, kc, vc, off, ring_at, lane);
            cp_async_commit();
            off = pa_offset<KT>(a, page1, key + step, first, k1);
            unsigned mask_next = __ballot_sync(0xffffffffu, off >= 0);
            if (key + step < k1) e.issue(a, kc, vc, off, ring_at + E::TILE_BYTES, lane);
            cp_async_commit();
            if (E::Q_BYTES) pa_group_sync(group, kwarps);
            for (int slot = 0;; slot ^= 1) {
                cp_async_wait<1>();
                unsigned char* from = ring + slot * E::TILE_BYTES + lane * 16;
                e.scores(qs, from, lane);
                e.weigh(mask, lane);
                e.values(from, lane);
                key += step;
                if (key >= k1) break;
                mask = mask_next;
                off = pa_offset<KT>(a, page, key + step, first, k1);
                mask_next = __ballot_sync(0xffffffffu, off >= 0);
                if (key + step < k1) e.issue(a, kc, vc, off, ring_at + slot * E::TILE_BYTES, lane);
                cp_async_commit();
                page = pa_page<KT>(a, row, key + 2 * step, k1);
            }
            cp_async_wait<0>();
        } else if (E::Q_BYTES) {
            pa_group_sync(group, kwarps);
        }
        __syncwarp();  // the warp's sums go where its tiles were
        e.finish(reinterpret_cast<float*>(ring), sm[warp], sl[warp], lane);
        __syncthreads();
        // each head's factors for its warps' sums
        if (tid < sh.groups * HW) {
            const int g = tid / HW, h = tid % HW;
            float top = -INFINITY, total = 0.f;
            for (int w = g; w < PA_WARPS; w += sh.groups) top = fmaxf(top, sm[w][h]);
            for (int w = g; w < PA_WARPS; w += sh.groups) {
                const float f = top == -INFINITY ? (sl[w][h] == 0.f ? 0.f : sl[w][h]) : exp2f(sm[w][h] - top);
                sf[w][h] = f;
                total = fmaf(f, sl[w][h], total);
            }
            const int head = head0 + tid;
            if (head < G) {
                if (take == units) {
                    const float inv = total == 0.f ? 0.f : 1.0f / total;
                    for (int w = g; w < PA_WARPS; w += sh.groups) sf[w][h] *= inv;
                    if (a.lse)
                        a.lse[(long long)b * a.Hq + hk * G + head] =
                            (top + log2f(total * (1.0f / E::SCALE))) * 0.693147180559945309f;
                } else {
                    parts.ml[((long long)blockIdx.x * 2 + (unit == 0)) * parts.heads + tid] = make_float2(top, total);
                }
            }
        }
        __syncthreads();
        const int n4 = a.dh / 4;
        for (int i = tid; i < sh.groups * HW * n4; i += PA_THREADS) {
            const int gh = i / n4, d = (i % n4) * 4, g = gh / HW, h = gh % HW;
            if (head0 + gh >= G) continue;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = g; w < PA_WARPS; w += sh.groups) {
                const float f = sf[w][h];
                const float4 x = *reinterpret_cast<const float4*>(smem + (size_t)w * PA_SLOTS * E::TILE_BYTES + (h * LD + d) * 4);
                o.x = fmaf(f, x.x, o.x);
                o.y = fmaf(f, x.y, o.y);
                o.z = fmaf(f, x.z, o.z);
                o.w = fmaf(f, x.w, o.w);
            }
            if (take == units)
                store4((T*)a.out + b * a.o_sb + ((long long)hk * G + head0 + gh) * a.o_sh + d, o);
            else
                *reinterpret_cast<float4*>(
                    parts.acc + (((long long)blockIdx.x * 2 + (unit == 0)) * parts.heads + gh) * a.dh + d) = o;
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
        __syncthreads();  // the next piece's queries go where this one's sums were
    }
    if (!sh.whole && tid == 0) parts.rec[blockIdx.x] = rec;
}

// Joins the partial results: block (c, h) looks whether block c of the
// attention began a (request, head) that it did not finish, and if so adds up
// query head h of it over the blocks c, c + 1, ... that worked on it.
template <typename T>
__global__ void __launch_bounds__(PA_THREADS) paged_join_kernel(const PagedAttnArgs a, const PagedShape sh,
                                                               const PagedParts parts, int blocks, int hw,
                                                               float scale) {
    __shared__ float weight[PA_MAX_BLOCKS + 1];
    __shared__ float red[2][PA_WARPS];
    __shared__ float4 sums[PA_THREADS];
    const int c = blockIdx.x, gh = blockIdx.y, tid = threadIdx.x;
    pdl_wait();
    const int item = parts.rec[c].y;
    if (item < 0) return;
    const int G = a.Hq / a.Hkv, pieces = a.Hkv * sh.per_kv;
    const int b = item / pieces, piece = item % pieces, hk = piece / sh.per_kv;
    const int head = (piece % sh.per_kv) * sh.groups * hw + gh;
    if (head >= G) return;
    int count = 1;  // the blocks of an item are neighbours
    for (int i = c + 1; i < blocks; i += PA_THREADS)
        count += __syncthreads_count(i + tid < blocks && parts.rec[min(i + tid, blocks - 1)].x == item);
    // weights 2^(m - top) and the sum
    float top = -INFINITY, total = 0.f;
    auto ml = [&](int i) { return parts.ml[((long long)(c + i) * 2 + (i == 0)) * parts.heads + gh]; };
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
                parts.acc + (((long long)(c + i) * 2 + (i == 0)) * parts.heads + gh) * a.dh + d);
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
        store4((T*)a.out + b * a.o_sb + ((long long)hk * G + head) * a.o_sh + d, o);
    }
    if (tid == 0 && a.lse)
        a.lse[(long long)b * a.Hq + hk * G + head] = (top + log2f(total * (1.0f / scale))) * 0.693147180559945309f;
}

int paged_sm_count();  // of the current device, 0 if it cannot be read

template <class E>
cudaError_t launch_paged_attn(const PagedAttnArgs& a, cudaStream_t s) {
    static DeviceOnce once;
    constexpr size_t kRing = (size_t)PA_WARPS * PA_SLOTS * E::TILE_BYTES;
    static_assert(E::HW * (E::DC + 4) * 4 <= PA_SLOTS * E::TILE_BYTES, "a warp's sums fit in its ring");
    const int G = a.Hq / a.Hkv;
    PagedShape sh{1, 1, 0};
    while (sh.groups < PA_WARPS && sh.groups * E::HW < G) sh.groups *= 2;
    sh.per_kv = (G + sh.groups * E::HW - 1) / (sh.groups * E::HW);
    const size_t smem = kRing + (size_t)sh.groups * E::Q_BYTES;
    cudaError_t e = once.set_smem((const void*)paged_attn_kernel<E>, kRing + PA_WARPS * E::Q_BYTES);
    if (e != cudaSuccess) return e;
    const long long items = (long long)a.B * a.Hkv * sh.per_kv;
    const int bound = a.window > 0 && a.window < a.max_len ? a.window + PA_ALIGN : a.max_len;
    const long long units = (bound + PA_UNIT - 1) / PA_UNIT;
    if (units <= PA_WHOLE_UNITS) {
        sh.whole = 1;
        paged_attn_kernel<E><<<(unsigned)items, PA_THREADS, smem, s>>>(a, sh, PagedParts{});
        add_launches(1);
        return cudaGetLastError();
    }
    const int sms = paged_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    int blocks = sms * E::BLOCKS < PA_MAX_BLOCKS ? sms * E::BLOCKS : PA_MAX_BLOCKS;
    if (items * units < blocks) blocks = (int)(items * units);
    PagedParts parts;
    parts.heads = sh.groups * E::HW;
    parts.acc = a.work;
    parts.ml = reinterpret_cast<float2*>(a.work + (size_t)PA_MAX_BLOCKS * 2 * parts.heads * a.dh);
    parts.rec = reinterpret_cast<int2*>(parts.ml + (size_t)PA_MAX_BLOCKS * 2 * parts.heads);
    paged_attn_kernel<E><<<blocks, PA_THREADS, smem, s>>>(a, sh, parts);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    add_launches(1);
    PdlScope pdl(true);
    e = launch_pdl(paged_join_kernel<typename E::Act>, dim3(blocks, G < parts.heads ? G : parts.heads),
                   dim3(PA_THREADS), 0, s, a, sh, parts, blocks, E::HW, E::SCALE);
    if (e == cudaSuccess) add_launches(1);
    return e;
}

}  // namespace krk
