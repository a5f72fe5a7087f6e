// Decode attention over half and bfloat16 pages: the engine on m16n8k16 matrix
// instructions.
//
// A warp's tile is 16 keys and 8 query heads that share them:
//   S = Q K^T        16 x 8 over k = 16: heads (two parts of each, or eight empty rows) x keys over dh
//   O^T = V^T P^T    16 x 8 over k = 16: elements of dh x heads over keys
// Rows of K are the second operand as they lie, rows of V the first one
// transposed by the load (ldmatrix), and P^T's operand layout is the one that S
// comes out in, so weights never leave their lane's registers.  The 16-byte
// pieces of a row are permuted by its number so that neither the copies nor the
// matrix loads meet in a bank.
//
// Keys and values are read once at up to the copy rate (bf16 128 x 32/8 x 128,
// up to 8192 keys, 2.15 GB: 331 us, 6.5 TB/s); with few keys a call, latency
// bounds it, and with 16 query heads a cache head, whose tiles two warps copy, L1
// (64 x 128/8 x 128, up to 8192 keys: 244 us for 168 us of bytes).  Rows that are not 16-byte
// aligned, or not a multiple of 8 elements, are shifted in place when all of a
// head's lie alike (bf16 64 x 32/8 x 76: 139 us for 100 us of bytes, 173 us when
// they were copied 8 bytes at a time, as they still are when tokens differ).
//
// Precision: the products are exact and added in 32 bits, and a tile's sum is
// folded into the float32 accumulators once a tile.  A float32 weight is the
// sum of two 16-bit parts (three when float32 results are wanted from bfloat16
// pages: 24 bits), and a float32 query of two half parts after scaling its row
// by a power of two (22 bits and a sign) or three bfloat16 parts (24 bits).
// Half weights are scaled by 2^14, so that a key 2^-24 as likely as the
// strongest still has 14 bits.  A part may be 0 where the weight is not: infinite
// values, which that would turn into NaN, are looked for in a second pass by warps
// whose sums are NaN.
#pragma once
#include "paged_attn.cuh"

namespace krk {
namespace {

KRK_DEV void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
KRK_DEV void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                 __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two floats rounded into one register (x in the low half), and what is left of them.
KRK_DEV uint32_t pack_rest(float& x, float& y, __half) {
    const __half2 h = __floats2half2_rn(x, y);
    x -= __low2float(h);
    y -= __high2float(h);
    return *reinterpret_cast<const uint32_t*>(&h);
}
KRK_DEV uint32_t pack_rest(float& x, float& y, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
    x -= __uint_as_float(u << 16);
    y -= __uint_as_float(u & 0xffff0000u);
    return u;
}

// The same onto zero.
KRK_DEV void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                       __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
KRK_DEV void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                       __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Four 8 x 8 matrices of 16-bit elements, lane l giving row l % 8 of matrix l / 8.
KRK_DEV void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
KRK_DEV void load_matrices_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

// How rows lie: 8-byte pieces only; every row of a cache head at the same place within 16 bytes; all on 16 bytes.
enum RowAlign { ROWS_NARROW, ROWS_SHIFTED, ROWS_WIDE };

// DC: the elements of a row that are worked on, a multiple of 32 that is at least dh (dh + 4 for shifted rows); SLOTS:
// of a warp's ring.  Shifted rows are copied from the 16-byte boundary before them, and everything -- queries, products,
// results -- is moved up by the `before` elements in between; what the copies bring along of other rows is cleared in
// the keys, where it would meet a query, and dropped with the results' columns in the values.
template <typename T, typename C, int DC_, int ALIGN, int SLOTS_, int HW_>
struct HalfEngine {
    using Act = T;
    using Cache = C;
    static constexpr bool kSame = sizeof(T) == 2, kHalf = sizeof(__half) == 2 && std::is_same<C, __half>::value;
    static constexpr int DC = DC_, KT = 16, HW = HW_;
    static constexpr bool kPacked = HW == PA_HEADS_PACKED;  // parts lie in the rows and columns of four heads that are not there
    static constexpr int NB = DC / 32, NV = DC / 16;     // steps of the two products
    static constexpr int CPR = DC <= 64 ? 8 : DC <= 128 ? 16 : 32, ROW = CPR * 16;  // a row's 16-byte pieces and bytes
    static constexpr int RPC = 32 / CPR;                  // rows of one copy
    static constexpr int QP = kSame ? 1 : kHalf ? 2 : 3;  // parts of a query
    static constexpr int PP = !kSame && !kHalf ? 3 : 2;   // parts of a weight
    static constexpr int QA = kPacked ? (QP + 1) / 2 : QP;  // eights of rows of the first operand
    static constexpr bool PARTS = true;
    static constexpr int Q_BYTES = QA * NB * 32 * 16;
    static constexpr int TILE_BYTES = KT * ROW, SLOTS = SLOTS_;
    static constexpr int BLOCKS = DC > 128 ? 2 : SLOTS == 1 ? 4 : 3;
    static constexpr float SCALE = kHalf ? 16384.f : 1.f;

    float acc[NV][4];
    float s[4], m, l, c, fade;
    int before_k, before_v;  // 0 or 4
    int dh;

    KRK_DEV void resume(const PagedAttnArgs& a, const C* kc, const C* vc, float scale) {
        dh = a.dh;
        before_k = ALIGN == ROWS_SHIFTED && (reinterpret_cast<uintptr_t>(kc) & 15) ? 4 : 0;
        before_v = ALIGN == ROWS_SHIFTED && (reinterpret_cast<uintptr_t>(vc) & 15) ? 4 : 0;
        c = scale;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[i][x] = 0.f;
    }
    // Lays the parts of the group's queries out as the first operand's registers.  Each warp of a group prepares
    // every kwarps-th head.
    KRK_DEV void init(const PagedAttnArgs& a, const T* q, const C* kc, const C* vc, int heads, unsigned char* qs,
                      int lane, int kwarp, int kwarps) {
        resume(a, kc, vc, a.scale * 1.44269504088896341f);
        for (int h = kwarp; h < HW; h += kwarps) {
            float4 x[(DC + 127) / 128];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < (DC + 127) / 128; ++i) {
                const int d = (i * 32 + lane) * 4 - before_k;
                x[i] = h < heads && d >= 0 && d < a.dh ? load4(q + h * a.q_sh + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                most = fmaxf(most, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
            }
            float up = 1.f;
            if (QP == 2) up = row_scale(warp_max(most));
#pragma unroll
            for (int i = 0; i < (DC + 127) / 128; ++i) {
                const int d = (i * 32 + lane) * 4;
                if (d >= DC) continue;
                float4 y = make_float4(x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up);
#pragma unroll
                for (int p = 0; p < (kPacked ? 2 * QA : QA); ++p) {  // (a part beyond the last is zero)
                    const int row = kPacked ? p * 4 + h : p * 8 + h;
                    uint32_t* to = reinterpret_cast<uint32_t*>(qs) +
                                   ((row / 8 * NB + d / 32) * 32 + row % 8 * 4 + d % 8 / 2) * 4 + d % 32 / 8;
                    to[0] = p < QP ? pack_rest(y.x, y.y, C()) : 0u;
                    to[4] = p < QP ? pack_rest(y.z, y.w, C()) : 0u;
                }
            }
            if (QP == 2 && lane / 4 % HW == h) c *= 1.0f / up;
        }
        if (QP == 2) {  // the other warps' heads: the same scales again
            for (int h = 0; h < HW; ++h) {
                if (h % kwarps == kwarp) continue;
                float most = 0.f;
                for (int d = lane * 4; h < heads && d < a.dh; d += 128) {
                    const float4 x = load4(q + h * a.q_sh + d);
                    most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                }
                const float up = row_scale(warp_max(most));
                if (lane / 4 % HW == h) c *= 1.0f / up;
            }
        }
    }
    // The power of two that brings the row's largest element to 2^14 .. 2^15 (at most 2^126, whose inverse is a normal
    // number; 1 for zeros, infinities and NaN).
    static KRK_DEV float row_scale(float most) {
        if (!(most > 0.f) || most == INFINITY) return 1.f;
        return exp2f((float)min(126, 14 - ilogbf(most)));
    }

    KRK_DEV void issue(const PagedAttnArgs& a, const C* base, const PagedTile& t, uint32_t to, int lane) {
        const int chunk = lane & (CPR - 1), row0 = lane / CPR;
        const int before = ALIGN == ROWS_SHIFTED && (reinterpret_cast<uintptr_t>(base) & 15) ? 4 : 0;
        const bool in = chunk * 8 < a.dh + before, more = chunk * 8 + 4 < a.dh;
        to += row0 * ROW;
        if (t.mask == 0xffffu && a.page_shift >= 4) {  // a whole tile on one page: an addition a copy
            const C* p = base + (t.off + row0 * a.c_st + chunk * 8 - before);
#pragma unroll
            for (int j = 0; j < KT / RPC; ++j) {
                const uint32_t at = to + j * RPC * ROW + (((chunk ^ row0) ^ (j * RPC & 7)) << 4);
                if (ALIGN != ROWS_NARROW) {
                    pa_copy<16>(at, p, in);
                } else {
                    pa_copy<8>(at, p, in);
                    pa_copy<8>(at + 8, p + 4, more);
                }
                p += RPC * a.c_st;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < KT / RPC; ++j) {
            const int row = j * RPC + row0;
            const bool seen = t.mask >> row & 1u;
            const long long off = pa_key(a, t, row);
            const C* p = seen ? base + off + chunk * 8 - before : base - before;
            const uint32_t at = to + j * RPC * ROW + (((chunk ^ row0) ^ (j * RPC & 7)) << 4);
            if (ALIGN != ROWS_NARROW) {
                pa_copy<16>(at, p, seen && in);
            } else {
                pa_copy<8>(at, p, seen && in);
                pa_copy<8>(at + 8, p + (seen ? 4 : 0), seen && more);
            }
        }
    }

    // Clears the four elements before and behind each of the tile's keys in their first and last 16 bytes.
    KRK_DEV void clear_edges(unsigned char* from, int lane) {
        const int end = dh + before_k;
        unsigned char* row = from + (lane & 15) * ROW;
        if (lane < 16) {
            if (before_k) *reinterpret_cast<uint2*>(row + ((lane & 7) << 4)) = make_uint2(0u, 0u);
        } else {
            if (end & 4) *reinterpret_cast<uint2*>(row + (((end >> 3) ^ (lane & 7)) << 4) + 8) = make_uint2(0u, 0u);
        }
        __syncwarp();
    }

    KRK_DEV void scores(const unsigned char* qs, unsigned char* from, int lane) {
        if (ALIGN == ROWS_SHIFTED) clear_edges(from, lane);
        float d0[4], d1[4], e0[4], e1[4];
        const uint4* qf = reinterpret_cast<const uint4*>(qs) + lane;
        const uint32_t at = smem_addr(from) + (lane & 7) * ROW;
        const int piece = lane >> 3, turn = lane & 7;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            uint32_t k0[4], k1[4];
            load_matrices(k0, at + (((i * 4 + piece) ^ turn) << 4));
            load_matrices(k1, at + 8 * ROW + (((i * 4 + piece) ^ turn) << 4));
            const uint4 h = qf[i * 32];
            const uint4 r = QA > 1 ? qf[(NB + i) * 32] : make_uint4(0u, 0u, 0u, 0u);
            if (i == 0) {
                mma_first(d0, h.x, r.x, h.y, r.y, k0[0], k0[1], C());
                mma_first(d1, h.x, r.x, h.y, r.y, k1[0], k1[1], C());
            } else {
                mma(d0, h.x, r.x, h.y, r.y, k0[0], k0[1], C());
                mma(d1, h.x, r.x, h.y, r.y, k1[0], k1[1], C());
            }
            mma(d0, h.z, r.z, h.w, r.w, k0[2], k0[3], C());
            mma(d1, h.z, r.z, h.w, r.w, k1[2], k1[3], C());
            if (QA > 2) {
                const uint4 t = qf[(2 * NB + i) * 32];
                if (i == 0) {
                    mma_first(e0, t.x, 0u, t.y, 0u, k0[0], k0[1], C());
                    mma_first(e1, t.x, 0u, t.y, 0u, k1[0], k1[1], C());
                } else {
                    mma(e0, t.x, 0u, t.y, 0u, k0[0], k0[1], C());
                    mma(e1, t.x, 0u, t.y, 0u, k1[0], k1[1], C());
                }
                mma(e0, t.z, 0u, t.w, 0u, k0[2], k0[3], C());
                mma(e1, t.z, 0u, t.w, 0u, k1[2], k1[3], C());
            }
        }
        if (QA <= 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) e0[i] = e1[i] = 0.f;
        }
        if (kPacked) {  // rows 0-3, 4-7 and 8-11 hold the parts of the same four heads: every lane gets all three
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                apart(d0[i], d0[2 + i], e0[i], lane);
                apart(d1[i], d1[2 + i], e1[i], lane);
            }
        }
        s[0] = joined(d0[0], d0[2], e0[0]);
        s[1] = joined(d0[1], d0[3], e0[1]);
        s[2] = joined(d1[0], d1[2], e1[0]);
        s[3] = joined(d1[1], d1[3], e1[1]);
    }
    static KRK_DEV void apart(float& low, float& high, float& third, int lane) {
        const float other = __shfl_xor_sync(0xffffffffu, low, 16);
        if (QP > 2) third = __shfl_sync(0xffffffffu, high, lane & 15);
        high = lane < 16 ? other : low;
        low = lane < 16 ? low : other;
    }
    // The parts' products; an infinite key's first part decides (the others may be infinite the other way, or NaN).
    static KRK_DEV float joined(float first, float second, float third) {
        if (QP == 1) return first;
        const float sum = QP > 2 ? first + (second + third) : first + second;
        return fabsf(first) == INFINITY ? first : sum;
    }

    KRK_DEV void weigh(unsigned mask, int lane) {
        const int t = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] *= c;
        if ((mask & 0xffffu) != 0xffffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(mask >> (2 * t + (i & 1) + (i >> 1) * 8) & 1u)) s[i] = -INFINITY;
        }
        float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m);
        const float ref = top == -INFINITY ? 0.f : top;
        fade = pa_exp2(m - ref);
        m = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = pa_exp2(s[i] - ref) * SCALE;
        l = l * fade + ((s[0] + s[1]) + (s[2] + s[3]));
    }

    // AGAIN: every weight that is not 0 taken for 2^-14 as well.  Where that product is infinite it is the result: a part
    // of the weight may be 0 there, or negative, and spoil it.
    template <bool AGAIN>
    KRK_DEV void values(const unsigned char* from, int lane) {
        // of the accumulators' columns 2 (lane % 4) and the one after it
        const float f0 = __shfl_sync(0xffffffffu, fade, (lane & 3) * 8 % (HW * 4));
        const float f1 = __shfl_sync(0xffffffffu, fade, ((lane & 3) * 8 + 4) % (HW * 4));
        uint32_t p[PP][2], some[2];
        if (AGAIN) {
            constexpr uint32_t kSmall = kHalf ? 0x0400u : 0x3880u;
#pragma unroll
            for (int x = 0; x < 2; ++x)
                some[x] = (s[2 * x] > 0.f ? kSmall : 0u) | (s[2 * x + 1] > 0.f ? kSmall << 16 : 0u);
        }
#pragma unroll
        for (int i = 0; i < PP; ++i) {
            p[i][0] = pack_rest(s[0], s[1], C());
            p[i][1] = pack_rest(s[2], s[3], C());
        }
        if (kPacked) {  // columns 0-3 take the first part, 4-7 the second, and the third goes by itself
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                p[0][x] = lane < 16 ? p[0][x] : p[1][x];
                if (PP > 2) p[1][x] = lane < 16 ? p[PP - 1][x] : 0u;
            }
        }
        constexpr int PA = kPacked ? PP - 1 : PP;
        // matrices: keys 0-7 and 8-15 of the pieces 2i and 2i + 1
        const int key = (lane >> 4) * 8 + (lane & 7), piece = lane >> 3 & 1, turn = lane & 7;
        const uint32_t at = smem_addr(from) + key * ROW;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint32_t v[4];
            load_matrices_t(v, at + (((i * 2 + piece) ^ turn) << 4));
            float d[4];
            mma_first(d, v[0], v[1], v[2], v[3], p[PA - 1][0], p[PA - 1][1], C());
#pragma unroll
            for (int x = PA - 2; x >= 0; --x) mma(d, v[0], v[1], v[2], v[3], p[x][0], p[x][1], C());
            if (AGAIN) {
                float y[4];
                mma_first(y, v[0], v[1], v[2], v[3], some[0], some[1], C());
#pragma unroll
                for (int x = 0; x < 4; ++x) d[x] = fabsf(y[x]) == INFINITY ? y[x] : d[x];
            }
            acc[i][0] = fmaf(acc[i][0], f0, d[0]);
            acc[i][1] = fmaf(acc[i][1], f1, d[1]);
            acc[i][2] = fmaf(acc[i][2], f0, d[2]);
            acc[i][3] = fmaf(acc[i][3], f1, d[3]);
        }
    }
    // NaN among the warp's sums: an infinite value may be behind it, and the tiles are taken once more, in parts.
    KRK_DEV bool spoilt() const {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) bad |= acc[i][x] != acc[i][x];
        return __any_sync(0xffffffffu, bad);
    }
    KRK_DEV void finish(float* obuf, float* sm, float* sl, int lane) {
        const int r = lane >> 2, t = lane & 3;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0 && r < HW) {
            sm[r] = m;
            sl[r] = l;
        }
        if (kPacked) {  // the columns of the parts
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float rest = __shfl_xor_sync(0xffffffffu, acc[i][x], 2);
                    acc[i][x] = fabsf(acc[i][x]) == INFINITY ? acc[i][x] : acc[i][x] + rest;
                }
            if (t > 1) return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float* o = obuf + 2 * t * (DC + 4) + i * 16 + r - before_v;
            if (ALIGN != ROWS_SHIFTED || i * 16 + r >= before_v) {
                o[0] = acc[i][0];
                o[DC + 4] = acc[i][1];
            }
            o[8] = acc[i][2];
            o[DC + 12] = acc[i][3];
        }
    }
};

template <typename T, typename C, int ALIGN, int HW>
cudaError_t by_width(const PagedAttnArgs& a, cudaStream_t s) {
    const int width = ALIGN == ROWS_SHIFTED ? a.dh + 4 : a.dh;
    if (width <= 64)
        return launch_paged_attn<HalfEngine<T, C, 64, ALIGN, 1, HW>, HalfEngine<T, C, 64, ALIGN, 2, HW>>(a, s);
    if (width <= 96)
        return launch_paged_attn<HalfEngine<T, C, 96, ALIGN, 1, HW>, HalfEngine<T, C, 96, ALIGN, 2, HW>>(a, s);
    if (width <= 128)
        return launch_paged_attn<HalfEngine<T, C, 128, ALIGN, 1, HW>, HalfEngine<T, C, 128, ALIGN, 2, HW>>(a, s);
    if (width <= 192)
        return launch_paged_attn<HalfEngine<T, C, 192, ALIGN, 1, HW>, HalfEngine<T, C, 192, ALIGN, 1, HW>>(a, s);
    return launch_paged_attn<HalfEngine<T, C, 256, ALIGN, 1, HW>, HalfEngine<T, C, 256, ALIGN, 1, HW>>(a, s);
}

// Up to four heads of float32 queries lie packed, their parts in the rows and columns of the four that are missing (f32
// queries on bf16 pages, 1024 x 8 x 76: 146 us, 161 us in eights; on f16 pages 147 and 162 us).
template <typename T, typename C, int ALIGN>
cudaError_t by_heads(const PagedAttnArgs& a, cudaStream_t s) {
    if constexpr (sizeof(T) == 4)
        if (a.Hq / a.Hkv <= PA_HEADS_PACKED) return by_width<T, C, ALIGN, PA_HEADS_PACKED>(a, s);
    return by_width<T, C, ALIGN, PA_HEADS_HALF>(a, s);
}

template <typename T, typename C>
cudaError_t by_alignment(const PagedAttnArgs& a, cudaStream_t s) {
    const bool same = a.c_sp % 8 == 0 && a.c_st % 8 == 0;
    const bool wide = same && a.dh % 8 == 0 && a.c_sh % 8 == 0 && (reinterpret_cast<uintptr_t>(a.kc) & 15) == 0 &&
                      (reinterpret_cast<uintptr_t>(a.vc) & 15) == 0;
    if (wide) return by_heads<T, C, ROWS_WIDE>(a, s);
    if (same && a.dh <= 252) return by_heads<T, C, ROWS_SHIFTED>(a, s);
    return by_width<T, C, ROWS_NARROW, PA_HEADS_HALF>(a, s);
}

}  // namespace

}  // namespace krk
