// Decode attention over float32 pages: the engine on float32 fused
// multiply-adds (as the framework's other float32 paths, no tensor cores: their
// 10-bit operands would change results).
//
// A warp's tile is eight 16-byte loads a lane of keys and eight of values: LPK
// lanes hold a key's elements four at a time, 32 / LPK keys side by side.  A
// lane multiplies its elements of eight (four) keys with its elements of a
// query; the eight partial sums are added over the LPK lanes by exchanging
// halves -- four, two, one, so that each lane ends with one key's score after
// 8 or 9 shuffles instead of 8 x 5 -- and one exponential a lane weighs the
// tile.  HBM bounds it (256 x 8 x 128 of 2048 keys, 4.3 GB: 619 us, 6.9 TB/s;
// 1024 x 8 x 76, whose rows share sectors: 235 us, 5.4 TB/s); with four query heads
// a warp the shuffles do (1024 x 8/2 x 76: 92 us for 51 us of bytes).
#include "paged_attn.cuh"

namespace krk {
namespace {

// PART: rows are not whole sectors of 32 bytes, and are copied through L1.
template <int DC_, int GW, int SLOTS_, bool PART>
struct F32Engine {
    using Act = float;
    using Cache = float;
    static constexpr int DC = DC_, HW = GW;
    static constexpr int LPK = DC >= 128 ? 32 : 16;    // lanes of a key
    static constexpr int NL = DC / (LPK * 4);          // 16-byte loads of a lane for a key
    static constexpr int J = 8 / NL;                   // key steps of a tile
    static constexpr int KPL = 32 / LPK;               // keys side by side
    static constexpr int KT = J * KPL;                 // 16, 8 or 4 keys
    static constexpr bool PARTS = false;
    static constexpr int Q_BYTES = 0;
    static constexpr int TILE_BYTES = 8 * 512, SLOTS = SLOTS_;
    static constexpr int BLOCKS = SLOTS == 1 ? 4 : 3;
    static constexpr float SCALE = 1.f;

    float2 q[GW][NL][2], acc[GW][NL][2];  // pairs for the packed multiply-adds
    float s[GW], m[GW], l[GW], fade[GW], c;

    KRK_DEV void init(const PagedAttnArgs& a, const float* qp, const float*, const float*, int heads, unsigned char*,
                      int lane, int, int) {
        c = a.scale * 1.44269504088896341f;
#pragma unroll
        for (int h = 0; h < GW; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int d = ((lane & (LPK - 1)) + i * LPK) * 4;
                const float4 x = h < heads && d < a.dh ? load4(qp + h * a.q_sh + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                acc[h][i][0] = acc[h][i][1] = make_float2(0.f, 0.f);
                q[h][i][0] = make_float2(x.x, x.y);
                q[h][i][1] = make_float2(x.z, x.w);
            }
        }
    }
    // A lane copies what it reads itself: load i of a tile fills 512 consecutive bytes.  A whole tile on one page
    // takes an addition a copy.
    KRK_DEV void issue(const PagedAttnArgs& a, const float* base, const PagedTile& t, uint32_t to, int lane) {
        constexpr unsigned kAll = (1u << KT) - 1;
        const int d = (lane & (LPK - 1)) * 4;
        to += lane * 16;
        if (t.mask == kAll && a.page_shift >= 4) {
            const float* p = base + (t.off + (lane / LPK) * a.c_st + d);
#pragma unroll
            for (int j = 0; j < J; ++j) {
#pragma unroll
                for (int i = 0; i < NL; ++i)
                    pa_copy<16, PART>(to + (j * NL + i) * 512, p + i * LPK * 4, d + i * LPK * 4 < a.dh);
                p += KPL * a.c_st;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int key = j * KPL + lane / LPK;
            const bool seen = t.mask >> key & 1u;
            const long long off = pa_key(a, t, key);
            const float* p = seen ? base + off + d : base;
#pragma unroll
            for (int i = 0; i < NL; ++i)
                pa_copy<16>(to + (j * NL + i) * 512, p + (seen ? i * LPK * 4 : 0), seen && d + i * LPK * 4 < a.dh);
        }
    }

    // The key step whose score this lane holds after `fold`, and the lane (of its half) that holds step j's.
    static KRK_DEV int step_of(int lane) {
        int j = 0;
#pragma unroll
        for (int o = LPK / 2, n = J / 2; n >= 1; o >>= 1, n >>= 1) j += (lane & o) ? n : 0;
        return j;
    }
    static KRK_DEV constexpr int lane_of(int j) {
        int lane = 0;
        for (int o = LPK / 2, n = J / 2; n >= 1; o >>= 1, n >>= 1) lane += (j & n) ? o : 0;
        return lane;
    }
    static KRK_DEV float fold(float (&x)[J], int lane) {
        int o = LPK / 2;
#pragma unroll
        for (int n = J / 2; n >= 1; n >>= 1, o >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const float give = up ? x[i] : x[i + n], keep = up ? x[i + n] : x[i];
                x[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        }
        float r = x[0];
#pragma unroll
        for (int p = LPK / 2 / J; p >= 1; p >>= 1) r += __shfl_xor_sync(0xffffffffu, r, p);
        return r;
    }

    KRK_DEV void scores(const unsigned char*, unsigned char* from, int lane) {
        float4 k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = *reinterpret_cast<const float4*>(from + lane * 16 + j * 512);
#pragma unroll
        for (int h = 0; h < GW; ++h) {
            float x[J];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                float2 y = make_float2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    y = __ffma2_rn(make_float2(k[j * NL + i].x, k[j * NL + i].y), q[h][i][0], y);
                    y = __ffma2_rn(make_float2(k[j * NL + i].z, k[j * NL + i].w), q[h][i][1], y);
                }
                x[j] = y.x + y.y;
            }
            s[h] = fold(x, lane);
        }
    }
    KRK_DEV void weigh(unsigned mask, int lane) {
        const bool seen = mask >> (step_of(lane) * KPL + lane / LPK) & 1u;
#pragma unroll
        for (int h = 0; h < GW; ++h) {
            const float x = seen ? s[h] * c : -INFINITY;
            float top = x;
#pragma unroll
            for (int o = LPK / 2, n = J / 2; n >= 1; o >>= 1, n >>= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (LPK == 16) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, m[h]);
            const float ref = top == -INFINITY ? 0.f : top;
            fade[h] = pa_exp2(m[h] - ref);
            m[h] = top;
            s[h] = pa_exp2(x - ref);
            l[h] = l[h] * fade[h] + s[h];
        }
    }
    KRK_DEV bool spoilt() const { return false; }
    KRK_DEV void resume(const PagedAttnArgs&, const float*, const float*, float) {}
    template <bool AGAIN>
    KRK_DEV void values(const unsigned char* from, int lane) {
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const float4*>(from + lane * 16 + j * 512);
        const int side = lane & ~(LPK - 1);
#pragma unroll
        for (int h = 0; h < GW; ++h) {
#pragma unroll
            for (int i = 0; i < NL; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    acc[h][i][e].x *= fade[h];
                    acc[h][i][e].y *= fade[h];
                }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float w = __shfl_sync(0xffffffffu, s[h], side + lane_of(j));
                const float2 p = make_float2(w, w);
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    acc[h][i][0] = __ffma2_rn(p, make_float2(v[j * NL + i].x, v[j * NL + i].y), acc[h][i][0]);
                    acc[h][i][1] = __ffma2_rn(p, make_float2(v[j * NL + i].z, v[j * NL + i].w), acc[h][i][1]);
                }
            }
        }
    }
    KRK_DEV void finish(float* obuf, float* sm, float* sl, int lane) {
#pragma unroll
        for (int h = 0; h < GW; ++h) {
            float sum = l[h];
#pragma unroll
            for (int o = LPK / 2, n = J / 2; n >= 1; o >>= 1, n >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (LPK == 16) sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            if (lane == 0) {
                sm[h] = m[h];
                sl[h] = sum;
            }
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                float4 o = make_float4(acc[h][i][0].x, acc[h][i][0].y, acc[h][i][1].x, acc[h][i][1].y);
                if (LPK == 16) {
                    o.x += __shfl_xor_sync(0xffffffffu, o.x, 16);
                    o.y += __shfl_xor_sync(0xffffffffu, o.y, 16);
                    o.z += __shfl_xor_sync(0xffffffffu, o.z, 16);
                    o.w += __shfl_xor_sync(0xffffffffu, o.w, 16);
                }
                if (lane < LPK) *reinterpret_cast<float4*>(obuf + h * (DC + 4) + (lane + i * LPK) * 4) = o;
            }
        }
    }
};

template <int GW, bool PART>
cudaError_t by_width(const PagedAttnArgs& a, cudaStream_t s) {
    if (a.dh <= 64) return launch_paged_attn<F32Engine<64, GW, 1, PART>, F32Engine<64, GW, 2, PART>>(a, s);
    if (a.dh <= 128) return launch_paged_attn<F32Engine<128, GW, 1, PART>, F32Engine<128, GW, 2, PART>>(a, s);
    return launch_paged_attn<F32Engine<256, GW, 1, PART>, F32Engine<256, GW, 2, PART>>(a, s);
}

}  // namespace

int paged_sm_count() {
    static int known[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = __atomic_load_n(&known[dev], __ATOMIC_RELAXED);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        __atomic_store_n(&known[dev], n, __ATOMIC_RELAXED);
    }
    return n;
}

size_t attn_paged_work_floats(int B, int Hq, int Hkv, int dh, int max_len, int window) {
    // the types are not known here: scratch if any engine takes shares, for as many rows as any makes
    const int sms = paged_sm_count(), share = Hq / Hkv, bound = pa_bound(max_len, window);
    const int rows = 4 * share < PA_MAX_ROWS ? 4 * share : PA_MAX_ROWS;
    const int heads[] = {pa_heads_f32(share), share <= PA_HEADS_PACKED ? PA_HEADS_PACKED : PA_HEADS_HALF, PA_HEADS_HALF};
    for (int h : heads)
        if (!pa_shape(B, Hq, Hkv, h, bound, sms > 0 ? sms : 148).cluster) return pa_scratch_floats(rows, dh);
    return 0;
}

cudaError_t attn_decode_paged_f32(const PagedAttnArgs& a, cudaStream_t s) {
    switch (pa_heads_f32(a.Hq / a.Hkv)) {
        case 1: return a.dh % 8 ? by_width<1, true>(a, s) : by_width<1, false>(a, s);
        case 2: return by_width<2, false>(a, s);
        default: return by_width<4, false>(a, s);
    }
}

cudaError_t attn_decode_paged_f16(const PagedAttnArgs& a, bool act_f32, cudaStream_t s);
cudaError_t attn_decode_paged_bf16(const PagedAttnArgs& a, bool act_f32, cudaStream_t s);

cudaError_t attn_decode_paged(const PagedAttnArgs& a, int act, int cache, cudaStream_t s) {
    if (cache == ELEM_F16) return attn_decode_paged_f16(a, act == ELEM_F32, s);
    if (cache == ELEM_BF16) return attn_decode_paged_bf16(a, act == ELEM_F32, s);
    return attn_decode_paged_f32(a, s);
}

}  // namespace krk
