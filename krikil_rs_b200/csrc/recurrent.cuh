// Device helpers of the recurrent layers: the rows and the state slots of a
// packed request, neither of which is trusted.
#pragma once
#include "elem.cuh"
#include "recurrent.h"

namespace krk {

struct Span {
    int begin, end;  // rows [begin, end) of the packed ones
};

KRK_DEV int clamp_row(int r, int T) { return r < 0 ? 0 : r > T ? T : r; }

KRK_DEV Span request_rows(const int32_t* cu, int s, int T) {
    const int i = cu[s], j = cu[s + 1], begin = clamp_row(i, T), end = clamp_row(j, T);
    if (begin != i || end != j || end < begin) check_fail(CHK_POSITION);
    return {begin, end < begin ? begin : end};
}

// The slot that a request leaves its state in and the one it continues from
// (below 0: nothing), of what its entries say; false for padding, whose rows are
// left alone.
KRK_DEV bool valid_slots(const SlotArgs& a, int to, int from) {
    if (to < 0) return false;
    if (to < a.num_slots && from < a.num_slots) return true;
    check_fail(CHK_TABLE);
    return false;
}
KRK_DEV bool request_slots(const SlotArgs& a, int s, int& to, int& from) {
    to = from = -1;
    if (!a.state) return true;
    to = a.slots ? a.slots[s] : s;
    from = a.init ? a.init[s] : to;
    return valid_slots(a, to, from);
}
// Those of R requests from s on (the last one's for those behind it), loaded
// without a wait in between.
template <int R>
KRK_DEV void load_slots(const SlotArgs& a, int s, int requests, int (&to)[R], int (&from)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = min(s + r, requests - 1);
        to[r] = a.slots ? a.slots[i] : i;
        from[r] = a.init ? a.init[i] : to[r];
    }
}

// x * sigmoid(x) on the exponential unit (ex2 and rcp, each within 2^-22).
KRK_DEV float fast_silu(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504088896341f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return x * r;
}
KRK_DEV float2 fast_silu(float2 x) {
    float2 e = __fmul2_rn(x, make_float2(-1.44269504088896341f, -1.44269504088896341f)), r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
    e = __fadd2_rn(e, make_float2(1.0f, 1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return __fmul2_rn(x, r);
}
KRK_DEV float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A decay in powers of two; finite, since rows that step by nothing step by 0 times it.
KRK_DEV float scan_rate(float a) {
    const float r = a * 1.44269504088896341f;
    return r < -3.0e38f ? -3.0e38f : r;
}

// log(1 + e^v) as max(v, 0) + 2 atanh(w / (2 + w)), w = e^-|v|, by atanh's series (its argument is at most 1/3: the
// first term left out is 2^-26 of the whole), which keeps the small steps that negative arguments make.
KRK_DEV float step_width(float v) {
    const float w = fast_exp2(fabsf(v) * -1.44269504088896341f);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(2.0f + w));
    const float s = w * r, q = s * s;
    float p = fmaf(q, 2.0f / 13.0f, 2.0f / 11.0f);
    p = fmaf(p, q, 2.0f / 9.0f);
    p = fmaf(p, q, 2.0f / 7.0f);
    p = fmaf(p, q, 2.0f / 5.0f);
    p = fmaf(p, q, 2.0f / 3.0f);
    p = fmaf(p, q, 2.0f);
    return fmaf(s, p, fmaxf(v, 0.0f));
}

// V consecutive elements in one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};
template <typename T, int V>
KRK_DEV Pack<T, V> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }
// V elements as packed pairs of float32 (a lone one in the first half), and back, each rounded once.
template <int V>
constexpr int pairs_of = (V + 1) / 2;
template <typename T, int V>
KRK_DEV void unpack(const Pack<T, V>& p, float2 (&x)[pairs_of<V>]) {
#pragma unroll
    for (int i = 0; i < pairs_of<V>; ++i)
        x[i] = make_float2(to_f32(p.v[2 * i]), 2 * i + 1 < V ? to_f32(p.v[V > 1 ? 2 * i + 1 : 0]) : 0.0f);
}
KRK_DEV void round_pair(float2 x, float* p) { p[0] = x.x, p[1] = x.y; }
KRK_DEV void round_pair(float2 x, __half* p) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x.x, x.y); }
KRK_DEV void round_pair(float2 x, __nv_bfloat16* p) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x.x, x.y); }
template <typename T, int V>
KRK_DEV Pack<T, V> pack(const float2 (&x)[pairs_of<V>]) {
    Pack<T, V> p;
    if constexpr (V == 1) {
        p.v[0] = from_f32<T>(x[0].x);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) round_pair(x[i], &p.v[2 * i]);
    }
    return p;
}
template <typename T, int V>
KRK_DEV void store_pack(T* p, const Pack<T, V>& x) { *reinterpret_cast<Pack<T, V>*>(p) = x; }

}  // namespace krk
