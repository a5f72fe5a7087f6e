// Element types of the paged cache kernels: 32-bit, half and bfloat16 values
// read four at a time into 32 bits and rounded once when they are written.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace krk {

KRK_DEV float to_f32(float x) { return x; }
KRK_DEV float to_f32(__half x) { return __half2float(x); }
KRK_DEV float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
KRK_DEV T from_f32(float x);
template <>
KRK_DEV float from_f32<float>(float x) { return x; }
template <>
KRK_DEV __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
KRK_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four consecutive elements (4 * sizeof(T) aligned).
KRK_DEV float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
KRK_DEV float4 load4(const __half* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
KRK_DEV float4 load4(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
KRK_DEV void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
KRK_DEV void store4(__half* p, float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
KRK_DEV void store4(__nv_bfloat16* p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

}  // namespace krk
