// Decode attention over bfloat16 pages.
#include "paged_attn_half.cuh"

namespace krk {

cudaError_t attn_decode_paged_bf16(const PagedAttnArgs& a, bool act_f32, cudaStream_t s) {
    return act_f32 ? by_alignment<float, __nv_bfloat16>(a, s) : by_alignment<__nv_bfloat16, __nv_bfloat16>(a, s);
}

}  // namespace krk
