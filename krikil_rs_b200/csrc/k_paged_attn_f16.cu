// Decode attention over half pages.
#include "paged_attn_half.cuh"

namespace krk {

cudaError_t attn_decode_paged_f16(const PagedAttnArgs& a, bool act_f32, cudaStream_t s) {
    return act_f32 ? by_alignment<float, __half>(a, s) : by_alignment<__half, __half>(a, s);
}

}  // namespace krk
