// The selective scan of bfloat16 activations.
#include "selective_scan.cuh"

namespace krk {
cudaError_t selective_scan_bf16(const ScanArgs& a, float* work, int rows, cudaStream_t s) {
    return scan_type<__nv_bfloat16>(a, work, rows, s);
}
}  // namespace krk
