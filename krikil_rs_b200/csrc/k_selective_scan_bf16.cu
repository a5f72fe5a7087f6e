// The selective scan of bfloat16 activations.
#include "selective_scan.cuh"

namespace krk {
cudaError_t selective_scan_bf16(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s) {
    return scan_type<__nv_bfloat16>(a, work, plan, s);
}
}  // namespace krk
