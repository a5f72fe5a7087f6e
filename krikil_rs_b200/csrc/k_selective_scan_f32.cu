// The selective scan of float32 activations.
#include "selective_scan.cuh"

namespace krk {
cudaError_t selective_scan_f32(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s) {
    return scan_type<float>(a, work, plan, s);
}
}  // namespace krk
