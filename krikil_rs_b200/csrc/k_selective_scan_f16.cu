// The selective scan of half activations.
#include "selective_scan.cuh"

namespace krk {
cudaError_t selective_scan_f16(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s) {
    return scan_type<__half>(a, work, plan, s);
}
}  // namespace krk
