// Gated scan kernels for x and g in f32.
#include "scan.cuh"

namespace gdn2 {
template int run_types<float, float>(const ScanParams&, const ScanPlan&, bool, bool, cudaStream_t, const char*);
}  // namespace gdn2
