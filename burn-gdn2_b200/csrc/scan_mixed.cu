// Gated scan kernels for x in bf16 and g in f32.
#include "scan.cuh"

namespace gdn2 {
template int run_types<__nv_bfloat16, float>(const ScanParams&, const ScanPlan&, bool, bool, cudaStream_t, const char*);
}  // namespace gdn2
