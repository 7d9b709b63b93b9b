// Gated scan kernels for x and g in bf16.
#include "scan.cuh"

namespace gdn2 {
template int run_types<__nv_bfloat16, __nv_bfloat16>(const ScanParams&, const ScanPlan&, bool, bool, cudaStream_t, const char*);
}  // namespace gdn2
