// The paged attention kernels for bf16, tile copies.
#include "fa_paged.cuh"

namespace fa {
template int launch_paged_kernels<__nv_bfloat16, true>(const PagedParams&, const PagedPlan&, int, cudaStream_t);
}  // namespace fa
