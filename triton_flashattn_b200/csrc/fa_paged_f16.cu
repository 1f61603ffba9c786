// The paged attention kernels for fp16, tile copies.
#include "fa_paged.cuh"

namespace fa {
template int launch_paged_kernels<__half, true>(const PagedParams&, const PagedPlan&, int, cudaStream_t);
}  // namespace fa
