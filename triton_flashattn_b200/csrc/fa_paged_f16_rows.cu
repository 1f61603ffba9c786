// The paged attention kernels for fp16, a copy for each row.
#include "fa_paged.cuh"

namespace fa {
template int launch_paged_kernels<__half, false>(const PagedParams&, const PagedPlan&, int, cudaStream_t);
}  // namespace fa
