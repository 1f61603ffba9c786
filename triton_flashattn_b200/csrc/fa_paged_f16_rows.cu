// The paged attention kernels for fp16, a copy for each row.
#include "fa_paged.cuh"

namespace fa {

int launch_paged_f16_rows(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  return launch_paged_kernels<__half, false>(d, x, bias_kind, stream);
}

}  // namespace fa
