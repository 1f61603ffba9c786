// The paged attention kernels for fp16, keys copied in rows.
#include "fa_paged.cuh"

namespace fa {

int launch_paged_f16_rows(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  return launch_paged_kernels<__half, 0>(d, x, bias_kind, stream);
}

}  // namespace fa
