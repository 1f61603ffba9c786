// The paged attention kernels for fp16, keys copied in boxes of 8 keys.
#include "fa_paged.cuh"

namespace fa {

int launch_paged_f16_box8(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  return launch_paged_kernels<__half, 8>(d, x, bias_kind, stream);
}

}  // namespace fa
