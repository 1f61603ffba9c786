// The paged attention kernels for bf16, keys copied in boxes of 16 keys.
#include "fa_paged.cuh"

namespace fa {

int launch_paged_bf16(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  return launch_paged_kernels<__nv_bfloat16, 16>(d, x, bias_kind, stream);
}

}  // namespace fa
