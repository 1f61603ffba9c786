// The paged attention kernels for bf16, tile copies.
#include "fa_paged.cuh"

namespace fa {

int launch_paged_bf16_tiles(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  return launch_paged_kernels<__nv_bfloat16, true>(d, x, bias_kind, stream);
}

}  // namespace fa
