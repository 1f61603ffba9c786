// Attention of one new token a sequence over a paged key / value cache.
//
//   s_n = sm_scale q . k_n + bias_n,   o = sum_n exp(s_n - m) v_n / sum_n exp(s_n - m)   over the keys n of the sequence,
// in one pass: a running maximum m, the sum and the weighted values of a stretch of keys are rescaled where m rises, and
// stretches are joined with the weights exp(m_i - m).  The simplest form: a CTA per (sequence, head), a key per warp and step.
#include "fa_common.cuh"
#include "fa_host.cuh"

namespace fa {
namespace {

struct PagedParams {
  const void* q;
  const void* k;
  const void* v;
  const void* bias;
  void* o;
  const int* table;
  const int* lens;
  int* status;
  int64_t q_sB, q_sH, o_sB, o_sH, k_sP, k_sT, k_sH, v_sP, v_sT, v_sH, bias_sB, bias_sH, table_s;
  int H, group, D, page_size, num_pages, width;
  float sm_scale;
};

constexpr int kWarps = 4;

template <typename T, int BIAS>
__global__ void __launch_bounds__(kWarps * 32) paged_kernel(const PagedParams p) {
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, hk = h / p.group;
  grid_dep_launch_next();
  grid_dep_wait();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  const int len = min(max(__ldcg(p.lens + b), 0), p.width * p.page_size);
  constexpr int kPer = 8;  // elements of a lane: lane, lane + 32, ...
  float q[kPer], o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < p.D ? static_cast<float>(static_cast<const T*>(p.q)[b * p.q_sB + h * p.q_sH + d]) : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int n = warp; n < len; n += kWarps) {
    const int page = __ldcg(p.table + b * p.table_s + n / p.page_size);
    if (page < 0 || page >= p.num_pages) continue;
    const int at = n % p.page_size;
    const T* k = static_cast<const T*>(p.k) + page * p.k_sP + at * p.k_sT + hk * p.k_sH;
    const T* v = static_cast<const T*>(p.v) + page * p.v_sP + at * p.v_sT + hk * p.v_sH;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (const int d = lane + 32 * i; d < p.D) s += q[i] * static_cast<float>(k[d]);
    for (int off = 1; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= p.sm_scale;
    const int64_t at_bias = b * p.bias_sB + h * p.bias_sH + n;
    if constexpr (BIAS == 1) s += static_cast<float>(static_cast<const T*>(p.bias)[at_bias]);
    if constexpr (BIAS == 2) s = static_cast<const uint8_t*>(p.bias)[at_bias] ? s : -INFINITY;
    if constexpr (BIAS == 3) s += static_cast<const float*>(p.bias)[at_bias];
    if (s == -INFINITY) continue;  // takes no part, whatever the value holds
    const float m_new = fmaxf(m, s);
    const float alpha = m == m_new ? 1.f : ex2((m - m_new) * kLog2e), w = ex2((s - m_new) * kLog2e);
    m = m_new;
    l = l * alpha + w;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (const int d = lane + 32 * i; d < p.D) o[i] = o[i] * alpha + w * static_cast<float>(v[d]);
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += kWarps * 32) {
    float top = -INFINITY, sum = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarps; ++w) {
      // (a stretch without a key counts for nothing; one whose scores are all NaN has a NaN sum, which stays)
      const float f = s_m[w] == -INFINITY ? (s_l[w] == 0.f ? 0.f : 1.f) : ex2((s_m[w] - top) * kLog2e);
      sum += f * s_l[w];
      acc += f * s_o[w][d];
    }
    static_cast<T*>(p.o)[b * p.o_sB + h * p.o_sH + d] = static_cast<T>(sum == 0.f ? 0.f : acc / sum);
  }
}

template <typename T>
int launch_typed(const PagedParams& d, int bias_kind, int64_t blocks, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (bias_kind) {
    case FA_BIAS_NONE: return launch_overlapped(paged_kernel<T, 0>, grid, kWarps * 32, 0, stream, d);
    case FA_BIAS_SAME: return launch_overlapped(paged_kernel<T, 1>, grid, kWarps * 32, 0, stream, d);
    case FA_BIAS_BOOL: return launch_overlapped(paged_kernel<T, 2>, grid, kWarps * 32, 0, stream, d);
    default: return launch_overlapped(paged_kernel<T, 3>, grid, kWarps * 32, 0, stream, d);
  }
}

}  // namespace

uint64_t paged_workspace_bytes(const fa_paged_params&) { return 0; }

int launch_paged(const fa_paged_params& p, void*, cudaStream_t stream, int* status) {
  PagedParams d;
  d.q = p.q, d.k = p.k_cache, d.v = p.v_cache, d.bias = p.bias, d.o = p.o;
  d.table = p.block_table, d.lens = p.seq_lens, d.status = status;
  d.q_sB = p.q_stride[0], d.q_sH = p.q_stride[1], d.o_sB = p.o_stride[0], d.o_sH = p.o_stride[1];
  d.k_sP = p.k_stride[0], d.k_sT = p.k_stride[1], d.k_sH = p.k_stride[2];
  d.v_sP = p.v_stride[0], d.v_sT = p.v_stride[1], d.v_sH = p.v_stride[2];
  d.bias_sB = p.bias_stride[0], d.bias_sH = p.bias_stride[1], d.table_s = p.table_stride;
  d.H = p.H, d.group = p.H / p.Hkv, d.D = p.D, d.page_size = p.page_size, d.num_pages = p.num_pages, d.width = p.width;
  d.sm_scale = p.sm_scale;
  const int64_t blocks = static_cast<int64_t>(p.B) * p.H;
  return p.dtype == FA_BF16 ? launch_typed<__nv_bfloat16>(d, p.bias_kind, blocks, stream)
                            : launch_typed<__half>(d, p.bias_kind, blocks, stream);
}

}  // namespace fa
