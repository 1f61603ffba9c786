// Upkeep of a paged key / value cache: rows into its pages by a slot map, block tables and slot maps from request lengths, and
// the pages of finished requests back on the stack of free ones.
#include <cooperative_groups.h>

#include "fa_common.cuh"
#include "fa_host.cuh"

namespace fa {
namespace {

namespace cg = cooperative_groups;

// ---- rows into the pages -----------------------------------------------------------------------
struct WriteParams {
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* k_cache;
  uint16_t* v_cache;
  const int64_t* slots;
  int* status;
  int64_t k_sT, k_sH, v_sT, v_sH;
  int64_t kc_sP, kc_sT, kc_sH, vc_sP, vc_sT, vc_sH;
  int64_t n_slots, chunks;  // slots of the cache; 16-byte pieces of a tensor of rows
  int page_size, Hkv, per_head;
};

__global__ void __launch_bounds__(256) kv_write_kernel(const WriteParams p) {
  grid_dep_launch_next();
  grid_dep_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.chunks || *reinterpret_cast<volatile int*>(p.status) != 0) return;
  const int64_t row = i / p.per_head;
  const int d = static_cast<int>(i - row * p.per_head) * 8;
  const int64_t t = row / p.Hkv;
  const int h = static_cast<int>(row - t * p.Hkv);
  const int64_t slot = __ldcg(p.slots + t);
  if (slot < 0 || slot >= p.n_slots) return;
  const int64_t page = slot / p.page_size;
  const int at = static_cast<int>(slot - page * p.page_size);
  const uint4 k = __ldcg(reinterpret_cast<const uint4*>(p.k + t * p.k_sT + h * p.k_sH + d));
  const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p.v + t * p.v_sT + h * p.v_sH + d));
  *reinterpret_cast<uint4*>(p.k_cache + page * p.kc_sP + at * p.kc_sT + h * p.kc_sH + d) = k;
  *reinterpret_cast<uint4*>(p.v_cache + page * p.vc_sP + at * p.vc_sT + h * p.vc_sH + d) = v;
}

// ---- tables ------------------------------------------------------------------------------------
// One cluster of CTAs does a call.  All of them look at all requests, kThreads at a time, and have the same running sums; what
// is written (pages, slots) is shared out over their threads.  The cluster barrier between looking and writing lets lens_out be
// lens and count_out be count.
constexpr int kThreads = 512;

struct TableParams {
  int32_t* table;
  const int32_t* lens;
  const int32_t* change;
  const uint8_t* finished;
  int32_t* free_pages;
  const int32_t* count;
  int32_t* lens_out;
  int32_t* count_out;
  int64_t* slots;
  int* status;
  int64_t table_stride;
  int B, width, page_size, capacity, T;
};

// Running sum of x over the threads of a CTA, x itself not included; *total is the sum of all.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* sums, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t y = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t z = __shfl_up_sync(0xffffffffu, y, off);
    if (lane >= off) y += z;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 31) sums[warp] = y;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int64_t s = sums[w];
    before += w < warp ? s : 0;
    all += s;
  }
  *total = all;
  return before + y - x;
}

// The last entry of first[0 .. n - 1], which does not fall, that is at most x (first[0] is).
__device__ __forceinline__ int find(const int64_t* first, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_size) { return (tokens + page_size - 1) / page_size; }

__global__ void __launch_bounds__(kThreads) kv_extend_kernel(const TableParams p) {
  __shared__ int64_t sums[kThreads / 32];
  __shared__ int64_t s_off[kThreads], s_rank[kThreads];  // tokens, pages wanted before each request
  __shared__ int s_old[kThreads];
  __shared__ uint8_t s_granted[kThreads];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const int me = blockIdx.x * kThreads + tid, all = gridDim.x * kThreads;
  grid_dep_launch_next();
  grid_dep_wait();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;  // (the same for all CTAs)
  const int64_t count = min(max(__ldcg(p.count), 0), p.capacity);
  int64_t tokens = 0, wanted = 0, taken = 0;  // of the requests looked at so far
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid, n = min(kThreads, p.B - b0);
    const int raw = b < p.B ? __ldcg(p.lens + b) : 0;
    const int64_t old = max(raw, 0), more = b < p.B ? max(__ldcg(p.change + b), 0) : 0;
    int64_t chunk_tokens, chunk_wanted, chunk_taken;
    const int64_t off = tokens + scan(more, sums, &chunk_tokens);
    const bool fits = old + more <= static_cast<int64_t>(p.width) * p.page_size && off + more <= p.T;
    const int64_t need = fits ? pages_of(old + more, p.page_size) - pages_of(old, p.page_size) : 0;
    const int64_t rank = wanted + scan(need, sums, &chunk_wanted);
    const bool granted = fits && (need == 0 || rank + need <= count);
    scan(granted ? need : 0, sums, &chunk_taken);
    s_off[tid] = off;
    s_rank[tid] = rank;
    s_old[tid] = static_cast<int>(old);
    s_granted[tid] = granted;
    cluster.sync();  // all have looked at these requests
    if (blockIdx.x == 0 && b < p.B) p.lens_out[b] = granted ? static_cast<int>(old + more) : raw;
    // granted requests take a run of pages from `wanted` on: behind the first that got none nobody gets any
    for (int64_t x = wanted + me; x < wanted + chunk_taken; x += all) {
      const int i = find(s_rank, n, x);
      const int64_t at = pages_of(s_old[i], p.page_size) + x - s_rank[i];
      p.table[(b0 + i) * p.table_stride + at] = __ldcg(p.free_pages + (count - 1 - x));
    }
    const int64_t end = min(tokens + chunk_tokens, static_cast<int64_t>(p.T));
    for (int64_t t = tokens + me; t < end; t += all) {
      const int i = find(s_off, n, t);
      int64_t slot = -1;
      if (s_granted[i]) {
        const int64_t pos = s_old[i] + t - s_off[i], at = pos / p.page_size, have = pages_of(s_old[i], p.page_size);
        const int page = at < have ? __ldcg(p.table + (b0 + i) * p.table_stride + at)
                                   : __ldcg(p.free_pages + (count - 1 - (s_rank[i] + at - have)));
        if (page >= 0) slot = static_cast<int64_t>(page) * p.page_size + pos % p.page_size;
      }
      p.slots[t] = slot;
    }
    tokens += chunk_tokens;
    wanted += chunk_wanted;
    taken += chunk_taken;
    __syncthreads();  // the next requests' sums go over these
  }
  for (int64_t t = min(tokens, static_cast<int64_t>(p.T)) + me; t < p.T; t += all) p.slots[t] = -1;
  cluster.sync();  // all have read the count
  if (me == 0) *p.count_out = static_cast<int>(count - taken);
}

__global__ void __launch_bounds__(kThreads) kv_release_kernel(const TableParams p) {
  __shared__ int64_t sums[kThreads / 32];
  __shared__ int64_t s_rank[kThreads];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const int me = blockIdx.x * kThreads + tid, all = gridDim.x * kThreads;
  grid_dep_launch_next();
  grid_dep_wait();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  int64_t top = min(max(__ldcg(p.count), 0), p.capacity);
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid, n = min(kThreads, p.B - b0);
    const int raw = b < p.B ? __ldcg(p.lens + b) : 0;
    const bool gone = b < p.B && __ldcg(p.finished + b) != 0;
    const int64_t give = gone ? min(pages_of(max(raw, 0), p.page_size), static_cast<int64_t>(p.width)) : 0;
    int64_t chunk;
    s_rank[tid] = scan(give, sums, &chunk);
    cluster.sync();
    if (blockIdx.x == 0 && b < p.B) p.lens_out[b] = gone ? 0 : raw;
    const int64_t end = min(chunk, p.capacity - top);
    for (int64_t x = me; x < end; x += all) {
      const int i = find(s_rank, n, x);
      p.free_pages[top + x] = __ldcg(p.table + (b0 + i) * p.table_stride + (x - s_rank[i]));
    }
    top = min(top + chunk, static_cast<int64_t>(p.capacity));
    __syncthreads();
  }
  cluster.sync();
  if (me == 0) *p.count_out = static_cast<int>(top);
}

TableParams table_params(const fa_kv_table_params& p, int* status) {
  TableParams t;
  t.table = p.block_table;
  t.lens = p.lens;
  t.change = p.change;
  t.finished = p.finished;
  t.free_pages = p.free_pages;
  t.count = p.count;
  t.lens_out = p.lens_out;
  t.count_out = p.count_out;
  t.slots = p.slots;
  t.status = status;
  t.table_stride = p.table_stride;
  t.B = p.B, t.width = p.width, t.page_size = p.page_size, t.capacity = p.capacity, t.T = p.T;
  return t;
}

}  // namespace

int launch_kv_write(const fa_kv_write_params& p, cudaStream_t stream, int* status) {
  WriteParams w;
  w.k = static_cast<const uint16_t*>(p.k);
  w.v = static_cast<const uint16_t*>(p.v);
  w.k_cache = static_cast<uint16_t*>(p.k_cache);
  w.v_cache = static_cast<uint16_t*>(p.v_cache);
  w.slots = p.slots;
  w.status = status;
  w.k_sT = p.k_stride[0], w.k_sH = p.k_stride[1], w.v_sT = p.v_stride[0], w.v_sH = p.v_stride[1];
  w.kc_sP = p.k_cache_stride[0], w.kc_sT = p.k_cache_stride[1], w.kc_sH = p.k_cache_stride[2];
  w.vc_sP = p.v_cache_stride[0], w.vc_sT = p.v_cache_stride[1], w.vc_sH = p.v_cache_stride[2];
  w.n_slots = static_cast<int64_t>(p.num_pages) * p.page_size;
  w.page_size = p.page_size, w.Hkv = p.Hkv, w.per_head = p.D / 8;
  w.chunks = static_cast<int64_t>(p.T) * p.Hkv * w.per_head;
  const int64_t blocks = (w.chunks + 255) / 256;
  if (blocks > INT32_MAX) return FA_ERR_TOO_LARGE;
  return launch_overlapped(kv_write_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, w);
}

int launch_kv_extend(const fa_kv_table_params& p, cudaStream_t stream, int* status) {
  const int ctas = p.T <= 4 * kThreads ? 1 : 8;
  return launch_overlapped(kv_extend_kernel, dim3(ctas), kThreads, 0, stream, table_params(p, status), ctas);
}

int launch_kv_release(const fa_kv_table_params& p, cudaStream_t stream, int* status) {
  const int ctas = static_cast<int64_t>(p.B) * p.width <= 4 * kThreads ? 1 : 8;
  return launch_overlapped(kv_release_kernel, dim3(ctas), kThreads, 0, stream, table_params(p, status), ctas);
}

}  // namespace fa
