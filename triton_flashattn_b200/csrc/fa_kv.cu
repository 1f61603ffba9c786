// Upkeep of a paged key / value cache: rows into its pages by a slot map, block tables and slot maps from request lengths, and
// the pages of finished requests back on the stack of free ones.
#include <cooperative_groups.h>

#include "fa_common.cuh"
#include "fa_host.cuh"

namespace fa {
namespace {

namespace cg = cooperative_groups;

// Division, rounded down, of x < 2^31 by 1 <= d < 2^31: with 2^(s - 1) < d <= 2^s it is (x + x * mul / 2^32) >> s,
// mul = 2^32 (2^s - d) / d + 1.
struct Divisor {
  uint32_t mul, shift;
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return (__umulhi(x, mul) + x) >> shift; }
};
Divisor divisor(uint64_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {static_cast<uint32_t>((((1ull << s) - d) << 32) / d + 1), s};
}

// ---- rows into the pages -----------------------------------------------------------------------
// A copy: what bounds it is the memory, read once, written once.  A thread moves 16 bytes of K and of V in kAhead places, and all its
// loads are under way before the first store.  16384 rows of 8 x 128 (134 MB): 22.5 us, 0.92 of a copy's rate; with one place a thread
// and 64-bit divisions 28.5.
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
  Divisor row, page;        // pieces of a token; tokens of a page
  int page_size, row_chunks, head_shift;  // 2^head_shift pieces of a head
};

constexpr int kWriteThreads = 256;
constexpr int kAhead = 4;

template <typename I>
__global__ void __launch_bounds__(kWriteThreads) kv_write_kernel(const WriteParams p) {
  grid_dep_launch_next();
  const I first = static_cast<I>(blockIdx.x) * (kWriteThreads * kAhead) + threadIdx.x;
  uint32_t token[kAhead], head[kAhead], d[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const I i = first + j * kWriteThreads;
    token[j] = sizeof(I) == 4 ? p.row.of(static_cast<uint32_t>(i)) : static_cast<uint32_t>(i / p.row_chunks);
    const uint32_t c = static_cast<uint32_t>(i - static_cast<I>(token[j]) * p.row_chunks);
    head[j] = c >> p.head_shift;
    d[j] = (c - (head[j] << p.head_shift)) * 8;
  }
  grid_dep_wait();
  const int status = *reinterpret_cast<volatile int*>(p.status);
  int64_t slot[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) slot[j] = first + j * kWriteThreads < static_cast<I>(p.chunks) ? __ldcg(p.slots + token[j]) : -1;
  if (status != 0) return;
  uint4 k[kAhead], v[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    if (slot[j] < 0 || slot[j] >= p.n_slots) continue;
    k[j] = __ldcg(reinterpret_cast<const uint4*>(p.k + token[j] * p.k_sT + head[j] * p.k_sH + d[j]));
    v[j] = __ldcg(reinterpret_cast<const uint4*>(p.v + token[j] * p.v_sT + head[j] * p.v_sH + d[j]));
  }
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    if (slot[j] < 0 || slot[j] >= p.n_slots) continue;
    const int64_t page = slot[j] >> 31 ? slot[j] / p.page_size : p.page.of(static_cast<uint32_t>(slot[j]));
    const int64_t at = slot[j] - page * p.page_size;
    *reinterpret_cast<uint4*>(p.k_cache + page * p.kc_sP + at * p.kc_sT + head[j] * p.kc_sH + d[j]) = k[j];
    *reinterpret_cast<uint4*>(p.v_cache + page * p.vc_sP + at * p.vc_sT + head[j] * p.vc_sH + d[j]) = v[j];
  }
}

// ---- tables ------------------------------------------------------------------------------------
// All CTAs of a call look at all requests, kThreads at a time, and have the same running sums; what is written (pages, slots) is
// shared out over their warps, a run of neighbours each, so that a lane looks for the request of its first one, and again only
// where its next one is another's.  Where lens_out is lens or count_out is count, the CTAs are one cluster, with a barrier between
// looking and writing.
// What bounds a call is latency: a launch, the lengths, the pages, the stores.  us in a captured graph, results apart / in place:
// 256 requests with a token each 5.1 / 5.1; prompts of 131 k tokens 7.1 / 18.0 (40 with a search for each token), of 1 M 17.7 / 97;
// 7 of 256 requests released 3.1 / 3.7, 131 k pages given back 5.3 / 12.7 (26).  In place, long lists wait for 8 CTAs where apart
// there are up to 64.
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
  int in_place;
  Divisor page;
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

__device__ __forceinline__ int64_t pages_of(int64_t tokens, const TableParams& p) {
  const int64_t x = tokens + p.page_size - 1;
  return x >> 31 ? x / p.page_size : p.page.of(static_cast<uint32_t>(x));
}

__device__ __forceinline__ void all_here(const TableParams& p) {
  if (p.in_place && gridDim.x > 1) cg::this_cluster().sync();
  else __syncthreads();
}

// What is between `from` and `to` (a list whose owners' first entries are in first[0 .. n - 1]) is dealt out to the warps of the
// call in runs, a lane an entry: into(owner, entry, *at(owner, entry)), where at() may be null (-1 then).  Four loads of a lane
// are under way at a time.
template <typename At, typename Into>
__device__ __forceinline__ void for_each(int64_t from, int64_t to, const int64_t* first, int n, At at, Into into) {
  constexpr int kAtOnce = 4;
  const int lane = threadIdx.x & 31;
  const int warp = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), warps = gridDim.x * (kThreads / 32);
  const int64_t run = ((to - from + warps - 1) / warps + 31) / 32 * 32;
  const int64_t begin = from + warp * run, end = min(begin + run, to);
  if (begin >= end) return;
  int owner = find(first, n, min(begin + lane, end - 1));
  int64_t next = owner + 1 < n ? first[owner + 1] : to;
  for (int64_t x0 = begin + lane; x0 < end; x0 += 32 * kAtOnce) {
    int owners[kAtOnce], value[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t x = x0 + 32 * j;
      if (x >= next && x < end) {
        owner += find(first + owner, n - owner, x);
        next = owner + 1 < n ? first[owner + 1] : to;
      }
      owners[j] = owner;
      const int* src = x < end ? at(owner, x) : nullptr;
      value[j] = src ? __ldcg(src) : -1;
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (x0 + 32 * j < end) into(owners[j], x0 + 32 * j, value[j]);
  }
}

__global__ void __launch_bounds__(kThreads) kv_extend_kernel(const TableParams p) {
  __shared__ int64_t sums[kThreads / 32];
  __shared__ int64_t s_off[kThreads], s_rank[kThreads];  // tokens, pages wanted before each request
  __shared__ int s_old[kThreads], s_have[kThreads];
  __shared__ uint8_t s_granted[kThreads];
  __shared__ int s_taken;
  const int tid = threadIdx.x;
  grid_dep_launch_next();
  if (tid == 0) s_taken = 0;
  grid_dep_wait();
  const int status = *reinterpret_cast<volatile int*>(p.status);
  const int64_t count = min(max(__ldcg(p.count), 0), p.capacity);
  int64_t tokens = 0, wanted = 0;  // of the requests looked at so far
  int taken = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid, n = min(kThreads, p.B - b0);
    const int raw = b < p.B ? __ldcg(p.lens + b) : 0, change = b < p.B ? __ldcg(p.change + b) : 0;
    if (status != 0) return;  // (the same for all CTAs)
    const int64_t old = max(raw, 0), more = max(change, 0);
    int64_t chunk_tokens, chunk_wanted;
    const int64_t off = tokens + scan(more, sums, &chunk_tokens);
    const bool fits = old + more <= static_cast<int64_t>(p.width) * p.page_size && off + more <= p.T;
    const int64_t have = pages_of(old, p), need = fits ? pages_of(old + more, p) - have : 0;
    const int64_t rank = wanted + scan(need, sums, &chunk_wanted);
    const bool granted = fits && (need == 0 || rank + need <= count);
    s_off[tid] = off;
    s_rank[tid] = rank;
    s_old[tid] = static_cast<int>(old);
    s_have[tid] = static_cast<int>(have);
    s_granted[tid] = granted;
    // granted requests take a run of pages from `wanted` on: behind the first that got none nobody gets any
    const int most = __reduce_max_sync(0xffffffffu, granted && need > 0 ? static_cast<int>(rank + need) : 0);
    if ((tid & 31) == 0 && most > 0) atomicMax(&s_taken, most);
    all_here(p);  // all have looked at these requests
    if (blockIdx.x == 0 && b < p.B) p.lens_out[b] = granted ? static_cast<int>(old + more) : raw;
    const int taken_now = s_taken;
    for_each(
        min(wanted, static_cast<int64_t>(taken_now)), taken_now, s_rank, n, [&](int, int64_t x) { return p.free_pages + (count - 1 - x); },
        [&](int i, int64_t x, int page) { p.table[(b0 + i) * p.table_stride + s_have[i] + (x - s_rank[i])] = page; });
    for_each(
        tokens, min(tokens + chunk_tokens, static_cast<int64_t>(p.T)), s_off, n,
        [&](int i, int64_t x) -> const int* {
          if (!s_granted[i]) return nullptr;
          const int at = static_cast<int>(p.page.of(static_cast<uint32_t>(s_old[i] + (x - s_off[i])))), have = s_have[i];
          return at < have ? p.table + (b0 + i) * p.table_stride + at : p.free_pages + (count - 1 - (s_rank[i] + at - have));
        },
        [&](int i, int64_t x, int page) {
          const uint32_t pos = static_cast<uint32_t>(s_old[i] + (x - s_off[i]));
          p.slots[x] = page < 0 ? -1 : static_cast<int64_t>(page) * p.page_size + (pos - p.page.of(pos) * p.page_size);
        });
    tokens += chunk_tokens;
    wanted += chunk_wanted;
    taken = taken_now;
    __syncthreads();  // the next requests' sums go over these
  }
  if (status != 0) return;
  const int64_t me = blockIdx.x * kThreads + tid, all = gridDim.x * kThreads;
  for (int64_t t = min(tokens, static_cast<int64_t>(p.T)) + me; t < p.T; t += all) p.slots[t] = -1;
  all_here(p);  // all have read the count
  if (me == 0) *p.count_out = static_cast<int>(count) - taken;
}

__global__ void __launch_bounds__(kThreads) kv_release_kernel(const TableParams p) {
  __shared__ int64_t sums[kThreads / 32];
  __shared__ int64_t s_rank[kThreads];
  const int tid = threadIdx.x;
  grid_dep_launch_next();
  grid_dep_wait();
  const int status = *reinterpret_cast<volatile int*>(p.status);
  int64_t top = min(max(__ldcg(p.count), 0), p.capacity);
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid, n = min(kThreads, p.B - b0);
    const int raw = b < p.B ? __ldcg(p.lens + b) : 0;
    const bool gone = b < p.B && __ldcg(p.finished + b) != 0;
    if (status != 0) return;
    const int64_t give = gone ? min(pages_of(max(raw, 0), p), static_cast<int64_t>(p.width)) : 0;
    int64_t chunk;
    s_rank[tid] = scan(give, sums, &chunk);
    all_here(p);
    if (blockIdx.x == 0 && b < p.B) p.lens_out[b] = gone ? 0 : raw;
    for_each(
        0, min(chunk, p.capacity - top), s_rank, n,
        [&](int i, int64_t x) { return p.table + (b0 + i) * p.table_stride + (x - s_rank[i]); },
        [&](int, int64_t x, int page) { p.free_pages[top + x] = page; });
    top = min(top + chunk, static_cast<int64_t>(p.capacity));
    __syncthreads();
  }
  if (status != 0) return;
  all_here(p);
  if (blockIdx.x == 0 && tid == 0) *p.count_out = static_cast<int>(top);
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
  t.page = divisor(p.page_size);
  t.in_place = p.lens_out == p.lens || p.count_out == p.count;
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
  w.page_size = p.page_size;
  for (w.head_shift = 1; 8 << w.head_shift < p.D;) ++w.head_shift;
  const int64_t row_chunks = static_cast<int64_t>(p.Hkv) << w.head_shift;
  if (row_chunks > INT32_MAX) return FA_ERR_TOO_LARGE;
  w.row_chunks = static_cast<int>(row_chunks);
  w.row = divisor(row_chunks), w.page = divisor(p.page_size);
  w.chunks = p.T * row_chunks;
  constexpr int kPerBlock = kWriteThreads * kAhead;
  const int64_t blocks = (w.chunks + kPerBlock - 1) / kPerBlock;
  if (blocks > INT32_MAX) return FA_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(blocks));
  return blocks * kPerBlock <= INT32_MAX ? launch_overlapped(kv_write_kernel<uint32_t>, grid, kWriteThreads, 0, stream, w)
                                         : launch_overlapped(kv_write_kernel<uint64_t>, grid, kWriteThreads, 0, stream, w);
}

// CTAs for so many entries: a run of 64 for each warp, as far as a cluster goes where one is needed.
static int table_ctas(int64_t entries, bool in_place) {
  const int64_t ctas = (entries + 64 * (kThreads / 32) - 1) / (64 * (kThreads / 32)), most = in_place ? 8 : 64;
  return static_cast<int>(ctas < 1 ? 1 : ctas < most ? ctas : most);
}

int launch_kv_extend(const fa_kv_table_params& p, cudaStream_t stream, int* status) {
  const TableParams t = table_params(p, status);
  const int ctas = table_ctas(p.T, t.in_place);
  return launch_overlapped(kv_extend_kernel, dim3(ctas), kThreads, 0, stream, t, t.in_place ? ctas : 1);
}

int launch_kv_release(const fa_kv_table_params& p, cudaStream_t stream, int* status) {
  const TableParams t = table_params(p, status);
  const int64_t pages = static_cast<int64_t>(p.B) * p.width;
  const int ctas = table_ctas(pages < p.capacity ? pages : p.capacity, t.in_place);
  return launch_overlapped(kv_release_kernel, dim3(ctas), kThreads, 0, stream, t, t.in_place ? ctas : 1);
}

}  // namespace fa
