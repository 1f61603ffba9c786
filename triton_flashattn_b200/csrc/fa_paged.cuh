// Attention of one new token a sequence over a paged key / value cache, on sm_100a.
//
//   s_n = sm_scale q . k_n + bias_n,   o = sum_n exp(s_n - m) v_n / sum_n exp(s_n - m)   over the keys n of the sequence,
// in one pass: a running maximum m, the sum and the weighted values of a stretch of keys are rescaled where m rises, and
// stretches are joined with the weights exp(m_i - m).
//
// What bounds it: the keys and values are read once and each takes part in a handful of products (one for each query head that
// shares it), so it is a stream from memory.  Each warp has a ring of tiles of 16 or 32 keys in shared memory that it fills itself,
// by tile copies where pages are whole boxes of 8 or 16 keys and else 16 bytes a lane, and empties with the warp-level matrix
// instruction: the heads that share a key head are the 8 or 16 columns of the product.  Its copies run ahead over the ends of
// sequences and heads, so the stream does not stop there.
//   tcgen05 would take the same products: 128 keys, or 128 elements of a value, as rows and 16 queries as columns.  Where the
// memory is the bound it has nothing to give (a tile's 32 products, at head dim 128 with up to 8 heads, keep the tensor pipe busy for a
// fifth of the time) and costs tiles of 128 keys and hand-offs between warps for each.  With 16 heads of 256 there are four warps,
// one a scheduler, each ready to issue in 15 % of the cycles: there the latency inside a tile is the bound, and tcgen05, or two
// warps a ring, could help.  Neither is built.
//
// Lengths are on the device and differ, and one long sequence must fill the SMs as well as thousands of short ones: the tiles of
// all sequences, in order, are one line, and each CTA takes an equal stretch of it with all key heads, a warp one head (or one
// head and a part of the stretch, or several).  So the warps of a CTA read neighbouring heads of the same tokens at the same
// time, which in a (page, token, head, element) cache are neighbours in memory.  A warp writes the sequences that lie whole in
// its stretch; of the others, at most two, it leaves the unfinished sums in the workspace, where a second kernel joins them in
// order.
//
// Measured, bf16, head dim 128, 32 query and 8 key heads, us (of the rate of a copy, 6453 GB/s):
//   64 sequences of 200 to 8192 keys 177 (1.07 GB, 0.94), one of 131072 91 (0.91), one of 20011 24 (0.52), one of 1000 8.3
// of which 5 pass before the first tile is there (lengths, pages, keys: one waits for the other) and 4 to 5 after the last one (the
// second kernel).  In a large call 24 of the 148 SMs take 15 % longer than the others for the same bytes.
//   What the forms before this one took, for the 64 sequences and the one of 20011: tiles in registers and one head a warp and
//   stretch 190, 26; a ring, one head a warp and stretch 186, 25.  Four times as many, smaller stretches than CTAs fit: 200; a sixth
//   of the line in small stretches for those who are done first: 180 to 188.
#pragma once

#include "fa_common.cuh"
#include "fa_host.cuh"
#include "fa_ring.h"

namespace fa {

struct PagedParams {
  CUtensorMap k_map, v_map;  // {D, Hkv, page_size, pages}, boxes of 64 elements and 8 or 16 tokens
  const void* q;
  const void* k;
  const void* v;
  const void* bias;
  void* o;
  const int* table;
  const int* lens;
  int* status;
  float* part;  // workspace: unfinished sums [stretch][2][unit][row]: of the sequence that began before, of the one that goes on
  int4* joint;  // workspace: a sequence that goes on: it (-1: none), the first and the last stretch that have some of it.  Null for
                // few sequences, where the joining kernel finds out itself, and where none goes on
  int64_t q_sB, q_sH, o_sB, o_sH, k_sP, k_sT, k_sH, v_sP, v_sT, v_sH, bias_sB, bias_sH, table_s;
  int B, H, Hkv, D;
  int page_size, num_pages, width, page_boxes;
  uint32_t div_mul, div_shift;        // division by the page size (in boxes where pages are whole boxes)
  uint32_t splits_mul, splits_shift;  // by `splits`
  int heads;   // query heads of a key head
  int rows;    // of them, those of a unit
  int splits;  // units of a key head
  int units;   // of a sequence
  int parts;   // stretches of a CTA
  int ring;    // tiles that a warp has room for
  int whole;   // stretches are whole sequences
  int ctas;    // of the first kernel
  int by_seq;  // joint has an entry for each sequence (else for each stretch: there are more sequences, so none is empty)
  int joints;  // entries of it
  int slices, teams;  // of a (sequence, head) in the joining kernel
  float scale;  // of the scores; in log2 units unless there is a float bias
};

// How a call is cut: rows a unit, units a key head, warps, their ring, the grid.
struct PagedPlan {
  int DP, NQ, rows, splits, units;
  int warps, ring, parts;
  int ctas, joints, slices, teams, ahead;
  bool whole, by_seq;
};
constexpr int kPagedSmem = 218 * 1024;  // shared memory for the warps' rooms

// An unfinished sum: per row DP values, their maximum and the sum of the weights (and two words to keep rows at 16 bytes).
__host__ __device__ constexpr int row_floats(int DP) { return DP + 4; }

// The kernels of a type and a kind of copies (boxes of 16 or 8 keys, or row by row), each in a translation unit of its own.
using PagedLaunch = int(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream);
PagedLaunch launch_paged_bf16, launch_paged_bf16_box8, launch_paged_bf16_rows;
PagedLaunch launch_paged_f16, launch_paged_f16_box8, launch_paged_f16_rows;

constexpr int kMostWarps = 8;
// Up to this many sequences a lane has one, and the places of the sequences are known without tables.
constexpr int kFew = 32;
constexpr int kJoinThreads = 256;

namespace {

constexpr int kKernelId = 20;  // in the status word

__device__ __forceinline__ void ldsm_x4(uint32_t (&a)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&a)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tma_load_4d_to(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// An arrival on the barrier once all copies that this thread has asked for so far have landed.
__device__ __forceinline__ void arrive_when_landed(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Pack2<T>::kIsBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Two 16-bit values with those that are infinite or NaN (all exponent bits set) replaced by 0.
template <typename T>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
  constexpr uint32_t kExp = Pack2<T>::kIsBf16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t kOne = Pack2<T>::kIsBf16 ? 0x00800080u : 0x04000400u;
  const uint32_t bad = (((w & kExp) + kOne) & 0x80008000u) >> 15;
  return w & ~(bad * 0xffffu);
}

// x / d for the divisor that `mul` and `shift` stand for (x below 2^31).
__device__ __forceinline__ int fast_div(int x, uint32_t mul, uint32_t shift) {
  return static_cast<int>((__umulhi(static_cast<uint32_t>(x), mul) + static_cast<uint32_t>(x)) >> shift);
}
// Quotients where both fit 32 bits, as they nearly always do.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
  return (x | y) >> 32 ? x / y : static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y));
}

// Scores are in log2 units, except with a float bias: the lowest number of its type, times log2 e, would be -inf.
template <int BIAS>
constexpr bool kNatural = BIAS == 1 || BIAS == 3;
template <int BIAS>
__device__ __forceinline__ float weight(float s, float m) {
  return ex2(kNatural<BIAS> ? (s - m) * kLog2e : s - m);
}
// How far a score may rise above the running maximum before that moves; and the power of two that all weights of a call, and
// their sums with them, are multiplied with.  fp16 ends at 2^16 and its steps at 2^-24: with weights up to 2^8 a factor of 2^7 is
// the most, and then a weight is kept, in its two terms, down to 2^-32 of the largest one and not to 2^-25 (65536 keys 17.9 below
// one more, in 5 stretches: the share of the stretch with that one, 1/5 of what they add up to, was lost).  The range of bf16 is
// that of fp32.
template <int BIAS, typename T>
constexpr float kRise = kNatural<BIAS> && !Pack2<T>::kIsBf16 ? 8 / kLog2e : 8;
template <typename T>
constexpr float kLift = Pack2<T>::kIsBf16 ? 0 : 7;
template <int BIAS, typename T>
__device__ __forceinline__ float lifted_weight(float s, float m) {
  if constexpr (Pack2<T>::kIsBf16) return weight<BIAS>(s, m);
  // (added to the difference: to m, which may be large, it would be rounded, to something else for each m)
  return ex2(kNatural<BIAS> ? fmaf(s - m, kLog2e, kLift<T>) : s - m + kLift<T>);
}
// What a stretch with maximum m counts beside one with m_all >= m; 0 where it has no key (its sums are zero then, or NaN, which
// stays).
template <int BIAS>
__device__ __forceinline__ float weight_of(float m, float m_all) {
  return m == -INFINITY ? 0.f : weight<BIAS>(m, m_all);
}
// What the sums are multiplied with in the end: 0 without a key; and where the sum is NaN, as those it belongs to then are.
__device__ __forceinline__ float inverse(float m, float sum) { return m != -INFINITY && sum > 0.f ? 1.f / sum : 0.f; }

// An element of a bias or mask as it lies in memory, and what it stands for.  (Loaded into whole registers: nothing waits for it
// before it is used.)
template <int BIAS>
constexpr int kBiasBytes = BIAS == 2 ? 1 : BIAS == 3 ? 4 : 2;
template <int BIAS>
__device__ __forceinline__ uint32_t load_bias(const void* p) {
  uint32_t x;
  if constexpr (BIAS == 2) asm volatile("ld.global.u8 %0, [%1];" : "=r"(x) : "l"(p));
  else if constexpr (BIAS == 3) asm volatile("ld.global.u32 %0, [%1];" : "=r"(x) : "l"(p));
  else asm volatile("ld.global.u16 %0, [%1];" : "=r"(x) : "l"(p));
  return x;
}
template <int BIAS, typename T>
__device__ __forceinline__ float bias_of(uint32_t x) {
  return BIAS == 3 ? __uint_as_float(x) : Pack2<T>::unpack(x).x;
}

// Shared memory of a kernel.  DP: head dim rounded up to 64, 128, 256; NQ: groups of 8 rows.  Tiles of 32 keys at DP 64: a tile
// costs a warp 1000 cycles whatever its width (waits, votes, the maximum), as much as 4 KB take of the memory rate.
template <int DP, int NQ>
struct Cfg {
  static constexpr int kPieces = DP == 64 ? 2 : 1;  // of 16 keys, in a tile: what a warp waits for and works on at once
  static constexpr int kKeys = 16 * kPieces;
  static constexpr int kPiece = 32 * DP;  // bytes of 16 keys of K or V: blocks of 64 elements, rows of 128 bytes, swizzled
  static constexpr int kTile = kPieces * kPiece;
  static constexpr int kQ = 8 * NQ * DP * 2;            // the queries
  static constexpr bool kQRegs = NQ == 1 && DP <= 128;  // are kept in registers over a sequence
  static constexpr int warp_bytes(int ring) { return (2 * ring * kTile + kQ + 1023) / 1024 * 1024; }
};

// The line of tiles, and how the CTAs, and the parts of their stretches, share it.
struct Line {
  int64_t tiles, share;
  int ctas, longer;  // the first `longer` CTAs take one tile more than `share`
  __device__ __forceinline__ Line(int64_t tiles, int most) : tiles(tiles) {
    ctas = static_cast<int>(min(static_cast<int64_t>(most), tiles));
    share = divide(tiles, ctas);
    longer = static_cast<int>(tiles - share * ctas);
  }
  __device__ __forceinline__ int64_t begin(int cta) const { return cta * share + min(cta, longer); }
  __device__ __forceinline__ int cta_of(int64_t x) const {
    const int64_t turn = longer * (share + 1);
    return static_cast<int>(x < turn ? divide(x, share + 1) : longer + divide(x - turn, share));
  }
  // The stretch that place x is in.
  __device__ __forceinline__ int stretch_of(int64_t x, int parts) const {
    const int cta = cta_of(x);
    if (parts == 1) return cta;
    const int64_t from = begin(cta);
    return cta * parts + static_cast<int>(divide((x - from + 1) * parts - 1, begin(cta + 1) - from));
  }
};

// The running sum over the lanes of a warp.
__device__ __forceinline__ int64_t warp_scan(int64_t x) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, off);
    if (static_cast<int>(threadIdx.x & 31) >= off) x += y;
  }
  return x;
}
// Keys of sequence b, and their tiles.  (An empty sequence has a tile, as it has its zeros to write.)
__device__ __forceinline__ int length_of(const PagedParams& p, int b) {
  return min(max(__ldcg(p.lens + b), 0), p.width * p.page_size);
}
template <int KEYS>
__device__ __forceinline__ int tiles_in(int len) {
  return max((len + KEYS - 1) / KEYS, 1);
}

template <int DP, int NQ, typename T, int BIAS, int BOX>
__global__ void __launch_bounds__(kMostWarps * 32, 1) paged_kernel(const __grid_constant__ PagedParams p) {
  using P2 = Pack2<T>;
  using C = Cfg<DP, NQ>;
  constexpr int KS = DP / 16;  // steps of 16 head-dim elements
  constexpr bool TILES = BOX > 0;
  constexpr int kBoxes = TILES ? C::kKeys / BOX : 1;  // of a tile
  constexpr int MB = C::kPieces, kMostRing = 8;
  constexpr int kMostThreads = kMostWarps * 32;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[kMostWarps][kMostRing];  // K and V of a ring place have landed
  __shared__ __align__(8) uint64_t s_q_full[kMostWarps];           // the next queries have
  // of the tile there: its keys that exist; 1 the last of its sequence, 2 of the item; the sequence's tiles
  __shared__ __align__(16) uint4 s_info[kMostWarps][kMostRing];
  __shared__ int64_t s_before[kMostThreads + 1];   // tiles of the sequences before a thread's
  __shared__ int64_t s_sum[kMostWarps];
  __shared__ int s_abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5, threads = blockDim.x;
  const int r = lane >> 2, t = lane & 3;
  const int cap = p.width * p.page_size, S = p.ring, units = p.units;
  if (TILES && tid == 0) {
    tma_prefetch_desc(&p.k_map);
    tma_prefetch_desc(&p.v_map);
  }

  // ---- this warp's room: a ring of tiles of K, one of V, queries
  const int warp_bytes = C::warp_bytes(S);
  uint8_t* const room = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023) + warp * warp_bytes;
  const uint32_t ring = smem_u32(room), q_room = ring + 2 * S * C::kTile;
  uint64_t(&full)[kMostRing] = s_full[warp];
  if (lane < S) mbar_init(&full[lane], TILES ? 1 : 32);
  if (lane == 0) mbar_init(&s_q_full[warp], 32);
  // What no copy writes is read all the same, times 0: columns behind the head dim, rows of queries that the unit has not, keys
  // behind the last one or on no page.  (What an earlier tile left is as good as zeros; an infinite or NaN value would be put right, slowly.)
  {
    const int from = kBoxes == 1 && TILES ? 2 * S * C::kTile : 0;
    for (int i = from / 16 + lane; i < (2 * S * C::kTile + C::kQ) / 16; i += 32)
      reinterpret_cast<uint4*>(room)[i] = make_uint4(0, 0, 0, 0);
  }
  if (tid == 0) s_abort = 0;
  mbar_fence_init();
  fence_proxy_async_smem();

  // (For few sequences the joining kernel reads the lengths before this one has ended, so it may start once whatever wrote them
  // has.)
  const bool late = !p.whole && !p.joint;
  if (!late) grid_dep_launch_next();
  grid_dep_wait();  // the previous kernel's results (and the status word) are visible from here
  if (late) grid_dep_launch_next();
  const int status = *reinterpret_cast<volatile int*>(p.status);
  const auto length = [&](int b) { return length_of(p, b); };
  const auto tiles_of = [&](int len) { return tiles_in<C::kKeys>(len); };

  // ---- the line.  Few sequences: a lane has one.  More: a thread has some, and a table what lies before.
  const bool few = p.B <= kFew;
  const int each = few ? 1 : (p.B + threads - 1) / threads;
  int64_t sum = 0;
  int len_l = 0;
  for (int b = (few ? lane : tid) * each, stop = min(b + each, p.B); b < stop; ++b) {
    len_l = length(b);
    sum += tiles_of(len_l);
  }
  const int64_t upto = warp_scan(sum);
  int64_t tiles = 0;
  if (few) {
    tiles = __shfl_sync(0xffffffffu, upto, 31);
    __syncthreads();  // s_abort
  } else {
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int64_t before = upto - sum;
    for (int w = 0; w < warps; ++w) {
      const int64_t x = s_sum[w];
      before += w < warp ? x : 0;
      tiles += x;
    }
    s_before[tid] = before;
    __syncthreads();
  }
  if (status != 0) return;
  const Line line(tiles, gridDim.x);
  const int me = blockIdx.x;
  if (me >= line.ctas) return;

  // A place on the line: a sequence and a tile of it.
  struct Place {
    int b, tile, len;
  };
  const auto locate = [&](int64_t x) {
    Place at;
    if (few) {
      at.b = __ffs(__ballot_sync(0xffffffffu, upto > x)) - 1;
      at.len = __shfl_sync(0xffffffffu, len_l, at.b);
      at.tile = static_cast<int>(x - __shfl_sync(0xffffffffu, upto - sum, at.b));
      return at;
    }
    int lo = 0, hi = threads;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_before[mid] <= x) lo = mid;
      else hi = mid;
    }
    int b = lo * each;
    int64_t before = s_before[lo];
    for (const int stop = min(b + each, p.B); b + 1 < stop;) {
      const int mine = b + lane < stop ? tiles_of(length(b + lane)) : 0;
      const int64_t sums = warp_scan(mine);
      const uint32_t beyond = __ballot_sync(0xffffffffu, before + sums > x);
      if (beyond) {
        const int k = __ffs(beyond) - 1;
        before += __shfl_sync(0xffffffffu, sums - mine, k);
        b += k;
        break;
      }
      before += __shfl_sync(0xffffffffu, sums, 31);
      b += 32;
    }
    at.b = b;
    at.len = length(b);
    at.tile = static_cast<int>(x - before);
    return at;
  };
  const auto begin_of = [&](int cta) {
    int64_t x = line.begin(cta);
    if (p.whole && x < line.tiles)
      if (const Place at = locate(x); at.tile > 0) x += tiles_of(at.len) - at.tile;
    return x;
  };
  const int64_t cta_first = begin_of(me), cta_tiles = begin_of(me + 1) - cta_first;

  // ---- this warp's items: a unit over a part of the stretch.  Items part * units + unit; warp w has w, w + warps, ...
  struct Item {
    int unit, part;
    int64_t first, tiles;
  };
  const int n_items = units * p.parts;
  const auto item_at = [&](int i) {
    Item x;
    x.part = i / units;
    x.unit = i - x.part * units;
    const int64_t from = divide(cta_tiles * x.part, p.parts);
    x.first = cta_first + from;
    x.tiles = divide(cta_tiles * (x.part + 1), p.parts) - from;
    return x;
  };
  const int64_t part_rows = static_cast<int64_t>(units) * p.rows * row_floats(DP);  // floats of a stretch and place
  const auto part_at = [&](int stretch, int place, int unit) {
    return p.part + (2 * static_cast<int64_t>(stretch) + place) * part_rows + static_cast<int64_t>(unit) * p.rows * row_floats(DP);
  };

  // ---- the copies, ahead of the products.  Pages: lane l knows that of the 16 keys (TILES; else of the key) number l of the
  // batch that begins at tile `batch` of sequence i_b, and the same of the batch after that.
  constexpr int kBatch = TILES ? 32 / kBoxes : 1;  // tiles
  const auto fetch_pages = [&](int b, int tile) {
    const int what = TILES ? tile * kBoxes + lane : tile * C::kKeys + (lane & (C::kKeys - 1));
    const int at_page = fast_div(what, p.div_mul, p.div_shift);
    return b < p.B && at_page < p.width ? __ldcg(p.table + b * p.table_s + at_page) : -1;
  };
  // (looked at only when it is needed: nothing waits for a batch that is fetched ahead)
  const auto in_cache = [&](int id) { return id >= 0 && id < p.num_pages ? id : -1; };
  int i_item = warp, i_unit = 0, i_head = 0;  // of the next tile to be copied: its item, ...
  int64_t i_left = 0;                         // tiles of the item that are not copied yet, it among them
  int i_b = 0, i_tile = 0, i_len = 0, i_tiles = 0;
  int batch = 0, page_l = -1, next_batch = 0, next_page = -1, next_len = 0;
  const auto fetch_next = [&] {  // the batch after the one at `batch`: of this sequence or the next
    next_batch = batch + kBatch;
    if (next_batch >= i_tiles) {
      next_batch = 0;
      next_len = i_b + 1 < p.B ? __ldcg(p.lens + i_b + 1) : 0;
    }
    next_page = fetch_pages(next_batch ? i_b : i_b + 1, next_batch);
  };
  Place start = {};    // where the items of part start_part begin
  int start_part = -1;
  const auto start_of = [&](const Item& x) {
    if (x.part != start_part) start = locate(x.first), start_part = x.part;
    return start;
  };
  // To the first tile of the next item that has one, from i_item on; an empty one says so to the kernel that joins.
  const auto open_item = [&] {
    for (; i_item < n_items; i_item += warps) {
      const Item x = item_at(i_item);
      if (x.tiles > 0) {
        const Place at = start_of(x);
        i_unit = x.unit, i_left = x.tiles;
        i_head = fast_div(i_unit, p.splits_mul, p.splits_shift);
        i_b = at.b, i_tile = at.tile, i_len = at.len, i_tiles = tiles_of(at.len);
        batch = i_tile / kBatch * kBatch;
        page_l = in_cache(fetch_pages(i_b, batch));
        fetch_next();
        return;
      }
      if (!p.whole && lane < p.rows)
        *reinterpret_cast<float2*>(part_at(me * p.parts + x.part, 0, x.unit) + lane * row_floats(DP) + DP) = make_float2(-INFINITY, 0.f);
    }
  };
  open_item();

  // The next tile: its key head, pages and first rows there (TILES: of each piece; else of the lane's key), its keys, and whether
  // it is the last one.
  int t_head = 0, t_page[kBoxes], t_row[kBoxes];
  uint32_t t_keys = 0, t_last = 0, t_tiles = 0;
  int t_rows = 0;      // with a bias: rows of its unit,
  int64_t t_bias = 0;  // and where theirs begins
  const auto turn_to_next = [&] {
    if (i_tile - batch >= kBatch || i_tile < batch) {
      batch = next_batch, page_l = in_cache(next_page);
      fetch_next();
    }
    t_head = i_head;
    const int behind = i_len - i_tile * C::kKeys;
    t_keys = behind >= C::kKeys ? 0xffffffffu >> (32 - C::kKeys) : (1u << max(behind, 0)) - 1u;
    if constexpr (TILES) {
#pragma unroll
      for (int i = 0; i < kBoxes; ++i) {
        const int box = i_tile * kBoxes + i;
        t_page[i] = __shfl_sync(0xffffffffu, page_l, box - batch * kBoxes);
        t_row[i] = (box - fast_div(box, p.div_mul, p.div_shift) * p.page_boxes) * BOX;
        if (t_page[i] < 0) t_keys &= ~(0xffffffffu >> (32 - BOX) << (BOX * i));
      }
    } else {
      const int key = i_tile * C::kKeys + (lane & (C::kKeys - 1));
      t_page[0] = page_l;
      t_row[0] = key - fast_div(key, p.div_mul, p.div_shift) * p.page_size;
      t_keys &= __ballot_sync(0xffffffffu, page_l >= 0);
    }
    t_tiles = i_tiles;
    t_last = (i_tile + 1 == i_tiles ? 1u : 0u) | (i_left == 1 ? 2u : 0u);
    if constexpr (BIAS != 0) {
      const int m0 = (i_unit - i_head * p.splits) * p.rows;
      t_rows = behind > 0 ? min(p.rows, p.heads - m0) : 0;
      t_bias = i_b * p.bias_sB + (i_head * p.heads + m0) * p.bias_sH + i_tile * C::kKeys;
    }
    ++i_tile;
    if (--i_left == 0) {
      i_item += warps;
      open_item();
    } else if (i_tile == i_tiles) {
      i_tile = 0;
      ++i_b;
      i_len = min(max(next_len, 0), cap);
      i_tiles = tiles_of(i_len);
      batch = -kBatch;  // of another sequence
    }
  };
  // Its keys and values into ring place `to`.
  const auto copy_tile = [&](int to) {
    const uint32_t k_dst = ring + to * C::kTile, v_dst = ring + (S + to) * C::kTile;
    if constexpr (TILES) {
      if (elect_one()) {
        s_info[warp][to] = make_uint4(t_keys, t_last, t_tiles, 0);
        // (a box without a key is left out: what lies there, finite or not, counts for nothing)
        int boxes = 1;
#pragma unroll
        for (int i = 1; i < kBoxes; ++i) boxes += t_keys >> (BOX * i) ? 1 : 0;
        mbar_expect_tx(&full[to], boxes * (2 * BOX * 2 * DP));
#pragma unroll
        for (int i = 0; i < kBoxes; ++i)
          if (i < boxes) {
            const uint32_t at = (i * BOX >> 4) * C::kPiece + (i * BOX & 15) * 128;
#pragma unroll
            for (int g = 0; g < DP / 64; ++g) {
              tma_load_4d_to(k_dst + at + g * 2048, &p.k_map, &full[to], g * 64, t_head, t_row[i], t_page[i]);
              tma_load_4d_to(v_dst + at + g * 2048, &p.v_map, &full[to], g * 64, t_head, t_row[i], t_page[i]);
            }
          }
      }
    } else {
      // 16 bytes a lane; a lane knows the addresses of its own key, and asks for those of the row that it copies from
      constexpr int kRow = DP / 8, kRows = 32 / kRow;  // pieces of a row, rows of a step
      if (lane == 0) s_info[warp][to] = make_uint4(t_keys, t_last, t_tiles, 0);
      const bool mine = t_keys >> lane & 1;
      const T* k_src = static_cast<const T*>(p.k) + (mine ? t_page[0] * p.k_sP + t_row[0] * p.k_sT : 0) + t_head * p.k_sH;
      const T* v_src = static_cast<const T*>(p.v) + (mine ? t_page[0] * p.v_sP + t_row[0] * p.v_sT : 0) + t_head * p.v_sH;
      const int c = lane % kRow;
#pragma unroll
      for (int i = 0; i < C::kKeys / kRows; ++i) {
        const int key = i * kRows + lane / kRow;
        const T* ks = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k_src), key));
        const T* vs = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v_src), key));
        const uint32_t at = (key >> 4) * C::kPiece + (c >> 3) * 2048 + (key & 15) * 128 + (((c & 7) ^ (key & 7)) << 4);
        if ((t_keys >> key & 1) && c * 8 < p.D) {
          copy16_async(k_dst + at, ks + c * 8);
          copy16_async(v_dst + at, vs + c * 8);
        }
      }
      arrive_when_landed(&full[to]);
    }
    __syncwarp();
  };
  // Its bias on the way to L2: a load a tile ahead would wait for memory.  (A row of a tile lies in one or two sectors.)
  const auto prefetch_bias = [&] {
    if constexpr (BIAS != 0) {
      if (lane < t_rows) {
        const char* src = static_cast<const char*>(p.bias) + (t_bias + lane * p.bias_sH) * kBiasBytes<BIAS>;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
      }
    }
  };
  // the queries of a unit into their room: 16-byte pieces, swizzled over the rows
  const auto fetch_q = [&](int b, int unit) {
    const int hk = fast_div(unit, p.splits_mul, p.splits_shift), m0 = (unit - hk * p.splits) * p.rows;
    const int rows = min(p.rows, p.heads - m0);
    const T* src = static_cast<const T*>(p.q) + b * p.q_sB + (hk * p.heads + m0) * p.q_sH;
#pragma unroll
    for (int i = lane; i < 8 * NQ * (DP / 8); i += 32) {
      const int m = i / (DP / 8), c = i % (DP / 8);
      if (m < rows && c * 8 < p.D) copy16_async(q_room + m * (2 * DP) + ((c ^ (m & 7)) << 4), src + m * p.q_sH + c * 8);
    }
    arrive_when_landed(&s_q_full[warp]);
  };

  // the item and the place on the line that the products are at
  int item = i_item;
  if (item >= n_items) return;
  int unit = i_unit, b = i_b, tile = i_tile;
  fetch_q(b, unit);
  __syncwarp();
  for (int i = 0; i < S && i_item < n_items; ++i) {
    turn_to_next();
    copy_tile(i);
    prefetch_bias();
  }

  // ---- the products
  const uint32_t lane_row = (lane >> 3 & 1) * 8 + (lane & 7);  // K: rows 0-7 and 8-15 of 16 elements, then those of the next
  const uint32_t lane_key = (lane >> 4) * 8 + (lane & 7);      // V: 8 elements and the next of keys 0-7, then of keys 8-15
  const uint32_t k_lane = lane_row * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_lane = lane_key * 128 + (((lane >> 3 & 1) ^ (lane & 7)) << 4);
  // elements 16 ks .. of the rows of a tile
  const auto step_at = [&](uint32_t tile_lane, int ks) { return (tile_lane ^ ((2 * ks & 7) << 4)) + (ks >> 2) * 2048; };
  // elements 32 j .. of the queries of a group: B operands of two steps
  const auto q_step = [&](int g, int j) {
    return q_room + (g * 8 + (lane & 7)) * (2 * DP) + (((4 * j + (lane >> 3)) ^ (lane & 7)) << 4);
  };

  const WaitCtx wait_ctx = {&s_abort, p.status, kKernelId};
  uint32_t q[C::kQRegs ? KS / 2 : 1][4];
  float o[NQ][KS][4];         // O^T: [query group][16 head-dim rows][fragment]
  float mx[NQ][2], l[NQ][2];  // of rows 2t, 2t+1: running maximum, this lane's part of the sum
  uint32_t bf[NQ][MB][4];     // bias of the next tile, as it lies in memory
  int h0 = 0, rows = 0;
  int64_t bias_bh = 0;
  const auto load_b = [&](int tile, uint32_t keys) {
    if constexpr (BIAS != 0) {
#pragma unroll
      for (int g = 0; g < NQ; ++g)
#pragma unroll
        for (int k = 0; k < MB; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = g * 8 + 2 * t + (i & 1), key = k * 16 + r + 8 * (i >> 1);
            if (m < rows && keys >> key & 1)
              bf[g][k][i] =
                  load_bias<BIAS>(static_cast<const char*>(p.bias) + (bias_bh + m * p.bias_sH + tile * C::kKeys + key) * kBiasBytes<BIAS>);
          }
    }
  };

  // What follows the sequence that the products are at, once its last tile is there: the next of the item, or the next item.
  int next_item = item, next_unit = unit, next_b = b + 1, next_tile = 0;
  const auto open_next = [&] {
    Item it;
    for (next_item = item + warps; next_item < n_items; next_item += warps) {
      it = item_at(next_item);
      if (it.tiles > 0) break;
    }
    if (next_item >= n_items) return;
    const Place at = start_of(it);
    next_unit = it.unit, next_b = at.b, next_tile = at.tile;
  };

  bool opens = true, begins = false;
  int place = 0;  // in the ring
  uint32_t phase = 0, q_phase = 0;
  int x = 0;  // tiles done
#pragma unroll 1
  while (true) {
    const uint4 info = s_info[warp][place];
    const uint32_t keys = info.x;
    const bool refill = i_item < n_items;
    if (refill) turn_to_next();
    if (opens) {
      const int hk = fast_div(unit, p.splits_mul, p.splits_shift), m0 = (unit - hk * p.splits) * p.rows;
      h0 = hk * p.heads + m0, rows = min(p.rows, p.heads - m0);
      bias_bh = b * p.bias_sB + h0 * p.bias_sH;
      begins = tile == 0;
      load_b(tile, keys);
      if (!wait_warp(&s_q_full[warp], q_phase, wait_ctx, 2, x)) break;
      q_phase ^= 1;
      if constexpr (C::kQRegs) {
#pragma unroll
        for (int j = 0; j < KS / 2; ++j) ldsm_x4(q[j], q_step(0, j));
      }
#pragma unroll
      for (int g = 0; g < NQ; ++g) {
        mx[g][0] = mx[g][1] = -INFINITY, l[g][0] = l[g][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[g][i][e] = 0.f;
      }
      opens = false;
    }
    // ---- S^T = K Q^T
    if (!wait_warp(&full[place], phase, wait_ctx, 1, x)) break;
    float s[NQ][MB][4];
    {
      const uint32_t k_tile = ring + place * C::kTile + k_lane;
      float s2[NQ][MB][4];  // (two chains of products)
#pragma unroll
      for (int g = 0; g < NQ; ++g)
#pragma unroll
        for (int k = 0; k < MB; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[g][k][e] = s2[g][k][e] = 0.f;
#pragma unroll
      for (int j = 0; j < KS / 2; ++j) {
        uint32_t a0[MB][4], a1[MB][4];
#pragma unroll
        for (int k = 0; k < MB; ++k) {
          ldsm_x4(a0[k], step_at(k_tile, 2 * j) + k * C::kPiece);
          ldsm_x4(a1[k], step_at(k_tile, 2 * j + 1) + k * C::kPiece);
        }
#pragma unroll
        for (int g = 0; g < NQ; ++g) {
          uint32_t y[4];
          if constexpr (C::kQRegs) y[0] = q[j][0], y[1] = q[j][1], y[2] = q[j][2], y[3] = q[j][3];
          else ldsm_x4(y, q_step(g, j));
#pragma unroll
          for (int k = 0; k < MB; ++k) {
            mma16816<T>(s[g][k], a0[k], y[0], y[1]);
            mma16816<T>(s2[g][k], a1[k], y[2], y[3]);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < NQ; ++g)
#pragma unroll
        for (int k = 0; k < MB; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[g][k][e] += s2[g][k][e];
    }
    if (info.y != 0) {  // the last tile of this sequence or item: the next queries may come
      __syncwarp();
      if (info.y >> 1) open_next();
      if (next_item < n_items) fetch_q(next_b, next_unit);
    }
    // ---- scores, -inf where a key takes no part
    bool need = false;
#pragma unroll
    for (int g = 0; g < NQ; ++g)
#pragma unroll
      for (int k = 0; k < MB; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = s[g][k][i] * p.scale;
          // a mask selects, and so does a bias of -inf: whatever the score of a key that is left out is (infinite, NaN), it takes
          // no part
          if constexpr (BIAS == 2) {
            y = bf[g][k][i] ? y : -INFINITY;
          } else if constexpr (BIAS != 0) {
            const float plus = bias_of<BIAS, T>(bf[g][k][i]);
            y = plus == -INFINITY ? -INFINITY : y + plus;
          }
          if (!(keys >> (k * 16 + r + 8 * (i >> 1)) & 1)) y = -INFINITY;
          s[g][k][i] = y;
          need = need || y - mx[g][i & 1] > kRise<BIAS, T>;  // (the difference that the weight is taken of)
        }
    if (BIAS != 0 && info.y == 0) load_b(tile + 1, s_info[warp][place + 1 == S ? 0 : place + 1].x);
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int g = 0; g < NQ; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float m_new = mx[g][j];
#pragma unroll
          for (int k = 0; k < MB; ++k) m_new = fmaxf(m_new, fmaxf(s[g][k][j], s[g][k][j + 2]));
          for (int off = 4; off < 32; off <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, off));
          const float alpha = m_new == -INFINITY ? 1.f : weight<BIAS>(mx[g][j], m_new);
          mx[g][j] = m_new;
          l[g][j] *= alpha;
#pragma unroll
          for (int i = 0; i < KS; ++i) o[g][i][j] *= alpha, o[g][i][j + 2] *= alpha;
        }
    }
    // Weights in two 16-bit terms, so that they lose 2^-17 (bf16) and not 2^-9: memory leaves the time for it.
    uint32_t hi[NQ][MB][2], lo[NQ][MB][2];
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
      const float m_0 = mx[g][0] == -INFINITY ? 0.f : mx[g][0], m_1 = mx[g][1] == -INFINITY ? 0.f : mx[g][1];
#pragma unroll
      for (int k = 0; k < MB; ++k) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = lifted_weight<BIAS, T>(s[g][k][i], i & 1 ? m_1 : m_0);
        l[g][0] += w[0] + w[2];
        l[g][1] += w[1] + w[3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t top = P2::pack(w[2 * i], w[2 * i + 1]);
          const float2 f = P2::unpack(top);
          hi[g][k][i] = transpose8x8(top);
          lo[g][k][i] = transpose8x8(P2::pack(w[2 * i] - f.x, w[2 * i + 1] - f.y));
        }
      }
    }
    // ---- O^T += V^T P^T
    // An infinite or NaN value: zero weights make it NaN.  So the values times zero are summed, and looked at.
    const uint32_t v_tile = ring + (S + place) * C::kTile + v_lane;
    float odd[4][4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd[c][e] = 0.f;
#pragma unroll
    for (int k = 0; k < MB; ++k)
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        uint32_t a[4];
        ldsm_x4_trans(a, step_at(v_tile, i) + k * C::kPiece);
        mma16816<T>(odd[i & 3], a, 0u, 0u);
      }
    if (__all_sync(0xffffffffu, (odd[0][0] + odd[1][0]) + (odd[2][0] + odd[3][0]) + ((odd[0][2] + odd[1][2]) + (odd[2][2] + odd[3][2])) == 0.f)) {
#pragma unroll
      for (int k = 0; k < MB; ++k)
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          uint32_t a[4];
          ldsm_x4_trans(a, step_at(v_tile, i) + k * C::kPiece);
#pragma unroll
          for (int g = 0; g < NQ; ++g) {
            mma16816<T>(o[g][i], a, hi[g][k][0], hi[g][k][1]);
            mma16816<T>(o[g][i], a, lo[g][k][0], lo[g][k][1]);
          }
        }
    } else {
      // Row by row of the queries: the values that its row leaves out as zeros, and without the infinite ones in the product
      // with the small terms (which may be 0, or of the other sign).  The same products in the same order otherwise.
#pragma unroll
      for (int k = 0; k < MB; ++k)
#pragma unroll
        for (int g = 0; g < NQ; ++g) {
          // lane 4 k' + t': key k' (+ 8) of the piece is left out by rows 2t', 2t' + 1
          const uint32_t out0 = __ballot_sync(0xffffffffu, s[g][k][0] == -INFINITY), out1 = __ballot_sync(0xffffffffu, s[g][k][1] == -INFINITY);
          const uint32_t out2 = __ballot_sync(0xffffffffu, s[g][k][2] == -INFINITY), out3 = __ballot_sync(0xffffffffu, s[g][k][3] == -INFINITY);
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            const uint32_t out_a = (c & 1 ? out1 : out0) >> (c >> 1), out_b = (c & 1 ? out3 : out2) >> (c >> 1);
            // halves of a word: keys 2t, 2t + 1 (+ 8)
            const uint32_t keep_a = (out_a >> (8 * t) & 1 ? 0u : 0xffffu) | (out_a >> (8 * t + 4) & 1 ? 0u : 0xffff0000u);
            const uint32_t keep_b = (out_b >> (8 * t) & 1 ? 0u : 0xffffu) | (out_b >> (8 * t + 4) & 1 ? 0u : 0xffff0000u);
            const bool even = t == c >> 1 && !(c & 1), uneven = t == c >> 1 && (c & 1);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              uint32_t a[4], f[4];
              ldsm_x4_trans(a, step_at(v_tile, i) + k * C::kPiece);
              a[0] &= keep_a, a[1] &= keep_a, a[2] &= keep_b, a[3] &= keep_b;
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = finite_or_zero<T>(a[e]);
              float y[4] = {o[g][i][0], o[g][i][1], o[g][i][2], o[g][i][3]};
              mma16816<T>(y, a, hi[g][k][0], hi[g][k][1]);
              mma16816<T>(y, f, lo[g][k][0], lo[g][k][1]);
              o[g][i][0] = even ? y[0] : o[g][i][0];
              o[g][i][1] = uneven ? y[1] : o[g][i][1];
              o[g][i][2] = even ? y[2] : o[g][i][2];
              o[g][i][3] = uneven ? y[3] : o[g][i][3];
            }
          }
        }
    }
    __syncwarp();
    if (refill) copy_tile(place), prefetch_bias();
    if (++place == S) place = 0, phase ^= 1;
    ++x, ++tile;
    if (info.y == 0) continue;

    // ---- the sequence, or what this item has of it
#pragma unroll
    for (int g = 0; g < NQ; ++g)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        for (int off = 4; off < 32; off <<= 1) l[g][j] += __shfl_xor_sync(0xffffffffu, l[g][j], off);
    const bool ends = info.y & 1;
    if (begins && ends) {
      // lane (r, t) has head-dim rows 16 i + r, + 8 of query rows 2t, 2t + 1; transposed: pairs of elements of query row r
#pragma unroll
      for (int g = 0; g < NQ; ++g) {
        const float i_0 = inverse(mx[g][0], l[g][0]), i_1 = inverse(mx[g][1], l[g][1]);
        T* dst = static_cast<T*>(p.o) + b * p.o_sB + (h0 + g * 8 + r) * p.o_sH + 2 * t;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const uint32_t w0 = transpose8x8(P2::pack(o[g][i][0] * i_0, o[g][i][1] * i_1));
          const uint32_t w1 = transpose8x8(P2::pack(o[g][i][2] * i_0, o[g][i][3] * i_1));
          if (g * 8 + r < rows && (DP > 64 || i * 16 < p.D)) {
            *reinterpret_cast<uint32_t*>(dst + i * 16) = w0;
            *reinterpret_cast<uint32_t*>(dst + i * 16 + 8) = w1;
          }
        }
      }
    } else {
      const int stretch = me * p.parts + item / units;
      float* part = part_at(stretch, begins ? 1 : 0, unit);
#pragma unroll
      for (int g = 0; g < NQ; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int m = g * 8 + 2 * t + j;
          if (m >= rows) continue;
          float* dst = part + m * row_floats(DP);
#pragma unroll
          for (int i = 0; i < KS; ++i) dst[i * 16 + r] = o[g][i][j], dst[i * 16 + 8 + r] = o[g][i][j + 2];
          if (r == 0) *reinterpret_cast<float2*>(dst + DP) = make_float2(mx[g][j], l[g][j]);
        }
    }
    if (p.joint && unit == 0 && lane == 0) {
      // the sequence that begins here: does it go on, and up to which stretch
      const int stretch = me * p.parts + item / units;
      if (begins && !ends) {
        const Item it = item_at(item);
        const int64_t last = it.first + it.tiles - tile + info.z - 1;  // its last tile on the line
        p.joint[p.by_seq ? b : stretch] = make_int4(b, stretch, line.stretch_of(last, p.parts), 0);
      } else if (p.by_seq ? begins : info.y >> 1) {
        p.joint[p.by_seq ? b : stretch] = make_int4(-1, 0, 0, 0);
      }
    }
    opens = true;
    if (next_item >= n_items) break;
    item = next_item, unit = next_unit, b = next_b, tile = next_tile;
    next_b = b + 1, next_tile = 0;
  }
  copies_landed();
  if (s_abort) {  // a copy never came: those that are still under way are waited for in their order, all together 0.1 s at most
    const uint64_t t0 = global_timer_ns();
#pragma unroll 1
    for (int j = 0; j < S; ++j) {
      const int i = place + j < S ? place + j : place + j - S;
      while (!mbar_try_wait(&full[i], ring_phase(i, place, phase)))
        if (global_timer_ns() - t0 > 100000000ull) return;
    }
  }
}

// Joins the sums of the sequences that go on.  A team of threads, four values each, adds up sums of a slice of a (sequence, head);
// where there are many sums, they are dealt out to teams, and where there are few heads, these to slices.  What bounds it is
// latency: 148 sums of 32 heads take 4 us from the first kernel's end, 1 of them before it sees that end, 1.5 for the loads; 64
// sequences of 2 to 6 sums 2 to 4.  With a block a sequence and row, its teams joined one by one, 8 and 7.
template <int DP, typename T, int BIAS, int AHEAD>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ PagedParams p) {
  __shared__ float4 s_acc[kJoinThreads / 32][32];
  __shared__ float2 s_ml[kJoinThreads / 32][32];
  const int tid = threadIdx.x, teams = p.teams, size = DP / 4 / p.slices;
  grid_dep_launch_next();
  const int team = tid / size, d0 = (tid - team * size) * 4, sub = team % teams;
  const int what = blockIdx.x * (kJoinThreads / (size * teams)) + team / teams;
  const int head = what / p.slices, d = (what - head * p.slices) * (DP / p.slices) + d0;
  const int which = head / p.H, h = head - which * p.H;
  const int hk = h / p.heads, split = (h - hk * p.heads) / p.rows;
  const int unit = hk * p.splits + split, m = h - hk * p.heads - split * p.rows;
  const int64_t step = 2ll * p.units * p.rows * row_floats(DP);  // from stretch to stretch
  const float* base = p.part + (static_cast<int64_t>(unit) * p.rows + m) * row_floats(DP);
  int4 joint = make_int4(-1, 0, 0, 0);
  if (!p.joint) {  // few sequences: by the lengths, while the sums are still being formed
    const int lane = tid & 31, n = lane < p.B ? tiles_in<DP == 64 ? 32 : 16>(length_of(p, lane)) : 0;
    const int64_t upto = warp_scan(n), tiles = __shfl_sync(0xffffffffu, upto, 31);
    const Line line(tiles, p.ctas);
    int from = 0, to = 0;
    if (lane < p.B) from = line.stretch_of(upto - n, p.parts), to = line.stretch_of(upto - 1, p.parts);
    joint = make_int4(which, __shfl_sync(0xffffffffu, from, which & 31), __shfl_sync(0xffffffffu, to, which & 31), 0);
    if (which >= p.joints || joint.y == joint.z) joint.x = -1;
  }
  grid_dep_wait();
  const int status = *reinterpret_cast<volatile int*>(p.status);
  if (p.joint && which < p.joints) joint = __ldcg(p.joint + which);
  if (status != 0) return;
  base += joint.y * step;
  const int n = joint.x < 0 ? 0 : joint.z - joint.y + 1;
  // a team takes every `teams`-th sum, AHEAD of them under way
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = -INFINITY, sum = 0.f;
  for (int i0 = sub; i0 < n; i0 += AHEAD * teams) {
    float4 x[AHEAD];
    float2 ml[AHEAD];
    float m_new = top;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * teams;
      const float* src = base + i * step + (i == 0 ? step / 2 : 0);
      x[k] = i < n ? __ldcg(reinterpret_cast<const float4*>(src + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
      ml[k] = i < n ? __ldcg(reinterpret_cast<const float2*>(src + DP)) : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) m_new = fmaxf(m_new, ml[k].x);
    const float f = weight_of<BIAS>(top, m_new);
    top = m_new;
    // (sums that are NaN under a maximum of -inf stay: times 0)
    acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f, sum *= f;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;  // no key; of an empty stretch nothing else is written
      const float w = weight_of<BIAS>(ml[k].x, m_new);
      acc.x += w * x[k].x, acc.y += w * x[k].y, acc.z += w * x[k].z, acc.w += w * x[k].w;
      sum += w * ml[k].y;
    }
  }
  // the teams of a warp, then the warps
  const auto add = [&](float m_x, float l_x, float4 x) {
    const float m_new = fmaxf(top, m_x), f = weight_of<BIAS>(top, m_new), w = weight_of<BIAS>(m_x, m_new);
    acc.x = f * acc.x + w * x.x, acc.y = f * acc.y + w * x.y, acc.z = f * acc.z + w * x.z, acc.w = f * acc.w + w * x.w;
    sum = f * sum + w * l_x;
    top = m_new;
  };
  const int lane = tid & 31, warp = tid >> 5;
  for (int off = size; off < 32 && off < size * teams; off <<= 1) {
    const float m_x = __shfl_down_sync(0xffffffffu, top, off), l_x = __shfl_down_sync(0xffffffffu, sum, off);
    float4 x;
    x.x = __shfl_down_sync(0xffffffffu, acc.x, off), x.y = __shfl_down_sync(0xffffffffu, acc.y, off);
    x.z = __shfl_down_sync(0xffffffffu, acc.z, off), x.w = __shfl_down_sync(0xffffffffu, acc.w, off);
    add(m_x, l_x, x);
  }
  if (const int warps = size * teams / 32; warps > 1) {
    const int one = size < 32 ? size : 32;  // lanes of a warp that hold a result
    if (lane < one) s_acc[warp][lane] = acc, s_ml[warp][lane] = make_float2(top, sum);
    __syncthreads();
    // (teams wider than a warp lie a few warps apart)
    const int stride = size > 32 ? size / 32 : 1;
    if (sub == 0 && lane < one)
      for (int w = warp + stride; w < warp - warp % stride + warps && w / warps == warp / warps; w += stride)
        add(s_ml[w][lane].x, s_ml[w][lane].y, s_acc[w][lane]);
  }
  if (sub != 0) return;
  if (n == 0 || (DP == 64 && d >= p.D)) return;
  const float inv = inverse(top, sum);
  *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + joint.x * p.o_sB + h * p.o_sH + d) =
      make_uint2(Pack2<T>::pack(acc.x * inv, acc.y * inv), Pack2<T>::pack(acc.z * inv, acc.w * inv));
}

template <int DP, int NQ, typename T, int BIAS, int BOX>
int launch_inst(const PagedParams& d, const PagedPlan& x, cudaStream_t stream) {
  using C = Cfg<DP, NQ>;
  static std::atomic<uint64_t> ready{0};  // devices whose kernel has its shared memory
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return FA_ERR_CUDA;
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(paged_kernel<DP, NQ, T, BIAS, BOX>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPagedSmem + 1024) != cudaSuccess)
      return FA_ERR_CUDA;
    ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int smem = x.warps * C::warp_bytes(x.ring) + 1024;
  if (int e = launch_overlapped(paged_kernel<DP, NQ, T, BIAS, BOX>, dim3(x.ctas), x.warps * 32, smem, stream, d)) return e;
  if (x.whole) return FA_OK;
  const int per_block = kJoinThreads / (DP / 4 / x.slices * x.teams);
  const int64_t blocks = (static_cast<int64_t>(x.joints) * d.H * x.slices + per_block - 1) / per_block;
  return x.ahead == 4 ? launch_overlapped(join_kernel<DP, T, BIAS, 4>, dim3(static_cast<unsigned>(blocks)), kJoinThreads, 0, stream, d)
                      : launch_overlapped(join_kernel<DP, T, BIAS, 8>, dim3(static_cast<unsigned>(blocks)), kJoinThreads, 0, stream, d);
}

template <int DP, int NQ, typename T, int BOX>
int launch_bias(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  switch (bias_kind) {
    case FA_BIAS_NONE: return launch_inst<DP, NQ, T, FA_BIAS_NONE, BOX>(d, x, stream);
    case FA_BIAS_SAME: return launch_inst<DP, NQ, T, FA_BIAS_SAME, BOX>(d, x, stream);
    case FA_BIAS_BOOL: return launch_inst<DP, NQ, T, FA_BIAS_BOOL, BOX>(d, x, stream);
    default: return launch_inst<DP, NQ, T, FA_BIAS_F32, BOX>(d, x, stream);
  }
}
template <int DP, typename T, int BOX>
int launch_rows(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  if (x.NQ == 1) return launch_bias<DP, 1, T, BOX>(d, x, bias_kind, stream);
  return launch_bias<DP, 2, T, BOX>(d, x, bias_kind, stream);
}
template <typename T, int BOX>
int launch_paged_kernels(const PagedParams& d, const PagedPlan& x, int bias_kind, cudaStream_t stream) {
  return x.DP == 256   ? launch_rows<256, T, BOX>(d, x, bias_kind, stream)
         : x.DP == 128 ? launch_rows<128, T, BOX>(d, x, bias_kind, stream)
                       : launch_rows<64, T, BOX>(d, x, bias_kind, stream);
}

}  // namespace
}  // namespace fa
