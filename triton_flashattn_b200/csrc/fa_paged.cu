// Attention of one new token a sequence over a paged key / value cache, on sm_100a.
//
//   s_n = sm_scale q . k_n + bias_n,   o = sum_n exp(s_n - m) v_n / sum_n exp(s_n - m)   over the keys n of the sequence,
// in one pass: a running maximum m, the sum and the weighted values of a stretch of keys are rescaled where m rises, and
// stretches are joined with the weights exp(m_i - m).
//
// What bounds it: the keys and values are read once and each takes part in a handful of products (one for each query head that
// shares it), so it is a stream from memory.  As in the forward for few query rows, K and V go from global memory straight into
// registers in the layout of the warp-level matrix instruction, a tile of 16 keys ahead, with the heads that share a key head
// as the 8 (or 16) columns of the product.
//
// Lengths are on the device and differ, and few heads must fill the SMs as well as thousands: the tiles of all (sequence, key
// head) units, in order, are one line, and each CTA takes an equal stretch of it, each of its warps an equal stretch of that.
// A warp writes the units that lie whole in its stretch; of the others, at most two, it leaves the unfinished sums in shared
// memory, the CTA joins those of its warps, and what goes on in the next CTA goes to the workspace (at most two partial results
// a CTA, so the traffic for it does not grow with the batch), where a second kernel joins it, in order.
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
  float* part;  // workspace: partial results, two a CTA
  int4* joint;  // workspace, one a CTA: the unit that begins there and goes on, and where its parts are
  int64_t q_sB, q_sH, o_sB, o_sH, k_sP, k_sT, k_sH, v_sP, v_sT, v_sH, bias_sB, bias_sH, table_s;
  int B, H, Hkv, D;
  int page_size, num_pages, width;
  uint32_t div_mul, div_shift;  // division by the page size (in tiles where pages are whole tiles)
  int heads;     // query heads of a key head
  int rows;      // of them, those of a unit
  int splits;    // units of a key head
  int whole;     // CTAs take whole units
  float scale;   // of the scores; in log2 units unless there is a float bias
};

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// Tiles that a CTA takes at least, where there are fewer CTAs for it.
constexpr int kLeastTiles = 8;
// Sequences of at most this many tiles are not split over CTAs: one launch less.
constexpr int kWholeTiles = 16;

__device__ __forceinline__ uint4 ldg_stream(const void* ptr, bool ok) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (ok)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(ptr));
  return v;
}

template <typename T>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (Pack2<T>::kIsBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Scores are in log2 units, except with a float bias: the lowest number of its type, times log2 e, would be -inf.
template <int BIAS>
constexpr bool kNatural = BIAS == 1 || BIAS == 3;
template <int BIAS>
__device__ __forceinline__ float weight(float s, float m) {
  return ex2(kNatural<BIAS> ? (s - m) * kLog2e : s - m);
}
// What a stretch with maximum m counts beside one with m_all >= m; 0 where it has no key (its sums are zero then, or NaN, which
// stays).
template <int BIAS>
__device__ __forceinline__ float weight_of(float m, float m_all) {
  return m == -INFINITY ? 0.f : weight<BIAS>(m, m_all);
}
// The result from sums: 0 without a key; a NaN stays (its sum is NaN, and 0 times its accumulator).
__device__ __forceinline__ float finish(float acc, float inv) { return acc * inv; }
__device__ __forceinline__ float inverse(float m, float sum) { return m != -INFINITY && sum > 0.f ? 1.f / sum : 0.f; }

// Registers decide how many warps an SM holds: K and V of a tile are 2 DP / 4 of a thread's, the accumulators NQ DP / 4, and
// at head dim 256 all of that fits with the queries in shared memory.
constexpr int ctas_per_sm(int DP, int NQ) { return DP == 256 ? 2 : DP == 128 ? (NQ == 1 ? 3 : 2) : (NQ == 1 ? 5 : 4); }

// Shared memory of a partial result: per row DP sums, their maximum and the sum of the weights.
constexpr int part_floats(int DP, int rows) { return rows * (DP + 2); }

// DP: head dim rounded up to 64, 128, 256; NQ: groups of 8 rows; ALIGNED: pages are whole tiles.
template <int DP, int NQ, typename T, int BIAS, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(DP, NQ)) paged_kernel(const PagedParams p) {
  using P2 = Pack2<T>;
  constexpr int KG = DP / 32;  // 16-byte loads per lane and key row of K
  constexpr int VG = DP / 64;  // ... of V
  constexpr bool kQShared = DP == 256;

  extern __shared__ __align__(16) float smem[];  // [2 * kWarps] partial results
  __shared__ int64_t s_before[kThreads + 1];     // tiles of a key head in the sequences before a thread's
  __shared__ int64_t s_sum[kWarps];
  __shared__ int s_first;  // the unit that begins where the CTA does, or -1
  __shared__ int s_unit[2 * kWarps], s_ends[2 * kWarps];  // of a partial result: its unit (-1: none); 1 it begins there, 2 it ends
  __shared__ __align__(16) T s_q[kQShared ? kWarps * NQ * 8 * DP : 8];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, t = lane & 3;
  const int cap = p.width * p.page_size;
  const int units = p.Hkv * p.splits;  // of a sequence
  grid_dep_launch_next();
  grid_dep_wait();  // the previous kernel's results (and the status word) are visible from here
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;

  const auto length = [&](int b) { return min(max(__ldcg(p.lens + b), 0), cap); };
  const auto tiles_of = [&](int len) { return max((len + 15) >> 4, 1); };  // (an empty sequence has its zeros to write)

  // ---- the line of tiles
  const int each = (p.B + kThreads - 1) / kThreads;
  {
    int64_t sum = 0;
    for (int b = tid * each; b < min((tid + 1) * each, p.B); ++b) sum += tiles_of(length(b));
    int64_t upto = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += x;
    }
    if (lane == 31) s_sum[warp] = upto;
    if (tid < 2 * kWarps) s_unit[tid] = -1;
    __syncthreads();
    int64_t before = upto - sum;
#pragma unroll
    for (int w = 0; w < kWarps - 1; ++w) before += w < warp ? s_sum[w] : 0;
    s_before[tid] = before;
    if (tid == kThreads - 1) s_before[kThreads] = before + sum;
    __syncthreads();
  }
  const int64_t line = s_before[kThreads] * units;
  const int64_t wanted = (line + kLeastTiles - 1) / kLeastTiles;
  const int ctas = static_cast<int>(min(static_cast<int64_t>(gridDim.x), wanted));
  if (static_cast<int>(blockIdx.x) >= ctas) {
    if (tid == 0 && !p.whole) p.joint[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }

  // A place on the line: sequence, unit of it, tile; and the sequence's first place.
  struct Place {
    int b, unit, tile, len;
    int64_t first;
  };
  const auto locate = [&](int64_t x) {
    const int64_t y = x / units;
    int lo = 0, hi = kThreads;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_before[mid] <= y) lo = mid;
      else hi = mid;
    }
    int b = lo * each;
    int64_t before = s_before[lo];
    for (const int stop = min(b + each, p.B); b + 1 < stop;) {
      const int mine = b + lane < stop ? tiles_of(length(b + lane)) : 0;
      int64_t upto = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int64_t z = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += z;
      }
      const uint32_t beyond = __ballot_sync(0xffffffffu, before + upto > y);
      if (beyond) {
        const int at = __ffs(beyond) - 1;
        before += __shfl_sync(0xffffffffu, upto - mine, at);
        b += at;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
      b += 32;
    }
    Place at;
    at.b = b;
    at.len = length(b);
    at.first = before * units;
    const int64_t rest = x - at.first;
    const int n = tiles_of(at.len);
    at.unit = static_cast<int>(rest / n);
    at.tile = static_cast<int>(rest - static_cast<int64_t>(at.unit) * n);
    return at;
  };
  // Where CTA c begins.
  const auto begin_of = [&](int64_t c) {
    int64_t x = c * line / ctas;
    if (p.whole && x < line)
      if (const Place at = locate(x); at.tile > 0) x += tiles_of(at.len) - at.tile;
    return x;
  };
  const int64_t cta_first = begin_of(blockIdx.x), cta_last = begin_of(blockIdx.x + 1);
  const int64_t mine = cta_last - cta_first;
  const int64_t x0 = cta_first + mine * warp / kWarps;
  int64_t left = cta_first + mine * (warp + 1) / kWarps - x0;

  Place at = {};
  if (left > 0) {
    at = locate(x0);
    if (x0 == cta_first && lane == 0) s_first = at.tile == 0 ? at.b * units + at.unit : -1;
  }
  int parts = 0;  // partial results that this warp has left
#pragma unroll 1
  while (left > 0) {
    const int n_tiles = tiles_of(at.len), first = at.tile;
    const int last = static_cast<int>(min(static_cast<int64_t>(n_tiles), first + left));
    const int b = at.b, len = at.len;
    const int hk = at.unit / p.splits, m0 = (at.unit - hk * p.splits) * p.rows;
    const int h0 = hk * p.heads + m0, rows = min(p.rows, p.heads - m0);

    // Q as the B operand: row = query head, the same 16-byte pieces of the head dim as a key's
    const T* qb = static_cast<const T*>(p.q) + b * p.q_sB + h0 * p.q_sH;
    uint4 q[NQ][kQShared ? 1 : KG];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const int m = n * 8 + r, d = g * 32 + t * 8;
        const uint4 x = m < rows && d < p.D ? __ldcg(reinterpret_cast<const uint4*>(qb + m * p.q_sH + d)) : make_uint4(0, 0, 0, 0);
        if constexpr (kQShared) *reinterpret_cast<uint4*>(s_q + ((warp * NQ + n) * KG + g) * 256 + lane * 8) = x;
        else q[n][g] = x;
      }

    const int* row = p.table + b * p.table_s;
    const T* kb = static_cast<const T*>(p.k) + hk * p.k_sH + t * 8;
    const T* vb = static_cast<const T*>(p.v) + hk * p.v_sH + r * 8;
    const int64_t bias_bh = b * p.bias_sB + h0 * p.bias_sH;

    // Pages.  ALIGNED: lane l knows page and first row of tile ids_from + l; else lane l that of key l % 16 of the next tile.
    int ids_from = 0, page_l = -1, row_l = 0;  // what the lane knows
    int page = -1, in_page = 0;                // of the tile that is loaded
    const auto look_up = [&](int tile) {
      if constexpr (ALIGNED) {
        ids_from = tile;
        const int mine = tile + lane, at_page = fast_div(mine, p.div_mul, p.div_shift);
        page_l = mine < last ? __ldcg(row + at_page) : -1;
        row_l = mine * 16 - at_page * p.page_size;
      } else {
        const int key = tile * 16 + (lane & 15), at_page = fast_div(key, p.div_mul, p.div_shift);
        page_l = tile < last && key < len ? __ldcg(row + at_page) : -1;
        row_l = key - at_page * p.page_size;
      }
      if (page_l >= p.num_pages) page_l = -1;
    };
    const auto turn_to = [&](int tile) {
      if constexpr (ALIGNED) {
        if (tile - ids_from >= 32) look_up(tile);
        page = __shfl_sync(0xffffffffu, page_l, tile - ids_from);
        in_page = __shfl_sync(0xffffffffu, row_l, tile - ids_from);
      } else {
        page = page_l;
        in_page = row_l;
        look_up(tile + 1);
      }
    };
    const auto page_of = [&](int key) { return ALIGNED ? page : __shfl_sync(0xffffffffu, page, key); };
    const auto row_of = [&](int key) { return ALIGNED ? in_page + key : __shfl_sync(0xffffffffu, in_page, key); };

    uint4 kf[2][KG], vf[4][VG];
    uint32_t there = 0;  // bit i: key r + 8 i of the tile whose K is loaded is one of the sequence's
    const auto load_k = [&](int tile) {
      there = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pg = page_of(r + 8 * i), at_row = row_of(r + 8 * i);
        const bool ok = tile * 16 + r + 8 * i < len && pg >= 0;
        there |= ok ? 1u << i : 0u;
        const T* src = kb + pg * p.k_sP + at_row * p.k_sT;
#pragma unroll
        for (int g = 0; g < KG; ++g) kf[i][g] = ldg_stream(src + g * 32, ok && (DP > 64 || g * 32 + t * 8 < p.D));
      }
    };
    const auto load_v = [&](int tile) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * t + (i & 1) + 8 * (i >> 1);
        const int pg = page_of(key), at_row = row_of(key);
        const bool ok = tile * 16 + key < len && pg >= 0;
        const T* src = vb + pg * p.v_sP + at_row * p.v_sT;
#pragma unroll
        for (int g = 0; g < VG; ++g) vf[i][g] = ldg_stream(src + g * 64, ok && (DP > 64 || r * 8 < p.D));
      }
    };
    float bf[NQ][4];
    const auto load_b = [&](int tile) {
      if constexpr (BIAS != 0) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = n * 8 + 2 * t + (i & 1), key = tile * 16 + r + 8 * (i >> 1);
            const int64_t at_b = bias_bh + m * p.bias_sH + key;
            float x = 0.f;
            if (m < rows && key < len) {
              if constexpr (BIAS == 1) x = static_cast<float>(static_cast<const T*>(p.bias)[at_b]);
              if constexpr (BIAS == 2) x = static_cast<const uint8_t*>(p.bias)[at_b] ? 1.f : 0.f;
              if constexpr (BIAS == 3) x = static_cast<const float*>(p.bias)[at_b];
            }
            bf[n][i] = x;
          }
      }
    };

    float o[NQ][VG * 4][4];  // O^T: [query group][16 head-dim rows][fragment]
    float mx[NQ][2], l[NQ][2];  // of rows 2t, 2t+1: running maximum, this lane's part of the sum
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      mx[n][0] = mx[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < VG * 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
    }

    look_up(first);
    turn_to(first);
    load_k(first);
    load_b(first);
    load_v(first);
    if constexpr (kQShared) __syncwarp();
#pragma unroll 1
    for (int tile = first; tile < last; ++tile) {
      const uint32_t here = there;
      float s[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const uint4 x = kQShared ? *reinterpret_cast<const uint4*>(s_q + ((warp * NQ + n) * KG + g) * 256 + lane * 8)
                                   : q[n][kQShared ? 0 : g];
          mma16816<T>(s[n], kf[0][g].x, kf[1][g].x, kf[0][g].y, kf[1][g].y, x.x, x.y);
          mma16816<T>(s[n], kf[0][g].z, kf[1][g].z, kf[0][g].w, kf[1][g].w, x.z, x.w);
        }
      }
      const bool more = tile + 1 < last;
      if (more) {
        turn_to(tile + 1);
        load_k(tile + 1);
      }
      // scores, -inf where a key takes no part
      bool need = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[n][i] * p.scale;
          // a mask selects: whatever the score of a masked key is (infinite, NaN), it takes no part
          if (BIAS == 2) x = bf[n][i] != 0.f ? x : -INFINITY;
          else if (BIAS != 0) x += bf[n][i];
          if (!(here >> (i >> 1) & 1)) x = -INFINITY;
          s[n][i] = x;
          need = need || x > mx[n][i & 1] + 8.f;
        }
      if (more) load_b(tile + 1);
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float m_new = fmaxf(mx[n][j], fmaxf(s[n][j], s[n][j + 2]));
            for (int off = 4; off < 32; off <<= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, off));
            const float alpha = m_new == -INFINITY ? 1.f : weight<BIAS>(mx[n][j], m_new);
            mx[n][j] = m_new;
            l[n][j] *= alpha;
#pragma unroll
            for (int i = 0; i < VG * 4; ++i) o[n][i][j] *= alpha, o[n][i][j + 2] *= alpha;
          }
      }
      // Weights in two 16-bit terms, so that they lose 2^-17 (bf16) and not 2^-9: memory leaves the time for it.
      uint32_t hi[NQ][2], lo[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float m_0 = mx[n][0] == -INFINITY ? 0.f : mx[n][0], m_1 = mx[n][1] == -INFINITY ? 0.f : mx[n][1];
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = weight<BIAS>(s[n][i], i & 1 ? m_1 : m_0);
        l[n][0] += w[0] + w[2];
        l[n][1] += w[1] + w[3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t top = P2::pack(w[2 * i], w[2 * i + 1]);
          const float2 f = P2::unpack(top);
          hi[n][i] = transpose8x8(top);
          lo[n][i] = transpose8x8(P2::pack(w[2 * i] - f.x, w[2 * i + 1] - f.y));
        }
      }
      // V^T of 16 head-dim rows: the halves of the words of keys 2t, 2t+1 and 2t+8, 2t+9
      const auto v_operand = [&](const uint4 (&v)[4][VG], int i, uint32_t (&a)[4]) {
        const auto word = [&](int k) {
          const uint4& x = v[k][i >> 2];
          return (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w;
        };
        a[0] = __byte_perm(word(0), word(1), 0x5410), a[1] = __byte_perm(word(0), word(1), 0x7632);
        a[2] = __byte_perm(word(2), word(3), 0x5410), a[3] = __byte_perm(word(2), word(3), 0x7632);
      };
      // An infinite or NaN value: zero weights make it NaN.  So the values times zero are summed, and looked at.
      float odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < VG * 4; ++i) {
        uint32_t a[4];
        v_operand(vf, i, a);
        mma16816<T>(odd, a[0], a[1], a[2], a[3], 0u, 0u);
      }
      const bool clean = odd[0] == 0.f && odd[2] == 0.f;
      if (__all_sync(0xffffffffu, clean)) {
#pragma unroll
        for (int i = 0; i < VG * 4; ++i) {
          uint32_t a[4];
          v_operand(vf, i, a);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma16816<T>(o[n][i], a[0], a[1], a[2], a[3], hi[n][0], hi[n][1]);
            mma16816<T>(o[n][i], a[0], a[1], a[2], a[3], lo[n][0], lo[n][1]);
          }
        }
      } else {
        // Row by row of the queries: the values that its row leaves out as zeros, and without the infinite ones in the product
        // with the small terms (which may be 0, or of the other sign).  The same products in the same order otherwise.
#pragma unroll 1
        for (int c = 0; c < 8 * NQ; ++c) {
          const int tc = (c & 7) >> 1;
          uint4 v1[4][VG], v2[4][VG];
          uint32_t out[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            bool left_out = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
              if (n == c >> 3) left_out = (c & 1 ? s[n][2 * half + 1] : s[n][2 * half]) == -INFINITY;
            out[half] = __ballot_sync(0xffffffffu, left_out) >> tc;  // bit 4 k: key k + 8 half
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int key = 2 * t + (k & 1);
            const uint32_t keep = out[k >> 1] >> (4 * key) & 1 ? 0u : 0xffffffffu;
#pragma unroll
            for (int g = 0; g < VG; ++g) {
              const uint4 x = vf[k][g];
              v1[k][g] = make_uint4(x.x & keep, x.y & keep, x.z & keep, x.w & keep);
              v2[k][g] = make_uint4(finite_or_zero<T>(x.x) & keep, finite_or_zero<T>(x.y) & keep, finite_or_zero<T>(x.z) & keep,
                                    finite_or_zero<T>(x.w) & keep);
            }
          }
#pragma unroll
          for (int i = 0; i < VG * 4; ++i) {
            uint32_t a1[4], a2[4];
            v_operand(v1, i, a1);
            v_operand(v2, i, a2);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              float x[4] = {o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]};
              mma16816<T>(x, a1[0], a1[1], a1[2], a1[3], hi[n][0], hi[n][1]);
              mma16816<T>(x, a2[0], a2[1], a2[2], a2[3], lo[n][0], lo[n][1]);
              const bool its = n == c >> 3 && t == tc;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (its && (e & 1) == (c & 1)) o[n][i][e] = x[e];
            }
          }
        }
      }
      if (more) load_v(tile + 1);
    }

    // ---- the unit, or what this warp has of it
    const bool begins = first == 0, ends = last == n_tiles;
    float* part = smem + (2 * warp + parts) * part_floats(DP, p.rows);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[n][j];
        for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int m = n * 8 + 2 * t + j;
        if (m >= rows) continue;
        // lane (r, t) holds head-dim elements 64 g + 8 r .. + 7 of its rows
        if (begins && ends) {
          const float inv = inverse(mx[n][j], sum);
          T* dst = static_cast<T*>(p.o) + b * p.o_sB + (h0 + m) * p.o_sH + r * 8;
#pragma unroll
          for (int g = 0; g < VG; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = P2::pack(finish(o[n][g * 4 + i][j], inv), finish(o[n][g * 4 + i][j + 2], inv));
            if (DP > 64 || r * 8 < p.D) *reinterpret_cast<uint4*>(dst + g * 64) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          float* dst = part + m * (DP + 2);
#pragma unroll
          for (int i = 0; i < VG * 4; ++i)
            *reinterpret_cast<float2*>(dst + (i >> 2) * 64 + r * 8 + (i & 3) * 2) = make_float2(o[n][i][j], o[n][i][j + 2]);
          if (r == 0) dst[DP] = mx[n][j], dst[DP + 1] = sum;
        }
      }
    if (!(begins && ends)) {
      if (lane == 0) s_unit[2 * warp + parts] = b * units + at.unit, s_ends[2 * warp + parts] = (begins ? 1 : 0) | (ends ? 2 : 0);
      ++parts;
    }
    // ---- on
    left -= last - first;
    at.tile = last;
    if (ends && left > 0) {
      at.tile = 0;
      if (++at.unit == units) {
        at.unit = 0;
        at.first += static_cast<int64_t>(n_tiles) * units;
        at.len = length(++at.b);
      }
    }
  }

  // ---- what the warps have of the same unit, in order
  __syncthreads();
  int4 joint = make_int4(-1, 0, 0, 0);
  for (int k = 0; k < 2 * kWarps;) {
    const int unit = s_unit[k];
    int stop = k + 1;
    if (unit >= 0) {
      int ends = s_ends[k];
      for (int j = k + 1; j < 2 * kWarps && (s_unit[j] < 0 || s_unit[j] == unit); ++j)
        if (s_unit[j] == unit) ends |= s_ends[j], stop = j + 1;
      const int b = unit / units, u = unit - b * units;
      const int hk = u / p.splits, m0 = (u - hk * p.splits) * p.rows;
      const int rows = min(p.rows, p.heads - m0);
      // the first unit of a CTA has its partial result in place 0, another one, which is the last, in place 1
      const int place = ends & 1 && unit != s_first ? 1 : 0;
      float* part = p.part + (2 * static_cast<int64_t>(blockIdx.x) + place) * part_floats(DP, p.rows);
      for (int e = tid; e < rows * DP; e += kThreads) {
        const int m = e / DP, d = e - m * DP;
        const float* src = smem + m * (DP + 2);
        float m_all = -INFINITY;
        for (int j = k; j < stop; ++j)
          if (s_unit[j] == unit) m_all = fmaxf(m_all, src[j * part_floats(DP, p.rows) + DP]);
        float acc = 0.f, sum = 0.f;
        for (int j = k; j < stop; ++j)
          if (s_unit[j] == unit) {
            const float* x = src + j * part_floats(DP, p.rows);
            const float f = weight_of<BIAS>(x[DP], m_all);
            acc += f * x[d];
            sum += f * x[DP + 1];
          }
        if (ends == 3) {
          if (d < p.D)
            (static_cast<T*>(p.o) + b * p.o_sB + (hk * p.heads + m0 + m) * p.o_sH)[d] = static_cast<T>(finish(acc, inverse(m_all, sum)));
        } else {
          part[m * (DP + 2) + d] = acc;
          if (d == 0) part[m * (DP + 2) + DP] = m_all, part[m * (DP + 2) + DP + 1] = sum;
        }
      }
      if (ends == 1) joint = make_int4(unit, place, 0, 0);
    }
    k = stop;
  }
  if (!p.whole && tid < 32) {
    if (joint.x >= 0) {  // the CTA that has the unit's last tile: the last one that begins at or before it
      const int b = joint.x / units, u = joint.x - b * units;
      const Place end = locate(cta_last - 1);
      const int64_t tile = (end.first + static_cast<int64_t>(u + 1) * tiles_of(length(b))) - 1;
      joint.z = static_cast<int>(((tile + 1) * ctas - 1) / line);
    }
    if (tid == 0) p.joint[blockIdx.x] = joint;
  }
}

// Joins the parts of the unit that begins in CTA blockIdx.x of the first kernel and goes on, a row of it a block.
constexpr int kJoinThreads = 256;
template <int DP, typename T, int BIAS>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const PagedParams p) {
  constexpr int kTeam = DP / 4;  // threads with four sums each
  constexpr int kTeams = kJoinThreads / kTeam;
  __shared__ float s_max[kJoinThreads / 32];
  __shared__ __align__(16) float s_acc[kTeams][DP];
  __shared__ float s_l[kTeams];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_launch_next();
  grid_dep_wait();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  const int4 joint = __ldcg(p.joint + blockIdx.x);
  if (joint.x < 0) return;
  const int units = p.Hkv * p.splits, row = blockIdx.y;
  const int b = joint.x / units, u = joint.x - b * units;
  const int hk = u / p.splits, m0 = (u - hk * p.splits) * p.rows;
  if (row >= min(p.rows, p.heads - m0)) return;
  const int n = joint.z - static_cast<int>(blockIdx.x) + 1;
  const int64_t step = part_floats(DP, p.rows);
  const float* base = p.part + 2 * static_cast<int64_t>(blockIdx.x) * step + row * (DP + 2);
  const auto part = [&](int i) { return base + (2 * i + (i == 0 ? joint.y : 0)) * step; };
  float top = -INFINITY;
  for (int i = tid; i < n; i += kJoinThreads) top = fmaxf(top, __ldcg(part(i) + DP));
  for (int off = 1; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, s_max[w]);
  const int team = tid / kTeam, d = (tid - team * kTeam) * 4;
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll 4
  for (int i = team; i < n; i += kTeams) {
    const float* x = part(i);
    const float2 a = __ldcg(reinterpret_cast<const float2*>(x + d)), c = __ldcg(reinterpret_cast<const float2*>(x + d + 2));
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(x + DP));
    const float f = weight_of<BIAS>(ml.x, top);
    acc[0] += f * a.x, acc[1] += f * a.y, acc[2] += f * c.x, acc[3] += f * c.y;
    sum += f * ml.y;
  }
  *reinterpret_cast<float4*>(&s_acc[team][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  if (d == 0) s_l[team] = sum;
  __syncthreads();
  for (int e = tid; e < p.D; e += kJoinThreads) {
    float a = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < kTeams; ++i) a += s_acc[i][e], s += s_l[i];
    (static_cast<T*>(p.o) + b * p.o_sB + (hk * p.heads + m0 + row) * p.o_sH)[e] = static_cast<T>(finish(a, inverse(top, s)));
  }
}

// How a call is cut: rows a unit, units a key head, the largest grid.
struct Plan {
  int DP, NQ, rows, splits, ctas;
  bool whole;
};
Plan plan_paged(const fa_paged_params& p) {
  Plan x;
  const int heads = p.H / p.Hkv;
  x.DP = padded_head_dim(p.D);
  x.NQ = heads <= 8 || x.DP == 256 ? 1 : 2;
  x.splits = (heads + 8 * x.NQ - 1) / (8 * x.NQ);
  x.rows = (heads + x.splits - 1) / x.splits;
  const int64_t cap = static_cast<int64_t>(p.width) * p.page_size;
  const int64_t most = (static_cast<int64_t>(p.B) * p.Hkv * x.splits * ((cap + 15) / 16) + kLeastTiles - 1) / kLeastTiles;
  const int64_t resident = static_cast<int64_t>(persistent_grid(1 << 30)) * ctas_per_sm(x.DP, x.NQ);
  x.ctas = static_cast<int>(most < resident ? most : resident);
  x.whole = cap <= 16 * kWholeTiles;
  return x;
}
uint64_t part_bytes(const Plan& x) { return (2ull * x.ctas * part_floats(x.DP, x.rows) * 4 + 15) / 16 * 16; }

template <int DP, int NQ, typename T, int BIAS, bool ALIGNED>
int launch_inst(const PagedParams& d, const Plan& x, cudaStream_t stream) {
  const int smem = 2 * kWarps * part_floats(DP, x.rows) * 4;
  static std::atomic<uint64_t> ready{0};  // devices whose kernel has its shared memory
  int dev = 0;
  cudaGetDevice(&dev);
  constexpr int kMost = 2 * kWarps * part_floats(DP, 8 * NQ) * 4;
  if (dev < 0 || dev >= 64) return FA_ERR_CUDA;
  if (kMost > 40 * 1024 && !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(paged_kernel<DP, NQ, T, BIAS, ALIGNED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess)
      return FA_ERR_CUDA;
    ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (int e = launch_overlapped(paged_kernel<DP, NQ, T, BIAS, ALIGNED>, dim3(x.ctas), kThreads, smem, stream, d)) return e;
  if (x.whole) return FA_OK;
  return launch_overlapped(join_kernel<DP, T, BIAS>, dim3(x.ctas, x.rows), kJoinThreads, 0, stream, d);
}

template <int DP, int NQ, typename T>
int launch_bias(const PagedParams& d, const Plan& x, int bias_kind, bool aligned, cudaStream_t stream) {
  switch (bias_kind) {
    case FA_BIAS_NONE: return aligned ? launch_inst<DP, NQ, T, 0, true>(d, x, stream) : launch_inst<DP, NQ, T, 0, false>(d, x, stream);
    case FA_BIAS_SAME: return aligned ? launch_inst<DP, NQ, T, 1, true>(d, x, stream) : launch_inst<DP, NQ, T, 1, false>(d, x, stream);
    case FA_BIAS_BOOL: return aligned ? launch_inst<DP, NQ, T, 2, true>(d, x, stream) : launch_inst<DP, NQ, T, 2, false>(d, x, stream);
    default: return aligned ? launch_inst<DP, NQ, T, 3, true>(d, x, stream) : launch_inst<DP, NQ, T, 3, false>(d, x, stream);
  }
}

template <typename T>
int launch_typed(const PagedParams& d, const Plan& x, int bias_kind, bool aligned, cudaStream_t stream) {
  if (x.DP == 256) return launch_bias<256, 1, T>(d, x, bias_kind, aligned, stream);
  if (x.DP == 128)
    return x.NQ == 1 ? launch_bias<128, 1, T>(d, x, bias_kind, aligned, stream) : launch_bias<128, 2, T>(d, x, bias_kind, aligned, stream);
  return x.NQ == 1 ? launch_bias<64, 1, T>(d, x, bias_kind, aligned, stream) : launch_bias<64, 2, T>(d, x, bias_kind, aligned, stream);
}

}  // namespace

uint64_t paged_workspace_bytes(const fa_paged_params& p) {
  const Plan x = plan_paged(p);
  return x.whole ? 0 : part_bytes(x) + 16ull * x.ctas;
}

int launch_paged(const fa_paged_params& p, void* workspace, cudaStream_t stream, int* status) {
  const Plan x = plan_paged(p);
  PagedParams d;
  d.q = p.q, d.k = p.k_cache, d.v = p.v_cache, d.bias = p.bias, d.o = p.o;
  d.table = p.block_table, d.lens = p.seq_lens, d.status = status;
  d.part = static_cast<float*>(workspace);
  d.joint = workspace ? reinterpret_cast<int4*>(static_cast<char*>(workspace) + part_bytes(x)) : nullptr;
  d.q_sB = p.q_stride[0], d.q_sH = p.q_stride[1], d.o_sB = p.o_stride[0], d.o_sH = p.o_stride[1];
  d.k_sP = p.k_stride[0], d.k_sT = p.k_stride[1], d.k_sH = p.k_stride[2];
  d.v_sP = p.v_stride[0], d.v_sT = p.v_stride[1], d.v_sH = p.v_stride[2];
  d.bias_sB = p.bias_stride[0], d.bias_sH = p.bias_stride[1], d.table_s = p.table_stride;
  d.B = p.B, d.H = p.H, d.Hkv = p.Hkv, d.D = p.D;
  d.page_size = p.page_size, d.num_pages = p.num_pages, d.width = p.width;
  d.heads = p.H / p.Hkv, d.rows = x.rows, d.splits = x.splits, d.whole = x.whole ? 1 : 0;
  d.scale = p.bias_kind == FA_BIAS_NONE || p.bias_kind == FA_BIAS_BOOL ? p.sm_scale * kLog2e : p.sm_scale;
  // Division by d, rounded down, of x < 2^31: with 2^(s - 1) < d <= 2^s it is (x + x * mul / 2^32) >> s, mul = 2^32 (2^s - d) / d + 1.
  const bool aligned = p.page_size % 16 == 0;
  const uint64_t by = static_cast<uint64_t>(aligned ? p.page_size / 16 : p.page_size);
  uint32_t s = 0;
  while ((1ull << s) < by) ++s;
  d.div_shift = s;
  d.div_mul = static_cast<uint32_t>((((1ull << s) - by) << 32) / by + 1);
  return p.dtype == FA_BF16 ? launch_typed<__nv_bfloat16>(d, x, p.bias_kind, aligned, stream)
                            : launch_typed<__half>(d, x, p.bias_kind, aligned, stream);
}

}  // namespace fa
