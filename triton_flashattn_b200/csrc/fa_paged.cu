// Attention of one new token a sequence over a paged cache: how a call is cut, its tile maps and its launch (the kernels are in
// fa_paged.cuh).
#include "fa_paged.cuh"

namespace fa {
namespace {

// Where no sequence is split over CTAs, there is one launch less.  Sequences of one tile cannot be.  Those of up to so many keys are
// not, unless that leaves warps idle (they have no parts of a stretch then) and there are more sequences than CTAs.  Whole / split,
// us, bf16, tables of 64 keys (8 key heads of 128 with 4 heads; 1 of 128 with 8; 12 of 64 with 1; 2 of 256 with 16):
//     1 sequence,  17 keys      6.5 / 7.3      5.7 / 7.1      7.9 / 8.9      8.7 / 8.8
//                  64           8.2 / 7.1      7.3 / 6.9     10.1 / 9.9     11.6 / 9.1
//    64 sequences, 17           9.1 / 10.6     8.1 / 9.6     10.4 / 10.2    11.0 / 13.9
//                  64          11.4 / 12.7     9.7 / 10.1    13.0 / 14.0    13.9 / 16.4
//   148 sequences, 64          14.1 / 15.9     9.8 / 10.0    14.0 / 14.2    15.9 / 22.6
//  1000 sequences, 64          55.0 / 57.8    37.0 / 21.6    51.0 / 52.2    62.8 / 53.0   (warps 8 of 8, 1 of 8, all, 2 of 4)
// and tables of 128, full: 1 sequence 11.8 / 7.5, 148 of up to 128 keys 19.9 / 21.6.
constexpr int kWholeKeys = 64;

PagedPlan plan_paged(const fa_paged_params& p) {
  PagedPlan x;
  const int heads = p.H / p.Hkv;
  x.DP = padded_head_dim(p.D);
  // Rows of a unit in groups of 8.  More heads than two groups are more units, which read the same keys side by side.
  // 16 sequences of 1000 to 8000 keys, 4 key heads, one group / two, us: 16 heads each 41 / 38.6 (D 64, 32 sequences 43 / 37); 32 heads
  // each 76 / 52, with four groups 56.
  x.NQ = heads <= 8 ? 1 : 2;
  x.splits = (heads + 8 * x.NQ - 1) / (8 * x.NQ);
  x.rows = (heads + x.splits - 1) / x.splits;
  x.units = p.Hkv * x.splits;
  const int tile = (x.DP == 64 ? 2 : 1) * 32 * x.DP, queries = 8 * x.NQ * x.DP * 2;  // bytes, as Cfg has them
  // Warps: as many as there is room for, fewer where that spares parts (each has units / gcd items over 1 / parts of the
  // stretch: a warp a unit, or some units, or some warps a unit).  Always the most: two units at head dim 256 (5 warps for 4) 28 -> 40
  // us, one unit at 128 (8 for 5) 24 -> 29.
  const auto ring_of = [&](int warps) { return ((kPagedSmem / warps) / 1024 * 1024 - queries) / (2 * tile); };
  int most = kMostWarps;
  while (most > 4 && ring_of(most) < 2) --most;
  x.warps = 0;
  for (int w = most; w >= 4 && w + 3 >= most; --w) {
    int a = x.units, g = w;
    while (a % g) {
      const int rest = a % g;
      a = g, g = rest;
    }
    if (x.warps == 0 || w / g < x.parts) x.warps = w, x.parts = w / g;
  }
  const int ring = ring_of(x.warps);
  x.ring = ring < 8 ? ring : 8;
  const int64_t cap = static_cast<int64_t>(p.width) * p.page_size;
  const int keys = x.DP == 64 ? 32 : 16;
  const int64_t most_ctas = p.B * ((cap + keys - 1) / keys);
  const int sms = persistent_grid(1 << 30);
  x.ctas = static_cast<int>(most_ctas < sms ? most_ctas : sms);
  x.whole = cap <= keys || (cap <= kWholeKeys && (x.parts == 1 || p.B <= sms));
  if (x.whole && cap > keys) x.parts = 1;
  const int stretches = x.ctas * x.parts;
  x.by_seq = p.B <= kFew || p.B <= stretches;
  x.joints = x.by_seq ? p.B : stretches;
  // More teams while a team has several rounds of sums and the SMs room for them; of smaller slices where a block holds no more.
  x.ahead = x.by_seq ? 8 : 4;  // (elsewhere a sequence has two sums, rarely more)
  const int64_t sums = p.B < stretches ? stretches / p.B : 1;
  const int64_t room_for = static_cast<int64_t>(sms) * 2 * kJoinThreads;
  int size = x.DP / 4;
  x.slices = x.teams = 1;
  while (sums > x.ahead * x.teams && static_cast<int64_t>(x.joints) * p.H * (x.DP / 4) * x.teams * 2 <= room_for &&
         (x.teams * size < kJoinThreads || size > 4)) {
    if (x.teams * size == kJoinThreads) x.slices *= 2, size /= 2;
    x.teams *= 2;
  }
  return x;
}
uint64_t part_bytes(const PagedPlan& x) {
  return x.whole ? 0 : 2ull * x.ctas * x.parts * x.units * x.rows * row_floats(x.DP) * 4;
}

// Tile map of a cache.  False where its layout has none (an expanded view): then its rows are copied one by one.
bool cache_map(CUtensorMap* out, const void* base, const fa_paged_params& p, const int64_t s[3], int box_keys) {
  const int extent[3] = {p.num_pages, p.page_size, p.Hkv};
  uint64_t bytes[3];
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of extent one does not matter
    const int64_t x = extent[i] == 1 ? 8 : s[i];
    if (x <= 0 || x >= 1ll << 38) return false;
    bytes[i] = static_cast<uint64_t>(x) * 2;
  }
  const uint64_t dims[4] = {static_cast<uint64_t>(p.D), static_cast<uint64_t>(p.Hkv), static_cast<uint64_t>(p.page_size),
                            static_cast<uint64_t>(p.num_pages)};
  const uint64_t strides[3] = {bytes[2], bytes[1], bytes[0]};
  const uint32_t box[4] = {64, 1, static_cast<uint32_t>(box_keys), 1};
  return make_tmap_4d(out, base, 2, dims, strides, box) == FA_OK;
}

}  // namespace

uint64_t paged_workspace_bytes(const fa_paged_params& p) {
  const PagedPlan x = plan_paged(p);
  return x.whole ? 0 : part_bytes(x) + 16ull * x.joints;
}

int launch_paged(const fa_paged_params& p, void* workspace, cudaStream_t stream, int* status) {
  PagedParams d;
  int box = p.page_size % 16 == 0 ? 16 : p.page_size % 8 == 0 ? 8 : 0;
  if (box && (!cache_map(&d.k_map, p.k_cache, p, p.k_stride, box) || !cache_map(&d.v_map, p.v_cache, p, p.v_stride, box))) box = 0;
  const PagedPlan x = plan_paged(p);
  d.q = p.q, d.k = p.k_cache, d.v = p.v_cache, d.bias = p.bias, d.o = p.o;
  d.table = p.block_table, d.lens = p.seq_lens, d.status = status;
  d.part = static_cast<float*>(workspace);
  d.joint = x.whole || p.B <= kFew ? nullptr : reinterpret_cast<int4*>(static_cast<char*>(workspace) + part_bytes(x));
  d.q_sB = p.q_stride[0], d.q_sH = p.q_stride[1], d.o_sB = p.o_stride[0], d.o_sH = p.o_stride[1];
  d.k_sP = p.k_stride[0], d.k_sT = p.k_stride[1], d.k_sH = p.k_stride[2];
  d.v_sP = p.v_stride[0], d.v_sT = p.v_stride[1], d.v_sH = p.v_stride[2];
  d.bias_sB = p.bias_stride[0], d.bias_sH = p.bias_stride[1], d.table_s = p.table_stride;
  d.B = p.B, d.H = p.H, d.Hkv = p.Hkv, d.D = p.D;
  d.page_size = p.page_size, d.num_pages = p.num_pages, d.width = p.width, d.page_boxes = box ? p.page_size / box : 0;
  d.heads = p.H / p.Hkv, d.rows = x.rows, d.splits = x.splits, d.units = x.units;
  d.parts = x.parts, d.ring = x.ring, d.whole = x.whole ? 1 : 0, d.by_seq = x.by_seq ? 1 : 0, d.joints = x.joints, d.ctas = x.ctas, d.slices = x.slices, d.teams = x.teams;
  d.scale = p.bias_kind == FA_BIAS_NONE || p.bias_kind == FA_BIAS_BOOL ? p.sm_scale * kLog2e : p.sm_scale;
  // Division by d, rounded down, of x < 2^31: with 2^(s - 1) < d <= 2^s it is (x + x * mul / 2^32) >> s, mul = 2^32 (2^s - d) / d + 1.
  const auto divisor = [](uint64_t by, uint32_t& mul, uint32_t& shift) {
    uint32_t s = 0;
    while ((1ull << s) < by) ++s;
    shift = s;
    mul = static_cast<uint32_t>((((1ull << s) - by) << 32) / by + 1);
  };
  divisor(box ? p.page_size / box : p.page_size, d.div_mul, d.div_shift);
  divisor(x.splits, d.splits_mul, d.splits_shift);
  const bool bf16 = p.dtype == FA_BF16;
  PagedLaunch* launch = box == 16  ? (bf16 ? launch_paged_bf16 : launch_paged_f16)
                        : box == 8 ? (bf16 ? launch_paged_bf16_box8 : launch_paged_f16_box8)
                                   : (bf16 ? launch_paged_bf16_rows : launch_paged_f16_rows);
  return launch(d, x, p.bias_kind, stream);
}

}  // namespace fa
