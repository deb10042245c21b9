// Attention over a paged cache for the rows of a serving batch, for gfx950: single tokens, prompt
// chunks and mixtures of them, over 16-bit, fp32 or MXFP4 pages, with an optional sliding window
// and first tokens that stay visible (sinks):
//     out[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j
// over the keys j <= p_r with j > p_r - window or j < sinks, j inside the request's block table and
// in a page whose table entry is a page of the pool. A row that sees no key gets zeros; a row with
// a negative position is left as it was.
//
// Query rows of one KV head are flattened as (row, q-head-in-group), so the heads of a group share
// every K / V row that is read. A row tile's keys are a list of key tiles: the sink tiles, then the
// tiles from the window's lower edge to the last position; what lies between is never read.
//
// Three kernels (plus one for other head sizes, alignments and scales):
//   * paged_decode_kernel: 16 flattened rows, 16-bit arithmetic. What bounds it is reading the
//     cache once; every wave walks its own key tiles with a softmax state of its own, so waves
//     never wait for each other, and the states meet in LDS at the end.
//   * paged_f32_kernel: the same for fp32 pages on the fp32 matrix cores.
//   * paged_rows_kernel: 256 flattened rows (8 waves x 32), 16-bit arithmetic; K / V tiles of 64
//     keys are staged in LDS for all of them. Matrix-core bound.
// Long key lists are split over workgroups; paged_merge_kernel joins the fp32 partials.
//
// Masked places may hold anything. A masked score is replaced, so K never leaks; a weight of zero
// times an infinite or NaN V would leak through the sum, so tiles that some row sees only in part
// have such values taken out of V before the products, and after the last tile they are added to
// the rows that do see them: whatever its (positive) weight, such a value decides a row's sum.
#include "sb_mma.h"

#include <algorithm>
#include <type_traits>

namespace sb {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kNoWindow = 0x7fffffff;
constexpr int kDecodeRows = 16;
constexpr int kDecodeWaves = 4;
constexpr int kFewSlots = 512;     // workgroups of the decode kernels at a time (two per CU)
constexpr int kFewTarget = 1536;   // balanced items of a launch
constexpr int kFewMinTiles = 8;    // fewest key tiles of an item (two per wave)
constexpr int kShortItem = 24;     // key tiles of an item up to which one round is cut
constexpr int64_t kLongTiles = 256;
constexpr int kBalancedRows = 2048;  // most rows of balanced items
constexpr int kDecodeAhead4 = 1;  // steps of 4-bit rows in flight per wave
constexpr int kRowsTile = 256;
constexpr int kRowsWaves = 8;
constexpr int kAhead = 2;  // fragments read ahead of their MFMA (ring of 4)

struct PagedArgs {
  const char* q;
  char* o;
  int64_t q_row, q_head, o_row, o_head;   // byte strides
  const char* k;                          // K plane (4 bit: codes)
  const char* v;
  int64_t c_head, c_pos;                  // byte strides
  const char* ks;                         // scale bytes of K and V (4 bit)
  const char* vs;
  int64_t s_head, s_pos;
  uint32_t c_block, s_block;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* positions;
  const int32_t* row_starts;              // nullptr: row i is request i's, or the only one's
  int num_rows, num_requests, num_kv_heads, group, head_dim;
  int block_size, num_blocks_total;
  uint32_t bs_magic;                      // key / block_size = (key * bs_magic) >> bs_shift
  int bs_shift;
  int kv_len;                             // keys that a block table can name
  int window, sinks;
  float scale, scale_log2, scale_log2_lo; // scale_log2_lo: what scale * log2(e) rounds off
  int flat_min, flat_max;                 // flattened rows of the requests this launch takes
  int num_tiles;                          // row tiles of the launch (bound)
  int nsplit, min_tiles;                  // key splits of a row tile; fewest key tiles of one
  int slots;                              // > 0: places of partials; nsplit is the most that they
                                          // allow the row tiles there are (counted on the device)
  int target;                             // > 0: items of about 1 / target of all key tiles (one
                                          // row per request), instead of nsplit per row tile
  float* part_o;                          // [tile][kv head][split][row][D]
  float* part_ml;                         // [tile][kv head][split][row][2]
  int2* part_item;                        // balanced items: [tile][kv head] first slot and splits
};

__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// First row, number of rows and number of row tiles of request r (with row_starts).
struct RequestRows {
  int start, rows, tiles;
};
template <int TR>
__device__ __forceinline__ RequestRows request_rows(const PagedArgs& a, int r) {
  RequestRows q = {0, 0, 0};
  if (r < a.num_requests) {
    q.start = min(max(a.row_starts[r], 0), a.num_rows);
    q.rows = max(min(a.row_starts[r + 1], a.num_rows) - q.start, 0);
    const int64_t flat = static_cast<int64_t>(q.rows) * a.group;
    if (flat > a.flat_min && flat <= a.flat_max) q.tiles = static_cast<int>((flat + TR - 1) / TR);
  }
  return q;
}

// Row tile `idx` of a launch: its request and which tile of TR flattened rows of it.
struct TileRef {
  int request;  // -1: behind the last tile
  int row0, rows, tile;
};
template <int TR>
__device__ __forceinline__ TileRef find_tile(const PagedArgs& a, int idx) {
  TileRef t = {-1, 0, 0, 0};
  if (!a.row_starts) {
    if (a.num_requests == 1) {
      if (static_cast<int64_t>(idx) * TR < static_cast<int64_t>(a.num_rows) * a.group)
        t = {0, 0, a.num_rows, idx};
      return t;
    }
    const int per = (a.group + TR - 1) / TR;
    const int r = idx / per;
    if (r < a.num_rows) t = {r, r, 1, idx - r * per};
    return t;
  }
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int c = 0; c < a.num_requests; c += 64) {
    const RequestRows q = request_rows<TR>(a, c + lane);
    int incl = q.tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(incl, d, 64);
      if (lane >= d) incl += y;
    }
    const uint64_t past = __ballot(idx < base + incl);
    if (past) {
      const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
      t.request = c + l;
      t.row0 = __builtin_amdgcn_readfirstlane(__shfl(q.start, l, 64));
      t.rows = __builtin_amdgcn_readfirstlane(__shfl(q.rows, l, 64));
      t.tile = idx - base -
               __builtin_amdgcn_readfirstlane(__shfl(incl, l, 64) - __shfl(q.tiles, l, 64));
      return t;
    }
    base += __builtin_amdgcn_readfirstlane(__shfl(incl, 63, 64));
  }
  return t;
}

// Row tiles of a launch and the most parts that the keys of one are cut into. The host knows how
// many row tiles a batch may have, and what its rows would fill if they were one request's; between
// the two lie factors of ten (one chunk among hundreds of single tokens). Partials are kept for
// `slots` (row tile, KV head, part) places, and the parts of a tile follow from the number of tiles
// that row_starts gives: one scan more per workgroup, of the launches that split only. (Bounds
// alone: 256 requests with a chunk of 512 rows, 32 / 8 heads x 128, up to 8192 tokens: 1022 MB of
// partials and 234 us of rows kernel and merge, 68 MB and 134 with the scan.)
struct Parts {
  int tiles, most;
};
template <int TR>
__device__ __forceinline__ Parts parts_of(const PagedArgs& a) {
  if constexpr (TR == kRowsTile) {
    if (a.slots > 0) {
      int n = 0;
      for (int c = 0; c < a.num_requests; c += 64)
        n += request_rows<TR>(a, c + (threadIdx.x & 63)).tiles;
      n = max(__builtin_amdgcn_readfirstlane(wave_sum_i(n)), 1);
      return {n, max(min(a.nsplit, a.slots / (n * a.num_kv_heads)), 1)};
    }
  }
  return {a.num_tiles, a.nsplit};
}

// The key tiles (of KT keys) that rows at positions [pmin, pmax] see: n_sink tiles from 0 on,
// then those from lo on; `total` of both.
struct KeyTiles {
  int n_sink, lo, total;
};
template <int KT>
__device__ __forceinline__ KeyTiles key_tiles(const PagedArgs& a, int pmin, int pmax) {
  const int hi_key = min(pmax, a.kv_len - 1);
  const int lo_key = max(0, pmin - a.window + 1);  // (a.window >= 1: no overflow)
  const int sink_keys = min(a.sinks, hi_key + 1);
  KeyTiles t;
  t.n_sink = (sink_keys + KT - 1) / KT;
  t.lo = lo_key / KT;
  int n_win = 0;
  if (lo_key <= hi_key) {
    n_win = hi_key / KT - t.lo + 1;
    t.n_sink = min(t.n_sink, t.lo);
  }
  t.total = t.n_sink + n_win;
  return t;
}
template <int KT>
__device__ __forceinline__ int tile_key(const KeyTiles& t, int i) {
  return (i < t.n_sink ? i : t.lo + i - t.n_sink) * KT;
}
__device__ __forceinline__ int split_count(const PagedArgs& a, int most, int total) {
  return max(1, min(most, total / a.min_tiles));
}

// Quotient of a key (31 bits) by the block size d: with l = ceil(log2 d) and m = ceil(2^(31+l) / d),
// m d - 2^(31+l) < d <= 2^l, so key * m >> (31 + l) is exact for keys below 2^31 (T. Granlund and
// P. Montgomery, "Division by invariant integers using multiplication", 1994).
__device__ __forceinline__ int block_of(const PagedArgs& a, int key) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(key)) * a.bs_magic) >>
                          a.bs_shift);
}
// Page of a key: its number in the pool, or -1 (outside the table, or no page of the pool).
// In two parts where it is requested ahead of its use: behind a branch, or compared at once, the load
// would be waited for, and with it all that were issued before it.
__device__ __forceinline__ int page_entry(const PagedArgs& a, const int32_t* table, int key) {
  return table[block_of(a, min(key, a.kv_len - 1))];
}
__device__ __forceinline__ int page_in(const PagedArgs& a, int entry, int key) {
  return key < a.kv_len && entry >= 0 && entry < a.num_blocks_total ? entry : -1;
}
__device__ __forceinline__ int page_of(const PagedArgs& a, const int32_t* table, int key) {
  return page_in(a, page_entry(a, table, key), key);
}
// Byte offset of a key's row from its plane and head (page given; no page: page 0, masked later).
__device__ __forceinline__ int64_t row_offset(const PagedArgs& a, int key, int pb, uint32_t s_block,
                                              int64_t s_pos) {
  const int slot = key - block_of(a, key) * a.block_size;
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(max(pb, 0))) * s_block) +
         slot * s_pos;
}
__device__ __forceinline__ bool sees(const PagedArgs& a, int p, int key) {
  return key <= p && (key > p - a.window || key < a.sinks);
}

// Bit r: a row at position p sees key k0 + r (0 <= r < 32), window, sinks and causality.
__device__ __forceinline__ uint32_t bits_to(int m) {  // bits 0 .. m (none below 0)
  return m < 0 ? 0u : m >= 31 ? ~0u : (2u << m) - 1u;
}
__device__ __forceinline__ uint32_t seen_bits(const PagedArgs& a, int p, int k0) {
  const int d = max(p - k0, -1);  // (below 0 no key is seen; p >= -1, so nothing overflows)
  return bits_to(d) & (~bits_to(d - a.window) | bits_to(a.sinks - k0 - 1));
}

template <int DT> struct Half;  // 16-bit arithmetic beyond Mma<DT>
template <> struct Half<SB_DTYPE_BF16> {
  static constexpr uint32_t kExp = 0x7f80u, kOne = 0x3f80u;
  static constexpr int kShift = 0;  // powers of two taken off 4-bit values
  // The first scale byte whose block can hold a value that converts to an infinity (4 * 2^126).
  static constexpr uint32_t kInfByte = 253;
  __device__ __forceinline__ static float to_f32(uint32_t x) { return bf16_to_f32(x); }
  __device__ __forceinline__ static f32x4 mma16(bf16x8_t a, bf16x8_t b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <int SEL>
  __device__ __forceinline__ static uint32_t fp4(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
  }
};
// fp16: 4-bit values are taken times 2^-2 and the scores and outputs times 2^2, so that a block
// whose largest value rounds to 65536 (its fp16 source was at most 65504) stays finite. Values below
// 2^18 are finite (larger ones, of pages written from wider tokens, become infinite), and exact where
// they have no bits below 2^-22; others are off by at most 2^-23.
template <> struct Half<SB_DTYPE_F16> {
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u;
  static constexpr int kShift = 2;
  static constexpr uint32_t kInfByte = 143;  // (4 * 2^(143 - 127 - 2) = 65536)
  __device__ __forceinline__ static float to_f32(uint32_t x) { return f16_to_f32(x); }
  __device__ __forceinline__ static f32x4 mma16(f16x8_t a, f16x8_t b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <int SEL>
  __device__ __forceinline__ static uint32_t fp4(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
  }
};

// The fp32 scale of a scale byte, for the conversions (which read the exponent field: 0 is 2^-127,
// 255 makes every value NaN).
template <int SHIFT>
__device__ __forceinline__ float scale_of(uint32_t byte) {
  if constexpr (SHIFT > 0) byte = byte == 255 ? 255 : static_cast<uint32_t>(max(static_cast<int>(byte) - SHIFT, 0));
  return __uint_as_float(byte << 23);
}

// 8 values (one word of codes) as packed 16-bit numbers.
template <int DT>
__device__ __forceinline__ u32x4_t fp4x8(uint32_t w, float scale) {
  using H = Half<DT>;
  const u32x4_t r = {H::template fp4<0>(w, scale), H::template fp4<1>(w, scale),
                     H::template fp4<2>(w, scale), H::template fp4<3>(w, scale)};
  return r;
}

// 4 values (16 bits of codes).
template <int DT>
__device__ __forceinline__ uint2 fp4x4(uint32_t w, float scale) {
  using H = Half<DT>;
  return make_uint2(H::template fp4<0>(w, scale), H::template fp4<1>(w, scale));
}

// Bits 15 and 31 of the result are set where a packed 16-bit value is infinite or NaN: adding one
// to an exponent field of all ones carries into the sign bit's place, and never past it.
template <int DT>
__device__ __forceinline__ uint32_t not_finite_bits(uint32_t w) {
  constexpr uint32_t e = Half<DT>::kExp | Half<DT>::kExp << 16;
  constexpr uint32_t one = (0x8000u - Half<DT>::kExp) | (0x8000u - Half<DT>::kExp) << 16;
  return (w & e) + one;
}
template <int DT>
__device__ __forceinline__ uint32_t not_finite_bits(u32x4_t v) {
  return not_finite_bits<DT>(v[0]) | not_finite_bits<DT>(v[1]) | not_finite_bits<DT>(v[2]) |
         not_finite_bits<DT>(v[3]);
}
constexpr uint32_t kNotFinite = 0x80008000u;

// The packed values where they are finite, 0 elsewhere.
template <int DT>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  constexpr uint32_t lo = Half<DT>::kExp, hi = lo << 16;
  return w & (((w & lo) == lo ? 0u : 0xffffu) | ((w & hi) == hi ? 0u : 0xffff0000u));
}
template <int DT>
__device__ __forceinline__ u32x4_t finite_part(u32x4_t v) {
  const u32x4_t r = {finite_part<DT>(v[0]), finite_part<DT>(v[1]), finite_part<DT>(v[2]),
                     finite_part<DT>(v[3])};
  return r;
}
// acc[0..3] += the four packed values that are not finite.
template <int DT, typename Acc>
__device__ __forceinline__ void add_not_finite(uint2 w, Acc& acc, int e) {
  if (((not_finite_bits<DT>(w.x) | not_finite_bits<DT>(w.y)) & kNotFinite) == 0) return;
  w.x &= ~finite_part<DT>(w.x), w.y &= ~finite_part<DT>(w.y);
  acc[e] += Half<DT>::to_f32(w.x & 0xffffu);
  acc[e + 1] += Half<DT>::to_f32(w.x >> 16);
  acc[e + 2] += Half<DT>::to_f32(w.y & 0xffffu);
  acc[e + 3] += Half<DT>::to_f32(w.y >> 16);
}

// The softmax state's reference of a row that has seen keys, but none with a score above -inf:
// the sum of its weights is zero and its output NaN, as the formula's 0 / 0.
constexpr float kSeenNothing = -3.0e38f;

// ---------------------------------------------------------------------------------------
// 16 flattened rows: one token's heads, or a few tokens'
// ---------------------------------------------------------------------------------------

// Work item of a workgroup: one KV head, a row tile, and which of its nsplit key splits; its partials
// are at rows slot * (rows of a tile) of the workspace.
struct Item {
  int kvh, nsplit, split;
  int64_t slot;
  TileRef t;
};

// Items of even splits: every row tile has its keys split nsplit ways (fewer if they are few); KV
// head fastest, then row tile (the last one, which sees most, first), then split. (nsplit is the most
// here; the tile's own follows once its positions are read.)
template <int TR>
__device__ __forceinline__ Item even_item(const PagedArgs& a, int b) {
  const Parts n = parts_of<TR>(a);
  const int rest = b / a.num_kv_heads, split = rest / n.tiles;
  const int kvh = b - rest * a.num_kv_heads;
  if (TR == kRowsTile && split >= n.most) return {kvh, n.most, split, 0, {-1, 0, 0, 0}};
  const int tile_idx = n.tiles - 1 - (rest - split * n.tiles);
  return {kvh, n.most, split,
          (static_cast<int64_t>(tile_idx) * a.num_kv_heads + kvh) * n.most + split,
          find_tile<TR>(a, tile_idx)};
}

// Items of one row per request, whose lengths may differ widely: all requests' key tiles together
// are cut into items of about 1 / target of them, so a long request has many and a short one has
// one. `c` counts the items of a KV head. Every wave goes through all positions (a load and two lane
// scans for 64 requests); a row tile's first item leaves its place for the merge, which would have to
// do the same (256 requests of up to 8300 tokens, 14 / 2 heads x 64: 17 us of merge, 1024: 112).
template <int KT>
__device__ __forceinline__ Item balanced_item(const PagedArgs& a, int c, int kvh) {
  const int lane = threadIdx.x & 63;
  const int per = (a.group + kDecodeRows - 1) / kDecodeRows;  // row tiles of a request
  auto tiles_of = [&](int r) -> int {
    const int p = r < a.num_rows ? a.positions[r] : -1;
    return p < 0 ? -1 : key_tiles<KT>(a, p, p).total;
  };
  const int first = tiles_of(lane);
  int64_t all = max(first, 0);
  for (int r = 64; r < a.num_rows; r += 64) all += max(tiles_of(r + lane), 0);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o, 64);
  // Key tiles of an item: one round of kFewSlots items while those are short, because there a
  // workgroup's fixed cost weighs; else `target` items, of which late ones make up for early ones.
  // (32 / 8 heads x 128, one round and 1536 items: 4 requests of up to 8300 tokens 18.7 and 23.5 us,
  // 32 requests 116 and 105, 32 of up to 32K over 4-bit pages 117 and 105.)
  all *= per * a.num_kv_heads;
  int64_t size64 = (all + kFewSlots - 1) / kFewSlots;
  if (size64 > kShortItem)
    size64 = max((all + a.target - 1) / a.target, static_cast<int64_t>(kShortItem));
  const int size = static_cast<int>(max(size64, static_cast<int64_t>(a.min_tiles)));
  Item it = {kvh, 0, 0, 0, {-1, 0, 0, 0}};
  int base = 0;  // items before this block of requests
  for (int r0 = 0; r0 < a.num_rows; r0 += 64) {
    const int tiles = r0 == 0 ? first : tiles_of(r0 + lane);
    const int n = tiles < 0 ? 0 : max((tiles + size - 1) / size, 1);  // items of a row tile
    int incl = n * per;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(incl, d, 64);
      if (lane >= d) incl += y;
    }
    const int before = incl - n * per;
    const uint64_t past = __ballot(c < base + incl);
    if (past) {
      const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
      const int r = r0 + l;
      const int nl = __builtin_amdgcn_readfirstlane(__shfl(n, l, 64));
      const int start = base + __builtin_amdgcn_readfirstlane(__shfl(before, l, 64));
      const int in = c - start;
      it.nsplit = nl;
      it.t = {r, r, 1, in / nl};
      it.split = in - it.t.tile * nl;
      it.slot = static_cast<int64_t>(start + in) * a.num_kv_heads + kvh;
      if (it.split == 0 && threadIdx.x == 0)
        a.part_item[(static_cast<int64_t>(r) * per + it.t.tile) * a.num_kv_heads + kvh] =
            make_int2(static_cast<int>(it.slot), nl);
      return it;
    }
    base += __builtin_amdgcn_readfirstlane(__shfl(incl, 63, 64));
  }
  return it;
}
// Distance of two splits' slots of one row tile.
__device__ __forceinline__ int slot_step(const PagedArgs& a) {
  return a.target > 0 ? a.num_kv_heads : 1;
}
template <int KT>
__device__ __forceinline__ Item decode_item(const PagedArgs& a, int b) {
  if (a.target > 0) {
    const int c = b / a.num_kv_heads;
    return balanced_item<KT>(a, c, b - c * a.num_kv_heads);
  }
  return even_item<kDecodeRows>(a, b);
}

// Joins the states of the workgroup's waves, which each hold (m, l, O) of the same 16 rows in
// `area` ([wave][16][D + 4] fp32, and [wave][16][2] in ml), and writes the output rows or this
// split's partials.
template <int DT, int D, int WAVES>
__device__ __forceinline__ void join_waves(const PagedArgs& a, const float* area, const float* ml,
                                           const Item& it, int nsplit, float out_scale) {
  constexpr int VPR = D / 4;  // float4 per row
  const TileRef& t = it.t;
  for (int i = threadIdx.x; i < kDecodeRows * VPR; i += WAVES * 64) {
    const int row = i / VPR, d = (i % VPR) * 4;
    const int flat = t.tile * kDecodeRows + row;
    if (flat >= t.rows * a.group) continue;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, ml[(w * kDecodeRows + row) * 2]);
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    if (m > -INFINITY) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float mw = ml[(w * kDecodeRows + row) * 2];
        if (mw == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(mw - m);
        l += f * ml[(w * kDecodeRows + row) * 2 + 1];
        const float4 x = *reinterpret_cast<const float4*>(
            area + (static_cast<size_t>(w) * kDecodeRows + row) * (D + 4) + d);
        o[0] += f * x.x, o[1] += f * x.y, o[2] += f * x.z, o[3] += f * x.w;
      }
    }
    const int pi = flat / a.group;
    if (nsplit > 1) {
      const int64_t slot = it.slot * kDecodeRows + row;
      *reinterpret_cast<float4*>(a.part_o + slot * D + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(m, l);
      continue;
    }
    if (a.positions[t.row0 + pi] < 0) continue;
    const float inv = m == -INFINITY ? 0.f : out_scale / l;
    char* op = a.o + (t.row0 + pi) * a.o_row + (it.kvh * a.group + flat - pi * a.group) * a.o_head;
    if constexpr (DT == SB_DTYPE_F32) {
      *reinterpret_cast<float4*>(op + d * 4) =
          make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    } else {
      const uint32_t w0 = Mma<DT>::cvt1(o[0] * inv) | Mma<DT>::cvt1(o[1] * inv) << 16;
      const uint32_t w1 = Mma<DT>::cvt1(o[2] * inv) | Mma<DT>::cvt1(o[3] * inv) << 16;
      *reinterpret_cast<uint2*>(op + d * 2) = make_uint2(w0, w1);
    }
  }
}

__device__ __forceinline__ int64_t lane64(int64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), l);
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// UNIFORM: pages of whole groups of 16 keys (block_size a multiple of 16). A group of 16 keys then
// lies in one page, so its offset is a scalar: the offsets of 32 steps are looked up at once, two
// per step in the lanes, and read from there (the scale bytes' are a sixteenth of the codes', as a
// row's bytes are). Other block sizes and strides look every lane's keys up.
// Four waves: a CU takes in about 40 GB/s whatever it runs, so a workgroup of eight is no faster
// (one row of 1000, 14 / 2 heads x 64: 9.1 against 7.8 us); few long rows are split instead.
// Bound by the pages' bytes: 64 requests under a window of 4096, 32 / 8 heads x 128, bf16, 1.03 GB
// in 171 us, 6.0 TB/s (a large copy reaches 6.6); 32 requests of up to 32K tokens over 4-bit pages
// 588 MB in 105 us, 5.6 TB/s (unpacking takes over 40% of the issue slots there). Few short rows: a
// chain of five memory latencies (arguments, positions, pages, rows, output), about 8 us.
template <int DT, int D, bool Q4, bool UNIFORM>
__global__ __launch_bounds__(kDecodeWaves * 64, Q4 ? 3 : 2) void paged_decode_kernel(const PagedArgs a) {
  using M = Mma<DT>;
  using H = Half<DT>;
  using vec8 = typename M::vec8;
  constexpr int KT = 32;             // keys of a wave's step: two MFMA key blocks
  constexpr int NKS = D / 32;        // QK^T k-steps
  constexpr int NDT = D / 16;        // output d-tiles
  constexpr int CH = D / 8;          // 16-byte chunks of a V row in LDS
  // V rows in LDS, 16-byte chunks XOR-swizzled by row (vchunk): sixteen rows' chunks of one column
  // fall on different banks (the writes), and so do four rows' two chunks of one 16-column tile
  // (the transposing reads). The same memory takes the waves' O at the end.
  constexpr int kArea = kDecodeRows * (D + 4) * 4;
  static_assert(kArea >= KT * D * 2, "O area covers the V stage");
  __shared__ __align__(16) char lds[kDecodeWaves][kArea];
  __shared__ float ml[kDecodeWaves][kDecodeRows][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lq = lane & 15, lg = lane >> 4;
  const Item it = decode_item<KT>(a, blockIdx.x);
  const TileRef& t = it.t;
  if (t.request < 0) return;
  const int kvh = it.kvh;
  const int flat = t.tile * kDecodeRows + lq;
  const bool valid = flat < t.rows * a.group;
  const int pi = valid ? flat / a.group : 0;
  const int p = valid ? a.positions[t.row0 + pi] : -1;
  int pmin = p >= 0 ? p : 0x7fffffff, pmax = p;
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) {
    pmin = min(pmin, __shfl_xor(pmin, o, 64));
    pmax = max(pmax, __shfl_xor(pmax, o, 64));
  }
  pmin = __builtin_amdgcn_readfirstlane(pmin);
  pmax = __builtin_amdgcn_readfirstlane(pmax);
  if (pmax < 0) return;
  const KeyTiles kt = key_tiles<KT>(a, pmin, pmax);
  const int nsplit = a.target > 0 ? it.nsplit : split_count(a, it.nsplit, kt.total);
  if (it.split >= nsplit) return;
  // this wave's share of the split's tiles
  const int64_t share = static_cast<int64_t>(it.split) * kDecodeWaves + wave;
  const int64_t shares = static_cast<int64_t>(nsplit) * kDecodeWaves;
  const int i0 = static_cast<int>(kt.total * share / shares);
  const int i1 = static_cast<int>(kt.total * (share + 1) / shares);

  const int32_t* table = a.tables + t.request * a.table_stride;
  const char* kbase = a.k + kvh * a.c_head;
  const char* vbase = a.v + kvh * a.c_head;
  const char* ksb = a.ks + kvh * a.s_head;
  const char* vsb = a.vs + kvh * a.s_head;

  // Query fragments (B operand). k-slot (step s, lane group lg, j) is dim 32 s + 8 lg + j over
  // 16-bit pages, and dim lg D/4 + 8 s + j over 4-bit ones, where a lane reads D/4 values at once.
  vec8 qf[NKS];
  {
    const char* qp = a.q + (t.row0 + pi) * a.q_row +
                     (kvh * a.group + flat - pi * a.group) * a.q_head;
#pragma unroll
    for (int s = 0; s < NKS; ++s) {
      vec8 v = {};
      const int dim = Q4 ? lg * (D / 4) + 8 * s : 32 * s + 8 * lg;
      if (p >= 0) v = *reinterpret_cast<const vec8*>(qp + dim * 2);
      qf[s] = v;
    }
  }

  // Registers of one step: the raw rows lq and lq + 16 of K and V, this lane's share of each.
  constexpr int RAW = Q4 ? 1 : NKS;
  using raw_t = std::conditional_t<Q4 && D == 64, u32x2_t, u32x4_t>;
  struct Stage {
    raw_t k[2][RAW], v[2][RAW];
    uint32_t sk[2], sv[2];
    uint32_t live;  // which of the step's keys have a page
  };
  const uint32_t lane_row = static_cast<uint32_t>(lq * a.c_pos) + (Q4 ? lg * (D / 8) : 16 * lg);
  const uint32_t lane_scale = static_cast<uint32_t>(lq * a.s_pos) + lg * (D / 32) / 4;
  int64_t group_off = 0;                   // UNIFORM: of group lane & 1 of step lane / 2
  uint64_t group_live = 0;
  // else the table's entries for keys lq and lq + 16 of the step that is fetched next, and of the one
  // behind it (requested before that fetch, whose loads need not be waited for then)
  int entry[2] = {-1, -1}, entry_next[2] = {-1, -1};
  auto lookup = [&](int idx) {
    if constexpr (UNIFORM) {
      if (((idx - i0) & 31) != 0 || idx >= i1) return;
      const int step = min(idx + (lane >> 1), i1 - 1);
      const int key = tile_key<KT>(kt, step) + 16 * (lane & 1);
      const int pb = page_of(a, table, key);
      group_off = row_offset(a, key, pb, a.c_block, a.c_pos);
      group_live = __ballot(pb >= 0);
    } else {
      const int k0 = tile_key<KT>(kt, min(idx, i1 - 1));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        entry[h] = entry_next[h];
        entry_next[h] = page_entry(a, table, k0 + 16 * h + lq);
      }
    }
  };
  auto fetch = [&](int idx, Stage& st) {  // (behind lookup(idx))
    if constexpr (UNIFORM) {
      const int at = 2 * ((idx - i0) & 31);
      const uint32_t two = static_cast<uint32_t>(group_live >> at) & 3u;
      st.live = (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // (the group's address stays in scalar registers, the lane's part is one of 32 bits)
        const int64_t off = lane64(group_off, at + h);
        const SB_GLOBAL char* kg = (const SB_GLOBAL char*)(kbase + off);
        const SB_GLOBAL char* vg = (const SB_GLOBAL char*)(vbase + off);
        asm volatile("" : "+s"(kg), "+s"(vg));
#pragma unroll
        for (int s = 0; s < RAW; ++s) {
          // (nontemporal for 4-bit rows: 32 requests of up to 32K tokens 119 -> 107 us; 16-bit
          // ones lose by it, 64 requests under a window of 4096 170 -> 181 us)
          const SB_GLOBAL raw_t* kr = (const SB_GLOBAL raw_t*)(kg + lane_row + 64 * s);
          const SB_GLOBAL raw_t* vr = (const SB_GLOBAL raw_t*)(vg + lane_row + 64 * s);
          st.k[h][s] = Q4 ? __builtin_nontemporal_load(kr) : *kr;
          st.v[h][s] = Q4 ? __builtin_nontemporal_load(vr) : *vr;
        }
        if constexpr (Q4) {
          const SB_GLOBAL char* ksg = (const SB_GLOBAL char*)(ksb + (off >> 4));
          const SB_GLOBAL char* vsg = (const SB_GLOBAL char*)(vsb + (off >> 4));
          asm volatile("" : "+s"(ksg), "+s"(vsg));
          st.sk[h] = static_cast<uint8_t>(ksg[lane_scale]);
          st.sv[h] = static_cast<uint8_t>(vsg[lane_scale]);
        }
      }
    } else {
      const int k0 = tile_key<KT>(kt, idx);
      const int page[2] = {page_in(a, entry[0], k0 + lq), page_in(a, entry[1], k0 + 16 + lq)};
      st.live = static_cast<uint32_t>(__ballot(page[0] >= 0) & 0xffffu) |
                static_cast<uint32_t>(__ballot(page[1] >= 0) & 0xffffu) << 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = k0 + 16 * h + lq;
        const int64_t off = row_offset(a, key, page[h], a.c_block, a.c_pos);
#pragma unroll
        for (int s = 0; s < RAW; ++s) {
          const int64_t at = off + (Q4 ? lg * (D / 8) : 64 * s + 16 * lg);
          st.k[h][s] = *reinterpret_cast<const raw_t*>(kbase + at);
          st.v[h][s] = *reinterpret_cast<const raw_t*>(vbase + at);
        }
        if constexpr (Q4) {
          const int64_t so =
              row_offset(a, key, page[h], a.s_block, a.s_pos) + lg * (D / 32) / 4;
          st.sk[h] = static_cast<uint8_t>(ksb[so]);
          st.sv[h] = static_cast<uint8_t>(vsb[so]);
        }
      }
    }
  };

  float m_ref = -INFINITY, negm = 0.f, l_run = 0.f;
  bool seen = false;
  f32x4 o[NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) o[d] = f32x4{};
  const float c_log2 = Q4 ? a.scale_log2 * (1 << H::kShift) : a.scale_log2;
  char* vst = lds[wave];
  auto vchunk = [&](int row, int c) -> int {  // byte offset of chunk c of a row
    const int y = CH >= 16 ? row & 15 : (row >> 1) & 7;
    const int x = CH >= 16 ? (y & 7) << 1 | y >> 3 : (y & 3) << 1 | y >> 2;
    return row * (D * 2) + 16 * (c ^ x);
  };

  int odd_first = 0x7fffffff, odd_last = -1;  // tiles that V values were taken out of
  auto step = [&](int idx, Stage& st) {
    const int k0 = tile_key<KT>(kt, idx);
    const uint32_t live = st.live;
    const bool whole = live == 0xffffffffu && k0 + KT - 1 <= pmin &&
                       (k0 > pmax - a.window || k0 + KT - 1 < a.sinks);
    bool taken = false;  // (wave-uniform) some of this tile's V is not finite and is taken out
    if (!whole) {  // values that are not finite are taken out of V, and added where they are seen
      bool odd;
      if constexpr (Q4) {
        // (the scale byte decides: the values are looked at below, where they are converted)
        odd = st.sv[0] >= H::kInfByte || st.sv[1] >= H::kInfByte;
      } else {
        uint32_t bits = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int s = 0; s < NKS; ++s) bits |= not_finite_bits<DT>(st.v[h][s]);
        odd = (bits & kNotFinite) != 0;
        if (odd) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < NKS; ++s) st.v[h][s] = finite_part<DT>(st.v[h][s]);
        }
      }
      taken = __any(odd);
      if (taken) {
        odd_first = min(odd_first, idx);
        odd_last = idx;
      }
    }
    // V rows to LDS
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * h + lq;
      if constexpr (Q4) {
        const float sc = scale_of<H::kShift>(st.sv[h]);
#pragma unroll
        for (int s = 0; s < NKS; ++s)
          *reinterpret_cast<u32x4_t*>(vst + vchunk(row, lg * NKS + s)) =
              fp4x8<DT>(st.v[h][0][s], sc);
      } else {
#pragma unroll
        for (int s = 0; s < NKS; ++s)
          *reinterpret_cast<u32x4_t*>(vst + vchunk(row, 4 * s + lg)) = st.v[h][s];
      }
    }
    if (Q4 && taken) {  // (the stage read back by words: values held in registers would spill)
      asm volatile("" ::: "memory");
#pragma unroll 1
      for (int c = 0; c < KT * D / 2; c += 64) {
        uint32_t* at = reinterpret_cast<uint32_t*>(vst) + c + lane;
        *at = finite_part<DT>(*at);
      }
      asm volatile("" ::: "memory");
    }
    // S^T = K Q^T: lane (lq, lg) gets row lq's scores of keys 16 h + 4 lg + 0..3
    f32x4 sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4{};
      const float ksc = Q4 ? scale_of<H::kShift>(st.sk[h]) : 0.f;
#pragma unroll
      for (int s = 0; s < NKS; ++s) {
        u32x4_t w;
        if constexpr (Q4) w = fp4x8<DT>(st.k[h][0][s], ksc);
        else w = st.k[h][s];
        sc[h] = H::mma16(__builtin_bit_cast(vec8, w), qf[s], sc[h]);
      }
    }
    if (whole) {
      seen = true;
    } else {
      const uint32_t on = (seen_bits(a, p, k0) & live) >> (4 * lg);
      seen |= (on & 0x000f000fu) != 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(on >> (16 * h + e) & 1u)) sc[h][e] = -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                      fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    // The reference moves only when a weight would pass 2^8: the row's largest score so far
    // otherwise lies within 2^8 of it, which costs no accuracy in fp32 sums.
    if (__any(__builtin_fmaf(c_log2, top, negm) > (m_ref == -INFINITY ? -INFINITY : 8.f))) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float x = c_log2 * top;
      if (x > m_ref) {
        const float f = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - x);
        l_run *= f;
#pragma unroll
        for (int d = 0; d < NDT; ++d) o[d] *= f;
        m_ref = x;
        negm = -x;
      }
    }
    float pf[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pf[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(c_log2, sc[0][e], negm));
      pf[4 + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(c_log2, sc[1][e], negm));
    }
    const vec8 pb = M::cvt8(pf);  // rounded weights, which the sum takes as well
    l_run = M::sum8(pb, l_run);
    // O^T += V^T P^T. Weight slot (lg, j) is key 4 lg + j, or 16 + 4 lg + j - 4: two transposing
    // reads give lane (lq, lg) its column of those keys.
    asm volatile("" ::: "memory");
#pragma unroll
    for (int d = 0; d < NDT; ++d) {
      u32x2_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = 16 * h + 4 * lg + (lq >> 2), col = 16 * d + 4 * (lq & 3);
        const char* src = vst + vchunk(row, col >> 3) + (col & 7) * 2;
        w[h] = __builtin_bit_cast(u32x2_t,
                                  __builtin_amdgcn_ds_read_tr16_b64_v4i16((SB_LDS s16x4_t*)src));
      }
      const u32x4_t v = {w[0].x, w[0].y, w[1].x, w[1].y};
      o[d] = H::mma16(__builtin_bit_cast(vec8, v), pb, o[d]);
    }
    asm volatile("" ::: "memory");
  };

  // Steps ahead in registers: 4-bit rows are an eighth of a step's registers and latency shows,
  // 16-bit ones fill them with one.
  constexpr int PD = UNIFORM && Q4 ? kDecodeAhead4 : 1;
  // Every trip issues its loads, past the end those of the last step again: behind a branch the
  // compiler would have to wait for all of them, the ones just issued as well.
  Stage st[PD + 1];
  if (i0 < i1) {
    lookup(i0);
#pragma unroll
    for (int x = 0; x < PD; ++x) {
      if (!UNIFORM) lookup(i0 + x + 1);
      fetch(min(i0 + x, i1 - 1), st[x]);
    }
    int i = i0;
    for (; i + PD < i1; i += PD + 1) {
#pragma unroll
      for (int u = 0; u <= PD; ++u) {
        lookup(UNIFORM ? i + u + PD : i + u + PD + 1);
        fetch(min(i + u + PD, i1 - 1), st[(u + PD) % (PD + 1)]);
        step(i + u, st[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < PD; ++u)
      if (i + u < i1) step(i + u, st[u]);
  }

  // What was taken out, added where it is seen: an infinity or a NaN of a seen key decides the sum,
  // whatever (positive) weight it has.
  for (int x = odd_first; x <= odd_last; ++x) {
    const int k0 = tile_key<KT>(kt, x);
    const uint64_t has = __ballot(page_of(a, table, k0 + (lane & 31)) >= 0);
    if (has == ~0ull && k0 + KT - 1 <= pmin && (k0 > pmax - a.window || k0 + KT - 1 < a.sinks))
      continue;  // (seen whole: nothing was taken out)
    for (int r = 0; r < KT; ++r) {
      const int key = k0 + r, pb = page_of(a, table, key);
      const bool on = pb >= 0 && sees(a, p, key);
      if (!__any(on)) continue;
      const char* row = vbase + row_offset(a, key, pb, a.c_block, a.c_pos);
      const char* sr = Q4 ? vsb + row_offset(a, key, pb, a.s_block, a.s_pos) : nullptr;
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        if constexpr (Q4) {
          const uint32_t byte = static_cast<uint8_t>(sr[d / 2]);
          if (on && byte >= H::kInfByte) {
            const uint32_t c = *reinterpret_cast<const uint16_t*>(row + 8 * d + 2 * lg);
            add_not_finite<DT>(fp4x4<DT>(c, scale_of<H::kShift>(byte)), o[d], 0);
          }
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(row + 2 * (16 * d + 4 * lg));
          if (on) add_not_finite<DT>(w, o[d], 0);
        }
      }
    }
  }

  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  const int any_seen = static_cast<int>(seen) | __shfl_xor(static_cast<int>(seen), 16, 64);
  const bool row_seen = (any_seen | __shfl_xor(any_seen, 32, 64)) != 0;
  if (lg == 0) {
    ml[wave][lq][0] = m_ref == -INFINITY && row_seen ? kSeenNothing : m_ref;
    ml[wave][lq][1] = l_run;
  }
  float* area = reinterpret_cast<float*>(vst);
#pragma unroll
  for (int d = 0; d < NDT; ++d)
    *reinterpret_cast<f32x4*>(area + lq * (D + 4) + 16 * d + 4 * lg) = o[d];
  __syncthreads();
  join_waves<DT, D, kDecodeWaves>(a, reinterpret_cast<const float*>(&lds[0][0]), &ml[0][0][0], it, nsplit,
                                  Q4 ? static_cast<float>(1 << H::kShift) : 1.f);
}

// fp32 pages: v_mfma_f32_16x16x4_f32, 16 keys a step. Lane (lq, lg) holds of K row lq the dims
// 16 c + 4 lg + 0..3 of every c (one 16-byte load each; k-step (c, e) multiplies dim
// 16 c + 4 lg + e), and of V rows 4 lg + s the dims 64 u + 4 lq + 0..3: element e of them is the A
// operand of output tile (u, e), whose row m is dim 64 u + 4 m + e, so V needs no transposition.
// Weight s of a lane is key 4 lg + s, as the scores leave it. (154 rows of a context of 1024, 14 / 2
// heads x 64, window 300: 10.5 us, the chain of latencies above and five key tiles per wave; with
// every lane looking its keys up, as for pages that are no multiple of 16 tokens, 11.2.)
template <int D, bool UNIFORM>
__global__ __launch_bounds__(kDecodeWaves * 64, 2) void paged_f32_kernel(const PagedArgs a) {
  constexpr int KT = 16;
  constexpr int NC = D / 16, NU = D / 64;
  __shared__ __align__(16) float area[kDecodeWaves][kDecodeRows][D + 4];
  __shared__ float ml[kDecodeWaves][kDecodeRows][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lq = lane & 15, lg = lane >> 4;
  const Item it = decode_item<KT>(a, blockIdx.x);
  const TileRef& t = it.t;
  if (t.request < 0) return;
  const int kvh = it.kvh;
  const int flat = t.tile * kDecodeRows + lq;
  const bool valid = flat < t.rows * a.group;
  const int pi = valid ? flat / a.group : 0;
  const int p = valid ? a.positions[t.row0 + pi] : -1;
  int pmin = p >= 0 ? p : 0x7fffffff, pmax = p;
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) {
    pmin = min(pmin, __shfl_xor(pmin, o, 64));
    pmax = max(pmax, __shfl_xor(pmax, o, 64));
  }
  pmin = __builtin_amdgcn_readfirstlane(pmin);
  pmax = __builtin_amdgcn_readfirstlane(pmax);
  if (pmax < 0) return;
  const KeyTiles kt = key_tiles<KT>(a, pmin, pmax);
  const int nsplit = a.target > 0 ? it.nsplit : split_count(a, it.nsplit, kt.total);
  if (it.split >= nsplit) return;
  const int64_t share = static_cast<int64_t>(it.split) * kDecodeWaves + wave;
  const int64_t shares = static_cast<int64_t>(nsplit) * kDecodeWaves;
  const int i0 = static_cast<int>(kt.total * share / shares);
  const int i1 = static_cast<int>(kt.total * (share + 1) / shares);

  const int32_t* table = a.tables + t.request * a.table_stride;
  const char* kbase = a.k + kvh * a.c_head;
  const char* vbase = a.v + kvh * a.c_head;
  f32x4 qf[NC];
  {
    const char* qp = a.q + (t.row0 + pi) * a.q_row +
                     (kvh * a.group + flat - pi * a.group) * a.q_head + 16 * lg;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      f32x4 v = {};
      if (p >= 0) v = *reinterpret_cast<const f32x4*>(qp + 64 * c);
      qf[c] = v;
    }
  }
  struct Stage {
    f32x4 k[NC], v[4][NU];
    uint32_t live;  // which of the step's keys have a page
  };
  // UNIFORM (as in paged_decode_kernel): the offsets of 64 steps, looked up at once, one per lane;
  // else the table's entries for key lq of the step that is fetched next and of the one behind it
  // (requested before that fetch, whose loads need not be waited for then).
  int64_t group_off = 0;
  uint64_t group_live = 0;
  int entry = -1, entry_next = -1;
  auto lookup = [&](int idx) {
    if constexpr (UNIFORM) {
      if (((idx - i0) & 63) != 0 || idx >= i1) return;
      const int key = tile_key<KT>(kt, min(idx + lane, i1 - 1));
      const int pb = page_of(a, table, key);
      group_off = row_offset(a, key, pb, a.c_block, a.c_pos);
      group_live = __ballot(pb >= 0);
    } else {
      entry = entry_next;
      entry_next = page_entry(a, table, tile_key<KT>(kt, min(idx, i1 - 1)) + lq);
    }
  };
  const uint32_t lane_k = static_cast<uint32_t>(lq * a.c_pos) + 16 * lg;
  auto fetch = [&](int idx, Stage& st) {  // (behind lookup(idx))
    if constexpr (UNIFORM) {
      const int at = (idx - i0) & 63;
      st.live = (group_live >> at & 1u) ? 0xffffu : 0u;
      const int64_t off = lane64(group_off, at);
      const SB_GLOBAL char* kg = (const SB_GLOBAL char*)(kbase + off);
      const SB_GLOBAL char* vg = (const SB_GLOBAL char*)(vbase + off);
      asm volatile("" : "+s"(kg), "+s"(vg));
#pragma unroll
      for (int c = 0; c < NC; ++c) st.k[c] = *(const SB_GLOBAL f32x4*)(kg + lane_k + 64 * c);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t lane_v = static_cast<uint32_t>((4 * lg + x) * a.c_pos) + 16 * lq;
#pragma unroll
        for (int u = 0; u < NU; ++u) st.v[x][u] = *(const SB_GLOBAL f32x4*)(vg + lane_v + 256 * u);
      }
    } else {
      const int key = tile_key<KT>(kt, idx) + lq;
      const int page = page_in(a, entry, key);
      st.live = static_cast<uint32_t>(__ballot(page >= 0) & 0xffffu);
      const int64_t off = row_offset(a, key, page, a.c_block, a.c_pos);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        st.k[c] = *reinterpret_cast<const f32x4*>(kbase + off + 16 * lg + 64 * c);
#pragma unroll
      for (int x = 0; x < 4; ++x) {  // the offset of key 4 lg + x is lane 4 lg + x's
        const int64_t vo = __shfl(off, 4 * lg + x, 64);
#pragma unroll
        for (int u = 0; u < NU; ++u)
          st.v[x][u] = *reinterpret_cast<const f32x4*>(vbase + vo + 16 * lq + 256 * u);
      }
    }
  };
  float m_ref = -INFINITY, negm = 0.f, l_run = 0.f;
  bool seen = false;
  f32x4 o[NU][4];
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[u][e] = f32x4{};
  const float c_hi = a.scale_log2, c_lo = a.scale_log2_lo;

  int odd_first = 0x7fffffff, odd_last = -1;
  auto step = [&](int idx, Stage& st, Stage& ahead) {
    const int k0 = tile_key<KT>(kt, idx);
    auto& v = st.v;
    lookup(UNIFORM ? idx + 1 : idx + 2);
    fetch(min(idx + 1, i1 - 1), ahead);
    f32x4 sc[2] = {f32x4{}, f32x4{}};  // two chains
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sc[c & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(st.k[c][e], qf[c][e], sc[c & 1], 0, 0, 0);
    f32x4 s = sc[0] + sc[1];
    const uint32_t live = st.live;
    const bool whole = live == 0xffffu && k0 + KT - 1 <= pmin &&
                       (k0 > pmax - a.window || k0 + KT - 1 < a.sinks);
    if (whole) {
      seen = true;
    } else {
      bool odd = false;  // as in paged_decode_kernel
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(fabsf(v[x][u][e]) < INFINITY)) odd = true, v[x][u][e] = 0.f;
      if (__any(odd)) {
        odd_first = min(odd_first, idx);
        odd_last = idx;
      }
      const uint32_t on = (seen_bits(a, p, k0) & live) >> (4 * lg);
      seen |= (on & 15u) != 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(on >> e & 1u)) s[e] = -INFINITY;
    }
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    if (__any(__builtin_fmaf(c_hi, top, negm) > (m_ref == -INFINITY ? -INFINITY : 8.f))) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float x = c_hi * top;
      if (x > m_ref) {
        const float f = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_ref - x);
        l_run *= f;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[u][e] *= f;
        m_ref = x;
        negm = -x;
      }
    }
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // (scale * log2(e) in two parts: rounded alone it would be off by 2^-25 of the score)
      w[e] = s[e] == -INFINITY
                 ? 0.f
                 : __builtin_amdgcn_exp2f(__builtin_fmaf(c_hi, s[e], __builtin_fmaf(c_lo, s[e], negm)));
      l_run += w[e];
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[u][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[x][u][e], w[x], o[u][e], 0, 0, 0);
  };

  // K and V one step ahead in registers, the pages two. (Loads past the end are those of the last
  // step again, as in paged_decode_kernel.)
  Stage st[2];
  if (i0 < i1) {
    lookup(i0);
    if (!UNIFORM) lookup(i0 + 1);
    fetch(i0, st[0]);
    int i = i0;
    for (; i + 1 < i1; i += 2) {
      step(i, st[0], st[1]);
      step(i + 1, st[1], st[0]);
    }
    if (i < i1) step(i, st[0], st[1]);
  }
  for (int x = odd_first; x <= odd_last; ++x) {
    const int k0 = tile_key<KT>(kt, x);
    const uint64_t has = __ballot(page_of(a, table, k0 + lq) >= 0);
    if (has == ~0ull && k0 + KT - 1 <= pmin && (k0 > pmax - a.window || k0 + KT - 1 < a.sinks))
      continue;
    for (int r = 0; r < KT; ++r) {
      const int key = k0 + r, pb = page_of(a, table, key);
      const bool on = pb >= 0 && sees(a, p, key);
      if (!__any(on)) continue;
      const char* row =
          a.v + kvh * a.c_head + row_offset(a, key, pb, a.c_block, a.c_pos);
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(row + 4 * (64 * u + 16 * lg + 4 * y));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (on && !(fabsf(w[e]) < INFINITY)) o[u][e][y] += w[e];
        }
    }
  }
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  const int any_seen = static_cast<int>(seen) | __shfl_xor(static_cast<int>(seen), 16, 64);
  const bool row_seen = (any_seen | __shfl_xor(any_seen, 32, 64)) != 0;
  if (lg == 0) {
    ml[wave][lq][0] = m_ref == -INFINITY && row_seen ? kSeenNothing : m_ref;
    ml[wave][lq][1] = l_run;
  }
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x4 w = {o[u][0][x], o[u][1][x], o[u][2][x], o[u][3][x]};
      *reinterpret_cast<f32x4*>(&area[wave][lq][64 * u + 16 * lg + 4 * x]) = w;
    }
  __syncthreads();
  join_waves<SB_DTYPE_F32, D, kDecodeWaves>(a, &area[0][0][0], &ml[0][0][0], it, nsplit, 1.f);
}

// ---------------------------------------------------------------------------------------
// 256 flattened rows: prompt chunks
// ---------------------------------------------------------------------------------------

// One workgroup of 8 waves, 32 rows each; K and V tiles of 64 keys in two LDS stages, filled while
// the stage before is multiplied: 16-bit rows by direct-to-LDS loads, 4-bit ones through registers
// (fetched a tile ahead, converted and written behind the products of the tile before). S^T = K Q^T
// and O^T += V^T P^T with v_mfma_f32_32x32x16 (a lane owns one row), V through transposing reads.
// Bound by instruction issue: 2.1 us a key tile at 28 / 4 heads x 128 (1.8 GHz under this load), of
// which the products take 1.1, and by the three dependent loads in front of a workgroup's first
// tile and its output, 10 us together (8192 rows under a window of 1024: 170-195 us by card, 18
// tiles a workgroup; 512 rows over 16384 keys of 4-bit pages: 144 us).
template <int DT, int D, bool Q4>
__global__ __launch_bounds__(kRowsWaves * 64, 1) void paged_rows_kernel(const PagedArgs a) {
  using M = Mma<DT>;
  using H = Half<DT>;
  using vec8 = typename M::vec8;
  constexpr int KT = 64;
  constexpr int THREADS = kRowsWaves * 64;
  constexpr int NKS = D / 16, NDT = D / 32, CH = D / 8;
  constexpr int NLD = KT * CH / THREADS;      // 16-byte loads per thread and plane
  __shared__ __align__(16) uint16_t Ks[2][KT * D];
  __shared__ __align__(16) uint16_t Vs[2][KT * D];
  __shared__ int red[2][kRowsWaves];
  __shared__ int odd_tiles[2];  // first and last tile that look_over took values out of

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, lq = lane & 31, lg = lane >> 5;
  const Item it = even_item<kRowsTile>(a, blockIdx.x);
  const TileRef& t = it.t;
  if (t.request < 0) return;
  const int flat = t.tile * kRowsTile + wave * 32 + lq;
  const bool valid = flat < static_cast<int64_t>(t.rows) * a.group;
  const int pi = valid ? flat / a.group : 0;
  const int head = it.kvh * a.group + (valid ? flat - pi * a.group : 0);
  const int p = valid ? a.positions[t.row0 + pi] : -1;
  const int pmin = __builtin_amdgcn_readfirstlane(wave_min_i(p >= 0 ? p : 0x7fffffff));
  const int pmax = __builtin_amdgcn_readfirstlane(wave_max_i(p));
  if (lane == 0) {
    red[0][wave] = pmin;
    red[1][wave] = pmax;
  }
  if (tid < 2) odd_tiles[tid] = tid ? -1 : 0x7fffffff;
  __syncthreads();
  int tmin = red[0][0], tmax = red[1][0];
#pragma unroll
  for (int w = 1; w < kRowsWaves; ++w) {
    tmin = min(tmin, red[0][w]);
    tmax = max(tmax, red[1][w]);
  }
  tmin = __builtin_amdgcn_readfirstlane(tmin);
  tmax = __builtin_amdgcn_readfirstlane(tmax);
  if (tmax < 0) return;  // uniform
  const KeyTiles kt = key_tiles<KT>(a, tmin, tmax);
  const int nsplit = split_count(a, it.nsplit, kt.total);
  if (it.split >= nsplit) return;  // uniform
  const int i0 = static_cast<int>(static_cast<int64_t>(kt.total) * it.split / nsplit);
  const int i1 = static_cast<int>(static_cast<int64_t>(kt.total) * (it.split + 1) / nsplit);

  const int32_t* table = a.tables + t.request * a.table_stride;
  const char* kbase = a.k + it.kvh * a.c_head;
  const char* vbase = a.v + it.kvh * a.c_head;
  const char* ksb = a.ks + it.kvh * a.s_head;
  const char* vsb = a.vs + it.kvh * a.s_head;

  vec8 qf[NKS];
  {
    const char* qp = a.q + (t.row0 + pi) * a.q_row + head * a.q_head;
#pragma unroll
    for (int s = 0; s < NKS; ++s) {
      vec8 v = {};
      if (p >= 0) v = *reinterpret_cast<const vec8*>(qp + (16 * s + 8 * lg) * 2);
      qf[s] = v;
    }
  }

  // Byte offsets of the keys' rows, in a ring of tiles (K and V rows share one; 4-bit pages have a
  // second for the scale bytes), and which keys have a page. One wave fills a tile's: it reads the
  // block table one iteration and writes the offsets the next. 4-bit codes are fetched an iteration
  // before they are written to LDS, so their offsets are needed one earlier.
  constexpr int RING = Q4 ? 4 : 3;
  __shared__ int64_t ofs[RING][KT];
  __shared__ int64_t sofs[Q4 ? RING : 1][Q4 ? KT : 1];
  __shared__ uint64_t paged[RING];
  auto slot_at = [](int slot, int x) { return slot + x >= RING ? slot + x - RING : slot + x; };
  const int n = i1 - i0;  // key tiles of this workgroup
  auto key_of = [&](int i) { return tile_key<KT>(kt, i0 + i); };
  auto fill = [&](int slot, int i, int key_in_tile, int page) {
    const int key = key_of(i) + key_in_tile;
    ofs[slot][key_in_tile] = row_offset(a, key, page, a.c_block, a.c_pos);
    if constexpr (Q4) sofs[slot][key_in_tile] = row_offset(a, key, page, a.s_block, a.s_pos);
    const uint64_t has = __ballot(page >= 0);
    if (lane == 0) paged[slot] = has;
  };
  if (wave < RING) fill(wave, wave, lane, wave < n ? page_of(a, table, key_of(wave) + lane) : -1);
  int ahead = -1;  // page of key `lane` of the tile that this wave fills next
  if (n > RING && wave == (RING & 3)) ahead = page_of(a, table, key_of(RING) + lane);

  // 16-bit pages: load q of a plane fills LDS slots q * THREADS + tid: row q * (THREADS / CH) +
  // tid / CH at chunk tid % CH, which holds the row's chunk that the swizzle puts there.
  const char* ksrc = kbase + 16 * kswz<CH>(tid / CH, tid % CH);
  const char* vsrc = vbase + 16 * vswz<CH>(tid / CH, tid % CH);
  auto read_ofs = [&](int slot, int64_t* ro) {
#pragma unroll
    for (int q = 0; q < NLD; ++q) ro[q] = ofs[slot][q * (THREADS / CH) + tid / CH];
  };
  auto dma_dst = [&](uint16_t* dst, int q) -> uint32_t {
    return lds_addr(dst) + (q * THREADS + wave * 64) * 16;
  };
  // 4-bit pages: thread tid converts D / 8 values of row tid / 8, read one tile ahead. (tid through
  // an empty asm: its addresses are formed anew in each iteration rather than held in registers
  // that the score block needs.)
  int tid4 = tid;
  constexpr int NW = D / 64;  // words of 8 codes
  using code_t = std::conditional_t<NW == 2, u32x2_t, uint32_t>;
  struct Codes {
    code_t w;
    uint32_t scale;
  };
  auto fetch = [&](const char* codes, const char* scales, int slot) -> Codes {
    Codes c;
    const int row = tid4 >> 3, part = tid4 & 7;
    c.w = *reinterpret_cast<const code_t*>(codes + ofs[slot][row] + part * (4 * NW));
    c.scale = static_cast<uint8_t>(scales[sofs[slot][row] + part * NW / 4]);
    return c;
  };
  auto unpack = [&](const Codes& c, uint16_t* dst, auto is_v) {
    const float sc = scale_of<H::kShift>(c.scale);
    uint32_t w[NW];
    __builtin_memcpy(w, &c.w, 4 * NW);
    const int row = tid4 >> 3, part = tid4 & 7;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const int ch = part * NW + x;
      const int at = decltype(is_v)::value ? vswz<CH>(row, ch) : kswz<CH>(row, ch);
      *reinterpret_cast<u32x4_t*>(reinterpret_cast<char*>(dst) + row * (D * 2) + 16 * at) =
          fp4x8<DT>(w[x], sc);
    }
  };
  using IsV = std::true_type;
  using IsK = std::false_type;

  // Looks this thread's part of V of tile i over, if the tile is one that some row of the
  // workgroup sees only in part (before the barrier that publishes the tile): values that are not
  // finite are taken out of it, and the tile is noted for `put_back`.
  auto in_part = [&](int k0, uint64_t has) -> bool {
    return !(has == ~0ull && k0 + KT - 1 <= tmin &&
             (k0 > tmax - a.window || k0 + KT - 1 < a.sinks));
  };
  auto look_over = [&](int i, int slot, int stage, uint32_t scale) {
    if (!in_part(key_of(i), paged[slot])) return;
    bool odd = false;
    if constexpr (Q4) {
      odd = scale >= H::kInfByte;
      if (odd) {
        const int row = tid4 >> 3, part = tid4 & 7;
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          u32x4_t* at = reinterpret_cast<u32x4_t*>(reinterpret_cast<char*>(Vs[stage]) + row * (D * 2) +
                                                   16 * vswz<CH>(row, part * NW + x));
          *at = finite_part<DT>(*at);
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < NLD; ++q) {
        u32x4_t* at = reinterpret_cast<u32x4_t*>(reinterpret_cast<char*>(Vs[stage]) +
                                                 (q * THREADS + tid) * 16);
        const u32x4_t v = *at;
        if ((not_finite_bits<DT>(v) & kNotFinite) == 0) continue;
        odd = true;
        *at = finite_part<DT>(v);
      }
    }
    if (odd) {
      atomicMin(&odd_tiles[0], i);
      atomicMax(&odd_tiles[1], i);
    }
  };

  // K fragment (half j, step k): row 32 j + lq, chunk 2 k + lg. V^T fragment (d-tile d, step s,
  // half j): keys 32 j + 16 s + {4 lg + 0..3, 8 + 4 lg + 0..3}, the order of the weights. Both
  // swizzles depend on the row modulo 16 at most: a lane's part of each address, and a constant.
  int kl[NKS], vl[NDT];
#pragma unroll
  for (int k = 0; k < NKS; ++k) kl[k] = lq * D * 2 + 16 * kswz<CH>(lq, 2 * k + lg);
  const int grp = lane >> 4, gi = lane & 15;
#pragma unroll
  for (int d = 0; d < NDT; ++d) {
    const int col = 32 * d + 16 * (grp & 1) + 4 * (gi & 3);
    const int row = 4 * lg + (gi >> 2);
    vl[d] = 2 * (row * D + 8 * vswz<CH>(row, col >> 3) + (col & 7));
  }
  auto kfrag = [&](int stage, int m) -> vec8 {  // m = 2 k + j
    return *reinterpret_cast<const vec8*>(reinterpret_cast<const char*>(&Ks[0][0]) +
                                          stage * (KT * D * 2) + (m & 1) * (32 * D * 2) +
                                          kl[m >> 1]);
  };
  auto vfrag = [&](int stage, int m) -> u32x4_t {  // m = (2 j + s) NDT + d
    const int d = m % NDT, s = (m / NDT) & 1, j = m / (2 * NDT);
    u32x2_t h[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const char* src = reinterpret_cast<const char*>(&Vs[0][0]) + stage * (KT * D * 2) +
                        (32 * j + 16 * s + 8 * e) * (D * 2) + vl[d];
      h[e] = __builtin_bit_cast(u32x2_t,
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((SB_LDS s16x4_t*)src));
    }
    const u32x4_t w = {h[0].x, h[0].y, h[1].x, h[1].y};
    return w;
  };

  const float c_log2 = Q4 ? a.scale_log2 * (1 << H::kShift) : a.scale_log2;
  float m_ref = 0.f, negm = 0.f, l_run = 0.f;
  bool seeded = p < 0, seen = false;
  f32x16_t o[NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) o[d] = f32x16_t{};
  using Scores = f32x16_t[2];
  constexpr int NQ = 2 * NKS, NV = 4 * NDT;

  // Whether every row of this wave sees all of tile i (then its scores are taken as they are).
  auto whole = [&](int i, int slot) -> bool {
    const int k0 = key_of(i);
    return paged[slot] == ~0ull && k0 + KT - 1 <= pmin &&
           (k0 > pmax - a.window || k0 + KT - 1 < a.sinks);
  };
  auto mask = [&](int i, int slot, Scores& sc) {
    if (__builtin_amdgcn_readfirstlane(whole(i, slot))) {
      seen = true;
      return;
    }
    const int k0 = key_of(i);
    const uint64_t has = paged[slot];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t on =
          (seen_bits(a, p, k0 + 32 * j) & static_cast<uint32_t>(has >> (32 * j))) >> (4 * lg);
      seen |= (on & 0x0f0f0f0fu) != 0;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(on >> (8 * (e >> 2) + (e & 3)) & 1u)) sc[j][e] = -INFINITY;
    }
  };
  vec8 pb[2][2];
  float tsum = 0.f;
  auto weights = [&](const Scores& sc) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          f[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(c_log2, sc[j][8 * s + e], negm));
        pb[j][s] = M::cvt8(f);
        t = M::sum8(pb[j][s], t);
      }
    tsum = t;
  };

  // Iteration i: S(i + 1) = K Q^T on the matrix cores while the weights of tile i are formed from
  // S(i), then O += V(i)^T P(i). K runs two tiles ahead of its use and V one, each in two LDS
  // stages; one barrier per tile. The first block is laid out by hand, as attn_mfma_kernel's is:
  // step m reads the K fragment of step m + kAhead, issues one MFMA, then fma, exp2 and packing of
  // three successive weight pairs, so that no instruction waits for another of its own step; tile
  // loads of 16-bit pages ride on the first steps.
  Codes ck = {}, cv = {};  // of K(i + 2) and V(i + 1) at the top of iteration i
  auto iteration = [&](int i, int slot, auto has_next, auto parity, auto swap, Scores& s_cur,
                       Scores& s_nxt, auto full) {
    constexpr bool NEXT = decltype(has_next)::value;
    constexpr bool FULL = decltype(full)::value;  // both loads are due
    constexpr int PAR = decltype(parity)::value;
    const int par = PAR >= 0 ? PAR : (i & 1);
    if (PAR >= 0) {
      // (carried through an empty asm, so that the stage constants fold into the LDS offsets)
#pragma unroll
      for (int k = 0; k < NKS; ++k) asm volatile("" : "+v"(kl[k]));
#pragma unroll
      for (int d = 0; d < NDT; ++d) asm volatile("" : "+v"(vl[d]));
    }
    const int slot1 = slot_at(slot, 1), slot2 = slot_at(slot, 2);
    int64_t ro_k[NLD], ro_v[NLD];
    const bool k_due = FULL || i + 2 < n, v_due = FULL || i + 1 < n;
    if constexpr (Q4) {
      asm volatile("" : "+v"(tid4));
      if (k_due) unpack(ck, Ks[par], IsK{});
      if (v_due) {
        unpack(cv, Vs[par ^ 1], IsV{});
        look_over(i + 1, slot1, par ^ 1, cv.scale);
      }
    } else {
      if (k_due) read_ofs(slot2, ro_k);
      if (v_due) read_ofs(slot1, ro_v);
      if (!FULL) {
#pragma unroll
        for (int q = 0; q < NLD; ++q) {
          if (k_due) dma_row_chunk(ksrc + ro_k[q], dma_dst(Ks[par], q));
          if (v_due) dma_row_chunk(vsrc + ro_v[q], dma_dst(Vs[par ^ 1], q));
        }
      }
    }
    if (i + RING < n && wave == ((i + RING) & 3)) fill(slot, i + RING, lane, ahead);
    if (i + RING + 1 < n && wave == ((i + RING + 1) & 3))
      ahead = page_of(a, table, key_of(i + RING + 1) + lane);

    if (NEXT) {
      constexpr int NPAIR = 16, PPS = NPAIR / NQ;  // weight pairs, and of them per step
      static_assert(NPAIR % NQ == 0, "pairs split evenly over the steps");
      vec8 ring[4];
#pragma unroll
      for (int m = 0; m < kAhead; ++m) ring[m] = kfrag(par ^ 1, m);
      uint32_t pw[2][2][4];
      float acc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
      auto s_at = [&](int q, int e) -> float { return s_cur[q / 8][2 * (q % 8) + e]; };
      auto pack = [&](int q, float e0, float e1) {
        const auto pr = M::cvt2(e0, e1);
        pw[q / 8][(q / 4) % 2][q % 4] = __builtin_bit_cast(uint32_t, pr);
        acc[q / 8][(q / 4) % 2] = M::sum2(pr, acc[q / 8][(q / 4) % 2]);
      };
      float f0[NPAIR], f1[NPAIR], e0[NPAIR], e1[NPAIR];
#pragma unroll
      for (int q = 0; q < PPS; ++q) {
        f0[q] = __builtin_fmaf(c_log2, s_at(q, 0), negm);
        f1[q] = __builtin_fmaf(c_log2, s_at(q, 1), negm);
      }
      auto load_dst = [&](int m) -> uint32_t {
        return m < NLD ? dma_dst(Ks[par], m) : dma_dst(Vs[par ^ 1], m - NLD);
      };
      if (!Q4 && FULL) dma_set_m0(load_dst(0));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < NQ; ++m) {
        if (m + kAhead < NQ) ring[(m + kAhead) & 3] = kfrag(par ^ 1, m + kAhead);
        s_nxt[m & 1] = M::mma(ring[m & 3], qf[m >> 1], m < 2 ? f32x16_t{} : s_nxt[m & 1]);
        if (!Q4 && FULL) {
          static_assert(2 * NLD <= NQ, "one load per step");
          if (m < NLD) dma_at_m0(ksrc + ro_k[m]);
          else if (m < 2 * NLD) dma_at_m0(vsrc + ro_v[m - NLD]);
          if (m + 1 < 2 * NLD) dma_set_m0(load_dst(m + 1));
        }
#pragma unroll
        for (int x = 0; x < PPS; ++x) {
          const int q = m * PPS + x;
          if (q + PPS < NPAIR) {
            f0[q + PPS] = __builtin_fmaf(c_log2, s_at(q + PPS, 0), negm);
            f1[q + PPS] = __builtin_fmaf(c_log2, s_at(q + PPS, 1), negm);
          }
          e0[q] = __builtin_amdgcn_exp2f(f0[q]);
          e1[q] = __builtin_amdgcn_exp2f(f1[q]);
          if (q >= PPS) pack(q - PPS, e0[q - PPS], e1[q - PPS]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int q = NPAIR - PPS; q < NPAIR; ++q) pack(q, e0[q], e1[q]);
      tsum = (acc[0][0] + acc[0][1]) + (acc[1][0] + acc[1][1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const u32x4_t w = {pw[j][s][0], pw[j][s][1], pw[j][s][2], pw[j][s][3]};
          pb[j][s] = __builtin_bit_cast(vec8, w);
        }
    } else {
      weights(s_cur);
    }
    // The reference moves only where the sum of the (rounded) weights shows that it must, or at
    // the row's first tile: no row maximum is formed otherwise.
    const float pair = tsum + xor32(tsum);
    const bool bad = !seeded || !(pair <= M::kPMax);
    if (NEXT) mask(i + 1, slot1, s_nxt);
    if (__any(bad)) {
      float v = s_cur[0][0];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) v = fmaxf(v, s_cur[j][e]);
      const float mx = __builtin_fmaf(c_log2, fmaxf(v, xor32(v)), negm);
      if (bad && mx != -INFINITY) {
        const float f = seeded ? __builtin_amdgcn_exp2f(-mx) : 0.f;
        l_run *= f;
#pragma unroll
        for (int d = 0; d < NDT; ++d) o[d] *= f;
        m_ref += mx;
        negm = -m_ref;
        seeded = true;
        weights(s_cur);
      }
    }
    l_run += tsum;
    if constexpr (Q4) {  // (behind the QK block, where registers are scarcest)
      asm volatile("" : "+v"(tid4));
      if (i + 3 < n) ck = fetch(kbase, ksb, slot_at(slot, 3));
      if (i + 2 < n) cv = fetch(vbase, vsb, slot2);
    }
    __builtin_amdgcn_s_setprio(1);
    {
      u32x4_t ring[4];
#pragma unroll
      for (int m = 0; m < kAhead; ++m) ring[m] = vfrag(par, m);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int m = 0; m < NV; ++m) {
        if (m + kAhead < NV) ring[(m + kAhead) & 3] = vfrag(par, m + kAhead);
        o[m % NDT] = M::mma(__builtin_bit_cast(vec8, ring[m & 3]),
                            pb[m / (2 * NDT)][(m / NDT) & 1], o[m % NDT]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (NEXT && !decltype(swap)::value) {
      s_cur[0] = s_nxt[0];
      s_cur[1] = s_nxt[1];
    }
    if constexpr (!Q4) {
      wait_vmem();
      if (v_due) look_over(i + 1, slot1, par ^ 1, 0);
    }
    __syncthreads();
  };

  __syncthreads();  // the first offsets
  Scores s_a, s_b;
  {
    uint32_t scale = 0;
    if constexpr (Q4) {
      const Codes k_first = fetch(kbase, ksb, 0), v_first = fetch(vbase, vsb, 0);
      Codes k_second = {};
      if (n > 1) k_second = fetch(kbase, ksb, 1);
      unpack(k_first, Ks[0], IsK{});
      unpack(v_first, Vs[0], IsV{});
      if (n > 1) unpack(k_second, Ks[1], IsK{});
      scale = v_first.scale;
      if (n > 2) ck = fetch(kbase, ksb, 2);
      if (n > 1) cv = fetch(vbase, vsb, 1);
    } else {
      int64_t ro[2][NLD];
      read_ofs(0, ro[0]);
      read_ofs(1, ro[1]);
#pragma unroll
      for (int q = 0; q < NLD; ++q) {
        dma_row_chunk(ksrc + ro[0][q], dma_dst(Ks[0], q));
        dma_row_chunk(vsrc + ro[0][q], dma_dst(Vs[0], q));
        if (n > 1) dma_row_chunk(ksrc + ro[1][q], dma_dst(Ks[1], q));
      }
      wait_vmem();
    }
    look_over(0, 0, 0, scale);
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < NQ; ++m)
    s_a[m & 1] = M::mma(kfrag(0, m), qf[m >> 1], m < 2 ? f32x16_t{} : s_a[m & 1]);
  mask(0, 0, s_a);
  __syncthreads();  // K stage 0 is refilled from here on

  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, 1>;
  using PR = std::integral_constant<int, -1>;
  using Yes = std::true_type;
  using No = std::false_type;
  auto next_slot = [&](int sl) { return slot_at(sl, 1); };
  int i = 0, slot = 0;
  for (; i + 3 < n; i += 2) {  // two tiles a trip: constant stages, score buffers in turn
    iteration(i, slot, Yes{}, P0{}, Yes{}, s_a, s_b, Yes{});
    slot = next_slot(slot);
    iteration(i + 1, slot, Yes{}, P1{}, Yes{}, s_b, s_a, Yes{});
    slot = next_slot(slot);
  }
  for (; i + 1 < n; ++i) {
    iteration(i, slot, Yes{}, PR{}, No{}, s_a, s_b, No{});
    slot = next_slot(slot);
  }
  iteration(i, slot, No{}, PR{}, No{}, s_a, s_b, No{});

  // What look_over took out, added where it is seen: an infinity or a NaN of a seen key decides the
  // sum, whatever (positive) weight it has.
  for (int x = odd_tiles[0]; x <= odd_tiles[1]; ++x) {
    const int k0 = key_of(x);
    const uint64_t has = __ballot(page_of(a, table, k0 + lane) >= 0);
    if (!in_part(k0, has)) continue;
    for (int r = 0; r < KT; ++r) {
      const int key = k0 + r;
      const bool on = (has >> r & 1u) && sees(a, p, key);
      if (!__any(on)) continue;
      const int page = page_of(a, table, key);
      const char* row = vbase + row_offset(a, key, page, a.c_block, a.c_pos);
      if constexpr (Q4) {
        const char* sr = vsb + row_offset(a, key, page, a.s_block, a.s_pos);
#pragma unroll
        for (int d = 0; d < NDT; ++d)
        {
          const uint32_t byte = static_cast<uint8_t>(sr[d]);
          if (!on || byte < H::kInfByte) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t c = *reinterpret_cast<const uint16_t*>(row + 16 * d + 4 * e + 2 * lg);
            add_not_finite<DT>(fp4x4<DT>(c, scale_of<H::kShift>(byte)), o[d], 4 * e);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < NDT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint2 w =
                *reinterpret_cast<const uint2*>(row + 2 * (32 * d + 8 * e + 4 * lg));
            if (on) add_not_finite<DT>(w, o[d], 4 * e);
          }
      }
    }
  }

  const float l_tot = l_run + xor32(l_run);
  const int other_seen = __shfl_xor(static_cast<int>(seen), 32, 64);  // (by every lane)
  const bool row_seen = seen || other_seen != 0;
  // The rows go out through LDS, a wave's 32 of them through its eighth of the tiles' memory, so
  // that a store instruction writes whole rows instead of eight bytes of each: 64 rows of 8 bytes
  // take 64 cycles of address processing, 16 KB 4 us of a CU (8192 rows of a window of 1: 64 -> 58 us).
  // 16-byte chunks XOR-swizzled by row.
  constexpr int kWaveBytes = 32 * D * 2;
  static_assert(sizeof(Ks) == kRowsWaves / 2 * kWaveBytes, "each of K and V holds half the waves");
  char* stage = (wave < kRowsWaves / 2 ? reinterpret_cast<char*>(Ks) : reinterpret_cast<char*>(Vs)) +
                wave % (kRowsWaves / 2) * kWaveBytes;
  if (nsplit > 1) {
    // fp32 partials, in two halves of the dims
    const int64_t slot = it.slot * kRowsTile + wave * 32;
    constexpr int PCH = D / 8;  // chunks of half a row
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int d = 0; d < NDT / 2; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int dd = half * (NDT / 2) + d;
          const int c = (32 * d + 8 * e + 4 * lg) / 4;
          *reinterpret_cast<float4*>(stage + lq * (D * 2) + 16 * (c ^ (lq & (PCH - 1)))) =
              make_float4(o[dd][4 * e], o[dd][4 * e + 1], o[dd][4 * e + 2], o[dd][4 * e + 3]);
        }
      asm volatile("" ::: "memory");
#pragma unroll
      for (int k = 0; k < 32 * PCH / 64; ++k) {
        const int r = (k * 64 + lane) / PCH, c = (k * 64 + lane) % PCH;
        *reinterpret_cast<float4*>(a.part_o + (slot + r) * D + half * (D / 2) + 4 * c) =
            *reinterpret_cast<const float4*>(stage + r * (D * 2) + 16 * (c ^ (r & (PCH - 1))));
      }
      asm volatile("" ::: "memory");
    }
    if (lg == 0)
      *reinterpret_cast<float2*>(a.part_ml + (slot + lq) * 2) =
          make_float2(seeded && p >= 0 ? m_ref : row_seen ? kSeenNothing : -INFINITY, l_tot);
    return;
  }
  const float out_scale = Q4 ? static_cast<float>(1 << H::kShift) : 1.f;
  const float inv = !row_seen ? 0.f : out_scale / l_tot;
#pragma unroll
  for (int d = 0; d < NDT; ++d)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = o[d][8 * h + e] * inv;
      const u32x4_t w = __builtin_bit_cast(u32x4_t, M::cvt8(f));
      const int c = 4 * d + 2 * h;  // dims 8 c + 4 lg + 0..3 and 8 (c + 1) + 4 lg + 0..3
      char* at = stage + lq * (D * 2) + 8 * lg;
      *reinterpret_cast<uint2*>(at + 16 * (c ^ (lq & (CH - 1)))) = make_uint2(w.x, w.y);
      *reinterpret_cast<uint2*>(at + 16 * ((c + 1) ^ (lq & (CH - 1)))) = make_uint2(w.z, w.w);
    }
  asm volatile("" ::: "memory");
  const int64_t row_at = p < 0 ? -1 : (t.row0 + pi) * a.o_row + head * a.o_head;
  const bool wide = (reinterpret_cast<uintptr_t>(a.o) | a.o_row | a.o_head) % 16 == 0;
#pragma unroll
  for (int k = 0; k < 32 * CH / 64; ++k) {
    const int r = (k * 64 + lane) / CH, c = (k * 64 + lane) % CH;
    const int64_t at = __shfl(row_at, r, 64);
    const uint4 w = *reinterpret_cast<const uint4*>(stage + r * (D * 2) + 16 * (c ^ (r & (CH - 1))));
    if (at < 0) continue;
    char* dst = a.o + at + 16 * c;
    if (wide) {
      *reinterpret_cast<uint4*>(dst) = w;
    } else {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w.x, w.y);
      *reinterpret_cast<uint2*>(dst + 8) = make_uint2(w.z, w.w);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Joins the partials of row tiles whose keys were split: blockIdx.x = (tile, KV head), blockIdx.y
// = which RPW rows of the tile. D / 4 lanes take a row, and the groups of them that RPW rows leave
// share the row's splits: a decode row of 60 splits is then one batch of loads each for 8 groups
// instead of eight batches in turn (28 / 4 heads x 128, one row of 16000: 8.5 -> 5.4 us; 4.0 since the
// places of balanced items are read instead of scanned for).
// ---------------------------------------------------------------------------------------
constexpr int kMergeThreads = 256;
template <int DT, int D, int TR, int KT, int RPW>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_kernel(const PagedArgs a,
                                                                   float out_scale) {
  constexpr int VPR = D / 4;                           // lanes of a row
  constexpr int G = kMergeThreads / (RPW * VPR);       // groups that share a row
  static_assert(G >= 1 && G * RPW * VPR == kMergeThreads, "every thread has a row");
  __shared__ int red[2][kMergeThreads / 64];
  __shared__ __align__(16) float4 part[G > 1 ? kMergeThreads : 1];
  __shared__ float2 part_ml[G > 1 ? RPW * G : 1];
  const int tile_idx = blockIdx.x / a.num_kv_heads;
  const int kvh = blockIdx.x - tile_idx * a.num_kv_heads;
  Item it;
  int most = 0;  // even splits: the most parts of a row tile
  if (TR == kDecodeRows && a.target > 0) {
    const int per = (a.group + TR - 1) / TR, r = tile_idx / per;
    if (r >= a.num_rows || a.positions[r] < 0) return;  // (no item, nothing written for it)
    const int2 first = a.part_item[blockIdx.x];
    it = {kvh, first.y, 0, first.x, {r, r, 1, tile_idx - r * per}};
  } else {
    most = parts_of<TR>(a).most;
    if (most <= 1) return;
    it = {kvh, 0, 0, (static_cast<int64_t>(tile_idx) * a.num_kv_heads + kvh) * most,
          find_tile<TR>(a, tile_idx)};
  }
  const TileRef& t = it.t;
  if (t.request < 0) return;
  const int nflat = static_cast<int>(
      min(static_cast<int64_t>(t.rows) * a.group - static_cast<int64_t>(t.tile) * TR,
          static_cast<int64_t>(TR)));
  const int row_base = blockIdx.y * RPW;
  if (row_base >= nflat) return;
  int nsplit = it.nsplit;
  if (nsplit == 0) {  // even splits: the tile's key range, as the attention kernel saw it
    int pmin = 0x7fffffff, pmax = -1;
    static_assert(TR <= kMergeThreads, "one row per thread");
    if (static_cast<int>(threadIdx.x) < nflat) {
      const int p = a.positions[t.row0 + (t.tile * TR + static_cast<int>(threadIdx.x)) / a.group];
      if (p >= 0) pmin = p;
      pmax = p;
    }
    pmin = wave_min_i(pmin);
    pmax = wave_max_i(pmax);
    if ((threadIdx.x & 63) == 0) {
      red[0][threadIdx.x >> 6] = pmin;
      red[1][threadIdx.x >> 6] = pmax;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMergeThreads / 64; ++w) {
      pmin = min(pmin, red[0][w]);
      pmax = max(pmax, red[1][w]);
    }
    if (pmax < 0) return;
    nsplit = split_count(a, most, key_tiles<KT>(a, pmin, pmax).total);
  }
  if (nsplit <= 1) return;
  const int lane = threadIdx.x % VPR, row_in = threadIdx.x / VPR % RPW;
  const int grp = threadIdx.x / (VPR * RPW);
  const int row = min(row_base + row_in, nflat - 1), d = lane * 4;
  const int flat = t.tile * TR + row, pi = flat / a.group;
  const int p = a.positions[t.row0 + pi];
  const int64_t slot0 = it.slot * TR + row;
  const int64_t step = static_cast<int64_t>(slot_step(a)) * TR;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int B = TR == kDecodeRows ? 8 : 4;  // splits in flight
  for (int s0 = grp; s0 < nsplit; s0 += B * G) {
    float2 ml[B];
    float4 x[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int64_t slot = slot0 + min(s0 + b * G, nsplit - 1) * step;
      ml[b] = *reinterpret_cast<const float2*>(a.part_ml + slot * 2);
      x[b] = *reinterpret_cast<const float4*>(a.part_o + slot * D + d);
    }
    float mb = m;
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (s0 + b * G < nsplit) mb = fmaxf(mb, ml[b].x);
    if (mb == -INFINITY) continue;
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mb);
    l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (s0 + b * G >= nsplit || ml[b].x == -INFINITY) continue;
      const float w = __builtin_amdgcn_exp2f(ml[b].x - mb);
      l += w * ml[b].y;
      o.x += w * x[b].x, o.y += w * x[b].y, o.z += w * x[b].z, o.w += w * x[b].w;
    }
    m = mb;
  }
  if constexpr (G > 1) {
    part[threadIdx.x] = o;
    if (lane == 0) part_ml[row_in * G + grp] = make_float2(m, l);
    __syncthreads();
    if (grp > 0) return;
    float mb = m;
#pragma unroll
    for (int g = 1; g < G; ++g) mb = fmaxf(mb, part_ml[row_in * G + g].x);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mb);
    l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
    for (int g = 1; g < G; ++g) {
      const float2 ml = part_ml[row_in * G + g];
      if (ml.x == -INFINITY) continue;
      const float w = __builtin_amdgcn_exp2f(ml.x - mb);
      const float4 x = part[g * VPR * RPW + threadIdx.x];
      l += w * ml.y;
      o.x += w * x.x, o.y += w * x.y, o.z += w * x.z, o.w += w * x.w;
    }
    m = mb;
  }
  if (row_base + row_in >= nflat || p < 0) return;
  const float inv = m == -INFINITY ? 0.f : out_scale / l;
  char* op = a.o + (t.row0 + pi) * a.o_row + (kvh * a.group + flat - pi * a.group) * a.o_head;
  if constexpr (DT == SB_DTYPE_F32) {
    *reinterpret_cast<float4*>(op + d * 4) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  } else {
    const uint32_t w0 = Mma<DT>::cvt1(o.x * inv) | Mma<DT>::cvt1(o.y * inv) << 16;
    const uint32_t w1 = Mma<DT>::cvt1(o.z * inv) | Mma<DT>::cvt1(o.w * inv) << 16;
    *reinterpret_cast<uint2*>(op + d * 2) = make_uint2(w0, w1);
  }
}

// ---------------------------------------------------------------------------------------
// Any other head size (at most 512), alignment or scale: one wave per (row, query head), a key per
// lane for the scores and a dim per lane for the output. For the calls that the matrix cores do not
// take; bound by the scores' unshared loads.
// ---------------------------------------------------------------------------------------
constexpr int kValuMaxDim = 512;
template <int DT>
__device__ __forceinline__ float load16(const char* p, int i) {
  if constexpr (DT == SB_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  else if constexpr (DT == SB_DTYPE_F16) return f16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
  else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}
template <int DT, bool Q4>
__device__ __forceinline__ float load_kv(const char* row, const char* scales, int i) {
  if constexpr (Q4) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const uint32_t w = static_cast<uint8_t>(row[i >> 1]);
    const float sc = scale_of<0>(static_cast<uint8_t>(scales[i >> 5]));
    const f32x2 r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0);
    return (i & 1) ? r.y : r.x;
  } else {
    return load16<DT>(row, i);
  }
}

template <int DT, bool Q4>
__global__ __launch_bounds__(64) void paged_valu_kernel(const PagedArgs a) {
  constexpr int KT = 64;
  constexpr int PER = kValuMaxDim / 64;
  __shared__ float qs[kValuMaxDim];
  __shared__ float ws[KT];
  __shared__ int ps[KT];
  const int lane = threadIdx.x;
  const int hq = a.num_kv_heads * a.group;
  const int row = blockIdx.x / hq, h = blockIdx.x - row * hq, kvh = h / a.group;
  const int p = a.positions[row];
  if (p < 0) return;
  int request = a.num_requests == 1 ? 0 : row;
  if (a.row_starts) {
    if (row >= a.row_starts[a.num_requests]) return;
    int lo = 0, hi = a.num_requests;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.row_starts[mid] <= row) lo = mid;
      else hi = mid;
    }
    request = lo;
    if (row < a.row_starts[lo]) return;
  }
  const int D = a.head_dim;
  const char* qp = a.q + row * a.q_row + h * a.q_head;
  for (int d = lane; d < D; d += 64) qs[d] = load16<DT>(qp, d);
  __syncthreads();
  const KeyTiles kt = key_tiles<KT>(a, p, p);
  const int32_t* table = a.tables + request * a.table_stride;
  const char* kbase = a.k + kvh * a.c_head;
  const char* vbase = a.v + kvh * a.c_head;
  const char* ksb = a.ks + kvh * a.s_head;
  const char* vsb = a.vs + kvh * a.s_head;
  float m = -INFINITY, l = 0.f, o[PER];
  bool seen = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) o[i] = 0.f;
  for (int idx = 0; idx < kt.total; ++idx) {
    const int k0 = tile_key<KT>(kt, idx), key = k0 + lane;
    const int pb = page_of(a, table, key);
    const bool on = pb >= 0 && sees(a, p, key);
    float s = -INFINITY;
    if (on) {
      const char* kr = kbase + row_offset(a, key, pb, a.c_block, a.c_pos);
      const char* sr = Q4 ? ksb + row_offset(a, key, pb, a.s_block, a.s_pos) : nullptr;
      float acc = 0.f;
      for (int d = 0; d < D; ++d) acc = __builtin_fmaf(qs[d], load_kv<DT, Q4>(kr, sr, d), acc);
      s = acc * a.scale;
    }
    seen |= __any(on) != 0;
    const float mt = fmaxf(m, wave_max(s));
    const float f = mt == -INFINITY || m == -INFINITY ? 0.f : expf(m - mt);
    // (a NaN score has a NaN weight, also while no other score is above -inf)
    const float w = !on || s == -INFINITY ? 0.f : expf(s - mt);
    l = l * f + wave_sum(w);
    m = mt;
    __syncthreads();
    ws[lane] = w;
    ps[lane] = on ? pb : -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int d = lane + 64 * i;
      if (d >= D) break;
      float acc = o[i] * f;
      for (int k = 0; k < KT; ++k) {
        if (ps[k] < 0) continue;
        const char* vr = vbase + row_offset(a, k0 + k, ps[k], a.c_block, a.c_pos);
        const char* sr = Q4 ? vsb + row_offset(a, k0 + k, ps[k], a.s_block, a.s_pos) : nullptr;
        acc = __builtin_fmaf(ws[k], load_kv<DT, Q4>(vr, sr, d), acc);
      }
      o[i] = acc;
    }
  }
  char* op = a.o + row * a.o_row + h * a.o_head;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = lane + 64 * i;
    if (d >= D) break;
    const float r = seen ? o[i] / l : 0.f;
    if constexpr (DT == SB_DTYPE_F32) reinterpret_cast<float*>(op)[d] = r;
    else if constexpr (DT == SB_DTYPE_F16) reinterpret_cast<uint16_t*>(op)[d] = f32_to_f16(r);
    else reinterpret_cast<uint16_t*>(op)[d] = f32_to_bf16(r);
  }
}

// ---------------------------------------------------------------------------------------
// Launch plan: which kernels a call takes, their tiles and splits, and the workspace.
// ---------------------------------------------------------------------------------------
struct PartPlan {  // one attention launch
  bool on;
  int64_t tiles, grid;
  int nsplit, min_tiles, target;
  int64_t slots;        // > 0: places of partials that row tiles counted on the device share
  int64_t merge_tiles;  // row tiles that may be split
  int64_t o_floats, ml_floats, items;
};
struct PagedPlan {
  bool matrix;          // the matrix-core kernels (else the VALU kernel)
  PartPlan few, rows;   // requests of few flattened rows, and the others
  int few_max;          // flattened rows up to which a request takes the `few` kernel
  int64_t bytes;
};

// Flattened rows up to which all requests take the decode kernel (16-bit arithmetic): three tiles, which
// read a request's keys three times. (Requests of 4000 tokens, 32 / 8 heads x 128, decode and rows
// kernel: 48 rows 4 requests 41 and 52 us, 32 requests 183 and 205; 64 rows 53 and 52, 234 and 192.
// One request alone crosses later, by its rows and its keys: 448 rows over 1000 tokens, 28 / 4 heads,
// 18.5 and 22.8 us; 1078 over 1024, 14 / 2 heads x 64, 11.2 and 16.8; 280 over 4096 29.3 and 32; 800
// over 2000, 32 / 8 heads, 42.8 and 26.7. The rule stays at the batches' figure; a caller that knows
// its rows to be few has max_rows.)
constexpr int kFewRows = 48;
// The same for a request of a call that launches the rows kernel anyway: one tile (40 requests of 700
// rows and up to 6000 tokens, 28 / 4 heads x 128: 177 us, with 32 rows 189; nine requests of 1801 rows,
// 32 / 8 heads, window 700: 57, with 32 rows 57, with 48 63).
constexpr int kFewBeside = kDecodeRows;
constexpr int kRowsMinTiles = 4;   // fewest 64-key tiles of a split of the rows kernel
// Places of partials of a batch of several requests: two rounds of workgroups, one per CU (40 requests
// of 17 rows, 28 / 4 heads x 128, up to 6000 tokens: 129 us, with one round 165; 68 MB at 128 dims).
constexpr int64_t kRowsSlots = 512;

// Splits of each of `items` row tiles over `tiles` key tiles: those that 256 CUs take the shortest
// for, in rounds of a workgroup's fixed time and its tiles' (which two workgroups of a CU share),
// and with more than one split the merge's, and `part` for a split's partials.
int split_for(int64_t items, int64_t tiles, int min_tiles, int64_t tile_ns, int64_t fixed_ns,
              int64_t merge_ns, int64_t part_ns) {
  constexpr int64_t kCus = 256;
  int64_t best = 1, cost = 0;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(tiles / min_tiles, 128));
  for (int64_t n = 1; n <= most && items * (n - 1) < 2 * kCus; ++n) {
    const int64_t rounds = (items * n + kCus - 1) / kCus;
    const int64_t c = rounds * ((tiles + n - 1) / n * tile_ns + fixed_ns) +
                      (n > 1 ? merge_ns + rounds * part_ns + items * n * part_ns / kCus : 0);
    if (n == 1 || c < cost) best = n, cost = c;
  }
  return static_cast<int>(best);
}

int64_t row_bytes(int64_t head_dim, int32_t dtype, bool q4) {
  return q4 ? head_dim / 2 + head_dim / 32 : head_dim * elem_size(dtype);
}

PagedPlan plan_paged(int64_t num_rows, int64_t num_requests, bool starts, int64_t max_rows,
                     int64_t num_kv_heads, int64_t group, int64_t head_dim, int64_t kv_len,
                     int64_t window, int64_t sinks, int32_t dtype, int64_t bytes_per_row,
                     bool matrix) {
  PagedPlan pl = {};
  pl.matrix = matrix && (head_dim == 64 || head_dim == 128);
  if (!pl.matrix) return pl;
  const bool f32 = dtype == SB_DTYPE_F32;
  const bool ragged = starts || num_requests == 1;  // else one row per request
  const bool one_each = !starts && (num_requests > 1 || num_rows == 1);  // row i is request i's
  // Keys that a row may see, tables taken as full: the host does not know the contexts. Parts that a
  // short key list has no tiles for end at once. (512 rows of 2000 tokens, 32 / 8 heads x 128: 35.5 us
  // under a table of 2000 keys, 34.5 under one of 131072.)
  const int64_t keys = std::min(kv_len, std::min<int64_t>(window, kv_len) + sinks + 64);
  const int64_t per_few = (group + kDecodeRows - 1) / kDecodeRows;
  const int64_t flat = num_rows * group;
  pl.few_max = 0x7fffffff;
  const bool rows_kernel = !f32 && ragged && max_rows * group > kFewRows;
  if (rows_kernel) pl.few_max = num_requests == 1 ? 0 : kFewBeside;
  const int64_t tiles_bound = (flat + kDecodeRows - 1) / kDecodeRows + num_requests;
  pl.few.on = !rows_kernel || num_requests > 1;
  if (pl.few.on) {
    // with both kernels a `few` request has one tile
    pl.few.tiles = one_each ? num_rows * per_few
                            : rows_kernel ? std::min<int64_t>(tiles_bound, num_requests)
                                         : std::min<int64_t>(tiles_bound, flat);
    const int64_t key_tiles = (keys + (f32 ? 15 : 31)) / (f32 ? 16 : 32);
    const int64_t items = pl.few.tiles * num_kv_heads;
    const int kt = f32 ? 16 : 32;
    const int64_t most_tiles =  // of any row
        std::min<int64_t>((kv_len + kt - 1) / kt,
                          (std::min(window, kv_len) + kt - 2) / kt + 1 + (sinks + kt - 1) / kt);
    pl.few.min_tiles = kFewMinTiles;
    // (a workgroup's start and end take about 4 us, the merge launch 5)
    const int64_t tile_ns = std::max<int64_t>(110, 2 * kt * bytes_per_row / 40);
    // (beside the rows kernel most of `tiles` are empty: one a request, about)
    pl.few.nsplit = split_for(rows_kernel ? std::min(items, num_requests * num_kv_heads) : items,
                              key_tiles, kFewMinTiles, tile_ns, 4000, 5000, 0);
    if (one_each) {
      // Balanced items, unless there are enough of them as they are and none is long, or so many rows
      // that going through their positions costs more: 14 / 2 heads x 64, rows of up to 8300 tokens,
      // balanced against one item each: 128 rows 66 and 73 us, 256 119 and 121, 1024 428 and 409,
      // 4096 1788 and 1546 (lengths spread evenly; a long row among short ones is one item's else).
      const bool split = (pl.few.nsplit > 1 || key_tiles > kLongTiles) && num_rows <= kBalancedRows;
      pl.few.target = split ? kFewTarget : 0;
      pl.few.nsplit = 1;
    }
    // (a row of t tiles has at most t / size + 1 items, of `size` tiles, and all tiles are at most
    // target * size)
    pl.few.grid = pl.few.target > 0
                      ? items + std::min<int64_t>(kFewTarget, items * (most_tiles / pl.few.min_tiles))
                      : items * pl.few.nsplit;
    const int64_t slots =
        pl.few.target > 0 || pl.few.nsplit > 1 ? pl.few.grid * kDecodeRows : 0;
    pl.few.o_floats = slots * head_dim;
    pl.few.ml_floats = slots * 2;
    pl.few.items = pl.few.target > 0 ? (items + 1) / 2 * 2 : 0;  // (keeps what follows aligned)
    pl.few.merge_tiles = pl.few.tiles;
  }
  pl.rows.on = rows_kernel;
  if (rows_kernel) {
    const int64_t filled = (flat + kRowsTile - 1) / kRowsTile;  // row tiles of one request's rows
    pl.rows.tiles = num_requests == 1 ? filled
                                      : std::min<int64_t>(flat / kRowsTile + num_requests,
                                                          (flat + kFewBeside - 1) / kFewBeside);
    pl.rows.min_tiles = kRowsMinTiles;
    // (a tile takes about 2.2 us at head_dim 128, a workgroup's start and end about 10)
    const int64_t tile_ns = 2200 * head_dim / 128;
    const int64_t items = filled * num_kv_heads, most_items = pl.rows.tiles * num_kv_heads;
    pl.rows.nsplit = split_for(items, (keys + 63) / 64, kRowsMinTiles, tile_ns, 10000, 5000, 6000);
    int64_t slots = 0;
    if (pl.rows.nsplit > 1) {
      // What the parts of `filled` tiles take, or kRowsSlots if that is more (rows of several requests
      // fill their tiles less), and no more than all parts of all tiles.
      slots = std::min(std::max<int64_t>(items * pl.rows.nsplit, kRowsSlots),
                       most_items * pl.rows.nsplit);
      if (num_requests > 1) pl.rows.slots = slots;
    }
    pl.rows.grid = std::max(most_items, slots);
    // (of more tiles than half the places none is split)
    pl.rows.merge_tiles = std::min(pl.rows.tiles, slots / (2 * num_kv_heads));
    pl.rows.o_floats = slots * kRowsTile * head_dim;
    pl.rows.ml_floats = slots * kRowsTile * 2;
  }
  pl.bytes = 4 * (pl.few.o_floats + pl.few.ml_floats + pl.rows.o_floats + pl.rows.ml_floats) +
             8 * pl.few.items;
  return pl;
}

}  // namespace
}  // namespace sb

extern "C" int64_t sb_paged_attention_workspace_size(int64_t num_rows, int64_t num_requests,
                                                     int32_t has_starts, int64_t max_rows,
                                                     int64_t num_q_heads, int64_t num_kv_heads,
                                                     int64_t head_dim, int64_t block_size,
                                                     int64_t num_blocks_per_seq, int64_t window,
                                                     int64_t sinks, int32_t dtype,
                                                     int32_t cache_dtype) {
  using namespace sb;
  if (num_rows <= 0 || num_requests <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 ||
      num_q_heads % num_kv_heads || block_size <= 0 || num_blocks_per_seq <= 0 || window < 0 ||
      sinks < 0 || block_size > 0x7fffffff || num_blocks_per_seq > 0x7fffffff)
    return 0;
  const int64_t kv_len = std::min<int64_t>(block_size * num_blocks_per_seq, 0x7fff0000);
  return plan_paged(num_rows, num_requests, has_starts != 0,
                    max_rows > 0 && max_rows < num_rows ? max_rows : num_rows, num_kv_heads,
                    num_q_heads / num_kv_heads, head_dim, kv_len,
                    window > 0 && window <= kNoWindow ? window : kNoWindow, sinks, dtype,
                    row_bytes(head_dim, dtype, cache_dtype == SB_DTYPE_MXFP4), true)
      .bytes;
}

extern "C" int sb_paged_attention(
    void* out, const void* q, const void* kv_cache, const void* kv_scales,
    const int32_t* block_tables, int64_t table_stride, const int32_t* positions,
    const int32_t* row_starts, void* workspace, int64_t workspace_bytes, int64_t num_rows,
    int64_t num_requests, int64_t max_rows, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks_total, int64_t num_blocks_per_seq,
    int64_t window, int64_t sinks, float scale, const int64_t* q_strides,
    const int64_t* o_strides, const int64_t* kv_strides, const int64_t* scale_strides,
    int32_t dtype, int32_t cache_dtype, void* stream) {
  using namespace sb;
  const char* fn = "sb_paged_attention";
  clear_error();
  if (num_rows == 0) return SB_OK;
  const int64_t es = elem_size(dtype);
  if (!es) return fail(fn, "invalid dtype");
  const bool q4 = cache_dtype == SB_DTYPE_MXFP4;
  if (!q4 && cache_dtype != dtype) return fail(fn, "the cache's dtype is neither the query's nor MXFP4");
  if (!out || !q || !kv_cache || !block_tables || !positions || !q_strides || !o_strides ||
      !kv_strides || (q4 && (!kv_scales || !scale_strides)))
    return fail(fn, "null pointer");
  if (num_rows < 0 || num_requests <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      block_size <= 0 || num_blocks_total <= 0 || num_blocks_per_seq <= 0)
    return fail(fn, "sizes must be positive");
  if (num_q_heads % num_kv_heads) return fail(fn, "num_q_heads must be a multiple of num_kv_heads");
  if (head_dim <= 0 || head_dim > kValuMaxDim || (q4 && head_dim % 32))
    return fail(fn, "head_dim must be at most 512, and a multiple of 32 over 4-bit pages");
  if (window < 0 || sinks < 0) return fail(fn, "window and sinks must not be negative");
  if (!row_starts && num_requests > 1 && num_rows > num_requests)
    return fail(fn, "without row_starts there is one row per request");
  const int64_t group = num_q_heads / num_kv_heads;
  if (num_rows * num_q_heads > 0x7fffffff - 0x10000 || num_requests > 0x3fffffff ||
      num_blocks_total > 0x7fffffff || block_size > 0x7fffffff ||
      num_blocks_per_seq > 0x7fffffff)
    return fail(fn, "size past 32 bits");
  if (q_strides[2] != 1 || o_strides[2] != 1 || kv_strides[4] != 1 ||
      (q4 && scale_strides[4] != 1))
    return fail(fn, "the last dimension must be contiguous");
  const int64_t cs = q4 ? 1 : es;
  if (kv_strides[0] < 0 || kv_strides[0] * cs > 0xffffffffll ||
      (q4 && (scale_strides[0] < 0 || scale_strides[0] > 0xffffffffll)))
    return fail(fn, "a page must be smaller than 4 GiB");

  PagedArgs a = {};
  a.q = static_cast<const char*>(q);
  a.o = static_cast<char*>(out);
  a.q_row = q_strides[0] * es, a.q_head = q_strides[1] * es;
  a.o_row = o_strides[0] * es, a.o_head = o_strides[1] * es;
  a.k = static_cast<const char*>(kv_cache);
  a.v = a.k + kv_strides[1] * cs;
  a.c_block = static_cast<uint32_t>(kv_strides[0] * cs);
  a.c_head = kv_strides[2] * cs, a.c_pos = kv_strides[3] * cs;
  if (q4) {
    a.ks = static_cast<const char*>(kv_scales);
    a.vs = a.ks + scale_strides[1];
    a.s_block = static_cast<uint32_t>(scale_strides[0]);
    a.s_head = scale_strides[2], a.s_pos = scale_strides[3];
  }
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.positions = positions;
  a.row_starts = row_starts;
  a.num_rows = static_cast<int>(num_rows);
  a.num_requests = static_cast<int>(num_requests);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.group = static_cast<int>(group);
  a.head_dim = static_cast<int>(head_dim);
  a.block_size = static_cast<int>(block_size);
  int log2_up = 0;
  while ((1ll << log2_up) < block_size) ++log2_up;
  a.bs_shift = 31 + log2_up;
  a.bs_magic = static_cast<uint32_t>(((1ull << a.bs_shift) + block_size - 1) / block_size);
  a.num_blocks_total = static_cast<int>(num_blocks_total);
  a.kv_len = static_cast<int>(std::min<int64_t>(block_size * num_blocks_per_seq, 0x7fff0000));
  // (no window: the last position's would end behind key 0, so every key is a first one as well)
  const bool windowed = window > 0 && window <= kNoWindow;
  a.window = windowed ? static_cast<int>(window) : kNoWindow;
  a.sinks = windowed ? static_cast<int>(std::min<int64_t>(sinks, a.kv_len)) : a.kv_len;
  a.scale = scale;
  const double sl = static_cast<double>(scale) * 1.4426950408889634;
  a.scale_log2 = static_cast<float>(sl);
  a.scale_log2_lo = static_cast<float>(sl - static_cast<double>(a.scale_log2));

  const auto addr = [](const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); };
  const int64_t c0 = addr(kv_cache), cell = q4 ? head_dim / 8 : 16;
  bool aligned = vec_bytes({addr(q), a.q_row, a.q_head}) == 16 &&
                 vec_bytes({addr(out), a.o_row, a.o_head}) >= (es == 4 ? 16 : 8);
  for (int64_t x : {c0, static_cast<int64_t>(a.c_block), kv_strides[1] * cs, a.c_head, a.c_pos})
    aligned = aligned && x % cell == 0;
  // (scales that 2^8 times a score's rounding could turn, and those of no sign, are the VALU's)
  const bool matrix = aligned && !(dtype == SB_DTYPE_F32 && q4) && a.scale_log2 > 1e-37f &&
                      a.scale_log2 < 1e30f;
  const PagedPlan pl = plan_paged(num_rows, num_requests, row_starts != nullptr,
                                  max_rows > 0 && max_rows < num_rows ? max_rows : num_rows,
                                  num_kv_heads, group, head_dim, a.kv_len, a.window, a.sinks,
                                  dtype, row_bytes(head_dim, dtype, q4), matrix);
  if (pl.bytes > workspace_bytes || (pl.bytes && !workspace))
    return fail(fn, "workspace too small");
  if (workspace && addr(workspace) % 16) return fail(fn, "workspace must be 16-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);

  if (!pl.matrix) {
    const int64_t g = num_rows * num_q_heads;
#define SB_VALU(DT)                                                                             \
  if (dtype == DT) {                                                                            \
    if (q4)                                                                                     \
      SB_LAUNCH("paged_valu", (paged_valu_kernel<DT, true>), dim3(static_cast<unsigned>(g)),    \
                dim3(64), st, a);                                                               \
    else                                                                                        \
      SB_LAUNCH("paged_valu", (paged_valu_kernel<DT, false>), dim3(static_cast<unsigned>(g)),   \
                dim3(64), st, a);                                                               \
  }
    SB_VALU(SB_DTYPE_F32)
    SB_VALU(SB_DTYPE_F16)
    SB_VALU(SB_DTYPE_BF16)
#undef SB_VALU
    return check_launch(fn);
  }

  float* ws = static_cast<float*>(workspace);
  const float out_scale = q4 && dtype == SB_DTYPE_F16 ? 4.f : 1.f;
  const auto part = [&](const PartPlan& p) {
    PagedArgs b = a;
    b.num_tiles = static_cast<int>(p.tiles);
    b.nsplit = p.nsplit;
    b.min_tiles = p.min_tiles;
    b.slots = static_cast<int>(p.slots);
    b.target = p.target;
    b.part_o = ws;
    b.part_ml = ws + p.o_floats;
    b.part_item = reinterpret_cast<int2*>(ws + p.o_floats + p.ml_floats);
    ws += p.o_floats + p.ml_floats + 2 * p.items;
    return b;
  };
#define SB_D(X)                     \
  if (head_dim == 64) { X(64) }     \
  else { X(128) }
#define SB_MERGE(DT, D, TR, KT, B, P)                                                           \
  if ((P).nsplit > 1 || (P).target > 0) {                                                       \
    constexpr int rpw = TR == kDecodeRows ? 1 : 1024 / D;                                       \
    const int live = (P).target > 0 ? std::min<int>(TR, static_cast<int>(group)) : TR;          \
    const dim3 mg(static_cast<unsigned>((P).merge_tiles * num_kv_heads), (live + rpw - 1) / rpw); \
    SB_LAUNCH("paged_merge", (paged_merge_kernel<DT, D, TR, KT, rpw>), mg, dim3(kMergeThreads), \
              st, B, out_scale);                                                                \
  }
  const int64_t most = 0x7fffffff;
  if (pl.few.grid > most || pl.rows.grid > most)
    return fail(fn, "grid too large");
  if (pl.rows.on) {
    PagedArgs b = part(pl.rows);
    b.flat_min = pl.few_max;
    b.flat_max = 0x7fffffff;
    const dim3 grid(static_cast<unsigned>(pl.rows.grid));
#define SB_ROWS(DT, D)                                                                          \
  {                                                                                             \
    if (q4)                                                                                     \
      SB_LAUNCH("paged_rows", (paged_rows_kernel<DT, D, true>), grid, dim3(kRowsWaves * 64), st, b); \
    else                                                                                        \
      SB_LAUNCH("paged_rows", (paged_rows_kernel<DT, D, false>), grid, dim3(kRowsWaves * 64), st, b); \
    SB_MERGE(DT, D, kRowsTile, 64, b, pl.rows)                                                  \
  }
#define SB_ROWS_BF16(D) SB_ROWS(SB_DTYPE_BF16, D)
#define SB_ROWS_F16(D) SB_ROWS(SB_DTYPE_F16, D)
    if (dtype == SB_DTYPE_BF16) { SB_D(SB_ROWS_BF16) }
    else { SB_D(SB_ROWS_F16) }
  }
  if (pl.few.on) {
    PagedArgs b = part(pl.few);
    b.flat_min = 0;
    b.flat_max = pl.few_max;
    const dim3 grid(static_cast<unsigned>(pl.few.grid));
    const dim3 block(kDecodeWaves * 64);
    // (a lane's offset inside a group of 16 keys is 32 bits there)
    const bool uniform = block_size % 16 == 0 && a.c_pos >= 0 && a.c_pos < (1 << 27) &&
                         (!q4 || (a.c_block == 16ull * a.s_block && a.c_pos == 16 * a.s_pos));
#define SB_FEW_K(DT, D, Q4, U)                                                                  \
  { SB_LAUNCH("paged_decode", (paged_decode_kernel<DT, D, Q4, U>), grid, block, st, b); }
#define SB_FEW(DT, D)                                                                           \
  {                                                                                             \
    if (q4 && uniform) SB_FEW_K(DT, D, true, true)                                              \
    else if (q4) SB_FEW_K(DT, D, true, false)                                                   \
    else if (uniform) SB_FEW_K(DT, D, false, true)                                              \
    else SB_FEW_K(DT, D, false, false)                                                          \
    SB_MERGE(DT, D, kDecodeRows, 32, b, pl.few)                                                 \
  }
#define SB_FEW_BF16(D) SB_FEW(SB_DTYPE_BF16, D)
#define SB_FEW_F16(D) SB_FEW(SB_DTYPE_F16, D)
#define SB_FEW_F32(D)                                                                           \
  {                                                                                             \
    if (uniform) SB_LAUNCH("paged_f32", (paged_f32_kernel<D, true>), grid, block, st, b);       \
    else SB_LAUNCH("paged_f32", (paged_f32_kernel<D, false>), grid, block, st, b);              \
    SB_MERGE(SB_DTYPE_F32, D, kDecodeRows, 16, b, pl.few)                                       \
  }
    if (dtype == SB_DTYPE_BF16) { SB_D(SB_FEW_BF16) }
    else if (dtype == SB_DTYPE_F16) { SB_D(SB_FEW_F16) }
    else { SB_D(SB_FEW_F32) }
  }
  return check_launch(fn);
}
