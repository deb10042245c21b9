// A model's rotary positions for gfx950: rows of Q and K turned by their positions, donor K/V
// scattered into paged caches with K turned on the way, and cached K shifted in place.
//
// The first 2 P elements of a row are turned in P pairs, interleaved (2i, 2i + 1) or half (i, i + P):
//   a' = a c - b s,  b' = a s + b c,  c, s = factor * cos, sin(p * f_i),
// p a position or a difference of two, f_i the model's fp32 frequencies (any scaling for long
// contexts is in them). The angle is formed and reduced in 64 bits; 16-bit rows are turned in fp32
// with one rounding, fp32 rows in 64 bits with one.
//
// What bounds it: bytes. A workgroup takes a few tokens and some of their rows (heads, or layers x
// K/V x heads): the sines of a (token, pair), about 45 fp64 instructions, are evaluated once in LDS
// and serve all of these, and one thread per row works out its addresses (sb_rows.h). Kernel times: 8192
// tokens of 32 / 8 heads x 128 in bf16 26.5 us (168 MB, 6.3 TB/s; a large copy reaches 6.6), in fp32 60.5
// (336 MB, 5.5); 28 layers x 6963 pairs of 4 heads scattered 137 us (799 MB, 5.8 TB/s: rows of 256 bytes, two
// dependent reads before them); 32 layers x 3001 positions of 8 heads shifted in place 74 us (393 MB, 5.3
// TB/s); 32 tokens 3.9 us, a launch and its chain.
#include "sb_rows.h"

namespace sb {
namespace {

// Tokens of a dense workgroup (8192 tokens of 32 / 8 heads x 128, bf16 / fp32: 1 31.8 / 61.5 us, 2 27.7 /
// 62.3, 4 27.7 / 66.2, 8 28.5 / 70.4), rows of a scattering one (28 layers x 6963 pairs of 4 heads x 128: 64
// 141 us, 128 145, 256 149) and of a shifting one (32 layers x 3001 positions of 8 heads x 128: 32 74 us, 64
// 76, 128 77, 256 79). Rows in flight of a thread, half pairs: 2 (scatter, 4: 155 us with 64 rows).
constexpr int kDenseTokens = 2;
constexpr int kScatterRows = 64, kShiftRows = 32;
enum RotaryMode : int { ROTARY_DENSE = 0, ROTARY_SCATTER = 1, ROTARY_SHIFT = 2 };

struct RotaryArgs {
  // dense: query rows, then key rows of a token
  const char* q;
  char* q_out;
  const char* k;
  char* k_out;
  int64_t q_tok, q_head, qo_tok, qo_head, k_tok, k_head, ko_tok, ko_head;  // byte strides
  int num_q_heads;
  // scatter, shift: rows are layers x (K, V) x heads, or layers x heads of K
  const uint64_t* layers;
  const uint64_t* donors;
  int64_t c_block, c_kv, c_head, c_pos, d_kv, d_head, d_pos;  // byte strides
  int64_t donor_len, num_blocks_total, num_blocks_per_seq;
  const int32_t* table;
  const int32_t* from;       // scatter: donor positions
  int num_heads, block_size;
  // all
  const int32_t* positions;  // of each token (scatter: target, shift: the slot's)
  const int32_t* deltas;     // shift
  const float* inv_freq;
  double factor;
  int64_t num_tokens;
  int head_dim, pairs;
  int rows_per_token, tokens_per_wg, rows_per_y;  // rows_per_y: of each token
  RowSplit split;
  Divisor pair_div, head_div;
};

// Positions and deltas carried in the launch itself (a short list of the host's).
struct RotaryInline {
  int32_t pos[SB_INLINE_POSITIONS_MAX];
  int32_t delta[SB_INLINE_POSITIONS_MAX];
};
struct NoInline {};

// ONCE: rows are read once (nontemporal); INLINE: positions and deltas in the launch.
template <int DT, int VEC, bool HALF, int MODE, bool ONCE, bool INLINE>
__global__ __launch_bounds__(kRowThreads) void rotary_rows_kernel(
    const RotaryArgs a, const std::conditional_t<INLINE, RotaryInline, NoInline> list) {
  using CS = std::conditional_t<DT == SB_DTYPE_F32, double, float>;
  __shared__ __align__(16) CS cs[2 * kTableEntries];
  __shared__ __align__(16) RowRef rows[kRowsMax];
  const int tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_wg;
  const int ntok = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_wg), a.num_tokens - t0));
  const int j0 = blockIdx.y * a.rows_per_y;
  const int per = min(a.rows_per_y, a.rows_per_token - j0);
  const int n = per * ntok;
  bool sines = true;

  // The angle of a token: its position, the way from the donor's, or its delta.
  auto angle = [&](int64_t t) -> int {
    if constexpr (INLINE) return list.delta[t];
    else if constexpr (MODE == ROTARY_SHIFT) return a.deltas[t];
    else if constexpr (MODE == ROTARY_SCATTER)  // (a pair left out may hold any numbers)
      return static_cast<int>(static_cast<uint32_t>(a.positions[t]) - static_cast<uint32_t>(a.from[t]));
    else return a.positions[t];
  };

  if (tid < n) {
    // rows in the order of memory: a token's heads, or one head (of a layer, of K or V) of all tokens
    const int major = tid / (MODE == ROTARY_DENSE ? per : ntok);
    const int minor = tid - major * (MODE == ROTARY_DENSE ? per : ntok);
    const int jr = MODE == ROTARY_DENSE ? minor : major, tok = MODE == ROTARY_DENSE ? major : minor;
    const int64_t t = t0 + tok;
    const int j = j0 + jr;
    RowRef ref = {nullptr, nullptr, nullptr, 0, 0};
    bool turn = true;
    if constexpr (MODE == ROTARY_DENSE) {
      const bool key = j >= a.num_q_heads;
      const int h = j - (key ? a.num_q_heads : 0);
      ref.src = key ? a.k + t * a.k_tok + h * a.k_head : a.q + t * a.q_tok + h * a.q_head;
      ref.dst = key ? a.k_out + t * a.ko_tok + h * a.ko_head : a.q_out + t * a.qo_tok + h * a.qo_head;
    } else {
      const int plane = a.head_div.of(j), h = j - plane * a.num_heads;
      const int layer = MODE == ROTARY_SCATTER ? plane >> 1 : plane;
      const int kv = MODE == ROTARY_SCATTER ? plane & 1 : 0;
      int p;
      if constexpr (INLINE) p = list.pos[t];
      else p = a.positions[t];
      const int d = MODE == ROTARY_SCATTER ? a.from[t] : 0;
      if (p >= 0 && (MODE != ROTARY_SCATTER || (d >= 0 && d < a.donor_len))) {
        const int lb = p / a.block_size, slot = p - lb * a.block_size;
        const int64_t pb = lb < a.num_blocks_per_seq ? a.table[lb] : -1;
        const int turned_by = angle(t);
        if (pb >= 0 && pb < a.num_blocks_total && (MODE == ROTARY_SCATTER || turned_by != 0)) {
          ref.dst = reinterpret_cast<char*>(a.layers[layer]) + pb * a.c_block + slot * a.c_pos +
                    kv * a.c_kv + h * a.c_head;
          ref.src = MODE == ROTARY_SCATTER
                        ? reinterpret_cast<const char*>(a.donors[layer]) + kv * a.d_kv + h * a.d_head +
                              d * a.d_pos
                        : ref.dst;
          turn = kv == 0 && turned_by != 0;
        }
      }
    }
    ref.info = static_cast<uint32_t>(2 * tok * a.pairs) << 2 | (turn ? 1u : 0u);
    rows[tid] = ref;
  }
  // (a workgroup of V rows alone turns none)
  if (MODE == ROTARY_SCATTER) {
    const int first = a.head_div.of(j0), last = a.head_div.of(j0 + per - 1);
    sines = first != last || (first & 1) == 0;
  }
  // (from the last wave down: the first ones work out the rows)
  for (int i = kRowThreads - 1 - tid; sines && i < ntok * a.pairs; i += kRowThreads) {
    const int tok = a.pair_div.of(i), f = i - tok * a.pairs;
    double s, c;
    sincos_cw(static_cast<double>(angle(t0 + tok)) * static_cast<double>(a.inv_freq[f]), &s, &c);
    CS* to = cs + 2 * tok * a.pairs + Sines<DT, VEC, HALF>::at(f, a.pairs);
    to[0] = static_cast<CS>(c * a.factor);
    to[1] = static_cast<CS>(s * a.factor);
  }
  __syncthreads();
  const int rpi = kRowThreads / a.split.units;
  const int rsub = tid / a.split.units, unit = tid - rsub * a.split.units;
  if (rsub >= rpi) return;
  turn_rows<DT, VEC, false, HALF, ONCE, HALF ? 2 : 4>(rows, n, cs, nullptr, a.split, a.head_dim,
                                                       a.pairs, rsub, rpi, unit);
}

int64_t address(const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); }

// `vb`: the widest vector that the rows and strides allow; list: positions in the launch, or nullptr.
template <int MODE, bool ONCE>
int launch_rotary(const char* fn, RotaryArgs a, int32_t layout, int32_t dtype, int vb,
                  const RotaryInline* list, hipStream_t st) {
  const bool half = layout == SB_ROTARY_HALF;
  const int64_t es = elem_size(dtype);
  const bool wide = vec_bytes({vb, a.head_dim * es, (half ? a.pairs : 2 * a.pairs) * es}) == 16;
  const int vec = wide ? static_cast<int>(16 / es) : 2;
  a.split = RowSplit::of(a.head_dim, a.pairs, vec, half);
  // Tokens of a workgroup: as many as its table of sines takes and as leave 1024 workgroups; few
  // tokens: one, and its rows spread over workgroups until there are 512.
  const int rpi = kRowThreads / a.split.units;
  int fit = std::min(MODE == ROTARY_DENSE ? kDenseTokens : kTokensMax, std::max(1, kTableEntries / a.pairs));
  if (MODE == ROTARY_DENSE) fit = std::max(1, std::min(fit, kRowsMax / a.rows_per_token));
  const int64_t units = a.num_tokens * ((a.rows_per_token + kRowsMax - 1) / kRowsMax);
  a.tokens_per_wg = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(fit, units / 1024)));
  const int64_t gx = (a.num_tokens + a.tokens_per_wg - 1) / a.tokens_per_wg;
  constexpr int kRows = MODE == ROTARY_SCATTER ? kScatterRows : MODE == ROTARY_SHIFT ? kShiftRows : kRowsMax;
  int per = std::max(1, kRows / a.tokens_per_wg);
  if (a.tokens_per_wg == 1) {
    const int steps = (a.rows_per_token + rpi - 1) / rpi;
    const int ny = static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, 512 / gx), steps));
    per = std::min(per, (steps + ny - 1) / ny * rpi);
  }
  a.rows_per_y = std::min(per, a.rows_per_token);
  const int64_t gy = (a.rows_per_token + a.rows_per_y - 1) / a.rows_per_y;
  if (gx > 0x7fffffff || gy > 65535) return fail(fn, "grid too large");
  a.pair_div = Divisor::by(a.pairs);
  a.head_div = Divisor::by(std::max(1, a.num_heads));
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
#define SB_ROTARY_(DT, VEC, HALF)                                                                \
  do {                                                                                           \
    if constexpr (MODE == ROTARY_SHIFT)                                                          \
      if (list) {                                                                                \
        SB_LAUNCH("rotary_rows", (rotary_rows_kernel<DT, VEC, HALF, MODE, ONCE, true>), grid,          \
                  dim3(kRowThreads), st, a, *list);                                              \
        break;                                                                                   \
      }                                                                                          \
    SB_LAUNCH("rotary_rows", (rotary_rows_kernel<DT, VEC, HALF, MODE, ONCE, false>), grid,             \
              dim3(kRowThreads), st, a, NoInline{});                                             \
  } while (0)
#define SB_ROTARY(DT, VEC)                  \
  if (dtype == DT && vec == VEC) {          \
    if (half) SB_ROTARY_(DT, VEC, true);    \
    else SB_ROTARY_(DT, VEC, false);        \
  }
  SB_ROTARY(SB_DTYPE_F32, 4)
  SB_ROTARY(SB_DTYPE_F32, 2)
  SB_ROTARY(SB_DTYPE_F16, 8)
  SB_ROTARY(SB_DTYPE_F16, 2)
  SB_ROTARY(SB_DTYPE_BF16, 8)
  SB_ROTARY(SB_DTYPE_BF16, 2)
#undef SB_ROTARY
#undef SB_ROTARY_
  return check_launch(fn);
}

// Checks and arguments that the paged forms share.
int paged_args(const char* fn, RotaryArgs* a, const uint64_t* layers, int64_t num_layers,
               const int32_t* table, const float* inv_freq, int64_t num, int64_t heads,
               int64_t block_size, int64_t head_dim, int64_t num_blocks_total,
               int64_t num_blocks_per_seq, int64_t pairs, int32_t layout, int32_t dtype) {
  if (!valid_dtype(dtype)) return fail(fn, "invalid dtype");
  if (!layers || !table || !inv_freq) return fail(fn, "null pointer");
  if (num < 0 || num_layers <= 0 || heads <= 0 || block_size <= 0 || num_blocks_total <= 0 ||
      num_blocks_per_seq <= 0)
    return fail(fn, "sizes must be positive");
  if (num > 0x7fffffff || num_layers > 4096 || heads > 65535 || block_size > 0x7fffffff)
    return fail(fn, "size past its limit");
  if (const char* why = rotary_fault(head_dim, pairs, layout, 1.0)) return fail(fn, why);
  a->layers = layers;
  a->table = table;
  a->inv_freq = inv_freq;
  a->factor = 1.0;
  a->num_tokens = num;
  a->num_heads = static_cast<int>(heads);
  a->block_size = static_cast<int>(block_size);
  a->head_dim = static_cast<int>(head_dim);
  a->pairs = static_cast<int>(pairs);
  a->num_blocks_total = num_blocks_total;
  a->num_blocks_per_seq = num_blocks_per_seq;
  return SB_OK;
}

int shift_layers(const char* fn, const uint64_t* layers, int64_t num_layers, const int32_t* table,
                 const int32_t* positions, const int32_t* deltas, const RotaryInline* list, int64_t num,
                 const float* inv_freq, int64_t heads, int64_t block_size, int64_t head_dim,
                 int64_t num_blocks_total, int64_t num_blocks_per_seq, const int64_t* kv_strides,
                 int64_t pairs, int32_t layout, int32_t dtype, hipStream_t st) {
  RotaryArgs a = {};
  const int rc = paged_args(fn, &a, layers, num_layers, table, inv_freq, num, heads, block_size,
                            head_dim, num_blocks_total, num_blocks_per_seq, pairs, layout, dtype);
  if (rc != SB_OK) return rc;
  if (!kv_strides || (!list && (!positions || !deltas))) return fail(fn, "null pointer");
  if (kv_strides[3] != 1) return fail(fn, "the last dimension must be contiguous");
  const int64_t es = elem_size(dtype);
  a.c_block = kv_strides[0] * es, a.c_head = kv_strides[1] * es, a.c_pos = kv_strides[2] * es;
  a.positions = positions;
  a.deltas = deltas;
  a.rows_per_token = static_cast<int>(num_layers * heads);
  return launch_rotary<ROTARY_SHIFT, true>(fn, a, layout, dtype,
                                           vec_bytes({a.c_block, a.c_head, a.c_pos}), list, st);
}

}  // namespace
}  // namespace sb

extern "C" int sb_apply_rotary(void* query_out, const void* query, void* key_out, const void* key,
                               const int32_t* positions, const float* inv_freq, int64_t num_tokens,
                               int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                               const int64_t* q_strides, const int64_t* qo_strides,
                               const int64_t* k_strides, const int64_t* ko_strides, int64_t pairs,
                               int32_t layout, double factor, int32_t dtype, void* stream) {
  using namespace sb;
  const char* fn = "sb_apply_rotary";
  clear_error();
  if (num_tokens == 0) return SB_OK;
  if (!valid_dtype(dtype)) return fail(fn, "invalid dtype");
  const bool has_k = key != nullptr;
  if (!query || !query_out || !positions || !inv_freq || !q_strides || !qo_strides ||
      (has_k && (!key_out || !k_strides || !ko_strides)))
    return fail(fn, "null pointer");
  if (num_tokens < 0 || num_q_heads <= 0 || (has_k && num_kv_heads <= 0))
    return fail(fn, "sizes must be positive");
  if (num_tokens > 0x7fffffff || num_q_heads > 65535 || num_kv_heads > 65535)
    return fail(fn, "size past its limit");
  if (const char* why = rotary_fault(head_dim, pairs, layout, factor)) return fail(fn, why);
  if (q_strides[2] != 1 || qo_strides[2] != 1 || (has_k && (k_strides[2] != 1 || ko_strides[2] != 1)))
    return fail(fn, "the last dimension must be contiguous");
  if (rows_overlap(num_tokens, num_q_heads, head_dim, qo_strides[0], qo_strides[1]) ||
      (has_k && rows_overlap(num_tokens, num_kv_heads, head_dim, ko_strides[0], ko_strides[1])))
    return fail(fn, "rows of an output must not overlap");
  const int64_t es = elem_size(dtype);
  RotaryArgs a = {};
  a.q = static_cast<const char*>(query);
  a.q_out = static_cast<char*>(query_out);
  a.q_tok = q_strides[0] * es, a.q_head = q_strides[1] * es;
  a.qo_tok = qo_strides[0] * es, a.qo_head = qo_strides[1] * es;
  a.num_q_heads = static_cast<int>(num_q_heads);
  a.rows_per_token = a.num_q_heads;
  if (has_k) {
    a.k = static_cast<const char*>(key);
    a.k_out = static_cast<char*>(key_out);
    a.k_tok = k_strides[0] * es, a.k_head = k_strides[1] * es;
    a.ko_tok = ko_strides[0] * es, a.ko_head = ko_strides[1] * es;
    a.rows_per_token += static_cast<int>(num_kv_heads);
  }
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.factor = factor;
  a.num_tokens = num_tokens;
  a.head_dim = static_cast<int>(head_dim);
  a.pairs = static_cast<int>(pairs);
  return launch_rotary<ROTARY_DENSE, false>(
      fn, a, layout, dtype,
      vec_bytes({address(query), address(query_out), address(key), address(key_out), a.q_tok, a.q_head,
                 a.qo_tok, a.qo_head, a.k_tok, a.k_head, a.ko_tok, a.ko_head}),
      nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int sb_rotary_scatter_paged_layers(
    const uint64_t* kv_layer_ptrs, const uint64_t* donor_layer_ptrs, int64_t num_layers,
    const int32_t* block_table, const int32_t* donor_pos, const int32_t* target_pos,
    const float* inv_freq, int64_t num_pairs, int64_t num_heads, int64_t block_size, int64_t head_dim,
    int64_t donor_seq_len, int64_t num_blocks_total, int64_t num_blocks_per_seq,
    const int64_t* kv_strides, const int64_t* d_strides, int64_t pairs, int32_t layout, int32_t dtype,
    int32_t flags, void* stream) {
  using namespace sb;
  const char* fn = "sb_rotary_scatter_paged_layers";
  clear_error();
  if (num_pairs == 0) return SB_OK;
  RotaryArgs a = {};
  const int rc = paged_args(fn, &a, kv_layer_ptrs, num_layers, block_table, inv_freq, num_pairs,
                            num_heads, block_size, head_dim, num_blocks_total, num_blocks_per_seq,
                            pairs, layout, dtype);
  if (rc != SB_OK) return rc;
  if (!donor_layer_ptrs || !donor_pos || !target_pos || !kv_strides || !d_strides)
    return fail(fn, "null pointer");
  if (donor_seq_len <= 0) return fail(fn, "sizes must be positive");
  if (flags & ~SB_SCATTER_FLAGS_ALL) return fail(fn, "unknown flags");
  if (kv_strides[4] != 1 || d_strides[3] != 1)
    return fail(fn, "the last dimension must be contiguous");
  const int64_t es = elem_size(dtype);
  a.donors = donor_layer_ptrs;
  a.c_block = kv_strides[0] * es, a.c_kv = kv_strides[1] * es, a.c_head = kv_strides[2] * es;
  a.c_pos = kv_strides[3] * es;
  a.d_kv = d_strides[0] * es, a.d_head = d_strides[1] * es, a.d_pos = d_strides[2] * es;
  a.donor_len = donor_seq_len;
  a.from = donor_pos;
  a.positions = target_pos;
  a.rows_per_token = static_cast<int>(2 * num_layers * num_heads);
  const int vb = vec_bytes({a.c_block, a.c_kv, a.c_head, a.c_pos, a.d_kv, a.d_head, a.d_pos});
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return flags & SB_SCATTER_REPEATED_DONOR_ROWS
             ? launch_rotary<ROTARY_SCATTER, false>(fn, a, layout, dtype, vb, nullptr, st)
             : launch_rotary<ROTARY_SCATTER, true>(fn, a, layout, dtype, vb, nullptr, st);
}

extern "C" int sb_rotary_shift_paged_layers(
    const uint64_t* kv_layer_ptrs, int64_t num_layers, const int32_t* block_table,
    const int32_t* positions, const int32_t* deltas, int64_t num_positions, const float* inv_freq,
    int64_t num_heads, int64_t block_size, int64_t head_dim, int64_t num_blocks_total,
    int64_t num_blocks_per_seq, const int64_t* kv_strides, int64_t pairs, int32_t layout, int32_t dtype,
    void* stream) {
  using namespace sb;
  clear_error();
  if (num_positions == 0) return SB_OK;
  return shift_layers("sb_rotary_shift_paged_layers", kv_layer_ptrs, num_layers, block_table, positions,
                      deltas, nullptr, num_positions, inv_freq, num_heads, block_size, head_dim,
                      num_blocks_total, num_blocks_per_seq, kv_strides, pairs, layout, dtype,
                      static_cast<hipStream_t>(stream));
}

extern "C" int sb_rotary_shift_paged_layers_host(
    const uint64_t* kv_layer_ptrs, int64_t num_layers, const int32_t* block_table,
    const int32_t* positions, const int32_t* deltas, int64_t num_positions, const float* inv_freq,
    int64_t num_heads, int64_t block_size, int64_t head_dim, int64_t num_blocks_total,
    int64_t num_blocks_per_seq, const int64_t* kv_strides, int64_t pairs, int32_t layout, int32_t dtype,
    void* stream) {
  using namespace sb;
  const char* fn = "sb_rotary_shift_paged_layers_host";
  clear_error();
  if (num_positions == 0) return SB_OK;
  if (!positions || !deltas) return fail(fn, "null pointer");
  if (num_positions < 0 || num_positions > SB_INLINE_POSITIONS_MAX)
    return fail(fn, "between 1 and " + std::to_string(SB_INLINE_POSITIONS_MAX) + " positions");
  RotaryInline list = {};
  std::copy(positions, positions + num_positions, list.pos);
  std::copy(deltas, deltas + num_positions, list.delta);
  return shift_layers(fn, kv_layer_ptrs, num_layers, block_table, nullptr, nullptr, &list,
                      num_positions, inv_freq, num_heads, block_size, head_dim, num_blocks_total,
                      num_blocks_per_seq, kv_strides, pairs, layout, dtype,
                      static_cast<hipStream_t>(stream));
}
