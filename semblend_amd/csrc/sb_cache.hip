// Appending new keys and values to a paged cache, and reading cache rows back, for gfx950.
//
// Append: token t of request r at position p goes to page table[r][p / bs], slot p % bs; K (and
// the query, written to a buffer of its own) is rotated by p on the way. Pages hold the tokens'
// own type, or MXFP4: 4-bit values (1 sign, 2 exponent, 1 mantissa bit: 0, 1/2, 1, 3/2, 2, 3, 4,
// 6) in blocks of 32 of a row that share a power of two 2^e, kept as the byte e + 127. With a the
// block's largest magnitude, e is the smallest integer with a <= 7 * 2^e: the step at a is then
// never wider than what rounding to 4 bits gives there (7 rounds to 6, off by half the step
// between 6 and 8), and no block is scaled one power further than that needs.
//
// Arithmetic: the angle p * f_i is formed and reduced in 64 bits (f_i the fp32 frequencies): its
// fp32 product is off by 2^-11 at position 16384, a quarter of a bf16 rounding. 16-bit pages take
// the rotation itself in fp32 with one rounding, fp32 pages in 64 bits. For 4-bit pages a value
// next to a border between two codes must fall on the side where its 64-bit value lies: blocks
// are rotated in fp32 and rounded to nearest even by v_cvt_scalef32_pk_fp4_f32, and again with
// the error's bound added and taken off; where the three agree on codes and scale the 64-bit
// result has the same ones. The others (one block in some thousands) are rotated in 64 bits and
// rounded to fp32 to odd, which keeps every comparison with a border (borders have few bits, an
// odd last bit never equals one), then rounded the same way. (16000 tokens of 8 heads x 128:
// 25.9 us.)
//
// What bounds it: bytes for prompts, the launch and one dependent chain (position, table entry,
// row) for decode steps. One workgroup takes a few tokens with all their heads, so that each
// (token, frequency) pair's sine and cosine (about 45 fp64 instructions) is evaluated once and
// shared through LDS by the K and query heads. Measured: 4587 tokens of 32 / 8 heads x 128, 113 MB
// in 20.7 us (5.4 TB/s; a large copy reaches 6.6); 16 tokens 4 us; 4099 tokens of 4 heads into 4-bit
// pages 8.4 us, 16000 of 8 heads 25.9 (instructions: a third sines and cosines, the rest rotation,
// scales and codes); reading 16384 of 8 heads back 18.6 us (85 MB, 4.6 TB/s).
#include "sb_rows.h"

namespace sb {
namespace {

// Rows in flight of a thread; half pairs, two vectors a row: 2 (4602 tokens of 32 / 8 heads x 128: 21.1 us,
// with 4 21.9).
constexpr int kRowsInFlight = 4, kHalfRowsInFlight = 2;

struct AppendArgs {
  const char* k;
  const char* v;
  const char* q;
  char* q_out;
  int64_t k_tok, k_head, v_tok, v_head, q_tok, q_head, qo_tok, qo_head;  // byte strides
  char* cache;
  char* scales;
  int64_t c_block, c_kv, c_head, c_pos;   // byte strides of the cache (4 bit: of the codes)
  int64_t s_block, s_kv, s_head, s_pos;   // byte strides of the scale bytes
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* positions;
  const int32_t* rotations;               // angle positions, or nullptr: the slot's position
  const int32_t* row_starts;              // nullptr: token t is request t's, or the only one's
  const float* inv_freq;                  // nullptr: no rotation
  int64_t num_tokens;
  int64_t num_blocks_total, num_blocks_per_seq;
  int num_requests, num_kv_heads, num_q_heads, head_dim, block_size;
  int tokens_per_wg, rows_per_y;
  int pairs;                              // pairs of a row that are turned
  double factor;                          // of the cosines and sines
  RowSplit split;
  Divisor row_div, half_div;              // by the rows of a token, by pairs
};

template <int DT, int VEC, bool Q4, bool HALF>
__global__ __launch_bounds__(kRowThreads) void append_kv_kernel(const AppendArgs a) {
  using CS = std::conditional_t<DT == SB_DTYPE_F32, double, float>;
  constexpr bool kBoth = Q4 && DT != SB_DTYPE_F32;         // 64-bit sines and cosines besides
  __shared__ __align__(16) CS cs[2 * kTableEntries];       // cosine, sine of each (token, pair)
  __shared__ double cs64[kBoth ? 2 * kTableEntries : 1];
  __shared__ __align__(16) RowRef rows[kRowsMax];
  const int tid = threadIdx.x;
  const int half = a.pairs;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_wg;
  const int ntok = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_wg), a.num_tokens - t0));

  const int upr = a.split.units;                // threads per row (at most kRowThreads)
  const int rpi = kRowThreads / upr;            // rows per step of the workgroup
  const int rsub = tid / upr, unit = tid - rsub * upr;
  const int hk = a.num_kv_heads;
  const int nrows = 2 * hk + a.num_q_heads;     // rows of a token
  // First of this workgroup's rows. (Several in y: of one token with many rows, or, where the rows of
  // a step do not divide kRowsMax, of tokens whose last rows a second workgroup takes.)
  const int j0 = blockIdx.y * a.rows_per_y;
  const int n = min(a.rows_per_y, ntok * nrows - j0);

  if (tid < n) {
    const int r0 = j0 + tid;
    const int tok = a.row_div.of(r0);
    const int j = r0 - tok * nrows;
    const int64_t t = t0 + tok;
    const int p = a.positions[t];
    RowRef ref = {nullptr, nullptr, nullptr, 0, 0};
    const int r = p < 0 ? -1
                  : a.row_starts ? request_of(a.row_starts, a.num_requests, static_cast<int>(t))
                  : a.num_requests == 1 ? 0 : static_cast<int>(t);
    if (r >= 0 && j >= 2 * hk) {
      ref.src = a.q + t * a.q_tok + (j - 2 * hk) * a.q_head;
      ref.dst = a.q_out + t * a.qo_tok + (j - 2 * hk) * a.qo_head;
    } else if (r >= 0) {
      const int kv = j >= hk, h = j - kv * hk;
      const int lb = p / a.block_size, slot = p - lb * a.block_size;
      const int64_t pb = lb < a.num_blocks_per_seq ? a.tables[r * a.table_stride + lb] : -1;
      if (pb >= 0 && pb < a.num_blocks_total) {
        ref.src = kv ? a.v + t * a.v_tok + h * a.v_head : a.k + t * a.k_tok + h * a.k_head;
        ref.dst = a.cache + pb * a.c_block + slot * a.c_pos + kv * a.c_kv + h * a.c_head;
        if (Q4) ref.sdst = a.scales + pb * a.s_block + slot * a.s_pos + kv * a.s_kv + h * a.s_head;
      }
    }
    const bool turn = a.inv_freq && (j < hk || j >= 2 * hk);
    ref.info = static_cast<uint32_t>(2 * tok * half) << 2 | (Q4 && j < 2 * hk ? 2u : 0u) |
               (turn ? 1u : 0u);
    rows[tid] = ref;
  }
  if (a.inv_freq) {
    // (from the last wave down: the first ones look the pages up)
    for (int i = kRowThreads - 1 - tid; i < ntok * half; i += kRowThreads) {
      const int tok = a.half_div.of(i), f = i - tok * half;
      const int p = (a.rotations ? a.rotations : a.positions)[t0 + tok];
      double s, c;
      sincos_cw(static_cast<double>(p) * static_cast<double>(a.inv_freq[f]), &s, &c);
      c *= a.factor, s *= a.factor;
      CS* to = cs + 2 * tok * half + Sines<DT, VEC, HALF>::at(f, half);
      to[0] = static_cast<CS>(c);
      to[1] = static_cast<CS>(s);
      if constexpr (kBoth) cs64[2 * i] = c, cs64[2 * i + 1] = s;
    }
  }
  __syncthreads();
  if (rsub >= rpi) return;

  constexpr int kFlight = HALF ? kHalfRowsInFlight : kRowsInFlight;
  turn_rows<DT, VEC, Q4, HALF, false, kFlight>(rows, n, cs, cs64, a.split, a.head_dim, a.pairs, rsub, rpi, unit);
}

// ---------------------------------------------------------------------------------------
// Rows read back: out[kv, h, i] = the cache row of position positions[i], in the output's type.
// ---------------------------------------------------------------------------------------
struct GatherArgs {
  char* out;
  int64_t o_kv, o_head, o_row;            // byte strides
  const char* cache;
  const char* scales;
  int64_t c_block, c_kv, c_head, c_pos;
  int64_t s_block, s_kv, s_head, s_pos;
  const int32_t* table;
  const int32_t* positions;               // nullptr: 0 .. num_rows - 1
  int64_t num_rows;
  int64_t num_blocks_total, num_blocks_per_seq;
  int num_kv_heads, head_dim, block_size;
  int planes_per_y;
};

constexpr int kGatherThreads = 256;

// VEC values of a word of codes; one instruction converts two (fp16: and rounds them).
template <int DT, int VEC>
__device__ __forceinline__ void unpack_codes(uint32_t w, float scale, typename Elem<DT>::T* e) {
  auto put = [&](int i, auto pair) { __builtin_memcpy(e + 2 * i, &pair, sizeof(pair)); };
#define SB_UNPACK(I)                                                                      \
  if constexpr (2 * I < VEC) {                                                            \
    if constexpr (DT == SB_DTYPE_F32) put(I, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, I)); \
    else if constexpr (DT == SB_DTYPE_F16)                                                \
      put(I, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, I));                      \
    else put(I, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I));                  \
  }
  SB_UNPACK(0)
  SB_UNPACK(1)
  SB_UNPACK(2)
  SB_UNPACK(3)
#undef SB_UNPACK
}

// A thread takes VEC elements of one position and some of its 2 Hkv rows, four in flight: the
// position and its table entry are read once. Positions without a page give zeros.
template <int DT, int VEC, bool Q4>
__global__ __launch_bounds__(kGatherThreads) void gather_kv_kernel(const GatherArgs a) {
  constexpr int ES = sizeof(typename Elem<DT>::T);
  const int vpr = a.head_dim / VEC;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * kGatherThreads + threadIdx.x;
  const int64_t i = idx <= 0xffffffffll
                        ? static_cast<int64_t>(static_cast<uint32_t>(idx) / static_cast<uint32_t>(vpr))
                        : idx / vpr;
  if (i >= a.num_rows) return;
  const int vec = static_cast<int>(idx - i * vpr);
  const int p = a.positions ? a.positions[i] : static_cast<int>(i);
  int64_t oc = -1, os = 0;
  if (p >= 0) {
    const int lb = p / a.block_size, slot = p - lb * a.block_size;
    if (lb < a.num_blocks_per_seq) {
      const int64_t pb = a.table[lb];
      if (pb >= 0 && pb < a.num_blocks_total) {
        oc = pb * a.c_block + slot * a.c_pos;
        os = pb * a.s_block + slot * a.s_pos + vec * VEC / 32;
      }
    }
  }
  const int j0 = blockIdx.y * a.planes_per_y;
  const int j1 = min(j0 + a.planes_per_y, 2 * a.num_kv_heads);
  char* dst = a.out + i * a.o_row + static_cast<int64_t>(vec) * VEC * ES;
  constexpr int U = 4;
  for (int jb = j0; jb < j1; jb += U) {
    RowVec<DT, VEC> x[U];
    uint32_t w[U], sb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(jb + u, j1 - 1);
      const int kv = j >= a.num_kv_heads, h = j - kv * a.num_kv_heads;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[u].e[e] = 0;
      w[u] = 0;
      sb[u] = 0;
      if (oc >= 0) {
        const char* src = a.cache + oc + kv * a.c_kv + h * a.c_head;
        if constexpr (Q4) {
          src += vec * (VEC / 2);
          if constexpr (VEC == 8) w[u] = *reinterpret_cast<const uint32_t*>(src);
          else if constexpr (VEC == 4) w[u] = *reinterpret_cast<const uint16_t*>(src);
          else w[u] = *reinterpret_cast<const uint8_t*>(src);
          sb[u] = static_cast<uint8_t>(a.scales[os + kv * a.s_kv + h * a.s_head]);
        } else {
          x[u].load(src + static_cast<int64_t>(vec) * VEC * ES);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jb + u;
      if (j >= j1) break;
      const int kv = j >= a.num_kv_heads, h = j - kv * a.num_kv_heads;
      if constexpr (Q4) {
        if (oc >= 0) {
          // (the exponent field alone is the scale: byte 0 is 2^-127, byte 255 gives NaN)
          unpack_codes<DT, VEC>(w[u], __uint_as_float(sb[u] << 23), x[u].e);
        }
      }
      x[u].store(dst + kv * a.o_kv + h * a.o_head);
    }
  }
}

// Byte strides of a cache given in elements (4 bit: codes in bytes, scales in bytes).
struct CacheStrides {
  int64_t block, kv, head, pos;
};
CacheStrides cache_strides(const int64_t* s, int64_t es) {
  return {s[0] * es, s[1] * es, s[2] * es, s[3] * es};
}

// Both append entries; `pairs` pairs of a row are turned (0: all of it).
int append_kv(
    const char* fn, void* kv_cache, void* kv_scales, const void* key, const void* value, const void* query,
    void* query_out, const int32_t* block_tables, int64_t table_stride, const int32_t* positions,
    const int32_t* rotations, const int32_t* row_starts, const float* inv_freq,
    int64_t num_tokens, int64_t num_requests, int64_t num_kv_heads, int64_t num_q_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks_total, int64_t num_blocks_per_seq,
    const int64_t* k_strides, const int64_t* v_strides, const int64_t* q_strides,
    const int64_t* qo_strides, const int64_t* kv_strides, const int64_t* scale_strides,
    int64_t pairs, int32_t layout, double factor, int32_t dtype, int32_t cache_dtype, void* stream) {
  clear_error();
  if (num_tokens == 0) return SB_OK;
  if (!valid_dtype(dtype)) return fail(fn, "invalid dtype");
  const bool q4 = cache_dtype == SB_DTYPE_MXFP4;
  if (!q4 && cache_dtype != dtype) return fail(fn, "the cache's dtype is neither the keys' nor MXFP4");
  const bool has_q = query != nullptr;
  if (!kv_cache || !key || !value || !block_tables || !positions || !k_strides || !v_strides ||
      !kv_strides || (q4 && (!kv_scales || !scale_strides)) ||
      (has_q && (!query_out || !q_strides || !qo_strides)))
    return fail(fn, "null pointer");
  if (num_tokens < 0 || num_requests <= 0 || num_kv_heads <= 0 || (has_q && num_q_heads <= 0) ||
      block_size <= 0 || num_blocks_total <= 0 || num_blocks_per_seq <= 0)
    return fail(fn, "sizes must be positive");
  if (num_tokens > 0x7fffffff || num_requests > 0x7fffffff || num_kv_heads > 65535 ||
      num_q_heads > 65535 || block_size > 0x7fffffff)
    return fail(fn, "size past 32 bits");
  if (head_dim <= 0 || head_dim % 2 || head_dim > 512)
    return fail(fn, "head_dim must be even and at most 512");
  if (q4 && head_dim % 32) return fail(fn, "4-bit pages need a head_dim that is a multiple of 32");
  const bool half = inv_freq && layout == SB_ROTARY_HALF;
  if (inv_freq) {
    if (const char* why = rotary_fault(head_dim, pairs, layout, factor)) return fail(fn, why);
    if (q4 && (half ? pairs % 32 || (head_dim - 2 * pairs) % 64 : pairs % 16))
      return fail(fn, "4-bit pages need whole blocks of 32 values in each half of what is rotated and of "
                      "what is not");
  } else {
    pairs = head_dim / 2;
  }
  if (!row_starts && num_requests > 1 && num_tokens > num_requests)
    return fail(fn, "without row_starts there is one token per request");
  if (k_strides[2] != 1 || v_strides[2] != 1 || kv_strides[4] != 1 ||
      (q4 && scale_strides[4] != 1) || (has_q && (q_strides[2] != 1 || qo_strides[2] != 1)))
    return fail(fn, "the last dimension must be contiguous");
  if (has_q && rows_overlap(num_tokens, num_q_heads, head_dim, qo_strides[0], qo_strides[1]))
    return fail(fn, "rows of query_out must not overlap");
  const int64_t es = elem_size(dtype);
  AppendArgs a = {};
  a.k = static_cast<const char*>(key);
  a.v = static_cast<const char*>(value);
  a.q = static_cast<const char*>(query);
  a.q_out = static_cast<char*>(query_out);
  a.k_tok = k_strides[0] * es, a.k_head = k_strides[1] * es;
  a.v_tok = v_strides[0] * es, a.v_head = v_strides[1] * es;
  if (has_q) {
    a.q_tok = q_strides[0] * es, a.q_head = q_strides[1] * es;
    a.qo_tok = qo_strides[0] * es, a.qo_head = qo_strides[1] * es;
  }
  const CacheStrides c = cache_strides(kv_strides, q4 ? 1 : es);
  a.cache = static_cast<char*>(kv_cache);
  a.c_block = c.block, a.c_kv = c.kv, a.c_head = c.head, a.c_pos = c.pos;
  if (q4) {
    a.scales = static_cast<char*>(kv_scales);
    a.s_block = scale_strides[0], a.s_kv = scale_strides[1];
    a.s_head = scale_strides[2], a.s_pos = scale_strides[3];
  }
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.positions = positions;
  a.rotations = rotations;
  a.row_starts = row_starts;
  a.inv_freq = inv_freq;
  a.pairs = static_cast<int>(pairs);
  a.factor = factor;
  a.num_tokens = num_tokens;
  a.num_requests = static_cast<int>(num_requests);
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.num_q_heads = has_q ? static_cast<int>(num_q_heads) : 0;
  a.head_dim = static_cast<int>(head_dim);
  a.block_size = static_cast<int>(block_size);
  a.num_blocks_total = num_blocks_total;
  a.num_blocks_per_seq = num_blocks_per_seq;

  const auto addr = [](const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); };
  int vb = vec_bytes({addr(key), addr(value), addr(query), addr(query_out), a.k_tok, a.k_head,
                      a.v_tok, a.v_head, a.q_tok, a.q_head, a.qo_tok, a.qo_head, head_dim * es,
                      (half ? pairs : 2 * pairs) * es});
  const int64_t cells[] = {addr(kv_cache), c.block, c.kv, c.head, c.pos};
  const int64_t cell = q4 ? 16 / es / 2 : 16;  // bytes of the cache that 16 bytes of a row become
  for (int64_t x : cells)
    if (x % cell) vb = 2;
  const bool wide = vb == 16;
  const int vec = wide ? static_cast<int>(16 / es) : 2;
  // Tokens per workgroup: as many as fill its threads' first rows in flight (and the table of sines
  // and cosines takes). Few tokens: one, and its rows spread over workgroups until there are 512
  // (each repeats the sines and cosines).
  const int nrows = 2 * a.num_kv_heads + a.num_q_heads;
  a.split = RowSplit::of(a.head_dim, a.pairs, vec, half);
  const int rpi = kRowThreads / a.split.units;
  const int fit = std::min(kTokensMax, std::max(1, kTableEntries / a.pairs));
  const int full = std::max(1, std::min(fit, std::min(kRowsInFlight * rpi, kRowsMax) / nrows));
  a.tokens_per_wg = num_tokens >= 512 * static_cast<int64_t>(full) ? full : 1;
  const int64_t gx = (num_tokens + a.tokens_per_wg - 1) / a.tokens_per_wg;
  const int all = a.tokens_per_wg * nrows;
  const int steps = (all + rpi - 1) / rpi;
  const int ny = a.tokens_per_wg > 1
                     ? 1 : static_cast<int>(std::min<int64_t>(std::max<int64_t>(1, 512 / gx), steps));
  a.rows_per_y = std::min((steps + ny - 1) / ny, kRowsMax / rpi) * rpi;
  a.row_div = Divisor::by(nrows);
  a.half_div = Divisor::by(a.pairs);
  const dim3 grid(static_cast<unsigned>(gx),
                  static_cast<unsigned>((all + a.rows_per_y - 1) / a.rows_per_y));
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SB_APPEND_(DT, VEC, Q4, HALF)                                                            \
  SB_LAUNCH("append_kv", (append_kv_kernel<DT, VEC, Q4, HALF>), grid, dim3(kRowThreads), st, a)
#define SB_APPEND(DT, VEC)                  \
  if (dtype == DT && vec == VEC) {          \
    if (q4 && half)                         \
      SB_APPEND_(DT, VEC, true, true);      \
    else if (q4)                            \
      SB_APPEND_(DT, VEC, true, false);     \
    else if (half)                          \
      SB_APPEND_(DT, VEC, false, true);     \
    else                                    \
      SB_APPEND_(DT, VEC, false, false);    \
  }
  SB_APPEND(SB_DTYPE_F32, 4)
  SB_APPEND(SB_DTYPE_F32, 2)
  SB_APPEND(SB_DTYPE_F16, 8)
  SB_APPEND(SB_DTYPE_F16, 2)
  SB_APPEND(SB_DTYPE_BF16, 8)
  SB_APPEND(SB_DTYPE_BF16, 2)
#undef SB_APPEND
#undef SB_APPEND_
  return check_launch(fn);
}

}  // namespace
}  // namespace sb

extern "C" int sb_append_kv_paged(
    void* kv_cache, void* kv_scales, const void* key, const void* value, const void* query,
    void* query_out, const int32_t* block_tables, int64_t table_stride, const int32_t* positions,
    const int32_t* rotations, const int32_t* row_starts, const float* inv_freq,
    int64_t num_tokens, int64_t num_requests, int64_t num_kv_heads, int64_t num_q_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks_total, int64_t num_blocks_per_seq,
    const int64_t* k_strides, const int64_t* v_strides, const int64_t* q_strides,
    const int64_t* qo_strides, const int64_t* kv_strides, const int64_t* scale_strides,
    int32_t dtype, int32_t cache_dtype, void* stream) {
  return sb::append_kv("sb_append_kv_paged", kv_cache, kv_scales, key, value, query, query_out,
                       block_tables, table_stride, positions, rotations, row_starts, inv_freq,
                       num_tokens, num_requests, num_kv_heads, num_q_heads, head_dim, block_size,
                       num_blocks_total, num_blocks_per_seq, k_strides, v_strides, q_strides,
                       qo_strides, kv_strides, scale_strides, head_dim / 2, SB_ROTARY_INTERLEAVED,
                       1.0, dtype, cache_dtype, stream);
}

extern "C" int sb_append_kv_rotary_paged(
    void* kv_cache, void* kv_scales, const void* key, const void* value, const void* query,
    void* query_out, const int32_t* block_tables, int64_t table_stride, const int32_t* positions,
    const int32_t* rotations, const int32_t* row_starts, const float* inv_freq,
    int64_t num_tokens, int64_t num_requests, int64_t num_kv_heads, int64_t num_q_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks_total, int64_t num_blocks_per_seq,
    const int64_t* k_strides, const int64_t* v_strides, const int64_t* q_strides,
    const int64_t* qo_strides, const int64_t* kv_strides, const int64_t* scale_strides,
    int64_t pairs, int32_t layout, double factor, int32_t dtype, int32_t cache_dtype, void* stream) {
  if (!inv_freq && num_tokens != 0)
    return sb::fail("sb_append_kv_rotary_paged", "null pointer");
  return sb::append_kv("sb_append_kv_rotary_paged", kv_cache, kv_scales, key, value, query, query_out,
                       block_tables, table_stride, positions, rotations, row_starts, inv_freq,
                       num_tokens, num_requests, num_kv_heads, num_q_heads, head_dim, block_size,
                       num_blocks_total, num_blocks_per_seq, k_strides, v_strides, q_strides,
                       qo_strides, kv_strides, scale_strides, pairs, layout, factor, dtype, cache_dtype,
                       stream);
}

extern "C" int sb_gather_kv_paged(void* out, const void* kv_cache, const void* kv_scales,
                                  const int32_t* block_table, const int32_t* positions,
                                  int64_t num_rows, int64_t num_kv_heads, int64_t head_dim,
                                  int64_t block_size, int64_t num_blocks_total,
                                  int64_t num_blocks_per_seq, const int64_t* o_strides,
                                  const int64_t* kv_strides, const int64_t* scale_strides,
                                  int32_t dtype, int32_t cache_dtype, void* stream) {
  using namespace sb;
  const char* fn = "sb_gather_kv_paged";
  clear_error();
  if (num_rows == 0) return SB_OK;
  if (!valid_dtype(dtype)) return fail(fn, "invalid dtype");
  const bool q4 = cache_dtype == SB_DTYPE_MXFP4;
  if (!q4 && cache_dtype != dtype) return fail(fn, "the cache's dtype is neither the output's nor MXFP4");
  if (!out || !kv_cache || !block_table || !o_strides || !kv_strides ||
      (q4 && (!kv_scales || !scale_strides)))
    return fail(fn, "null pointer");
  if (num_rows < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks_total <= 0 ||
      num_blocks_per_seq <= 0)
    return fail(fn, "sizes must be positive");
  if (num_rows > 0x7fffffff || num_kv_heads > 65535 || block_size > 0x7fffffff)
    return fail(fn, "size past 32 bits");
  if (head_dim <= 0 || head_dim % 2 || head_dim > 512)
    return fail(fn, "head_dim must be even and at most 512");
  if (q4 && head_dim % 32) return fail(fn, "4-bit pages need a head_dim that is a multiple of 32");
  if (o_strides[3] != 1 || kv_strides[4] != 1 || (q4 && scale_strides[4] != 1))
    return fail(fn, "the last dimension must be contiguous");
  const int64_t es = elem_size(dtype);
  GatherArgs a = {};
  a.out = static_cast<char*>(out);
  a.o_kv = o_strides[0] * es, a.o_head = o_strides[1] * es, a.o_row = o_strides[2] * es;
  const CacheStrides c = cache_strides(kv_strides, q4 ? 1 : es);
  a.cache = static_cast<const char*>(kv_cache);
  a.c_block = c.block, a.c_kv = c.kv, a.c_head = c.head, a.c_pos = c.pos;
  if (q4) {
    a.scales = static_cast<const char*>(kv_scales);
    a.s_block = scale_strides[0], a.s_kv = scale_strides[1];
    a.s_head = scale_strides[2], a.s_pos = scale_strides[3];
  }
  a.table = block_table;
  a.positions = positions;
  a.num_rows = num_rows;
  a.num_blocks_total = num_blocks_total;
  a.num_blocks_per_seq = num_blocks_per_seq;
  a.num_kv_heads = static_cast<int>(num_kv_heads);
  a.head_dim = static_cast<int>(head_dim);
  a.block_size = static_cast<int>(block_size);
  const auto addr = [](const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); };
  int vb = vec_bytes({addr(out), a.o_kv, a.o_head, a.o_row, head_dim * es});
  const int64_t cell = q4 ? 16 / es / 2 : 16;
  const int64_t cells[] = {addr(kv_cache), c.block, c.kv, c.head, c.pos};
  for (int64_t x : cells)
    if (x % cell) vb = 2;
  const int vec = vb == 16 ? static_cast<int>(16 / es) : 2;
  const int64_t gx = (num_rows * (head_dim / vec) + kGatherThreads - 1) / kGatherThreads;
  if (gx > 0x7fffffff) return fail(fn, "grid too large");
  const int planes = 2 * a.num_kv_heads;
  // Up to eight rows a thread behind one lookup, fewer until there are 2048 workgroups.
  const int64_t want = std::max<int64_t>(1, 2048 / gx);
  a.planes_per_y = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, planes / want)));
  const dim3 grid(static_cast<unsigned>(gx),
                  static_cast<unsigned>((planes + a.planes_per_y - 1) / a.planes_per_y));
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SB_GATHER(DT, VEC)                                                                      \
  if (dtype == DT && vec == VEC) {                                                              \
    if (q4)                                                                                     \
      SB_LAUNCH("gather_kv", (gather_kv_kernel<DT, VEC, true>), grid, dim3(kGatherThreads), st, a); \
    else                                                                                        \
      SB_LAUNCH("gather_kv", (gather_kv_kernel<DT, VEC, false>), grid, dim3(kGatherThreads), st, a); \
  }
  SB_GATHER(SB_DTYPE_F32, 4)
  SB_GATHER(SB_DTYPE_F32, 2)
  SB_GATHER(SB_DTYPE_F16, 8)
  SB_GATHER(SB_DTYPE_F16, 2)
  SB_GATHER(SB_DTYPE_BF16, 8)
  SB_GATHER(SB_DTYPE_BF16, 2)
#undef SB_GATHER
  return check_launch(fn);
}
