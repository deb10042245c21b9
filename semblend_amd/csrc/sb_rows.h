// Rows of a head's elements moved from one place to another and turned on the way: what the kernels
// of the paged cache (sb_cache.hip) and of the rotary positions (sb_rotary.hip) share (gfx950).
//
// A pair (a, b) of a row becomes (a c - b s, a s + b c), c and s the cosine and sine of its token's
// angle. Interleaved pairs (2i, 2i + 1) lie in one 16-byte vector. Half pairs (i, i + pairs) lie
// `pairs` elements apart, so a thread takes two vectors of a row, one of each half: both outputs of a
// pair come from registers of one thread, a row may be turned in place, and no value is loaded twice.
#pragma once

#include "sb_common.h"
#include "sb_overlap.h"

#include <algorithm>
#include <type_traits>

namespace sb {
namespace {

constexpr int kRowThreads = 256;
constexpr int kTableEntries = 512;   // (token, frequency) pairs of one workgroup
constexpr int kTokensMax = 8;
constexpr int kRowsMax = 256;        // rows (K, V and query heads of its tokens) of one workgroup

// x / d for 0 <= x < 2^31: with l = ceil(log2 d) and m = ceil(2^(31+l) / d), m d - 2^(31+l) < d <=
// 2^l, so x * m >> (31 + l) is exact (T. Granlund and P. Montgomery, "Division by invariant integers
// using multiplication", 1994).
struct Divisor {
  uint32_t magic;
  int shift;
  static Divisor by(int d) {
    int shift = 31;
    while ((1ll << (shift - 31)) < d) ++shift;
    return {static_cast<uint32_t>(((1ull << shift) + d - 1) / d), shift};
  }
  __device__ __forceinline__ int of(int x) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * magic) >> shift);
  }
};

// Request of row t, or -1 before the first and behind the last one: the last r with
// row_starts[r] <= t.
__device__ __forceinline__ int request_of(const int32_t* row_starts, int num_requests, int t) {
  if (t < row_starts[0] || t >= row_starts[num_requests]) return -1;
  int lo = 0, hi = num_requests;  // row_starts[lo] <= t < row_starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row_starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// An element's value, and two values rounded to elements.
template <int DT> struct Elem;
template <> struct Elem<SB_DTYPE_F32> {
  using T = float;
  __device__ static float get(float x) { return x; }
  __device__ static void put2(float a, float b, float* e) { e[0] = a, e[1] = b; }
};
template <> struct Elem<SB_DTYPE_F16> {
  using T = uint16_t;
  __device__ static float get(uint16_t x) { return f16_to_f32(x); }
  __device__ static void put2(float a, float b, uint16_t* e) {
    e[0] = f32_to_f16(a), e[1] = f32_to_f16(b);
  }
};
template <> struct Elem<SB_DTYPE_BF16> {
  using T = uint16_t;
  __device__ static float get(uint16_t x) { return bf16_to_f32(x); }
  __device__ static void put2(float a, float b, uint16_t* e) {
    const uint32_t w = pack2_bf16(a, b);
    e[0] = static_cast<uint16_t>(w), e[1] = static_cast<uint16_t>(w >> 16);
  }
};

// Device memory (a pointer that went through LDS would be taken for any kind, and its loads wait
// with LDS's).
#define SB_GLOBAL __attribute__((address_space(1)))
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// VEC elements of a row: 16 bytes, or (VEC 2) a pair, element by element at any alignment.
template <int DT, int VEC> struct RowVec {
  using T = typename Elem<DT>::T;
  static constexpr bool kWide = VEC * sizeof(T) == 16;
  T e[VEC];
  template <bool ONCE = false>  // ONCE: no other thread reads it, nontemporal
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (kWide) {
      const u32x4_t w = ONCE ? __builtin_nontemporal_load((const SB_GLOBAL u32x4_t*)p)
                             : *(const SB_GLOBAL u32x4_t*)p;
      __builtin_memcpy(e, &w, 16);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = ((const SB_GLOBAL T*)p)[i];
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (kWide) {
      // (nontemporal: append of 4587 tokens of 32 / 8 heads x 128 24.4 -> 21.1 us)
      u32x4_t w;
      __builtin_memcpy(&w, e, 16);
      __builtin_nontemporal_store(w, (SB_GLOBAL u32x4_t*)p);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) ((SB_GLOBAL T*)p)[i] = e[i];
    }
  }
};

// x rounded to fp32 to odd: the result's comparisons with fp32 values of an even last bit are x's.
__device__ __forceinline__ float round_to_odd(double x) {
  const float f = static_cast<float>(x);
  uint32_t u = __float_as_uint(f);
  const double back = static_cast<double>(f);
  if (back != x && (u & 1u) == 0 && (u & 0x7fffffffu) < 0x7f800000u)
    u += (fabs(x) > fabs(back)) ? 1u : 0xffffffffu;  // (toward x; f = 0 only moves outwards)
  return __uint_as_float(u);
}

// The scale byte of a block whose largest magnitude is `top`, a number: top in
// [4, 8) * 2^(E - 2 - 127), and one power more above 7 (mantissa above 1.75).
__device__ __forceinline__ int scale_byte(float top) {
  const uint32_t u = __float_as_uint(top);
  return max(static_cast<int>(u >> 23) - 2 + ((u & 0x7fffffu) > 0x600000u), 0);
}
template <int VEC>
__device__ __forceinline__ uint32_t pack_codes(const float (&f)[VEC], float scale) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], scale, 0);
  if constexpr (VEC >= 4) w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[2], f[3], scale, 1);
  if constexpr (VEC >= 8) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[4], f[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[6], f[7], scale, 3);
  }
  return w;
}
// Largest of the 32 / VEC lanes that share a block of 32 values, in all of them: neighbours inside
// four lanes, then the mirror image inside eight and sixteen (DPP moves, no trip through LDS; with the
// two packings below instead of three, 16000 tokens of 8 heads 27.3 -> 25.9 us).
template <int VEC>
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 15, 15, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4e, 15, 15, true)));
  if constexpr (VEC <= 4)
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 15, 15, true)));
  if constexpr (VEC <= 2)
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 15, 15, true)));
  return v;
}
// The scale of a block; one that holds an infinity or a NaN is marked as one by scale byte 255.
struct Scale {
  int byte;
  bool bad;
  float top, value;
};
template <int VEC>
__device__ __forceinline__ Scale block_scale(const float (&f)[VEC]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  top = block_max<VEC>(top);
  Scale b;
  b.top = __uint_as_float(top);
  b.bad = top >= 0x7f800000u;
  b.byte = b.bad ? 255 : scale_byte(b.top);
  // (byte 0 is 2^-127, below fp32's normal numbers)
  b.value = __uint_as_float(b.byte > 0 && !b.bad ? static_cast<uint32_t>(b.byte) << 23 : 0x00400000u);
  return b;
}

// One thread per row works out where the row comes from and goes to, for all lanes of it: worked out
// by every lane, that (selects, divisions, 64-bit products) was most of the kernel's instructions: 4587 tokens of 32 / 8
// heads x 128 22.9 -> 20.9 us, 16000 of 8 heads into 4-bit pages 31.2 -> 27.0.
struct RowRef {
  const char* src;  // nullptr: left out (padding, or no slot)
  char* dst;
  char* sdst;       // scale bytes of a 4-bit row
  uint32_t info;    // index of the token's sines and cosines << 2 | a 4-bit row << 1 | rotated
  uint32_t pad;
};
// How a row's vectors fall to threads. Interleaved: thread u takes vector u. Half: u < P (P vectors in
// a half) takes vectors u and u + P, the others two of the rest (the last of them maybe one).
struct RowSplit {
  int half;    // vectors of a half (0: interleaved)
  int rest;    // units of two vectors behind the halves
  int units;   // threads a row takes
  static RowSplit of(int head_dim, int pairs, int vec, bool half_pairs) {
    const int v = head_dim / vec;
    if (!half_pairs) return {0, 0, v};
    const int p = pairs / vec;
    return {p, (v - 2 * p + 1) / 2, p + (v - 2 * p + 1) / 2};
  }
};

// A token's cosines and sines in LDS, 2 * pairs numbers. A thread's pairs are 32 or 64 bytes; they lie in
// pieces of 16, piece after piece of all threads of a row, so that the threads' reads of a piece are 16 bytes
// apart and fall on all banks.
template <int DT, int VEC, bool HALF> struct Sines {
  using CS = std::conditional_t<DT == SB_DTYPE_F32, double, float>;
  static constexpr int kPairs = HALF ? VEC : VEC / 2;  // of a thread
  static constexpr int kPiece = 16 / sizeof(CS);       // numbers
  static constexpr int kPieces = 2 * kPairs / kPiece;  // (0, 1: as they come)
  // Place of pair f's cosine (its sine follows), of `pairs`.
  __device__ __forceinline__ static int at(int f, int pairs) {
    if constexpr (kPieces <= 1) return 2 * f;
    const int e = f % kPairs * 2;
    return (e / kPiece * (pairs / kPairs) + f / kPairs) * kPiece + e % kPiece;
  }
  const CS* first;
  int step;
  __device__ __forceinline__ Sines(const CS* token, int unit, int pairs)
      : first(token + (kPieces <= 1 ? 2 * kPairs : kPiece) * unit), step(pairs / kPairs * kPiece) {}
  // Cosine and sine of the thread's pair i.
  template <typename T> __device__ __forceinline__ void get(int i, T* c, T* s) const {
    const CS* p = kPieces <= 1 ? first + 2 * i : first + 2 * i / kPiece * step + 2 * i % kPiece;
    *c = p[0], *s = p[1];
  }
};

// Rows rows[0 .. n) by a workgroup: thread `unit` of a row takes rows rsub + k rpi, FLIGHT of them at
// a time. cs: cosine and sine of each (token, pair), in Sines' order; cs64: the same in 64 bits, pair after pair
// (4-bit rows).
template <int DT, int VEC, bool Q4, bool HALF, bool ONCE, int FLIGHT>
__device__ __forceinline__ void turn_rows(
    const RowRef* rows, int n, const std::conditional_t<DT == SB_DTYPE_F32, double, float>* cs,
    const double* cs64, const RowSplit& split, int head_dim, int pairs, int rsub, int rpi, int unit) {
  using CS = std::conditional_t<DT == SB_DTYPE_F32, double, float>;
  constexpr bool kBoth = Q4 && DT != SB_DTYPE_F32;
  constexpr int ES = sizeof(typename Elem<DT>::T);
  constexpr int NV = HALF ? 2 : 1;
  // this thread's vectors, whether they are turned, and its first sine
  const bool paired = HALF ? unit < split.half : unit * VEC < 2 * pairs;
  int at[NV];
  at[0] = HALF && !paired ? unit + split.half : unit;
  if constexpr (HALF) at[1] = at[0] + (paired ? split.half : split.rest);
  const bool second = HALF && at[NV - 1] * VEC < head_dim;

  for (int ib = rsub; ib < n; ib += FLIGHT * rpi) {
    RowVec<DT, VEC> x[FLIGHT][NV];
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const char* src = rows[min(ib + u * rpi, n - 1)].src;
      if (src) {
        x[u][0].template load<ONCE>(src + at[0] * (VEC * ES));
        if constexpr (HALF)
          if (second) x[u][1].template load<ONCE>(src + at[1] * (VEC * ES));
      }
    }
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      if (ib + u * rpi >= n) break;
      const RowRef ref = rows[ib + u * rpi];
      if (!ref.src) continue;
      const Sines<DT, VEC, HALF> trig(cs + (ref.info >> 2), unit, pairs);
      const bool turn = (ref.info & 1u) && paired;
      float f[NV][VEC];
      if constexpr (HALF) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const CS e = Elem<DT>::get(x[u][0].e[i]), o = Elem<DT>::get(x[u][NV - 1].e[i]);
          if (turn) {
            CS c, s;
            trig.get(i, &c, &s);
            f[0][i] = static_cast<float>(e * c - o * s);
            f[NV - 1][i] = static_cast<float>(e * s + o * c);
          } else {
            f[0][i] = static_cast<float>(e);
            f[NV - 1][i] = static_cast<float>(o);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const CS e = Elem<DT>::get(x[u][0].e[i]), o = Elem<DT>::get(x[u][0].e[i + 1]);
          if (turn) {
            CS c, s;
            trig.get(i / 2, &c, &s);
            f[0][i] = static_cast<float>(e * c - o * s);
            f[0][i + 1] = static_cast<float>(e * s + o * c);
          } else {
            f[0][i] = static_cast<float>(e);
            f[0][i + 1] = static_cast<float>(o);
          }
        }
      }
      if (Q4 && (ref.info & 2u)) {
        Scale b[NV];
        uint32_t w[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) b[v] = block_scale(f[v]);
        if (turn) {
          // A rotated fp32 value is off by at most 2^-22 of its pair's norm (products and sum
          // 2^-24 each, sine and cosine 2^-24): 2^-21 of the largest magnitude of the blocks that
          // its pair lies in (one block, or with half pairs one of each half), which is below 2^-18
          // of the larger scale. Codes that agree at both ends agree between.
          const float top = HALF ? fmaxf(b[0].top, b[NV - 1].top) : b[0].top;
          const float off = 0x1p-18f * (HALF ? fmaxf(b[0].value, b[NV - 1].value) : b[0].value);
          uint32_t unsure = 0;
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            if constexpr (HALF)
              unsure |= b[v].bad || scale_byte(fmaxf(b[v].top - top * 0x1p-20f, 0.f)) !=
                                        scale_byte(b[v].top + top * 0x1p-20f);
            else
              unsure |= b[v].bad || scale_byte(b[v].top * (1.f - 0x1p-20f)) !=
                                        scale_byte(b[v].top * (1.f + 0x1p-20f));
            float lo[VEC], hi[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) lo[i] = f[v][i] - off, hi[i] = f[v][i] + off;
            w[v] = pack_codes(lo, b[v].value);
            unsure |= w[v] ^ pack_codes(hi, b[v].value);
          }
          if (block_max<VEC>(unsure)) {
            const double* t64 = kBoth ? cs64 + (ref.info >> 2) + unit * VEC * NV : nullptr;
            // (a sum of two values of the largest fp32 exponent may pass fp32, but not 7 * 2^126: such a
            // block, not finite above, is taken times 2^-2)
            const double down = b[0].bad ? 0.25 : 1.0, down_2 = b[NV - 1].bad ? 0.25 : 1.0;
            const int up[2] = {b[0].bad ? 2 : 0, b[NV - 1].bad ? 2 : 0};
#pragma unroll
            for (int i = 0; i < VEC; i += HALF ? 1 : 2) {
              const int j = HALF ? i : i + 1, t = HALF ? 2 * i : i;
              const double e = Elem<DT>::get(x[u][0].e[i]), o = Elem<DT>::get(x[u][NV - 1].e[j]);
              double c, s;
              if constexpr (kBoth) c = t64[t], s = t64[t + 1];
              else trig.get(t / 2, &c, &s);
              f[0][i] = round_to_odd((e * c - o * s) * down);
              f[NV - 1][j] = round_to_odd((e * s + o * c) * down_2);
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) {
              b[v] = block_scale(f[v]);
              w[v] = b[v].bad ? 0u : pack_codes(f[v], b[v].value);
              if (!b[v].bad) b[v].byte += up[v];
            }
          }
        } else {
#pragma unroll
          for (int v = 0; v < NV; ++v) w[v] = b[v].bad ? 0u : pack_codes(f[v], b[v].value);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          char* dst = ref.dst + at[v] * (VEC / 2);
          if constexpr (VEC == 8) *(SB_GLOBAL uint32_t*)dst = w[v];
          else if constexpr (VEC == 4) *(SB_GLOBAL uint16_t*)dst = static_cast<uint16_t>(w[v]);
          else *(SB_GLOBAL uint8_t*)dst = static_cast<uint8_t>(w[v]);
          if ((at[v] & (32 / VEC - 1)) == 0)
            ((SB_GLOBAL char*)ref.sdst)[at[v] / (32 / VEC)] = static_cast<char>(b[v].byte);
        }
      } else {
        if (turn) {
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) Elem<DT>::put2(f[v][i], f[v][i + 1], x[u][v].e + i);
        }
        x[u][0].store(ref.dst + at[0] * (VEC * ES));
        if constexpr (HALF)
          if (second) x[u][1].store(ref.dst + at[1] * (VEC * ES));
      }
    }
  }
}

inline bool valid_dtype(int32_t dt) {
  return dt == SB_DTYPE_F32 || dt == SB_DTYPE_F16 || dt == SB_DTYPE_BF16;
}

// Why a rotary embedding cannot turn rows of head_dim elements, or nullptr.
inline const char* rotary_fault(int64_t head_dim, int64_t pairs, int32_t layout, double factor) {
  if (head_dim <= 0 || head_dim % 2 || head_dim > 512) return "head_dim must be even and at most 512";
  if (layout != SB_ROTARY_INTERLEAVED && layout != SB_ROTARY_HALF) return "invalid rotary layout";
  if (pairs <= 0 || 2 * pairs > head_dim) return "between one pair and head_dim / 2 must be rotated";
  if (layout == SB_ROTARY_HALF && pairs % 2)
    return "the half layout needs an even number of pairs";
  if (!(factor > 0.0) || factor > 1e4) return "the factor must be positive and at most 1e4";
  return nullptr;
}

}  // namespace
}  // namespace sb
