// Products with 4-bit weights for gfx950: y = x w^T + bias, w[n, k] = (code[n, k] - zero[n, k / g]) *
// scale[n, k / g] with 16-bit scales, one per group of g inputs.
//
// Arithmetic. A code c becomes the 16-bit float B + c by putting its four bits into the mantissa of B
// (two instructions a pair): B = 16 in bf16, 128 in fp16. For one group, with P = sum x (B + c) and
// S = sum x from the matrix cores, sum x w = scale (P - (B + zero) S). Nothing is rounded on the way but
// the fp32 sums, so that the result is that of the 16-bit inputs and the exact weights, rounded once; B + c
// against c - zero costs the sums two or three of their 24 bits (six in fp16). fp16 has a packed
// subtraction: with 64 rows a workgroup and in tiles, where S costs more than it, P = sum x (c - zero) and
// sum x w = scale P.
//
// Layout, made once (w4_pack_kernel): 16 features x 128 inputs are 1 KiB, lane l of a wave holding 16
// bytes: word j the codes of feature l % 16, inputs 32 j + 8 (l / 16) + 0 .. 7, which is the operand of one
// 16x16x32 matrix instruction. A wave loads a tile with one 16-byte load a lane, 1 KiB in a row. Scales
// and zeros share words (scale's bits, 16 + zero as the upper half of an fp32) per feature and group of
// 32, 64 or 128 inputs, 16 features in a row.
#include "sb_common.h"
#include "sb_w4_plan.h"

#include <algorithm>

namespace sb {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int64_t kInputsMax = int64_t{1} << 22;  // inputs, and row stride: 128 rows stay within 2^31 bytes

// A constant that the compiler does not know as one, in a scalar or a vector register: (w & mask) | base
// is one instruction then, with a literal each they are two.
__device__ __forceinline__ uint32_t scalar_constant(uint32_t x) {
  asm("" : "+s"(x));
  return x;
}
__device__ __forceinline__ uint32_t vector_constant(uint32_t x) {
  asm("" : "+v"(x));
  return x;
}

// The eight codes of a word as 16-bit floats kBase + c: pair p's lie at bits 4p + 3 .. 4p + 6 of both
// halves (modulo 32) and go to bits 3 .. 6 of kBase.
__device__ __forceinline__ u32x4_t w4_words(uint32_t w, uint32_t base_bits) {
  const uint32_t m = scalar_constant(0x00780078u), base = vector_constant(base_bits);
  const u32x4_t r = {(w & m) | base, ((w >> 4) & m) | base, ((w >> 8) & m) | base,
                     (__builtin_amdgcn_alignbit(w, w, 12) & m) | base};
  return r;
}

template <int DT> struct W4;
template <> struct W4<SB_DTYPE_BF16> {
  using vec8 = bf16x8_t;
  static constexpr uint32_t kOnes = 0x3f803f80u;
  // There is no packed bf16 addition: the values stay 16 + c, and the offset goes to the sums.
  static constexpr float kBase = 16.f;
  static constexpr bool kExact = false;
  __device__ __forceinline__ static vec8 minus(vec8 v, float) { return v; }
  __device__ __forceinline__ static f32x4_t mma(vec8 a, vec8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static vec8 values(uint32_t w) {
    return __builtin_bit_cast(vec8, w4_words(w, 0x41804180u));
  }
  __device__ __forceinline__ static uint16_t round(float f) { return f32_to_bf16(f); }
  __device__ __forceinline__ static float value(uint16_t h) { return bf16_to_f32(h); }
};
template <> struct W4<SB_DTYPE_F16> {
  using vec8 = f16x8_t;
  static constexpr uint32_t kOnes = 0x3c003c00u;
  // Ten bits of mantissa: the same bits are 128 + c. (128 + c) - (128 + zero) is exact too, one packed
  // addition for two codes.
  static constexpr float kBase = 128.f;
  static constexpr bool kExact = true;
  __device__ __forceinline__ static vec8 minus(vec8 v, float off) {
    const _Float16 h = static_cast<_Float16>(off);
    const vec8 o = {h, h, h, h, h, h, h, h};
    return v - o;
  }
  __device__ __forceinline__ static f32x4_t mma(vec8 a, vec8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static vec8 values(uint32_t w) {
    return __builtin_bit_cast(vec8, w4_words(w, 0x58005800u));
  }
  __device__ __forceinline__ static uint16_t round(float f) { return f32_to_f16(f); }
  __device__ __forceinline__ static float value(uint16_t h) { return f16_to_f32(h); }
};

// The scale of a table word, and DT's kBase + zero.
__device__ __forceinline__ float scale_of(uint32_t w, bool f16) {
  const float h = f16_to_f32(static_cast<uint16_t>(w));
  return f16 ? h : __uint_as_float(w << 16);
}
template <int DT> __device__ __forceinline__ float offset_of(uint32_t w) {
  return __uint_as_float(w & 0xffff0000u) + (W4<DT>::kBase - 16.f);
}

struct W4Args {
  char* y;
  const char* x;
  const u32x4_t* codes;   // [tiles of features][tiles of inputs][64]
  const uint32_t* table;  // [tiles of features][groups][16]
  const uint16_t* bias;   // or nullptr
  int64_t x_row, y_row;   // bytes
  int64_t num_rows;
  int n, k, k_tiles;
  bool scales_f16;
  // many rows
  const char* sums;       // [rows][sum_blocks][4][32] bf16
  int sum_blocks;
  bool wide_out;          // rows of y take 16-byte stores
  // split inputs: slice s of the steps gives its sums to part [splits][rows][n], and no y
  float* part;
  int splits, split_steps;
  uint32_t tiles;         // workgroups of a slice
};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Copies global -> LDS without registers, 16 or 4 bytes a lane, lane i's to lds_wave + 16 i (4 i);
// assembly so that the compiler does not order later LDS reads behind them (the kernels wait
// themselves: vector memory operations end in order).
__device__ __forceinline__ void w4_dma(const void* src, uint32_t lds_wave) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(lds_wave), "v"(src)
      : "memory", "m0");
}
__device__ __forceinline__ void w4_dma_once(const void* src, uint32_t lds_wave) {  // nontemporal
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off nt"
      :
      : "s"(lds_wave), "v"(src)
      : "memory", "m0");
}
__device__ __forceinline__ void w4_dma4(const void* src, uint32_t lds_wave) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off"
      :
      : "s"(lds_wave), "v"(src)
      : "memory", "m0");
}
// Rows of x: `rows` describes up to 2^32 bytes from a workgroup's first row to the end of the last one
// (a load behind it gives zeros or nothing), `at` is a lane's offset, `add` one for all lanes. One
// register where addresses take two for every four rows. The offsets are added here and not by the load:
// its scalar offset may be left out of the check against the end. (In the assembly, or the sums of all
// copies would be kept in registers.)
__device__ __forceinline__ u32x4_t w4_rows_of(const char* first, int64_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(first);
  const u32x4_t r = {static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32) & 0xffffu,
                     static_cast<uint32_t>(min(bytes, static_cast<int64_t>(0xffffffffll))), 0x00020000u};
  return r;
}
__device__ __forceinline__ void w4_dma_row(uint32_t at, u32x4_t rows, uint32_t add, uint32_t lds_wave) {
  uint32_t sum;
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "v_add_u32 %0, %4, %2\n\t"
      "buffer_load_dwordx4 %0, %3, 0 offen lds"
      : "=&v"(sum)
      : "s"(lds_wave), "v"(at), "s"(rows), "s"(add)
      : "memory", "m0");
}
// Until at most N vector memory operations of the wave are under way; later LDS reads stay behind it.
template <int N>
__device__ __forceinline__ void w4_wait_vm() {
  static_assert(N >= 0 && N < 64, "a six-bit count");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// Until every LDS read of the wave has its values.
__device__ __forceinline__ void w4_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }
__device__ __forceinline__ uint32_t w4_lds_addr(const void* p) {
  using lds_ptr = __attribute__((address_space(3))) const void*;
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)p));
}
#pragma clang diagnostic pop

// Few rows. A workgroup takes 16 J features and up to R rows (4, or 16 MI); its WAVES waves take every
// WAVES'th tile of inputs each for itself, and add their sums up in LDS at the end, in order. What a step
// needs (codes, table words and the rows' 128 inputs) is copied into a stage of the wave's own LDS, AHEAD
// steps in flight, with no register and no barrier between. Rows are copied 256 bytes at a time: read by
// lanes as the matrix operand has them (64 bytes of 16 rows), the rows alone took twice as long as all
// else (16 rows of 3584 -> 4608: 9.2 us, with one row's address for all of them 4.9). GPT: groups of a
// tile of inputs.
//
// What bounds it: the codes' bytes where these are many (one row of 4096 -> 131072 in fp16, 277 MB in 43 us,
// 6.4 TB/s; 8 rows of 3584 -> 37888, 72 MB in no cache in 18.1, 4.0 TB/s, in 14.5 where the last cache holds a
// part), else the rows, which every workgroup copies again (64 rows of 3584 -> 4608: 7.7 us, 96 x 2 workgroups
// of 32 rows, 45 MB of rows and 17 of codes), and a launch with one chain of copies (one row of 3584 -> 4608
// 4.5 us). Halves of a tile as steps of their own, so that one is copied under the other (64 rows, 128 bytes of
// eight rows a copy): 8.9 -> 11.0 us.
template <int R, int J, int GPT> struct RowsStage {
  static constexpr int kMi = R < 16 ? 1 : R / 16;
  static constexpr int kTableCopies = (J * GPT + 3) / 4;
  static constexpr int kRowCopies = R / 4;
  static constexpr int kCopies = J + kTableCopies + kRowCopies;
  static constexpr int kBytes = J * 1024 + kTableCopies * 256 + R * 256;
};
// ONCE: codes nontemporal.
template <int DT, int R, int J, int GPT, int WAVES, int AHEAD, bool ONCE>
__global__ __launch_bounds__(64 * WAVES, 2) void w4_rows_kernel(const W4Args a) {
  using T = W4<DT>;
  using S = RowsStage<R, J, GPT>;
  using vec8 = typename T::vec8;
  constexpr int MI = S::kMi;
  // (up to 32 rows: the products with ones cost less than the additions of exact differences; one row of
  // 4096 -> 131072 in fp16 46 against 55-58 us)
  constexpr bool kExact = T::kExact && MI == 4;
  constexpr int kRing = WAVES * AHEAD * S::kBytes, kParts = WAVES * MI * J * 1024;
  __shared__ __align__(16) char smem[kRing > kParts ? kRing : kParts];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_n = (a.n + kTileN - 1) / kTileN;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * R;
  // (tiles of features behind the last one: the last one)
  const u32x4_t* codes[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int64_t nt = min(static_cast<int>(blockIdx.x) * J + j, tiles_n - 1);
    codes[j] = a.codes + nt * a.k_tiles * 64 + lane;
  }
  const uint32_t* table[S::kTableCopies];
#pragma unroll
  for (int t = 0; t < S::kTableCopies; ++t) {
    const int word = min(lane + 64 * t, J * GPT * 16 - 1);
    const int64_t nt = min(static_cast<int>(blockIdx.x) * J + word / (GPT * 16), tiles_n - 1);
    table[t] = a.table + nt * a.k_tiles * GPT * 16 + word % (GPT * 16);
  }
  const uint32_t x_row = static_cast<uint32_t>(a.x_row);
  const u32x4_t rows = w4_rows_of(a.x + m0 * a.x_row, (a.num_rows - 1 - m0) * a.x_row + a.k * 2);
  const uint32_t row_at = (lane >> 4) * x_row;
  int chunk[R < 16 ? 1 : 4];  // 16 inputs' place of a row: position ^ row
#pragma unroll
  for (int c = 0; c < (R < 16 ? 1 : 4); ++c) chunk[c] = (lane & 15) ^ (4 * c + (lane >> 4));
  char* mine = smem + wave * (AHEAD * S::kBytes);
  const uint32_t mine_lds = w4_lds_addr(mine);
  auto copy = [&](int stage, int kt) {
    uint32_t at = mine_lds + stage * S::kBytes;
#pragma unroll
    for (int j = 0; j < J; ++j, at += 1024) {
      if (ONCE) w4_dma_once(codes[j] + static_cast<int64_t>(kt) * 64, at);
      else w4_dma(codes[j] + static_cast<int64_t>(kt) * 64, at);
    }
#pragma unroll
    for (int t = 0; t < S::kTableCopies; ++t, at += 256)
      w4_dma4(table[t] + static_cast<int64_t>(kt) * (GPT * 16), at);
#pragma unroll
    for (int c = 0; c < S::kRowCopies; ++c, at += 1024) {
      int k8 = kt * 16 + chunk[c & 3 & (R < 16 ? 0 : 3)];
      if (GPT > 1) k8 = min(k8, a.k / 8 - 1);  // (behind the last input: the last ones, of scale 0)
      w4_dma_row(row_at + k8 * 16, rows, 4 * c * x_row, at);
    }
  };
  const u32x4_t one4 = {T::kOnes, T::kOnes, T::kOnes, T::kOnes};
  const vec8 ones = __builtin_bit_cast(vec8, one4);
  f32x4_t acc[MI][J] = {};
  auto multiply = [&](int stage) {
    const char* at = mine + stage * S::kBytes;
    const char* xs = at + J * 1024 + S::kTableCopies * 256;
    u32x4_t w[J];
#pragma unroll
    for (int j = 0; j < J; ++j) w[j] = *reinterpret_cast<const u32x4_t*>(at + j * 1024 + lane * 16);
    constexpr int kSteps = 4 / GPT;
#pragma unroll
    for (int g = 0; g < GPT; ++g) {
      float s[J], off[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t sz =
            *reinterpret_cast<const uint32_t*>(at + J * 1024 + ((j * GPT + g) * 16 + (lane & 15)) * 4);
        s[j] = scale_of(sz, a.scales_f16), off[j] = offset_of<DT>(sz);
      }
      f32x4_t p[MI][J] = {}, sum[MI] = {};
#pragma unroll
      for (int q = g * kSteps; q < (g + 1) * kSteps; ++q) {
        vec8 b[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          b[j] = T::values(w[j][q]);
          if (kExact) b[j] = T::minus(b[j], off[j]);
        }
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int r = R < 16 ? lane & 3 : 16 * i + (lane & 15);
          const vec8 x =
              *reinterpret_cast<const vec8*>(xs + r * 256 + (((4 * q + (lane >> 4)) ^ r) & 15) * 16);
#pragma unroll
          for (int j = 0; j < J; ++j) p[i][j] = T::mma(x, b[j], p[i][j]);
          if (!kExact) sum[i] = T::mma(x, ones, sum[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i][j][r] = fmaf(s[j], kExact ? p[i][j][r] : fmaf(-off[j], sum[i][r], p[i][j][r]),
                                acc[i][j][r]);
      // (64 rows: a group's sums go to the accumulators now; left to the compiler those of all groups
      // wait behind the next copies, in more registers than there are)
      if constexpr (MI == 4 && GPT > 1)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < J; ++j) asm volatile("" : "+v"(acc[i][j]));
    }
  };
#pragma unroll
  for (int p = 0; p < AHEAD; ++p)
    if (wave + p * WAVES < a.k_tiles) copy(p, wave + p * WAVES);
  int stage = 0;
  for (int kt = wave; kt < a.k_tiles; kt += WAVES) {
    // (the last steps wait for all that is left)
    if (kt + (AHEAD - 1) * WAVES < a.k_tiles) w4_wait_vm<(AHEAD - 1) * S::kCopies>();
    else w4_wait_vm<0>();
    multiply(stage);
    if (kt + AHEAD * WAVES < a.k_tiles) {
      w4_wait_lds();  // the stage is read before it is written again
      copy(stage, kt + AHEAD * WAVES);
    }
    stage = stage + 1 == AHEAD ? 0 : stage + 1;
  }
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);  // [wave][row tile, feature tile, register][lane]
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        part[((wave * MI + i) * J + j) * 256 + r * 64 + lane] = acc[i][j][r];
  __syncthreads();
  for (int e = threadIdx.x; e < MI * J * 256; e += 64 * WAVES) {
    const int l = e & 63, ir = e >> 6, ij = ir >> 2;
    const int64_t row = m0 + 16 * (ij / J) + 4 * (l >> 4) + (ir & 3);
    const int64_t f = (static_cast<int64_t>(blockIdx.x) * J + ij % J) * kTileN + (l & 15);
    if (row < a.num_rows && f < a.n && row < m0 + R) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) v += part[w * (MI * J * 256) + e];
      if (a.bias) v += T::value(a.bias[f]);
      reinterpret_cast<uint16_t*>(a.y + row * a.y_row)[f] = T::round(v);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Many rows. A workgroup of four waves takes 128 rows x 128 features, each wave all the rows and 32
// features, so that a code is unpacked once for 128 rows and weights never pass through LDS: a wave
// loads its 32 x 128 codes of a step straight into registers, two steps ahead. Rows go global -> LDS, 128
// inputs a step, two stages. A group's sum P of one 32 x 32 block is a chain of matrix instructions from
// zero, then acc += scale P. bf16: the offsets' share, sum over groups of S (16 + zero) scale, is a
// product over the groups: S as three bf16 values and (16 + zero) scale as two (exact: 5 bits times 11 at
// most), the five largest of their six products, 2^-24 of the largest left out. w4_sums_kernel writes the S of
// 32 groups as one more step of 128 columns of a row ([part][group], the last quarter unused).
//
// What bounds it: the issue of instructions. Of the cycles of a SIMD with one wave, 39% are matrix
// instructions and 49% the issue of all others (a matrix instruction of 32 cycles comes with two fmas, an
// LDS read and its wait, and two to three to unpack codes), and little of one runs under the other; a
// second wave gains a quarter. Waves of 64 x 64 (half the LDS reads, twice the unpacking) were slower
// (2458 rows of 3584 -> 4608 103 against 95 us), so were copies spread over the step (92-94 against 90);
// reads 3, 4 and 6 ahead instead of 2 changed nothing, but for groups of 32 (131 -> 128 us).
// ---------------------------------------------------------------------------------------
typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ f32x16_t mma32(typename W4<DT>::vec8 a, typename W4<DT>::vec8 b, f32x16_t c) {
  if constexpr (DT == SB_DTYPE_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// x as three bf16 values that add up to it.
__device__ __forceinline__ void split3(float x, uint16_t* p) {
  p[0] = f32_to_bf16(x);
  const float r = x - bf16_to_f32(p[0]);
  p[1] = f32_to_bf16(r);
  p[2] = f32_to_bf16(r - bf16_to_f32(p[1]));
}

// sums [rows][blocks of 32 groups][4][32]: thread (kSumRows rows, 8 inputs of a group of STEP).
constexpr int kSumRows = 4;
template <int DT, int STEP>
__global__ __launch_bounds__(256) void w4_sums_kernel(uint16_t* sums, const char* x, int64_t x_row,
                                                      int64_t num_rows, int k, int blocks) {
  constexpr int kLanes = STEP / 8;  // lanes of a group
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per = static_cast<int64_t>(blocks) * 32 * kLanes;
  const int64_t row0 = idx / per * kSumRows;
  const int64_t rest = idx - idx / per * per;
  const int64_t k0 = rest * 8;
  u32x4_t w[kSumRows];
#pragma unroll
  for (int r = 0; r < kSumRows; ++r) {
    w[r] = u32x4_t{};
    if (row0 + r < num_rows && k0 < k) w[r] = *reinterpret_cast<const u32x4_t*>(x + (row0 + r) * x_row + k0 * 2);
  }
  const int64_t g = rest / kLanes;
  const int sub = static_cast<int>(rest % kLanes);
#pragma unroll
  for (int r = 0; r < kSumRows; ++r) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v += W4<DT>::value(static_cast<uint16_t>(w[r][i])) + W4<DT>::value(static_cast<uint16_t>(w[r][i] >> 16));
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) v += __shfl_xor(v, o, 64);
    uint16_t p[3];
    split3(v, p);
    // (lanes of the group share the stores: parts, and zeros behind them)
    if (row0 + r < num_rows && sub < 4)
      sums[((row0 + r) * blocks + g / 32) * 128 + g % 32 + sub * 32] =
          sub == 0 ? p[0] : sub == 1 ? p[1] : sub == 2 ? p[2] : 0;
  }
}

constexpr int kXcds = 8;
constexpr int kBand = 8;       // row tiles of a band of the tile order

// Tile of workgroup b: workgroups go round-robin to the XCDs, each of which gets a contiguous range of
// an order that walks bands of kBand row tiles, feature tile by feature tile, so that the workgroups of
// an XCD share rows and weights in its L2.
__device__ __forceinline__ void w4_tile(uint32_t b, uint32_t n_ft, uint32_t n_rt, uint32_t* ft, uint32_t* rt) {
  const uint32_t total = n_ft * n_rt, x = b % kXcds, i = b / kXcds;
  const uint32_t q = x * (total / kXcds) + min(x, total % kXcds) + i;
  const uint32_t band = q / (kBand * n_ft), in_band = q - band * kBand * n_ft;
  const uint32_t rows_in_band = min<uint32_t>(kBand, n_rt - band * kBand);
  *rt = band * kBand + in_band % rows_in_band;
  *ft = in_band / rows_in_band;
}

// One wave's 32 x 32 blocks of a slice's sums.
__device__ __forceinline__ void store_part(const W4Args& a, const f32x16_t (&acc)[4], int slice, int64_t m0,
                                           int f, int lg) {
  if (f >= a.n) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t row = m0 + 32 * i + 8 * (r >> 2) + 4 * lg + (r & 3);
      if (row < a.num_rows) a.part[(slice * a.num_rows + row) * a.n + f] = acc[i][r];
    }
}

// y = the slices' sums, in order, + bias. A thread takes VEC features of a row.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void w4_merge_kernel(const W4Args a) {
  const int per = (a.n + VEC - 1) / VEC;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / per;
  if (row >= a.num_rows) return;
  const int f = static_cast<int>(i - row * per) * VEC;
  const float* p = a.part + row * a.n + f;
  const int64_t step = a.num_rows * a.n;
  float v[VEC] = {};
  for (int s0 = 0; s0 < a.splits; s0 += 4) {
    float x[4][VEC];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float* at = p + min(s0 + s, a.splits - 1) * step;
      if constexpr (VEC == 4) {
        const f32x4_t w = *reinterpret_cast<const f32x4_t*>(at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[s][e] = w[e];
      } else {
        x[s][0] = *at;
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] += s0 + s < a.splits ? x[s][e] : 0.f;
  }
  uint16_t h[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) h[e] = W4<DT>::round(v[e] + (a.bias ? W4<DT>::value(a.bias[f + e]) : 0.f));
  uint16_t* out = reinterpret_cast<uint16_t*>(a.y + row * a.y_row) + f;
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] = h[e];
}

template <int DT, int GPT>
__global__ __launch_bounds__(256, 2) void w4_tiles_kernel(const W4Args a) {
  using T = W4<DT>;
  using vec8 = typename T::vec8;
  constexpr int kLoads = kBM * 16 / 256;  // 16-byte copies of a thread a step
  __shared__ __align__(16) uint16_t ring[2][kBM * kTileK];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, lq = lane & 31, lg = lane >> 5;
  const uint32_t n_ft = (a.n + kBN - 1) / kBN;
  const uint32_t n_rt = static_cast<uint32_t>((a.num_rows + kBM - 1) / kBM);
  uint32_t ft, rt;
  const int slice = static_cast<int>(blockIdx.x / a.tiles);
  w4_tile(blockIdx.x % a.tiles, n_ft, n_rt, &ft, &rt);
  const int64_t m0 = static_cast<int64_t>(rt) * kBM;
  const int64_t f0 = static_cast<int64_t>(ft) * kBN;
  const int begin = slice * a.split_steps, steps = min(begin + a.split_steps, a.k_tiles + a.sum_blocks);

  // Copies: slot q * 256 + tid of a stage is row (slot / 16), position slot % 16, and holds chunk
  // position ^ (row & 15) of the row: the 16-byte reads of 16 consecutive rows fall on all banks. Chunks
  // behind the last input are the last ones (their scale is 0).
  const int chunk = (tid & 15) ^ ((tid >> 4) & 15);
  const uint32_t x_row = static_cast<uint32_t>(a.x_row), s_row = static_cast<uint32_t>(a.sum_blocks) * 256;
  const u32x4_t rows = w4_rows_of(a.x + m0 * a.x_row, (a.num_rows - 1 - m0) * a.x_row + a.k * 2);
  auto copy = [&](int stage, int kt) {
    const uint32_t to = w4_lds_addr(ring[stage]) + wave * 1024;
    if (kt < a.k_tiles) {
      const uint32_t at = (tid >> 4) * x_row + (GPT == 1 ? kt * 16 + chunk : min(kt * 16 + chunk, a.k / 8 - 1)) * 16;
#pragma unroll
      for (int q = 0; q < kLoads; ++q) w4_dma_row(at, rows, 16 * q * x_row, to + q * 4096);
    } else {
      const u32x4_t sums = w4_rows_of(a.sums + m0 * s_row, (a.num_rows - m0) * s_row);
      const uint32_t at = (tid >> 4) * s_row + (kt - a.k_tiles) * 256 + chunk * 16;
#pragma unroll
      for (int q = 0; q < kLoads; ++q) w4_dma_row(at, sums, 16 * q * s_row, to + q * 4096);
    }
  };
  // This wave's features: two tiles of the packed order (past the last one: the last one's).
  const int64_t tiles_n = (a.n + kTileN - 1) / kTileN;
  const int64_t nt = min(f0 / kTileN + 2 * wave + (lq >> 4), tiles_n - 1);
  const u32x4_t* codes = a.codes + nt * a.k_tiles * 64 + (lq & 15) + 16 * lg;
  const uint32_t* table = a.table + nt * a.k_tiles * GPT * 16 + (lq & 15);

  f32x16_t acc[4] = {};
  // Codes and table words of step kt: in `next` from the step before it on, in `coming` the one before.
  struct Codes {
    u32x4_t w[2];
    uint32_t sz[GPT];
  } next, coming;
  const int last = min(steps, a.k_tiles) - 1;  // (the last step with codes; maybe below begin)
  auto fetch = [&](Codes& c, int kt) {
    kt = max(min(kt, last), 0);
    c.w[0] = codes[static_cast<int64_t>(kt) * 64];
    c.w[1] = codes[static_cast<int64_t>(kt) * 64 + 32];
#pragma unroll
    for (int g = 0; g < GPT; ++g) c.sz[g] = table[(static_cast<int64_t>(kt) * GPT + g) * 16];
  };
  auto read = [&](int stage, int i, int s) {
    const int r = 32 * i + lq;
    return *reinterpret_cast<const vec8*>(ring[stage] + r * kTileK + 8 * ((2 * s + lg) ^ (r & 15)));
  };
  fetch(next, begin);
  copy(begin & 1, begin);
  fetch(coming, begin + 1);
  vec8 b[8];
  float scale[GPT];
  auto unpack = [&](int s) {
    b[s] = T::minus(T::values(next.w[s & 1][s >> 1]), offset_of<DT>(next.sz[s * GPT / 8]));
  };
#pragma unroll
  for (int s = 0; s < 8; ++s) unpack(s);
#pragma unroll
  for (int g = 0; g < GPT; ++g) scale[g] = scale_of(next.sz[g], a.scales_f16);
  // A block is a group's chain of matrix instructions for 32 rows. Its sums p go to the accumulators
  // under the next block's chain, and a step's codes are unpacked for the next step behind their last use,
  // so that every matrix instruction has its share of vector ones; rows are read kReads ahead.
  constexpr int kChain = 8 / GPT, kBlocks = 4 * GPT, kReads = GPT == 4 ? 4 : 2;
  f32x16_t p[2] = {};
  float p_scale = 0.f;  // of the block whose sums are waiting
  for (int kt = begin; kt <= last; ++kt) {
    const int stage = kt & 1;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this step's rows and the next one's codes are here
    __syncthreads();
    next = coming;
    fetch(coming, kt + 2);
    if (kt + 1 < steps) copy(stage ^ 1, kt + 1);
    vec8 x[kReads + 1];
#pragma unroll
    for (int c = 0; c < kReads; ++c) x[c] = read(stage, 0, c);
#pragma unroll
    for (int blk = 0; blk < kBlocks; ++blk) {
      const int i = blk / GPT, g = blk % GPT, prev = (blk + kBlocks - 1) % kBlocks / GPT;
      f32x16_t q = {};
#pragma unroll
      for (int c = 0; c < kChain; ++c) {
        const int s = g * kChain + c, at = blk * kChain + c, ahead = at + kReads;
        if (ahead < kBlocks * kChain) x[ahead % (kReads + 1)] = read(stage, ahead / 8, ahead % 8);
        __builtin_amdgcn_sched_barrier(0);
        q = mma32<DT>(x[at % (kReads + 1)], b[s], q);
#pragma unroll
        for (int r = c * 16 / kChain; r < (c + 1) * 16 / kChain; ++r)
          acc[prev][r] = fmaf(p_scale, p[(blk & 1) ^ 1][r], acc[prev][r]);
        if (i == 3) unpack(s);
        __builtin_amdgcn_sched_barrier(0);
      }
      p[blk & 1] = q;
      p_scale = scale[g];
      if (i == 3) scale[g] = scale_of(next.sz[g], a.scales_f16);
    }
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[3][r] = fmaf(p_scale, p[1][r], acc[3][r]);
  // bf16: the offsets' share, 32 groups a step.
  if constexpr (!T::kExact) {
    using B = W4<SB_DTYPE_BF16>;
    for (int kt = max(begin, a.k_tiles); kt < steps; ++kt) {
      const int blk = kt - a.k_tiles, stage = kt & 1;
      B::vec8 z[2][2];  // [16 groups][upper, lower part of -(16 + zero) scale]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int g = blk * 32 + 16 * h + 8 * lg + e;
          const uint32_t t = table[static_cast<int64_t>(min(g, a.k_tiles * GPT - 1)) * 16];
          const float v = -offset_of<SB_DTYPE_BF16>(t) * scale_of(t, a.scales_f16);
          const uint32_t up = f32_to_bf16(v), low = f32_to_bf16(v - bf16_to_f32(static_cast<uint16_t>(up)));
          if (e & 1) hi[e >> 1] |= up << 16, lo[e >> 1] |= low << 16;
          else hi[e >> 1] = up, lo[e >> 1] = low;
        }
        const u32x4_t hv = {hi[0], hi[1], hi[2], hi[3]}, lv = {lo[0], lo[1], lo[2], lo[3]};
        z[h][0] = __builtin_bit_cast(B::vec8, hv);
        z[h][1] = __builtin_bit_cast(B::vec8, lv);
      }
      w4_wait_vm<0>();
      __syncthreads();
      if (kt + 1 < steps) copy(stage ^ 1, kt + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const auto s = __builtin_bit_cast(B::vec8, read(stage, i, 2 * part + h));
            acc[i] = mma32<SB_DTYPE_BF16>(s, z[h][0], acc[i]);
            if (part < 2) acc[i] = mma32<SB_DTYPE_BF16>(s, z[h][1], acc[i]);
          }
    }
  }

  if (a.part) {  // (uniform)
    store_part(a, acc, slice, m0, static_cast<int>(f0) + 32 * wave + lq, lg);
    return;
  }
  // Out: through LDS, so that a row's features are stored together.
  __syncthreads();
  uint16_t* tile = ring[0];
  const int64_t f = f0 + 32 * wave + lq;
  const float bias = a.bias && f < a.n ? T::value(a.bias[f]) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * i + 8 * (r >> 2) + 4 * lg + (r & 3);
      tile[row * kBN + 32 * wave + lq] = T::round(acc[i][r] + bias);
    }
  __syncthreads();
  const int live = static_cast<int>(min(static_cast<int64_t>(kBM), a.num_rows - m0));
  if (a.wide_out && f0 + kBN <= a.n) {  // (uniform)
    for (int e = tid; e < live * (kBN / 8); e += 256) {
      const int row = e / (kBN / 8), c = e % (kBN / 8) * 8;
      *reinterpret_cast<u32x4_t*>(a.y + (m0 + row) * a.y_row + (f0 + c) * 2) =
          *reinterpret_cast<const u32x4_t*>(tile + row * kBN + c);
    }
  } else {
    for (int e = tid; e < live * kBN; e += 256) {
      const int row = e / kBN, c = e % kBN;
      if (f0 + c < a.n) *reinterpret_cast<uint16_t*>(a.y + (m0 + row) * a.y_row + (f0 + c) * 2) = tile[e];
    }
  }
}

// One 16-byte piece of packed codes a thread.
__global__ __launch_bounds__(256) void w4_pack_kernel(u32x4_t* out, const uint8_t* codes, int64_t stride,
                                                      int64_t n, int64_t k, int64_t k_tiles,
                                                      int64_t pieces) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= pieces) return;
  const int lane = static_cast<int>(i & 63);
  const int64_t tile = i >> 6, nt = tile / k_tiles, kt = tile - nt * k_tiles;
  const int64_t f = nt * kTileN + (lane & 15);
  u32x4_t r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t k0 = kt * kTileK + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    if (f < n && k0 < k) {  // (k is a multiple of 32)
      const uint8_t* c = codes + f * stride + k0;
#pragma unroll
      for (int e = 0; e < 8; ++e) w |= static_cast<uint32_t>(c[e] & 15) << (4 * (e >> 1) + 16 * (e & 1));
    }
    r[j] = w << 3 | w >> 29;
  }
  out[i] = r;
}

// One table word a thread: a scale's 16 bits and 16 + zero.
__global__ __launch_bounds__(256) void w4_table_kernel(uint32_t* out, const uint16_t* scales,
                                                       const uint8_t* zeros, int64_t s_stride,
                                                       int64_t z_stride, int64_t n, int64_t k,
                                                       int64_t group, int64_t step, int64_t steps,
                                                       int64_t words) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= words) return;
  const int64_t nt = i / (steps * kTileN), rest = i - nt * steps * kTileN;
  const int64_t f = nt * kTileN + (rest & 15), k0 = (rest >> 4) * step;
  uint32_t w = 0x41800000u;  // scale 0 behind the last feature and input
  if (f < n && k0 < k) {
    const float off = 16.f + (zeros ? zeros[f * z_stride + k0 / group] & 15 : 8);
    w = __float_as_uint(off) | scales[f * s_stride + k0 / group];
  }
  out[i] = w;
}

// The weights themselves, rounded once: eight of a row a thread.
template <int DT>
__global__ __launch_bounds__(256) void w4_unpack_kernel(char* out, const uint32_t* codes,
                                                        const uint32_t* table, int64_t o_row, int64_t n,
                                                        int64_t k, int64_t k_tiles, int gpt,
                                                        bool scales_f16) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per = k / 8, f = i / per;
  if (f >= n) return;
  const int64_t k0 = (i - f * per) * 8, kt = k0 / kTileK;
  const int in = static_cast<int>(k0 - kt * kTileK);
  const int64_t nt = f / kTileN;
  const int lane = static_cast<int>(f - nt * kTileN) + 16 * ((in & 31) >> 3);
  uint32_t w = codes[((nt * k_tiles + kt) * 64 + lane) * 4 + (in >> 5)];
  const uint32_t t = table[((nt * k_tiles + kt) * gpt + in * gpt / kTileK) * 16 + (lane & 15)];
  const float s = scale_of(t, scales_f16), off = offset_of<SB_DTYPE_BF16>(t) - 16.f;
  w = w >> 3 | w << 29;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = static_cast<float>((w >> (4 * (e >> 1) + 16 * (e & 1))) & 15u);
    const float v = (c - off) * s;
    char* at = out + f * o_row + (k0 + e) * (DT == SB_DTYPE_F32 ? 4 : 2);
    if constexpr (DT == SB_DTYPE_F32) *reinterpret_cast<float*>(at) = v;
    else *reinterpret_cast<uint16_t*>(at) = W4<DT>::round(v);
  }
}

const char* shape_fault(int64_t n, int64_t k, int64_t group) {
  if (n <= 0 || k <= 0 || group <= 0) return "sizes must be positive";
  if (n > 0x7fffffe0 || k > kInputsMax) return "size past its limit";
  if (group % 32 || k % group) return "the group must be a multiple of 32 that divides the inputs";
  return nullptr;
}

}  // namespace
}  // namespace sb

extern "C" int64_t sb_w4_codes_size(int64_t out_features, int64_t in_features) {
  return sb::tiles(out_features, sb::kTileN) * sb::tiles(in_features, sb::kTileK) * 1024;
}

extern "C" int64_t sb_w4_table_size(int64_t out_features, int64_t in_features, int64_t group) {
  return sb::tiles(out_features, sb::kTileN) * sb::tiles(in_features, sb::kTileK) *
         (sb::kTileK / sb::table_step(group)) * 64;
}

extern "C" int sb_w4_pack(void* packed, void* table, const uint8_t* codes, const void* scales,
                          const uint8_t* zeros, int64_t out_features, int64_t in_features, int64_t group,
                          int64_t codes_stride, int64_t scales_stride, int64_t zeros_stride,
                          void* stream) {
  using namespace sb;
  const char* fn = "sb_w4_pack";
  clear_error();
  if (!packed || !table || !codes || !scales) return fail(fn, "null pointer");
  if (const char* why = shape_fault(out_features, in_features, group)) return fail(fn, why);
  if (reinterpret_cast<uintptr_t>(packed) % 16 || reinterpret_cast<uintptr_t>(table) % 16)
    return fail(fn, "packed codes and table must be 16-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t kt = tiles(in_features, kTileK), step = table_step(group), steps = kt * (kTileK / step);
  const int64_t pieces = tiles(out_features, kTileN) * kt * 64;
  const int64_t words = tiles(out_features, kTileN) * steps * kTileN;
  if (tiles(pieces, 256) > 0x7fffffff) return fail(fn, "grid too large");
  SB_LAUNCH("w4_pack", w4_pack_kernel, dim3(static_cast<unsigned>(tiles(pieces, 256))), dim3(256), st,
            static_cast<u32x4_t*>(packed), codes, codes_stride, out_features, in_features, kt, pieces);
  SB_LAUNCH("w4_pack", w4_table_kernel, dim3(static_cast<unsigned>(tiles(words, 256))), dim3(256), st,
            static_cast<uint32_t*>(table), static_cast<const uint16_t*>(scales), zeros, scales_stride,
            zeros_stride, out_features, in_features, group, step, steps, words);
  return check_launch(fn);
}

extern "C" int sb_w4_dequantize(void* out, const void* packed, const void* table, int64_t out_features,
                                int64_t in_features, int64_t group, int64_t out_stride,
                                int32_t scale_dtype, int32_t dtype, void* stream) {
  using namespace sb;
  const char* fn = "sb_w4_dequantize";
  clear_error();
  if (!out || !packed || !table) return fail(fn, "null pointer");
  if (const char* why = shape_fault(out_features, in_features, group)) return fail(fn, why);
  if (elem_size(dtype) == 0) return fail(fn, "invalid dtype");
  if (scale_dtype != SB_DTYPE_F16 && scale_dtype != SB_DTYPE_BF16) return fail(fn, "invalid dtype of scales");
  if (reinterpret_cast<uintptr_t>(packed) % 16 || reinterpret_cast<uintptr_t>(table) % 16)
    return fail(fn, "packed codes and table must be 16-byte aligned");
  if (out_features > 1 && out_stride < in_features) return fail(fn, "rows of out must not overlap");
  const int64_t gx = tiles(out_features * (in_features / 8), 256);
  if (gx > 0x7fffffff) return fail(fn, "grid too large");
  const hipStream_t st = static_cast<hipStream_t>(stream);
#define SB_W4_UNPACK(DT)                                                                              \
  if (dtype == DT)                                                                                    \
    SB_LAUNCH("w4_unpack", w4_unpack_kernel<DT>, dim3(static_cast<unsigned>(gx)), dim3(256), st,      \
              static_cast<char*>(out), static_cast<const uint32_t*>(packed),                          \
              static_cast<const uint32_t*>(table), out_stride * elem_size(DT), out_features,          \
              in_features, tiles(in_features, kTileK),                                                \
              static_cast<int>(kTileK / table_step(group)), scale_dtype == SB_DTYPE_F16);
  SB_W4_UNPACK(SB_DTYPE_F32)
  SB_W4_UNPACK(SB_DTYPE_F16)
  SB_W4_UNPACK(SB_DTYPE_BF16)
#undef SB_W4_UNPACK
  return check_launch(fn);
}

namespace sb {
namespace {

int64_t sums_bytes(const W4Plan& p, int64_t m) { return m * p.sum_blocks * 256; }

}  // namespace
}  // namespace sb

extern "C" int64_t sb_w4_linear_workspace_size(int64_t num_rows, int64_t out_features, int64_t in_features,
                                               int64_t group, int32_t dtype) {
  using namespace sb;
  if (num_rows <= 0 || shape_fault(out_features, in_features, group)) return 0;
  const W4Plan p = w4_plan(num_rows, out_features, in_features, group, dtype == SB_DTYPE_BF16);
  return sums_bytes(p, num_rows) + (p.splits > 1 ? p.splits * num_rows * out_features * 4 : 0);
}

extern "C" int sb_w4_linear(void* y, const void* x, const void* packed, const void* table,
                            const void* bias, int64_t num_rows, int64_t out_features,
                            int64_t in_features, int64_t group, int64_t x_stride, int64_t y_stride,
                            void* workspace, int64_t workspace_bytes, int32_t scale_dtype,
                            int32_t dtype, void* stream) {
  using namespace sb;
  const char* fn = "sb_w4_linear";
  clear_error();
  if (num_rows == 0) return SB_OK;
  if (dtype != SB_DTYPE_F16 && dtype != SB_DTYPE_BF16) return fail(fn, "rows must be bf16 or fp16");
  if (scale_dtype != SB_DTYPE_F16 && scale_dtype != SB_DTYPE_BF16) return fail(fn, "invalid dtype of scales");
  if (!y || !x || !packed || !table) return fail(fn, "null pointer");
  if (const char* why = shape_fault(out_features, in_features, group)) return fail(fn, why);
  if (num_rows < 0) return fail(fn, "sizes must be positive");
  if (num_rows > 0x7fffff00) return fail(fn, "size past its limit");
  if (x_stride < 0 || x_stride > kInputsMax) return fail(fn, "row stride past its limit");
  if (reinterpret_cast<uintptr_t>(x) % 16 || x_stride * 2 % 16)
    return fail(fn, "rows of x must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(packed) % 16 || reinterpret_cast<uintptr_t>(table) % 16)
    return fail(fn, "packed codes and table must be 16-byte aligned");
  W4Args a = {};
  a.y = static_cast<char*>(y);
  a.x = static_cast<const char*>(x);
  a.codes = static_cast<const u32x4_t*>(packed);
  a.table = static_cast<const uint32_t*>(table);
  a.bias = static_cast<const uint16_t*>(bias);
  a.x_row = x_stride * 2;
  a.y_row = y_stride * 2;
  a.num_rows = num_rows;
  a.n = static_cast<int>(out_features);
  a.k = static_cast<int>(in_features);
  a.k_tiles = static_cast<int>(tiles(in_features, kTileK));
  a.scales_f16 = scale_dtype == SB_DTYPE_F16;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int gpt = static_cast<int>(kTileK / table_step(group));
  const W4Plan plan = w4_plan(num_rows, out_features, in_features, group, dtype == SB_DTYPE_BF16);
  const int64_t need = sb_w4_linear_workspace_size(num_rows, out_features, in_features, group, dtype);
  if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need))
    return fail(fn, "workspace too small or not 16-byte aligned");
  if (num_rows > 1 && y_stride < out_features) return fail(fn, "rows of y must not overlap");
  a.wide_out = reinterpret_cast<uintptr_t>(y) % 16 == 0 && a.y_row % 16 == 0;
  a.sums = static_cast<const char*>(workspace);
  a.sum_blocks = plan.sum_blocks;
  a.splits = plan.splits;
  a.split_steps = plan.split_steps;
  if (plan.splits > 1)
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums_bytes(plan, num_rows));
  if (!plan.tiled) {
    const int64_t gy = tiles(num_rows, plan.r);
    const int64_t nt = tiles(out_features, kTileN);
    // Two steps in flight where a CU's LDS holds two such workgroups, else one (other waves run meanwhile).
#define SB_W4_L(DT, R, J, GPT, W, ONCE)                                                               \
  do {                                                                                                \
    constexpr int kAhead = 2 * W * RowsStage<R, J, GPT>::kBytes <= 80 * 1024 ? 2 : 1;                 \
    const dim3 grid(static_cast<unsigned>(tiles(nt, J)), static_cast<unsigned>(gy));                  \
    SB_LAUNCH("w4_rows", (w4_rows_kernel<DT, R, J, GPT, W, kAhead, ONCE>), grid, dim3(64 * W), st, a); \
  } while (0)
#define SB_W4(DT, R, J, GPT)                                                                          \
  if (dtype == DT && plan.r == R && plan.j == J && gpt == GPT) {                                      \
    if constexpr (R <= 16) {                                                                          \
      if (J == 1 && plan.waves == 16) SB_W4_L(DT, R, 1, GPT, 16, false);                              \
      else if (J > 1 && plan.once) SB_W4_L(DT, R, (J > 1 ? J : 2), GPT, 8, true);                     \
      else SB_W4_L(DT, R, J, GPT, 8, false);                                                          \
    } else {                                                                                          \
      SB_W4_L(DT, R, J, GPT, (R == 64 && J == 4 ? 7 : 8), false);                                     \
    }                                                                                                 \
  }
#define SB_W4_(DT, R, J) SB_W4(DT, R, J, 1) SB_W4(DT, R, J, 2) SB_W4(DT, R, J, 4)
#define SB_W4_R(DT, J) SB_W4_(DT, 16, J) SB_W4_(DT, 32, J) SB_W4_(DT, 64, J)
#define SB_W4_D(DT)                                                                                  \
  SB_W4_(DT, 4, 1) SB_W4_(DT, 4, 2) SB_W4_R(DT, 1) SB_W4_R(DT, 2) SB_W4_R(DT, 3) SB_W4_R(DT, 4)
    SB_W4_D(SB_DTYPE_BF16)
    SB_W4_D(SB_DTYPE_F16)
#undef SB_W4_D
#undef SB_W4_R
#undef SB_W4_
#undef SB_W4
#undef SB_W4_L
    return check_launch(fn);
  }
  const int64_t grid_tiles = tiles(num_rows, kBM) * tiles(out_features, kBN);
  const int64_t grid = grid_tiles * plan.splits;
  if (grid > 0x7fffffff) return fail(fn, "grid too large");
  a.tiles = static_cast<uint32_t>(grid_tiles);
  const int64_t work = tiles(num_rows, kSumRows) * a.sum_blocks * 32 * (table_step(group) / 8);
  if (tiles(work, 256) > 0x7fffffff) return fail(fn, "grid too large");
#define SB_W4(DT, GPT)                                                                                \
  if (dtype == DT && gpt == GPT) {                                                                    \
    if (a.sum_blocks)                                                                                 \
      SB_LAUNCH("w4_sums", (w4_sums_kernel<DT, kTileK / GPT>), dim3(static_cast<unsigned>(tiles(work, 256))), \
              dim3(256), st, static_cast<uint16_t*>(workspace), a.x, a.x_row, a.num_rows, a.k,        \
              a.sum_blocks);                                                                          \
    SB_LAUNCH("w4_tiles", (w4_tiles_kernel<DT, GPT>), dim3(static_cast<unsigned>(grid)), dim3(256), st, a); \
  }
  SB_W4(SB_DTYPE_BF16, 1) SB_W4(SB_DTYPE_BF16, 2) SB_W4(SB_DTYPE_BF16, 4)
  SB_W4(SB_DTYPE_F16, 1) SB_W4(SB_DTYPE_F16, 2) SB_W4(SB_DTYPE_F16, 4)
#undef SB_W4
  if (plan.splits > 1) {
    const int vec = out_features % 4 == 0 ? 4 : 1;
    const int64_t gx = tiles(num_rows * tiles(out_features, vec), 256);
    if (gx > 0x7fffffff) return fail(fn, "grid too large");
#define SB_W4(DT, VEC)                                                                                \
  if (dtype == DT && vec == VEC)                                                                      \
    SB_LAUNCH("w4_merge", (w4_merge_kernel<DT, VEC>), dim3(static_cast<unsigned>(gx)), dim3(256), st, a);
    SB_W4(SB_DTYPE_BF16, 4) SB_W4(SB_DTYPE_BF16, 1) SB_W4(SB_DTYPE_F16, 4) SB_W4(SB_DTYPE_F16, 1)
#undef SB_W4
  }
  return check_launch(fn);
}
