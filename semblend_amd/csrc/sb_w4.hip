// Products with 4-bit weights for gfx950: y = x w^T + bias, w[n, k] = (code[n, k] - zero[n, k / g]) *
// scale[n, k / g] with 16-bit scales, one per group of g inputs.
//
// Arithmetic. A code c becomes the 16-bit float 16 + c by putting its four bits at the top of the
// mantissa of 16.0 (two instructions a pair). For one group, with P = sum x (16 + c) and S = sum x from the
// matrix cores (S a product with ones), sum x w = scale (P - (16 + zero) S). Nothing is rounded on the
// way but the fp32 sums, so that the result is that of the 16-bit inputs and the exact weights, rounded
// once; 16 + c against c - zero costs the sums two or three of their 24 bits.
//
// Layout, made once (w4_pack_kernel): 16 features x 128 inputs are 1 KiB, lane l of a wave holding 16
// bytes: word j the codes of feature l % 16, inputs 32 j + 8 (l / 16) + 0 .. 7, which is the operand of one
// 16x16x32 matrix instruction. A wave loads a tile with one 16-byte load a lane, 1 KiB in a row. Scales
// and zeros share words (scale's bits, 16 + zero as the upper half of an fp32) per feature and group of
// 32, 64 or 128 inputs, 16 features in a row.
#include "sb_common.h"

#include <algorithm>

namespace sb {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTileN = 16;    // features of a tile
constexpr int kTileK = 128;   // inputs of a tile

template <int DT> struct W4;
template <> struct W4<SB_DTYPE_BF16> {
  using vec8 = bf16x8_t;
  static constexpr uint32_t kOnes = 0x3f803f80u;
  __device__ __forceinline__ static f32x4_t mma(vec8 a, vec8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // 16 + c for the eight codes of a word: pair p's codes lie at bits 4p + 3 .. 4p + 6 of both halves
  // (modulo 32).
  __device__ __forceinline__ static vec8 values(uint32_t w) {
    const u32x4_t r = {(w & 0x00780078u) | 0x41804180u, ((w >> 4) & 0x00780078u) | 0x41804180u,
                       ((w >> 8) & 0x00780078u) | 0x41804180u,
                       (__builtin_amdgcn_alignbit(w, w, 12) & 0x00780078u) | 0x41804180u};
    return __builtin_bit_cast(vec8, r);
  }
  __device__ __forceinline__ static uint16_t round(float f) { return f32_to_bf16(f); }
  __device__ __forceinline__ static float value(uint16_t h) { return bf16_to_f32(h); }
};
template <> struct W4<SB_DTYPE_F16> {
  using vec8 = f16x8_t;
  static constexpr uint32_t kOnes = 0x3c003c00u;
  __device__ __forceinline__ static f32x4_t mma(vec8 a, vec8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static vec8 values(uint32_t w) {
    const u32x4_t r = {((w << 3) & 0x03c003c0u) | 0x4c004c00u, ((w >> 1) & 0x03c003c0u) | 0x4c004c00u,
                       ((w >> 5) & 0x03c003c0u) | 0x4c004c00u,
                       (__builtin_amdgcn_alignbit(w, w, 9) & 0x03c003c0u) | 0x4c004c00u};
    return __builtin_bit_cast(vec8, r);
  }
  __device__ __forceinline__ static uint16_t round(float f) { return f32_to_f16(f); }
  __device__ __forceinline__ static float value(uint16_t h) { return f16_to_f32(h); }
};

// The scale and 16 + zero of a table word.
__device__ __forceinline__ float scale_of(uint32_t w, bool f16) {
  const float h = f16_to_f32(static_cast<uint16_t>(w));
  return f16 ? h : __uint_as_float(w << 16);
}
__device__ __forceinline__ float offset_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

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
};

// A workgroup takes 16 features and 16 MI rows; its waves take every kWaves'th tile of inputs and add
// their sums up in LDS at the end, in order. GPT: groups of a tile of inputs.
constexpr int kWaves = 8;
template <int DT, int MI, int GPT>
__global__ __launch_bounds__(64 * kWaves) void w4_rows_kernel(const W4Args a) {
  using T = W4<DT>;
  using vec8 = typename T::vec8;
  __shared__ float part[kWaves][MI * 4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t nt = blockIdx.x;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * MI);
  const u32x4_t* codes = a.codes + nt * a.k_tiles * 64 + lane;
  const uint32_t* table = a.table + nt * a.k_tiles * GPT * 16 + (lane & 15);
  const char* xr[MI];
  bool live[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t row = m0 + 16 * i + (lane & 15);
    live[i] = row < a.num_rows;
    xr[i] = a.x + (live[i] ? row : 0) * a.x_row + (lane >> 4) * 16;
  }
  const u32x4_t one4 = {T::kOnes, T::kOnes, T::kOnes, T::kOnes};
  const vec8 ones = __builtin_bit_cast(vec8, one4);

  f32x4_t acc[MI] = {};
  for (int kt = wave; kt < a.k_tiles; kt += kWaves) {
    const u32x4_t w = codes[static_cast<int64_t>(kt) * 64];
    uint32_t sz[GPT];
#pragma unroll
    for (int g = 0; g < GPT; ++g) sz[g] = table[(static_cast<int64_t>(kt) * GPT + g) * 16];
    vec8 xv[MI][4];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (live[i] && kt * kTileK + 32 * j < a.k)
          v = *reinterpret_cast<const u32x4_t*>(xr[i] + (static_cast<int64_t>(kt) * kTileK + 32 * j) * 2);
        xv[i][j] = __builtin_bit_cast(vec8, v);
      }
    constexpr int kSteps = 4 / GPT;
#pragma unroll
    for (int g = 0; g < GPT; ++g) {
      const float s = scale_of(sz[g], a.scales_f16), off = offset_of(sz[g]);
      f32x4_t p[MI] = {}, sum[MI] = {};
#pragma unroll
      for (int j = g * kSteps; j < (g + 1) * kSteps; ++j) {
        const vec8 b = T::values(w[j]);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          p[i] = T::mma(xv[i][j], b, p[i]);
          sum[i] = T::mma(xv[i][j], ones, sum[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(s, fmaf(-off, sum[i][r], p[i][r]), acc[i][r]);
    }
  }
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][4 * i + r][lane] = acc[i][r];
  __syncthreads();
  for (int e = threadIdx.x; e < MI * 4 * 64; e += 64 * kWaves) {
    const int l = e & 63, ir = e >> 6;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += part[w][ir][l];
    const int64_t row = m0 + 16 * (ir >> 2) + 4 * (l >> 4) + (ir & 3);
    const int64_t f = nt * kTileN + (l & 15);
    if (row < a.num_rows && f < a.n) {
      if (a.bias) v += T::value(a.bias[f]);
      reinterpret_cast<uint16_t*>(a.y + row * a.y_row)[f] = T::round(v);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Many rows. A workgroup of four waves takes 128 rows x 128 features, each wave all the rows and 32
// features, so that a code is unpacked once for 128 rows and weights never pass through LDS: a wave
// loads its 32 x 128 codes of a step straight into registers, a step ahead. Rows go global -> LDS, 128
// inputs a step, two stages. A group's sum P of one 32 x 32 block is a chain of matrix instructions from
// zero, then acc += scale P. The offsets' share, sum over groups of S (16 + zero) scale, is a product
// over the groups: S as three bf16 values and (16 + zero) scale as two (exact: 5 bits times 11 at
// most), the five largest of their six products, 2^-24 of the largest left out. w4_sums_kernel writes the
// S of 32 groups as one more step of 128 columns of a row ([part][group], the last quarter unused).
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

// sums [rows][blocks of 32 groups][4][32]: thread (row, group of `step` inputs). 8 lanes a group and up.
template <int DT, int STEP>
__global__ __launch_bounds__(256) void w4_sums_kernel(uint16_t* sums, const char* x, int64_t x_row,
                                                      int64_t num_rows, int k, int blocks) {
  constexpr int kLanes = STEP / 8;  // lanes of a group, 8 values each
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per = static_cast<int64_t>(blocks) * 32 * kLanes;
  const int64_t row = idx / per;
  const int64_t rest = idx - row * per;
  const int64_t k0 = rest * 8;
  float v = 0.f;
  if (row < num_rows && k0 < k) {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(x + row * x_row + k0 * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v += W4<DT>::value(static_cast<uint16_t>(w[i])) + W4<DT>::value(static_cast<uint16_t>(w[i] >> 16));
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) v += __shfl_xor(v, o, 64);
  if (row >= num_rows) return;
  const int64_t g = rest / kLanes;
  uint16_t p[3];
  split3(v, p);
  uint16_t* out = sums + (row * blocks + g / 32) * 128 + g % 32;
  // (lanes of the group share the stores: parts, and zeros behind them)
  const int sub = static_cast<int>(rest % kLanes);
  if (sub < 4) out[sub * 32] = sub == 0 ? p[0] : sub == 1 ? p[1] : sub == 2 ? p[2] : 0;
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// One 16-byte global -> LDS copy per lane, lane i's chunk to lds_wave + 16 i; assembly so that the
// compiler does not order later LDS reads behind it (the kernel waits before its barriers).
__device__ __forceinline__ void w4_dma(const char* src, uint32_t lds_wave) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(lds_wave), "v"(src)
      : "memory", "m0");
}
__device__ __forceinline__ uint32_t w4_lds_addr(const void* p) {
  using lds_ptr = __attribute__((address_space(3))) const void*;
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)p));
}
#pragma clang diagnostic pop

constexpr int kXcds = 8;
constexpr int kBand = 8;       // row tiles of a band of the tile order
constexpr int kBM = 128, kBN = 128;

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
  w4_tile(blockIdx.x, n_ft, n_rt, &ft, &rt);
  const int64_t m0 = static_cast<int64_t>(rt) * kBM;
  const int64_t f0 = static_cast<int64_t>(ft) * kBN;
  const int steps = a.k_tiles + a.sum_blocks;

  // Copies: slot q * 256 + tid of a stage is row (slot / 16), position slot % 16, and holds chunk
  // position ^ (row & 15) of the row: the 16-byte reads of 16 consecutive rows fall on all banks. Rows
  // behind the last are the last one's, chunks behind the last input too (their scale is 0).
  const int chunk = (tid & 15) ^ ((tid >> 4) & 15);
  auto copy = [&](int stage, int kt, int q) {
    const int64_t row = min(m0 + q * 16 + (tid >> 4), a.num_rows - 1);
    const char* src;
    if (kt < a.k_tiles)
      src = a.x + row * a.x_row + static_cast<int64_t>(min(kt * 16 + chunk, a.k / 8 - 1)) * 16;
    else
      src = a.sums + (row * a.sum_blocks + (kt - a.k_tiles)) * 256 + chunk * 16;
    w4_dma(src, w4_lds_addr(ring[stage]) + (q * 256 + wave * 64) * 16);
  };
  // This wave's features: two tiles of the packed order (past the last one: the last one's).
  const int64_t tiles_n = (a.n + kTileN - 1) / kTileN;
  const int64_t nt = min(f0 / kTileN + 2 * wave + (lq >> 4), tiles_n - 1);
  const u32x4_t* codes = a.codes + nt * a.k_tiles * 64 + (lq & 15) + 16 * lg;
  const uint32_t* table = a.table + nt * a.k_tiles * GPT * 16 + (lq & 15);

  f32x16_t acc[4] = {};
  u32x4_t w[2];
  uint32_t sz[GPT];
  auto fetch = [&](int kt) {
    w[0] = codes[static_cast<int64_t>(kt) * 64];
    w[1] = codes[static_cast<int64_t>(kt) * 64 + 32];
#pragma unroll
    for (int g = 0; g < GPT; ++g) sz[g] = table[(static_cast<int64_t>(kt) * GPT + g) * 16];
  };
  auto read = [&](int stage, int i, int s) {
    const int r = 32 * i + lq;
    return *reinterpret_cast<const vec8*>(ring[stage] + r * kTileK + 8 * ((2 * s + lg) ^ (r & 15)));
  };
#pragma unroll
  for (int q = 0; q < kLoads; ++q) copy(0, 0, q);
  fetch(0);
  for (int kt = 0; kt < a.k_tiles; ++kt) {
    const int stage = kt & 1;
    vec8 b[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) b[s] = T::values(w[s & 1][s >> 1]);
    float scale[GPT];
#pragma unroll
    for (int g = 0; g < GPT; ++g) scale[g] = scale_of(sz[g], a.scales_f16);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this step's rows have landed
    __syncthreads();
    if (kt + 1 < steps) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) copy(stage ^ 1, kt + 1, q);
    }
    if (kt + 1 < a.k_tiles) fetch(kt + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int g = 0; g < GPT; ++g) {
        f32x16_t p = {};
#pragma unroll
        for (int s = g * (8 / GPT); s < (g + 1) * (8 / GPT); ++s) p = mma32<DT>(read(stage, i, s), b[s], p);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = fmaf(scale[g], p[r], acc[i][r]);
      }
    }
  }
  // The offsets' share, 32 groups a step.
  using B = W4<SB_DTYPE_BF16>;
  for (int blk = 0; blk < a.sum_blocks; ++blk) {
    const int kt = a.k_tiles + blk, stage = kt & 1;
    B::vec8 z[2][2];  // [16 groups][upper, lower part of -(16 + zero) scale]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int g = blk * 32 + 16 * h + 8 * lg + e;
        const uint32_t t = table[static_cast<int64_t>(min(g, a.k_tiles * GPT - 1)) * 16];
        const float v = -offset_of(t) * scale_of(t, a.scales_f16);
        const uint32_t up = f32_to_bf16(v), low = f32_to_bf16(v - bf16_to_f32(static_cast<uint16_t>(up)));
        if (e & 1) hi[e >> 1] |= up << 16, lo[e >> 1] |= low << 16;
        else hi[e >> 1] = up, lo[e >> 1] = low;
      }
      const u32x4_t hv = {hi[0], hi[1], hi[2], hi[3]}, lv = {lo[0], lo[1], lo[2], lo[3]};
      z[h][0] = __builtin_bit_cast(B::vec8, hv);
      z[h][1] = __builtin_bit_cast(B::vec8, lv);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    if (kt + 1 < steps) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) copy(stage ^ 1, kt + 1, q);
    }
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
  for (int e = tid; e < kBM * kBN / 8; e += 256) {
    const int row = e / (kBN / 8), c = e % (kBN / 8) * 8;
    if (m0 + row >= a.num_rows) break;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.y + (m0 + row) * a.y_row) + f0 + c;
    if (a.wide_out && f0 + c + 8 <= a.n) {
      *reinterpret_cast<u32x4_t*>(out) = *reinterpret_cast<const u32x4_t*>(tile + row * kBN + c);
    } else {
      for (int j = 0; j < 8 && f0 + c + j < a.n; ++j) out[j] = tile[row * kBN + c + j];
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
  const float s = scale_of(t, scales_f16), off = offset_of(t) - 16.f;
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

int64_t tiles(int64_t x, int64_t by) { return (x + by - 1) / by; }

// Inputs that share a table word: the group, or the largest of 32, 64 and 128 that divides it.
int64_t table_step(int64_t group) { return group % 128 == 0 ? 128 : group % 64 == 0 ? 64 : 32; }

const char* shape_fault(int64_t n, int64_t k, int64_t group) {
  if (n <= 0 || k <= 0 || group <= 0) return "sizes must be positive";
  if (n > 0x7fffffe0 || k > 0x7fffff00) return "size past 32 bits";
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
// Rows from which a call takes 128 x 128 tiles.
constexpr int64_t kTiledRows = 65;
int64_t sum_blocks(int64_t k, int64_t group) { return tiles(tiles(k, kTileK) * (kTileK / table_step(group)), 32); }
}  // namespace
}  // namespace sb

extern "C" int64_t sb_w4_linear_workspace_size(int64_t num_rows, int64_t out_features, int64_t in_features,
                                               int64_t group) {
  using namespace sb;
  if (num_rows < kTiledRows || shape_fault(out_features, in_features, group)) return 0;
  return num_rows * sum_blocks(in_features, group) * 256;
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
  if (num_rows > 0x7fffff00) return fail(fn, "size past 32 bits");
  if (reinterpret_cast<uintptr_t>(x) % 16 || x_stride * 2 % 16)
    return fail(fn, "rows of x must be 16-byte aligned");
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
  if (num_rows >= kTiledRows) {
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
        workspace_bytes < sb_w4_linear_workspace_size(num_rows, out_features, in_features, group))
      return fail(fn, "workspace too small or not 16-byte aligned");
    a.sums = static_cast<const char*>(workspace);
    a.sum_blocks = static_cast<int>(sum_blocks(in_features, group));
    a.wide_out = reinterpret_cast<uintptr_t>(y) % 16 == 0 && a.y_row % 16 == 0;
    const int64_t work = num_rows * a.sum_blocks * 32 * (table_step(group) / 8);
    const int64_t grid = tiles(num_rows, kBM) * tiles(out_features, kBN);
    if (tiles(work, 256) > 0x7fffffff || grid > 0x7fffffff) return fail(fn, "grid too large");
#define SB_W4(DT, GPT)                                                                                \
  if (dtype == DT && gpt == GPT) {                                                                    \
    SB_LAUNCH("w4_sums", (w4_sums_kernel<DT, kTileK / GPT>), dim3(static_cast<unsigned>(tiles(work, 256))), \
              dim3(256), st, static_cast<uint16_t*>(workspace), a.x, a.x_row, a.num_rows, a.k,        \
              a.sum_blocks);                                                                          \
    SB_LAUNCH("w4_tiles", (w4_tiles_kernel<DT, GPT>), dim3(static_cast<unsigned>(grid)), dim3(256), st, a); \
  }
    SB_W4(SB_DTYPE_BF16, 1) SB_W4(SB_DTYPE_BF16, 2) SB_W4(SB_DTYPE_BF16, 4)
    SB_W4(SB_DTYPE_F16, 1) SB_W4(SB_DTYPE_F16, 2) SB_W4(SB_DTYPE_F16, 4)
#undef SB_W4
    return check_launch(fn);
  }
  const int mi = num_rows <= 16 ? 1 : num_rows <= 32 ? 2 : 4;
  const int64_t gy = tiles(num_rows, 16 * mi);
  if (gy > 65535) return fail(fn, "too many rows");
  const dim3 grid(static_cast<unsigned>(tiles(out_features, kTileN)), static_cast<unsigned>(gy));
#define SB_W4(DT, MI, GPT)                                                                            \
  if (dtype == DT && mi == MI && gpt == GPT)                                                          \
    SB_LAUNCH("w4_rows", (w4_rows_kernel<DT, MI, GPT>), grid, dim3(64 * kWaves), st, a);
#define SB_W4_(DT)                                    \
  SB_W4(DT, 1, 1) SB_W4(DT, 1, 2) SB_W4(DT, 1, 4)     \
  SB_W4(DT, 2, 1) SB_W4(DT, 2, 2) SB_W4(DT, 2, 4)     \
  SB_W4(DT, 4, 1) SB_W4(DT, 4, 2) SB_W4(DT, 4, 4)
  SB_W4_(SB_DTYPE_BF16)
  SB_W4_(SB_DTYPE_F16)
#undef SB_W4_
#undef SB_W4
  return check_launch(fn);
}
