// Matrix-core and LDS helpers shared by the attention kernels (gfx950, wave64).
#pragma once

#include "sb_common.h"

namespace sb {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}

// Value of v in lane (lane ^ 32): v_permlane32_swap exchanges the upper half of one register
// with the lower half of another, so swapping v with itself and picking the moved half gives
// the partner lane's value without a round trip through LDS.
__device__ __forceinline__ float xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

template <int DT> struct Mma;
template <> struct Mma<SB_DTYPE_BF16> {
  using vec8 = bf16x8_t;
  using elem = __bf16;
  __device__ __forceinline__ static f32x16_t mma(vec8 a, vec8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static vec8 cvt8(const float* f) {
    vec8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = static_cast<__bf16>(f[e]);
    return r;
  }
  __device__ __forceinline__ static uint16_t cvt1(float f) { return f32_to_bf16(f); }
  // Two values rounded to a packed pair (one v_cvt_pk_bf16_f32), and acc + their sum.
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  __device__ __forceinline__ static x2 cvt2(float a, float b) {
    const x2 r = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return r;
  }
  __device__ __forceinline__ static float sum2(x2 v, float acc) {
    const x2 one = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
    return __builtin_amdgcn_fdot2_f32_bf16(v, one, acc, false);
  }
  // 0 + the sum of v, the zero as an inline constant of the VOP3 form (no zeroed register).
  __device__ __forceinline__ static float sum2z(x2 v, uint32_t one) {
    float r;
    asm volatile("v_dot2_f32_bf16 %0, %1, %2, 0" : "=v"(r) : "v"(v), "v"(one));
    return r;
  }
  static constexpr uint32_t kOnePair = 0x3f803f80u;
  // acc + sum of the 8 (rounded) elements of v, two per v_dot2.
  __device__ __forceinline__ static float sum8(vec8 v, float acc) {
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
    const x2 one = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const x2 pr = {v[2 * e], v[2 * e + 1]};
      acc = __builtin_amdgcn_fdot2_f32_bf16(pr, one, acc, false);
    }
    return acc;
  }
  // Largest tile sum of P accepted without moving the reference max (bf16 keeps fp32's
  // exponent range, so only fp32 overflow of O bounds it).
  static constexpr float kPMax = 0x1p64f;
};
template <> struct Mma<SB_DTYPE_F16> {
  using vec8 = f16x8_t;
  using elem = _Float16;
  __device__ __forceinline__ static f32x16_t mma(vec8 a, vec8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static vec8 cvt8(const float* f) {
    vec8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = static_cast<_Float16>(f[e]);
    return r;
  }
  __device__ __forceinline__ static uint16_t cvt1(float f) { return f32_to_f16(f); }
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  __device__ __forceinline__ static x2 cvt2(float a, float b) {
    const x2 r = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return r;
  }
  __device__ __forceinline__ static float sum2(x2 v, float acc) {
    const x2 one = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
    return __builtin_amdgcn_fdot2(v, one, acc, false);
  }
  __device__ __forceinline__ static float sum2z(x2 v, uint32_t one) {
    float r;
    asm volatile("v_dot2_f32_f16 %0, %1, %2, 0" : "=v"(r) : "v"(v), "v"(one));
    return r;
  }
  static constexpr uint32_t kOnePair = 0x3c003c00u;
  __device__ __forceinline__ static float sum8(vec8 v, float acc) {
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
    const x2 one = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const x2 pr = {v[2 * e], v[2 * e + 1]};
      acc = __builtin_amdgcn_fdot2(pr, one, acc, false);
    }
    return acc;
  }
  // fp16 P saturates at 65504: keep every p below 2^8.
  static constexpr float kPMax = 256.f;
};

// 16-byte chunk position of chunk c of row r in the swizzled K and V tiles (CH chunks per
// row). K fragments are read as 16 bytes per lane from 32 consecutive rows at one chunk:
// rows r..r+15 land on distinct chunk positions. V is read with transpose loads that touch
// 4 consecutive rows x 32-64 bytes: rows r..r+3 land on disjoint 64-byte bank ranges.
template <int CH>
__device__ __forceinline__ int kswz(int r, int c) {
  return c ^ (r & (CH - 1));
}
template <int CH>
__device__ __forceinline__ int vswz(int r, int c) {
  return CH >= 16 ? c ^ (4 * (r & 3)) : c ^ (4 * ((r >> 1) & 1));
}

#define SB_GLOBAL __attribute__((address_space(1)))
#define SB_LDS __attribute__((address_space(3)))
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Waits until this wave's outstanding vector-memory operations (including direct-to-LDS
// loads) are complete: s_waitcnt vmcnt(0), other counters untouched.
__device__ __forceinline__ void wait_vmem() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// One 16-byte global -> LDS copy per lane (global_load_lds_dwordx4): lane i's chunk lands at
// LDS byte address lds_wave + 16 i, where lds_wave is wave-uniform. Written as inline
// assembly on purpose:
// the compiler treats a direct-to-LDS load it knows about as a pending write to the whole LDS
// variable and waits for it (vmcnt(0)) before any later read of that variable, which would
// serialise every prefetch with the tile being computed. Hidden from it, the loads overlap
// the compute; the kernel orders them itself with wait_vmem() before each barrier that
// publishes a tile. (Waits the compiler places for its own vector-memory loads stay safe:
// completions are counted in order, so extra outstanding loads only make them stricter.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is named as clobbered on purpose
__device__ __forceinline__ void dma_row_chunk(const char* src, uint32_t lds_wave) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(lds_wave), "v"(src)
      : "memory", "m0");
}
// The same load in two parts, for callers that keep the M0 write and the load apart: the LDS
// destination goes to M0 first, and the load (which reads M0) must follow at least one other
// instruction later (the M0 write-to-use wait state). Nothing between them may write M0.
__device__ __forceinline__ void dma_set_m0(uint32_t lds_wave) {
  asm volatile("s_mov_b32 m0, %0" : : "s"(lds_wave) : "m0");
}
__device__ __forceinline__ void dma_at_m0(const char* src) {
  asm volatile("global_load_lds_dwordx4 %0, off" : : "v"(src) : "memory");
}
// The same with the wave's base address in scalar registers and a 32-bit byte offset per lane.
__device__ __forceinline__ void dma_at_m0_s(const char* base, uint32_t voff) {
  asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(base) : "memory");
}
// LDS byte address of a pointer into a __shared__ array (wave-uniform arithmetic on it stays
// in scalar registers).
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SB_LDS const void*)p));
}
#pragma clang diagnostic pop

}  // namespace sb
