// The 8-bit form of the norm, dense and cache operators: OCP e4m3 codes times a power of two per
// block. The power is held in one byte b (E8M0: 2^(b - 127)), the least for which the block's largest
// magnitude is at most 448, e4m3's largest number. A power of two costs a floating-point code none of
// its relative precision, raising it later changes no code that stays normal, and it is the form that
// the scale operand of the gfx950 matrix instructions takes.
#pragma once

#include "common.h"

namespace ldx {

constexpr int kBlock8 = LDX_BLOCK8;   // columns of a row that share a scale
constexpr int kPage8 = LDX_PAGE8;     // tokens of a cache page

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// The scale byte of a block with largest magnitude amax = 1.m * 2^(E - 127): amax <= 1.75 * 2^(b - 119)
// holds from b = E - 8 on where 1.m <= 1.75, from E - 7 where it is larger. All-zero and subnormal
// blocks get 1 (2^-126); an infinite amax gets 247, under which infinities become NaN codes.
__device__ __forceinline__ int scale_byte(float amax) {
  const int bits = __float_as_int(amax);
  const int b = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return b > 1 ? b : 1;
}

// 2^(b - 127) and 2^(127 - b) for 1 <= b <= 253.
__device__ __forceinline__ float scale_of(int b) { return __int_as_float(b << 23); }
__device__ __forceinline__ float inverse_of(int b) { return __int_as_float((254 - b) << 23); }

// Four values times the inverse scale as four codes (round to nearest even; v_cvt_pk_fp8_f32 gives
// subnormal codes their correct rounding, and NaN codes for infinities and NaN).
__device__ __forceinline__ int encode4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
}

// Eight consecutive values of T from memory of any alignment (gfx950 reads unaligned vectors).
template <typename T>
struct Load8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  Load8<T> u;
  __builtin_memcpy(&u, p, sizeof(u));
#pragma unroll
  for (int i = 0; i < 8; i++) f[i] = (float)u.v[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  Load8<T> u;
#pragma unroll
  for (int i = 0; i < 8; i++) u.v[i] = (T)f[i];
  __builtin_memcpy(p, &u, sizeof(u));
}

// The same past the caches' retention, for results that leave the kernel: they go out while it works, where
// dirty lines wait in the XCDs' caches for the launch's end.
template <typename T>
__device__ __forceinline__ void stream8(T* p, const float (&f)[8]) {
  typedef T V __attribute__((ext_vector_type(8)));
  typedef V Unaligned __attribute__((aligned(sizeof(T))));
  V v;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (T)f[i];
  __builtin_nontemporal_store(v, reinterpret_cast<Unaligned*>(p));
}

// Largest of v over the 16 lanes of a DPP row, on every one of them.
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp_f<0x128>(v));   // row_ror:8
  v = fmaxf(v, dpp_f<0x124>(v));
  v = fmaxf(v, dpp_f<0x122>(v));
  return fmaxf(v, dpp_f<0x121>(v));
}

__device__ __forceinline__ float wave_max(float v) {
  v = row16_max(v);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
// v's counterpart under a DPP row operation, and v and its partner half a row pair (a wave) away.
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  const i32x2 w = __builtin_bit_cast(i32x2, v);
  const i32x2 r = {__builtin_amdgcn_update_dpp(0, w[0], CTRL, 0xf, 0xf, false),
                   __builtin_amdgcn_update_dpp(0, w[1], CTRL, 0xf, 0xf, false)};
  return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double wave_sum(double v) {
  v += dpp_d<0x128>(v);
  v += dpp_d<0x124>(v);
  v += dpp_d<0x122>(v);
  v += dpp_d<0x121>(v);
  i32x2 w = __builtin_bit_cast(i32x2, v);
  const auto a0 = __builtin_amdgcn_permlane16_swap(w[0], w[0], false, false), a1 = __builtin_amdgcn_permlane16_swap(w[1], w[1], false, false);
  v = __builtin_bit_cast(double, (i32x2){(int)a0[0], (int)a1[0]}) + __builtin_bit_cast(double, (i32x2){(int)a0[1], (int)a1[1]});
  w = __builtin_bit_cast(i32x2, v);
  const auto b0 = __builtin_amdgcn_permlane32_swap(w[0], w[0], false, false), b1 = __builtin_amdgcn_permlane32_swap(w[1], w[1], false, false);
  return __builtin_bit_cast(double, (i32x2){(int)b0[0], (int)b1[0]}) + __builtin_bit_cast(double, (i32x2){(int)b0[1], (int)b1[1]});
}
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_f<0x128>(v);
  v += dpp_f<0x124>(v);
  v += dpp_f<0x122>(v);
  v += dpp_f<0x121>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = __int_as_float(a[0]) + __int_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// Four bytes per lane from a buffer (byte offset voff + soff; out of range reads zeros) straight into
// LDS at lds + 4 * lane; awaited like dma_buffer_b128.
__device__ __forceinline__ void dma_buffer_b32(i32x4 rs, unsigned voff, unsigned soff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(rs),
               "s"(soff), "s"(lds)
               : "memory");
}

}  // namespace ldx
