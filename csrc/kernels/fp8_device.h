// Device code that the 8-bit kernels share: magnitudes, a block's scale, conversions.
#pragma once

#include "fp8_launch.h"

namespace gpuexp {

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
typedef __attribute__((ext_vector_type(2))) short s16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// The byte e + 127 of a block whose largest finite magnitude has these bits (of a 32-bit float).
template <int kType>
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  constexpr int p = kType == kE4M3 ? 8 : 15;
  const int byte = int(amax >> 23) - p + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax == 0 ? 127 : byte < 0 ? 0 : byte;  // (a subnormal amax too: its exponent field is 0)
}
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float(uint32_t(byte) << 23); }

__device__ __forceinline__ uint32_t max2x16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// Magnitudes order as their bits.  `mags` of 16-bit values keeps two columns in a word; the first infinity
// has the bits kInf.
template <int kX>
constexpr uint32_t kInf = kX == kBF16 ? 0x7f80u : kX == kF16 ? 0x7c00u : 0x7f800000u;

template <int kX>
__device__ __forceinline__ uint32_t mag(uint32_t w) {
  return w & (kX == kF32 ? 0x7fffffffu : 0x7fff7fffu);
}
template <int kX>
__device__ __forceinline__ uint32_t max_mag(uint32_t a, uint32_t b) {
  if constexpr (kX == kF32) return max(a, b);
  else return max2x16(a, b);
}
// the same without what is not finite
template <int kX>
__device__ __forceinline__ uint32_t finite_mag(uint32_t w) {
  const uint32_t m = mag<kX>(w);
  if constexpr (kX == kF32) return m < kInf<kX> ? m : 0;
  else return ((m & 0xffffu) < kInf<kX> ? m & 0xffffu : 0) | ((m >> 16) < kInf<kX> ? m & 0xffff0000u : 0);
}
// the larger of the two in a word
template <int kX>
__device__ __forceinline__ uint32_t widest(uint32_t m) {
  if constexpr (kX == kF32) return m;
  else return max(m & 0xffffu, m >> 16);
}
// a magnitude as the bits of a 32-bit float
template <int kX>
__device__ __forceinline__ uint32_t mag_bits(uint32_t m) {
  if constexpr (kX == kF32) return m;
  if constexpr (kX == kBF16) return m << 16;
  if constexpr (kX == kF16) return __float_as_uint(float(__builtin_bit_cast(_Float16, uint16_t(m))));
}

// two values in 8 bits, into the low or high half of a word
template <int kX, int kType, bool kHigh>
__device__ __forceinline__ s16x2 convert2(s16x2 old, uint32_t w, float scale) {
  if constexpr (kX == kBF16) {
    const bf16x2 v = __builtin_bit_cast(bf16x2, w);
    if constexpr (kType == kE4M3) return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, v, scale, kHigh);
    else return __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(old, v, scale, kHigh);
  } else {
    const f16x2 v = __builtin_bit_cast(f16x2, w);
    if constexpr (kType == kE4M3) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, v, scale, kHigh);
    else return __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(old, v, scale, kHigh);
  }
}
template <int kType, bool kHigh>
__device__ __forceinline__ s16x2 convert2(s16x2 old, float a, float b, float scale) {
  if constexpr (kType == kE4M3) return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(old, a, b, scale, kHigh);
  else return __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(old, a, b, scale, kHigh);
}
// four values: words of two 16-bit values each, or floats
template <int kX, int kType>
__device__ __forceinline__ uint32_t convert4(uint32_t a, uint32_t b, float scale) {
  const s16x2 lo = convert2<kX, kType, false>(s16x2{0, 0}, a, scale);
  return __builtin_bit_cast(uint32_t, convert2<kX, kType, true>(lo, b, scale));
}
template <int kType>
__device__ __forceinline__ uint32_t convert4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, float scale) {
  const s16x2 lo = convert2<kType, false>(s16x2{0, 0}, __uint_as_float(a), __uint_as_float(b), scale);
  return __builtin_bit_cast(uint32_t, convert2<kType, true>(lo, __uint_as_float(c), __uint_as_float(d), scale));
}
}  // namespace gpuexp
