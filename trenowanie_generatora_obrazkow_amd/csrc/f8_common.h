// 8-bit floating point with block scales (e4m3 values, power-of-two scales as e8m0 bytes: exponent + 127).
//
// A block's scale is 2^e with the least e >= -126 such that its largest finite value is at most 448 * 2^e (448: the largest
// e4m3 number), and its values are x * 2^-e rounded to nearest even.  With a power of two the product is exact and only that
// one rounding is made, so a value keeps its rounding whichever block it stands in (but near the format's smallest steps),
// and the scaled MFMA takes the scales as they are.  Infinities and NaNs become NaN and take no part in the scale.
#pragma once
#include "hmoe_common.h"

namespace hmoe {

constexpr int kF8Block = 128;       // columns per scale of the products' operands
constexpr int kF8ScaleAlign = 16;   // scale rows are whole 16-byte pieces: one load serves 16 blocks

inline int64_t f8_scale_ld(int64_t K) {
  return ((K + kF8Block - 1) / kF8Block + kF8ScaleAlign - 1) / kF8ScaleAlign * kF8ScaleAlign;
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

// |x| of a finite x, else 0
__device__ __forceinline__ float f8_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < __builtin_inff() ? a : 0.0f;
}
// amax finite and >= 0 (1.75 * 2^8 = 448)
__device__ __forceinline__ int f8_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  return max((int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
}
__device__ __forceinline__ float f8_inv(int e) { return __uint_as_float((uint32_t)(127 - e) << 23); }  // 2^-e
__device__ __forceinline__ float f8_pow(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // 2^e
// the conversion's input: x * 2^-e, or NaN
__device__ __forceinline__ float f8_arg(float x, float inv) {
  const float t = x * inv;
  return __builtin_fabsf(t) < __builtin_inff() ? t : __builtin_nanf("");
}
// four values -> four e4m3 bytes (v_cvt_pk_fp8_f32: to nearest even; the arguments are at most 448)
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(f8_arg(a, inv), f8_arg(b, inv), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(f8_arg(c, inv), f8_arg(d, inv), r, true);
  return (uint32_t)r;
}
// bytes 2 H and 2 H + 1 of w as floats
template <int H>
__device__ __forceinline__ void f8_unpack2(uint32_t w, float& a, float& b) {
  const auto v = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, H != 0);
  a = v[0];
  b = v[1];
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// eight e4m3 values times 2^e as bf16, exactly
__device__ __forceinline__ u32x4 f8_widen(uint2 v, float scale) {
  u32x4 f;
  f[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.x, scale, false));
  f[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.x, scale, true));
  f[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.y, scale, false));
  f[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.y, scale, true));
  return f;
}

}  // namespace hmoe
