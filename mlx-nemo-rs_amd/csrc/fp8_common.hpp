// Device helpers of the e4m3 block format.
#pragma once

#include "common.hpp"

namespace mhsa {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// |v| for the block's maximum; infinities and NaNs do not count (they are
// coded NaN whatever the scale).
__device__ __forceinline__ float fp8_mag(float v) {
  const float a = __builtin_fabsf(v);
  return a < __builtin_inff() ? a : 0.f;
}

// Scale byte of a block with maximum m: the smallest s >= 0 with
// m <= 448 * 2^(s - 127). 448 = 1.75 * 2^8, so the exponent field drops by 8
// and rises by one past a mantissa of 0.75. A block of zeros has s = 127.
__device__ __forceinline__ int fp8_scale_byte(float m) {
  const uint32_t u = __builtin_bit_cast(uint32_t, m);
  const int s = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return u == 0 ? 127 : (s > 0 ? s : 0);
}
// 2^(s - 127); the smallest, 2^-127, is a subnormal.
__device__ __forceinline__ float fp8_scale(int s) {
  return __builtin_bit_cast(float, s > 0 ? (uint32_t)s << 23 : 0x00400000u);
}
// Four values over a power of two to codes, in one step of rounding (to
// nearest even; past 448 and NaN: NaN).
__device__ __forceinline__ uint32_t fp8_pack4_scaled(float a, float b, float c, float d, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, r);
}
// Eight codes (two words) as bf16, exactly.
__device__ __forceinline__ bf16x8 fp8_to_bf16(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace mhsa
