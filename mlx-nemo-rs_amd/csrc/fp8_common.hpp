// Device helpers of the e4m3 block format.
#pragma once

#include <type_traits>

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
// Eight codes (two words) times a power of two as bf16: exact but for what
// lies below bf16's smallest subnormal, 2^-133.
__device__ __forceinline__ bf16x8 fp8_to_bf16(uint32_t lo, uint32_t hi, float scale = 1.f) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 values from x on. The loads need no more alignment than an element (the
// memory unit takes 16 bytes at any address).
template <typename T>
__device__ __forceinline__ void load_run(const T* x, float v[8]) {
  T t[8];
  __builtin_memcpy(t, x, sizeof t);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
}
// 8 values of row x from column c on, zero past K.
template <typename T>
__device__ __forceinline__ void load8(const T* x, int c, int K, float v[8]) {
  if (c + 8 <= K) {
    load_run(x + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? (float)x[c + i] : 0.f;
  }
}

// Each row of 16 lanes' values under `o`, in all of the row's lanes: the first
// N steps of: lanes xor 1, xor 2 (quad permutations), half rows and rows
// mirrored.
template <int N = 4, typename T, typename O>
__device__ __forceinline__ T row_reduce(T v, O o) {
  auto move = [](T x, auto ctrl) {
    constexpr int C = decltype(ctrl)::value;
    if constexpr (sizeof(T) == 4) {
      const int u = __builtin_bit_cast(int, x);
      return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(u, u, C, 0xF, 0xF, false));
    } else {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      i32x2 u = __builtin_bit_cast(i32x2, x);
      u[0] = __builtin_amdgcn_update_dpp(u[0], u[0], C, 0xF, 0xF, false);
      u[1] = __builtin_amdgcn_update_dpp(u[1], u[1], C, 0xF, 0xF, false);
      return __builtin_bit_cast(T, u);
    }
  };
  using std::integral_constant;
  if constexpr (N > 0) v = o(v, move(v, integral_constant<int, 0xB1>{}));
  if constexpr (N > 1) v = o(v, move(v, integral_constant<int, 0x4E>{}));
  if constexpr (N > 2) v = o(v, move(v, integral_constant<int, 0x141>{}));
  if constexpr (N > 3) v = o(v, move(v, integral_constant<int, 0x140>{}));
  return v;
}
// The wave's: one lane of each row.
template <typename T, typename O>
__device__ __forceinline__ T wave_reduce(T v, O o) {
  v = row_reduce(v, o);
  auto at = [&](int l) {
    if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
    } else {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      const i32x2 u = __builtin_bit_cast(i32x2, v);
      return __builtin_bit_cast(T, i32x2{__builtin_amdgcn_readlane(u[0], l), __builtin_amdgcn_readlane(u[1], l)});
    }
  };
  return o(o(at(0), at(16)), o(at(32), at(48)));
}

// A wave rounds 4 blocks of a row, 16 lanes of 8 values to a block; item `id`
// of rows * ceil(K / 512).
template <typename T>
__device__ __forceinline__ void quantize_blocks(const T* x, int64_t ldx, int64_t rows, int K, uint8_t* codes, uint8_t* scales,
                                                int64_t id) {
  const int kb = (K + 127) / 128, items = (kb + 3) / 4;
  if (id >= rows * items) return;
  const int64_t row = id / items;
  const int lane = threadIdx.x & 63, blk = (int)(id % items) * 4 + (lane >> 4);
  float v[8];
  load8(x + row * ldx, blk * 128 + (lane & 15) * 8, blk < kb ? K : 0, v);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fp8_mag(v[i]));
#pragma unroll
  for (int o = 1; o < 16; o *= 2) m = fmaxf(m, __shfl_xor(m, o, 64));
  if (blk >= kb) return;
  const int s = fp8_scale_byte(m);
  const float scale = fp8_scale(s);
  const u32x2 q = {fp8_pack4_scaled(v[0], v[1], v[2], v[3], scale), fp8_pack4_scaled(v[4], v[5], v[6], v[7], scale)};
  *reinterpret_cast<u32x2*>(codes + row * ((int64_t)kb * 128) + blk * 128 + (lane & 15) * 8) = q;
  if ((lane & 15) == 0) scales[row * (items * 4) + blk] = (uint8_t)s;
}

}  // namespace mhsa
