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

// 8 values of a row of K from column c on as they lie in memory, in one load, so
// that many are on their way at a time (load8's branches wait for each). Where
// the row ends before them the row's last 8 are loaded; trim, where something
// waits for them anyway, puts them in their places and zeros behind them. Rows of
// whole runs (c a multiple of 8) need neither; rows of under 8 are loaded one by
// one, in a form of their own: a branch on K beside the load had every load waited
// for (2^25 bf16 in rows of 2047 with their norm: 84 -> 42 us).
enum RowForm { kRagged, kWhole, kTiny };
inline RowForm row_form(int64_t k) { return k % 8 == 0 ? kWhole : k >= 8 ? kRagged : kTiny; }
template <typename T, RowForm FORM> struct Run {
  static constexpr int N = 2 * (int)sizeof(T);
  uint32_t u[N];
  __device__ __forceinline__ float operator[](int e) const {
    T t[8];
    __builtin_memcpy(t, u, sizeof t);
    return (float)t[e];
  }
  __device__ __forceinline__ void load(const T* row, int c, int K) {
    if constexpr (FORM != kTiny) {
      __builtin_memcpy(u, row + min(c, K - 8), sizeof u);
    } else {
      T t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = row[min(e, K - 1)];
      __builtin_memcpy(u, t, sizeof u);
    }
  }
  __device__ __forceinline__ void trim(int c, int K) {
    if constexpr (FORM == kWhole) {
#pragma unroll
      for (int e = 0; e < N; ++e) u[e] = c < K ? u[e] : 0;
      return;
    }
    // elements too many (of a row of under 8, whose only run begins with it: past its end)
    int s = min(max(c + 8 - K, 0), 8) * (int)sizeof(T) / 2;  // in half words
    if (__ballot(s != 0) == 0) return;
    if constexpr (FORM == kRagged) {
#pragma unroll
      for (int step = N; step; step /= 2)  // words: N, N / 2, ..., 1
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (s & 2 * step) u[e] = e + step < N ? u[e + step] : 0;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (s & 1) u[e] = u[e] >> 16 | (e + 1 < N ? u[e + 1] << 16 : 0);
      }
    } else {
      s = 2 * N - s;  // half words left
#pragma unroll
      for (int e = 0; e < N; ++e) u[e] = 2 * e + 2 <= s ? u[e] : 2 * e < s ? u[e] & 0xFFFF : 0;
    }
  }
};

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

// The largest finite magnitude of a block, 16 lanes' runs of 8 values. An
// infinity or a NaN in one of the wave's blocks costs a second look.
__device__ __forceinline__ float block_max(const float v[8]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, __builtin_fabsf(v[e]));  // (a NaN does not count)
  auto larger = [](float a, float b) { return fmaxf(a, b); };
  m = row_reduce(m, larger);
  if (__any(!(m < __builtin_inff()))) {
    m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fp8_mag(v[e]));
    m = row_reduce(m, larger);
  }
  return m;
}
template <RowForm FORM>
__device__ __forceinline__ float block_max(const Run<float, FORM>& x) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[e];
  return block_max(v);
}
// bf16 magnitudes have the order of their bits.
template <RowForm FORM>
__device__ __forceinline__ float block_max(const Run<bf16, FORM>& x) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x.u[e] & 0x7FFF7FFFu));
  auto larger = [](uint32_t a, uint32_t b) { return max(a, b); };
  uint32_t t = row_reduce((uint32_t)max(m[0], m[1]), larger);
  if (__any(t >= 0x7F80u)) {
    t = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t a = x.u[e / 2] >> 16 * (e % 2) & 0x7FFFu;
      t = max(t, a < 0x7F80u ? a : 0);
    }
    t = row_reduce(t, larger);
  }
  return __builtin_bit_cast(float, t << 16);
}
// Its codes.
template <RowForm FORM>
__device__ __forceinline__ u32x2 fp8_pack8_scaled(const Run<float, FORM>& x, float scale) {
  return u32x2{fp8_pack4_scaled(x[0], x[1], x[2], x[3], scale), fp8_pack4_scaled(x[4], x[5], x[6], x[7], scale)};
}
template <RowForm FORM>
__device__ __forceinline__ u32x2 fp8_pack8_scaled(const Run<bf16, FORM>& x, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  u32x2 q;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, x.u[2 * e]), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, x.u[2 * e + 1]), scale, true);
    q[e] = __builtin_bit_cast(uint32_t, r);
  }
  return q;
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
