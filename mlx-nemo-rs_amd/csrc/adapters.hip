// Low-rank adapters beside a shared 8-bit projection, the first product:
// t_r = s_a A_a x_r for each row r with its adapter a = which[r]. (The second,
// B_a t_r, begins the projection's sums in fp8_gemm.hip.)
//
// A wave takes 16 RG rows and every WK-th block of 128 inputs; the MFMA's first
// operand is 16 ranks of A, its second 16 rows, of which those of other adapters
// count as zero, so that one set of sums serves all of a group's adapters, which
// go through their A one by one. bf16 rows (and codes, which bf16 holds) multiply
// exactly, f32 rows as three bf16 parts; sums are f32, joined over the waves in
// their order. The projection needs the rows' codes where it runs in tiles: they
// are made here, from the same registers, so that x is read once and the
// adapters cost no launch. Bound: x's bytes from HBM, A's from the L2 once per
// 16 RG rows.
#include <algorithm>
#include <type_traits>

#include "../../include/relpos_mhsa.h"
#include "fp8_common.hpp"
#include "fp8_kernels.hpp"

namespace mhsa {
namespace {

template <typename TX, int RT, int RG, int WK>
__global__ __launch_bounds__(WK * 64) void adapter_rows_kernel(AdapterRows p) {
  constexpr bool CODES = std::is_same_v<TX, uint8_t>, F32 = std::is_same_v<TX, float>;
  __shared__ floatx4 red[WK][RG * RT][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, c4 = lane >> 4;
  const int kb = (p.K + 127) / 128, kp = kb * 128, kbp = (kb + 3) / 4 * 4;
  int64_t row[RG];
  int mine[RG];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    row[g] = ((int64_t)blockIdx.x * RG + g) * 16 + r;
    mine[g] = row[g] < p.rows ? p.which[row[g]] : -1;
    if (mine[g] >= p.n) mine[g] = -1;
  }
  floatx4 acc[RG][RT];
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[g][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int b = w; b < kb; b += WK) {
    // this lane's inputs: 8 of each run of 32, from 8 c4 on
    uint32_t part[RG][F32 ? 3 : 1][4][4];
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int64_t at = min(row[g], p.rows - 1);
      if constexpr (CODES) {
        const float scale = fp8_scale(p.scales[at * kbp + b]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x2 c;
          __builtin_memcpy(&c, p.codes + at * kp + b * 128 + 32 * i + 8 * c4, 8);
          const bf16x8 v = fp8_to_bf16(c[0], c[1], scale);
          __builtin_memcpy(part[g][0][i], &v, 16);
        }
      } else {
        const TX* x = static_cast<const TX*>(p.x) + at * p.ldx;
        float v[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) load8(x, b * 128 + 32 * i + 8 * c4, p.K, v[i]);
        if (p.q_codes) {
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fp8_mag(v[i][e]));
          m = fmaxf(m, __shfl_xor(m, 16, 64));
          m = fmaxf(m, __shfl_xor(m, 32, 64));
          const int s = fp8_scale_byte(m);
          const float scale = fp8_scale(s);
          if (row[g] < p.rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<u32x2*>(p.q_codes + row[g] * kp + b * 128 + 32 * i + 8 * c4) =
                  u32x2{fp8_pack4_scaled(v[i][0], v[i][1], v[i][2], v[i][3], scale),
                        fp8_pack4_scaled(v[i][4], v[i][5], v[i][6], v[i][7], scale)};
            if (c4 == 0) p.q_scales[row[g] * kbp + b] = (uint8_t)s;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (F32) split_pair(v[i][2 * e], v[i][2 * e + 1], part[g][0][i][e], part[g][1][i][e], part[g][2][i][e]);
            else part[g][0][i][e] = pack_bf16(v[i][2 * e], v[i][2 * e + 1]);
          }
      }
    }
    uint64_t left[RG];
#pragma unroll
    for (int g = 0; g < RG; ++g) left[g] = __ballot(mine[g] >= 0);
    for (;;) {
      int d = -1;
#pragma unroll
      for (int g = RG - 1; g >= 0; --g)
        if (left[g]) d = __builtin_amdgcn_readlane(mine[g], __builtin_ctzll(left[g]));
      if (d < 0) break;
#pragma unroll
      for (int g = 0; g < RG; ++g) left[g] &= ~__ballot(mine[g] == d);
      const uint16_t* a = p.a + ((int64_t)d * p.rank + r) * kp + b * 128 + 8 * c4;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          const bf16x8 fa = *reinterpret_cast<const bf16x8*>(a + (int64_t)16 * j * kp + 32 * i);
#pragma unroll
          for (int g = 0; g < RG; ++g)
#pragma unroll
            for (int q = 0; q < (F32 ? 3 : 1); ++q) {
              u32x4 f = {};
              if (mine[g] == d) f = u32x4{part[g][q][i][0], part[g][q][i][1], part[g][q][i][2], part[g][q][i][3]};
              acc[g][j] = mma16(fa, __builtin_bit_cast(bf16x8, f), acc[g][j]);
            }
        }
    }
  }
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int j = 0; j < RT; ++j) red[w][g * RT + j][lane] = acc[g][j];
  __syncthreads();
  // lane: row r, ranks 16 j + 4 c4 + [0, 4)
  const int ext = p.parts * p.rank;
  for (int q = w; q < RG * RT; q += WK) {
    const int64_t to = ((int64_t)blockIdx.x * RG + q / RT) * 16 + r;
    if (to >= p.rows) continue;
    const int d = p.which[to], j = q % RT;
    const float s = d >= 0 && d < p.n ? p.scale[d] : 0.f;  // (of no adapter: the sums are 0)
    floatx4 v = red[0][q][lane];
#pragma unroll
    for (int i = 1; i < WK; ++i) v += red[i][q][lane];
    uint16_t* t = p.t + to * ext + 16 * j + 4 * c4;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= s;
    if (p.parts == 1) {
      *reinterpret_cast<u32x2*>(t) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    } else {
      uint32_t h[2], m[2], l[2];
      split_pair(v[0], v[1], h[0], m[0], l[0]);
      split_pair(v[2], v[3], h[1], m[1], l[1]);
      *reinterpret_cast<u32x2*>(t) = u32x2{h[0], h[1]};
      *reinterpret_cast<u32x2*>(t + p.rank) = u32x2{m[0], m[1]};
      *reinterpret_cast<u32x2*>(t + 2 * p.rank) = u32x2{l[0], l[1]};
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void adapter_weights_kernel(const T* from, int rows, int cols, uint16_t* to, int cols_to,
                                                              int64_t n, int* bad) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  const int row = (int)(at / cols_to), col = (int)(at % cols_to);
  const bf16 v = row < rows && col < cols ? (bf16)(float)from[(int64_t)row * cols + col] : (bf16)0.f;
  if (!(__builtin_fabsf((float)v) < __builtin_inff())) *bad = 1;
  if (to) to[at] = __builtin_bit_cast(uint16_t, v);
}

template <typename TX, int RT>
hipError_t go(const AdapterRows& p, hipStream_t s) {
  constexpr int RG = RT <= 4 ? 2 : 1;
  const unsigned grid = (unsigned)((p.rows + 16 * RG - 1) / (16 * RG));
  adapter_rows_kernel<TX, RT, RG, 8><<<grid, 512, 0, s>>>(p);
  return hipGetLastError();
}
template <typename TX>
hipError_t by_rank(const AdapterRows& p, hipStream_t s) {
  switch (p.rank) {
    case 16: return go<TX, 1>(p, s);
    case 32: return go<TX, 2>(p, s);
    case 64: return go<TX, 4>(p, s);
    case 128: return go<TX, 8>(p, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t adapter_rows(const AdapterRows& p, hipStream_t s) {
  if (p.rows <= 0 || p.rows > (int64_t)1 << 26 || p.K <= 0 || p.K > kFp8MaxK || p.n <= 0 || !p.which || !p.a || !p.scale || !p.t ||
      (p.parts != 1 && p.parts != 3) || (!p.x && (!p.codes || !p.scales || p.q_codes)) || !p.q_codes != !p.q_scales)
    return hipErrorInvalidValue;
  if (!p.x) return by_rank<uint8_t>(p, s);
  return p.x_dt == kBF16 ? by_rank<bf16>(p, s) : by_rank<float>(p, s);
}

hipError_t adapter_weights(int data_dtype, const void* from, int rows, int cols, uint16_t* to, int rows_to, int cols_to,
                           int* bad, hipStream_t s) {
  if (rows <= 0 || cols <= 0 || rows > rows_to || cols > cols_to || !from || !bad) return hipErrorInvalidValue;
  const int64_t n = (int64_t)rows_to * cols_to;
  if (n > (int64_t)1 << 31) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)((n + 255) / 256);
  switch (data_dtype) {
    case MHSA_F32: adapter_weights_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(from), rows, cols, to, cols_to, n, bad); break;
    case MHSA_BF16: adapter_weights_kernel<<<grid, 256, 0, s>>>(static_cast<const bf16*>(from), rows, cols, to, cols_to, n, bad); break;
    case MHSA_F16: adapter_weights_kernel<<<grid, 256, 0, s>>>(static_cast<const _Float16*>(from), rows, cols, to, cols_to, n, bad); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mhsa
