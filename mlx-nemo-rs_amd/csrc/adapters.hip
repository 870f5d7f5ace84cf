// Low-rank adapters beside a shared 8-bit projection, the first product:
// t_r = s_a A_a x_r for each row r with its adapter a = which[r]. (The second,
// B_a t_r, begins the projection's sums in fp8_gemm.hip.)
//
// 8 waves take R rows, KC inputs at a time: each reads whole lines of its rows
// (the next ones while these are worked on), rounds them to the codes that the
// projection needs where it runs in tiles, so that x is read once and the
// adapters cost no launch, and leaves them in LDS, from where the MFMA's second
// operand, 32 inputs of 16 rows, is read; the first is 16 ranks of A, held in the
// order of the instruction's lanes. Waves share out the steps of 32 inputs, and
// their sums are joined in their order at the end. The adapters of a group of
// rows are gone through one by one, rows of others as zeros, so that one set of
// sums serves all. bf16 rows (and codes, which bf16 holds) multiply exactly, f32
// rows as three bf16 parts; sums are f32. Bound: x's bytes and the codes' from
// and to HBM, A's from the L2 once per R rows.
#include <algorithm>
#include <type_traits>

#include "../../include/relpos_mhsa.h"
#include "fp8_common.hpp"
#include "fp8_kernels.hpp"

namespace mhsa {
namespace {

// A is held in fragments: step k / 32, block of 16 ranks, lane, 8 values; lane l
// has rank l % 16 and inputs 32 step + 8 (l / 16) on.
__device__ __host__ inline int64_t fragment(int step, int block, int rank) { return ((int64_t)step * (rank / 16) + block) * 512; }

template <typename TX, int RT, int R, int KC>
struct RowsCfg {
  using TL = std::conditional_t<std::is_same_v<TX, float>, float, bf16>;  // in LDS
  static constexpr int RG = R / 16, RUNS = R * KC / 8 / 512, PARTS = KC / 512, STEPS = KC / 32 / 8;
  static constexpr int PITCH = KC * (int)sizeof(TL) + 16, BUF = R * PITCH;
  static constexpr int RED = 8 * RG * RT * 1024;
  static constexpr int LDS = 2 * BUF > RED ? 2 * BUF : RED;
};

// VEC: rows of whole runs of 8 inputs.
template <typename TX, int RT, int R, int KC, bool VEC>
__global__ __launch_bounds__(512, 4) void adapter_rows_kernel(AdapterRows p) {
  using C = RowsCfg<TX, RT, R, KC>;
  using TL = typename C::TL;
  constexpr bool CODES = std::is_same_v<TX, uint8_t>, F32 = std::is_same_v<TX, float>;
  constexpr int RG = C::RG;
  __shared__ __attribute__((aligned(16))) char smem[C::LDS];
  const int lane = threadIdx.x & 63, r = lane & 15, c4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kb = (p.K + 127) / 128, kp = kb * 128, kbp = (kb + 3) / 4 * 4;
  const int64_t row0 = (int64_t)blockIdx.x * R;
  const int rows = (int)min<int64_t>(p.rows - row0, R);
  int mine[RG];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    mine[g] = 16 * g + r < rows ? p.which[row0 + 16 * g + r] : -1;
    if (mine[g] >= p.n) mine[g] = -1;
  }
  // Run u of this wave: a row's 512 inputs, 8 to a lane.
  auto run_row = [&](int u) { return (w * C::RUNS + u) / C::PARTS; };
  auto run_col = [&](int u, int k0) { return k0 + (w * C::RUNS + u) % C::PARTS * 512 + 8 * lane; };
  Run<TL, VEC> x[C::RUNS];  // (codes: two words of it, and their scale)
  auto fetch = [&](int k0) {
#pragma unroll
    for (int u = 0; u < C::RUNS; ++u) {
      const int c = run_col(u, k0);
      if (run_row(u) >= rows || c - 8 * lane >= kp) continue;
      const int64_t row = row0 + run_row(u);
      if constexpr (CODES) {
        __builtin_memcpy(x[u].u, p.codes + row * kp + min(c, kp - 8), 8);
        x[u].u[2] = p.scales[row * kbp + min(c / 128, kb - 1)];
      } else {
        x[u].load(static_cast<const TX*>(p.x) + row * p.ldx, c, p.K);
      }
    }
  };
  floatx4 acc[RG][RT];
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[g][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  uint64_t any = 0;
#pragma unroll
  for (int g = 0; g < RG; ++g) any |= __ballot(mine[g] >= 0);

  fetch(0);
#pragma unroll 1
  for (int k0 = 0, turn = 0; k0 < kp; k0 += KC, turn ^= 1) {
    char* buf = smem + turn * C::BUF;
#pragma unroll
    for (int u = 0; u < C::RUNS; ++u) {
      const int c = run_col(u, k0), row = run_row(u);
      if (row >= rows || c - 8 * lane >= kp) continue;
      char* to = buf + row * C::PITCH + (c - k0) * (int)sizeof(TL);
      if constexpr (CODES) {
        bf16x8 v = fp8_to_bf16(x[u].u[0], x[u].u[1], fp8_scale((int)x[u].u[2]));
        *reinterpret_cast<bf16x8*>(to) = v;
      } else {
        x[u].trim(c, p.K);
#pragma unroll
        for (int q = 0; q < Run<TX, VEC>::N / 4; ++q) *reinterpret_cast<u32x4*>(to + 16 * q) = u32x4{x[u].u[4 * q], x[u].u[4 * q + 1], x[u].u[4 * q + 2], x[u].u[4 * q + 3]};
        if (p.q_codes) {
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmaxf(m, fp8_mag(x[u][e]));
          m = row_reduce(m, [](float a, float b) { return fmaxf(a, b); });
          const int s = fp8_scale_byte(m);
          const float scale = fp8_scale(s);
          uint8_t* q = p.q_codes + (row0 + row) * kp + c;
          if (c < kp)
            *reinterpret_cast<u32x2*>(q) = u32x2{fp8_pack4_scaled(x[u][0], x[u][1], x[u][2], x[u][3], scale),
                                                 fp8_pack4_scaled(x[u][4], x[u][5], x[u][6], x[u][7], scale)};
          uint32_t bytes = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) bytes |= (uint32_t)__builtin_amdgcn_readlane(s, 16 * i) << 8 * i;
          if (lane == 0) *reinterpret_cast<uint32_t*>(p.q_scales + (row0 + row) * kbp + c / 128) = bytes;
        }
      }
    }
    if (k0 + KC < kp) fetch(k0 + KC);
    __syncthreads();
    if (any == 0) continue;
    // steps w, w + 8, ... of this wave
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
      const uint16_t* a = p.a + (int64_t)d * p.rank * kp + 8 * lane;
#pragma unroll
      for (int st = 0; st < C::STEPS; ++st) {
        const int k = k0 + 32 * (w + 8 * st);
        if (k >= kp) break;
        bf16x8 fa[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) fa[j] = *reinterpret_cast<const bf16x8*>(a + fragment(k / 32, j, p.rank));
#pragma unroll
        for (int g = 0; g < RG; ++g) {
          const char* from = buf + (16 * g + r) * C::PITCH + (k - k0 + 8 * c4) * (int)sizeof(TL);
          u32x4 f[F32 ? 3 : 1];
          if constexpr (F32) {
            const floatx4 lo = *reinterpret_cast<const floatx4*>(from), hi = *reinterpret_cast<const floatx4*>(from + 16);
            uint32_t h, m, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v0 = e < 2 ? lo[2 * e] : hi[2 * e - 4], v1 = e < 2 ? lo[2 * e + 1] : hi[2 * e - 3];
              split_pair(mine[g] == d ? v0 : 0.f, mine[g] == d ? v1 : 0.f, h, m, l);
              f[0][e] = h;
              f[1][e] = m;
              f[2][e] = l;
            }
          } else {
            f[0] = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[0][e] = mine[g] == d ? f[0][e] : 0;
          }
#pragma unroll
          for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int q = 0; q < (F32 ? 3 : 1); ++q) acc[g][j] = mma16(fa[j], __builtin_bit_cast(bf16x8, f[q]), acc[g][j]);
        }
      }
    }
  }
  if (any == 0) return;  // (nobody reads their t)
  __syncthreads();
  floatx4* red = reinterpret_cast<floatx4*>(smem);
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int j = 0; j < RT; ++j) red[(w * RG * RT + g * RT + j) * 64 + lane] = acc[g][j];
  __syncthreads();
  // lane: row r, ranks 16 j + 4 c4 + [0, 4)
  const int ext = p.parts * p.rank;
  for (int q = w; q < RG * RT; q += 8) {
    const int row = q / RT * 16 + r, j = q % RT;
    if (row >= rows) continue;
    const int d = p.which[row0 + row];
    const float s = d >= 0 && d < p.n ? p.scale[d] : 0.f;  // (of no adapter: the sums are 0)
    floatx4 v = red[q * 64 + lane];
#pragma unroll
    for (int i = 1; i < 8; ++i) v += red[(i * RG * RT + q) * 64 + lane];
    uint16_t* t = p.t + (row0 + row) * ext + 16 * j + 4 * c4;
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

// FRAGMENTS: `to` as A is held (rows_to ranks of cols_to inputs).
template <typename T, bool FRAGMENTS>
__global__ __launch_bounds__(256) void adapter_weights_kernel(const T* from, int rows, int cols, uint16_t* to, int rows_to,
                                                              int cols_to, int* bad) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)rows_to * cols_to) return;
  const int row = (int)(at / cols_to), col = (int)(at % cols_to);
  const bf16 v = row < rows && col < cols ? (bf16)(float)from[(int64_t)row * cols + col] : (bf16)0.f;
  if (!(__builtin_fabsf((float)v) < __builtin_inff())) *bad = 1;
  if (!to) return;
  const int64_t f = fragment(col / 32, row / 16, rows_to) + (row % 16 + col % 32 / 8 * 16) * 8 + col % 8;
  to[FRAGMENTS ? f : at] = __builtin_bit_cast(uint16_t, v);
}

// 32 rows to a workgroup halve A's way from the L2; up to RULE rows 16, which
// leaves more of them.
template <typename TX, int RT, int R, int KC>
hipError_t launch(const AdapterRows& p, hipStream_t s) {
  const unsigned grid = (unsigned)((p.rows + R - 1) / R);
  if (std::is_same_v<TX, uint8_t> || p.K % 8 == 0) adapter_rows_kernel<TX, RT, R, KC, true><<<grid, 512, 0, s>>>(p);
  else if constexpr (!std::is_same_v<TX, uint8_t>) adapter_rows_kernel<TX, RT, R, KC, false><<<grid, 512, 0, s>>>(p);
  return hipGetLastError();
}
template <typename TX, int RT>
hipError_t go(const AdapterRows& p, hipStream_t s) {
  if constexpr (RT <= 4 && !std::is_same_v<TX, float>)
    return p.rows > 16 * device_cus() ? launch<TX, RT, 32, 512>(p, s) : launch<TX, RT, 16, 1024>(p, s);
  else
    return launch<TX, RT, 16, 512>(p, s);
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
                           bool fragments, int* bad, hipStream_t s) {
  if (rows <= 0 || cols <= 0 || rows > rows_to || cols > cols_to || !from || !bad) return hipErrorInvalidValue;
  if (fragments && (rows_to % 16 || cols_to % 32)) return hipErrorInvalidValue;
  const int64_t n = (int64_t)rows_to * cols_to;
  if (n > (int64_t)1 << 31) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)((n + 255) / 256);
  auto go = [&](auto t) {
    const auto* f = static_cast<const decltype(t)*>(from);
    if (fragments) adapter_weights_kernel<decltype(t), true><<<grid, 256, 0, s>>>(f, rows, cols, to, rows_to, cols_to, bad);
    else adapter_weights_kernel<decltype(t), false><<<grid, 256, 0, s>>>(f, rows, cols, to, rows_to, cols_to, bad);
  };
  switch (data_dtype) {
    case MHSA_F32: go(0.f); break;
    case MHSA_BF16: go(bf16(0.f)); break;
    case MHSA_F16: go(_Float16(0.f)); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mhsa
