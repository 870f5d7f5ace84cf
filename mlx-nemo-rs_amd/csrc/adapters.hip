// Low-rank adapters beside a shared 8-bit projection, the first product:
// t_r = s_a A_a x_r for each row r with its adapter a = which[r]. (The second,
// B_a t_r, begins the projection's sums in fp8_gemm.hip.)
//
// The 8 waves of a workgroup take 16 rows, and each of them every 8th block of
// 128 inputs, without waiting for one another: 16 lanes read a row's block in
// whole lines (the next one's on its way while this is worked on) and round it
// to the codes that the projection needs where it runs in tiles, so that x is
// read once and the adapters cost no launch; the block passes through the wave's
// own LDS into the MFMA's second operand, 32 inputs of 16 rows. The first operand
// is 16 ranks of A, held in the order of the instruction's lanes. The adapters of
// the rows are gone through one by one, rows of others as zeros, so that one set
// of sums serves all; the waves' sums are joined in their order at the end. bf16
// rows (and codes, which bf16 holds) multiply exactly, f32 rows as three bf16
// parts; sums are f32.
//
// Bound: x's bytes and the codes' from and to HBM, and A's from the L2 once per
// 16 rows, which comes at about 19 TB/s: 15001 rows x 4096 take 36 us without an
// adapter (184 MB), 62 with adapters of rank 64 (480 MB more). 32 or 64 rows to a
// workgroup read A less often, but leave fewer waves (40 and 54 us without an
// adapter) and make more of the rows where one request ends (67 and 83 us with).
//
// Up to 4 rows a CU are 4 to a workgroup, of 16 waves: there a wave's blocks and the
// adapters of its rows, one behind the other, are what the launch lasts. With the
// projection 16 rows of 4096 -> 1024 with 16 adapters of rank 16 take 18 us instead
// of 37, 256 rows with 64 of rank 64 37 instead of 60, 1000 rows of 1024 -> 1024 f32
// with 10 14.0 instead of 15.3; 3000 rows of 1024 -> 4096, rank 32, would take 32.2
// instead of 30.7, for A is read four times as often.
//
// The sums' order, and with it t's last bits, go by the row's place in the call and
// by the number of rows: which block a workgroup begins with, and how many waves it
// has.
#include <algorithm>
#include <type_traits>

#include "../../include/relpos_mhsa.h"
#include "fp8_common.hpp"
#include "fp8_kernels.hpp"

namespace mhsa {
namespace {

// Registers for 4 waves a SIMD: at rank 128 f32 rows have 16 to 20 bytes a lane in
// scratch.
template <typename TX, int RT, RowForm FORM, bool FEW>
__global__ __launch_bounds__(FEW ? 1024 : 512, 4) void adapter_rows_kernel(AdapterRows p) {
  constexpr int NW = FEW ? 16 : 8, ROWS = FEW ? 4 : 16;
  constexpr bool CODES = std::is_same_v<TX, uint8_t>, F32 = std::is_same_v<TX, float>;
  using TL = std::conditional_t<F32, float, bf16>;  // in LDS
  constexpr int PITCH = 128 * (int)sizeof(TL) + 16, BUF = ROWS * PITCH, RED = NW * RT * 1024;
  __shared__ __attribute__((aligned(16))) char smem[NW * BUF > RED ? NW * BUF : RED];
  const int lane = threadIdx.x & 63, r = lane & 15, c4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kb = (p.K + 127) / 128, kp = kb * 128, kbp = (kb + 3) / 4 * 4;
  // a stretch of rows to each XCD, whose L2 then holds few adapters' A
  const unsigned per = gridDim.x / 8;
  const int64_t group = blockIdx.x % 8 * per + blockIdx.x / 8, row0 = group * ROWS;
  if (row0 >= p.rows) return;
  const int rows = (int)min<int64_t>(p.rows - row0, ROWS);
  int mine = r < rows ? p.which[row0 + r] : -1;
  if (mine >= p.n) mine = -1;
  const uint64_t some = __ballot(mine >= 0);
  // Run u of a block: row 4 u + lane / 16 (past the last: the last), 8 inputs.
  // (Rows' addresses are made again for each block, which takes no registers.)
  Run<TL, FORM> x[ROWS / 4];  // (codes: two words of it, and their scale)
  auto fetch = [&](int b) {
    int at = c4;
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int u = 0; u < ROWS / 4; ++u) {
      const int64_t row = row0 + min(4 * u + at, rows - 1);
      if constexpr (CODES) {
        __builtin_memcpy(x[u].u, p.codes + row * kp + b * 128 + 8 * r, 8);
        x[u].u[2] = p.scales[row * kbp + b];
      } else {
        x[u].load(static_cast<const TX*>(p.x) + row * p.ldx, b * 128 + 8 * r, p.K);
      }
    }
  };
  floatx4 acc[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
  char* buf = smem + w * BUF;
  // Workgroups begin at different blocks: with rows of some KB, the same ones of
  // all rows lie on few of the memory's channels (15001 rows x 4096 without an
  // adapter 58 -> 36 us).
  const int turn = (int)(group % ((kb + NW - 1) / NW)) * NW;
  auto block = [&](int i) { return i + turn < kb ? i + turn : i + turn - kb; };
  if (w < kb) fetch(block(w));
#pragma unroll 1
  for (int i = w; i < kb; i += NW) {
    const int b = block(i);
    int at = c4;
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int u = 0; u < ROWS / 4; ++u) {
      char* to = buf + (4 * u + c4) * PITCH + 8 * r * (int)sizeof(TL);
      if constexpr (CODES) {
        *reinterpret_cast<bf16x8*>(to) = fp8_to_bf16(x[u].u[0], x[u].u[1], fp8_scale((int)x[u].u[2]));
      } else {
        x[u].trim(b * 128 + 8 * r, p.K);
#pragma unroll
        for (int q = 0; q < x[u].N / 4; ++q)
          *reinterpret_cast<u32x4*>(to + 16 * q) = u32x4{x[u].u[4 * q], x[u].u[4 * q + 1], x[u].u[4 * q + 2], x[u].u[4 * q + 3]};
        if (p.q_codes) {
          const int s = fp8_scale_byte(block_max(x[u]));
          const u32x2 codes = fp8_pack8_scaled(x[u], fp8_scale(s));
          if (4 * u + at < rows) {
            const int64_t row = row0 + 4 * u + at;
            *reinterpret_cast<u32x2*>(p.q_codes + row * kp + b * 128 + 8 * r) = codes;
            if (r == 0) p.q_scales[row * kbp + b] = (uint8_t)s;
          }
        }
      }
    }
    if (i + NW < kb) fetch(block(i + NW));
    for (uint64_t todo = some; todo;) {
      const int d = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
      todo &= ~__ballot(mine == d);
      const uint16_t* a = p.a + (int64_t)d * p.rank * kp + 8 * lane;
      constexpr int AHEAD = RT <= 4 ? 2 : 1;
      bf16x8 fa[AHEAD][RT];
      auto fetch_a = [&](int st) {
#pragma unroll
        for (int j = 0; j < RT; ++j) fa[st % AHEAD][j] = *reinterpret_cast<const bf16x8*>(a + adapter_fragment(4 * b + st, j, 16 * RT));
      };
      fetch_a(0);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (AHEAD == 2 ? st < 3 : st > 0) fetch_a(st + AHEAD - 1);
        const char* from = buf + r % ROWS * PITCH + (32 * st + 8 * c4) * (int)sizeof(TL);
        u32x4 f[F32 ? 3 : 1];
        if constexpr (F32) {
          const floatx4 lo = *reinterpret_cast<const floatx4*>(from), hi = *reinterpret_cast<const floatx4*>(from + 16);
          uint32_t h, m, l;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v0 = e < 2 ? lo[2 * e] : hi[2 * e - 4], v1 = e < 2 ? lo[2 * e + 1] : hi[2 * e - 3];
            split_pair(mine == d ? v0 : 0.f, mine == d ? v1 : 0.f, h, m, l);
            f[0][e] = h;
            f[1][e] = m;
            f[2][e] = l;
          }
        } else {
          f[0] = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[0][e] = mine == d ? f[0][e] : 0;
        }
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int q = 0; q < (F32 ? 3 : 1); ++q) acc[j] = mma16(fa[st % AHEAD][j], __builtin_bit_cast(bf16x8, f[q]), acc[j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  if (!some) return;  // (nobody reads their t)
  __syncthreads();
  floatx4* red = reinterpret_cast<floatx4*>(smem);
#pragma unroll
  for (int j = 0; j < RT; ++j) red[(w * RT + j) * 64 + lane] = acc[j];
  __syncthreads();
  // lane: row r, ranks 16 j + 4 c4 + [0, 4)
  if (r >= rows) return;
  const int ext = p.parts * p.rank;
  const float s = mine >= 0 ? p.scale[mine] : 0.f;  // (of no adapter: the sums are 0)
  for (int j = w; j < RT; j += NW) {
    floatx4 v = red[j * 64 + lane];
#pragma unroll
    for (int i = 1; i < NW; ++i) v += red[(i * RT + j) * 64 + lane];
    uint16_t* t = p.t + (row0 + r) * ext + 16 * j + 4 * c4;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= s;
    uint32_t h[2], m[2], l[2];
    split_pair(v[0], v[1], h[0], m[0], l[0]);
    split_pair(v[2], v[3], h[1], m[1], l[1]);
    *reinterpret_cast<u32x2*>(t) = u32x2{h[0], h[1]};
    *reinterpret_cast<u32x2*>(t + p.rank) = u32x2{m[0], m[1]};
    if (p.parts == 3) *reinterpret_cast<u32x2*>(t + 2 * p.rank) = u32x2{l[0], l[1]};
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
  const int64_t f = adapter_fragment(col / 32, row / 16, rows_to) + (row % 16 + col % 32 / 8 * 16) * 8 + col % 8;
  to[FRAGMENTS ? f : at] = __builtin_bit_cast(uint16_t, v);
}

template <typename TX, int RT>
hipError_t go(const AdapterRows& p, hipStream_t s) {
  const bool few = p.rows <= 4 * device_cus();
  const unsigned grid = (unsigned)((p.rows + (few ? 31 : 127)) / (few ? 32 : 128) * 8);
  auto run = [&](auto form) {
    if (few) adapter_rows_kernel<TX, RT, decltype(form)::value, true><<<grid, 1024, 0, s>>>(p);
    else adapter_rows_kernel<TX, RT, decltype(form)::value, false><<<grid, 512, 0, s>>>(p);
  };
  const RowForm form = std::is_same_v<TX, uint8_t> ? kWhole : row_form(p.K);
  if (form == kWhole) run(std::integral_constant<RowForm, kWhole>());
  else if constexpr (!std::is_same_v<TX, uint8_t>) {
    if (form == kRagged) run(std::integral_constant<RowForm, kRagged>());
    else run(std::integral_constant<RowForm, kTiny>());
  }
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
      (p.parts != 2 && p.parts != 3) || (!p.x && (!p.codes || !p.scales || p.q_codes)) || !p.q_codes != !p.q_scales)
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
