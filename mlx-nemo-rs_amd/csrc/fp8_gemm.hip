// Products of e4m3 codes with a power of two for each block of 128
// (fp8_kernels.hpp has the format): y = (2^s_x q_x) (2^s_w q_w)^T.
//
// The scaled fp8 MFMA multiplies codes and applies both powers of two inside
// the instruction, so a chain over K needs no work between blocks. It adds
// products in groups of 8, in which it drops what lies under 2^-13 of the
// largest product's power of two: a sum is off by at most 7 * 2^-13 of its
// terms' magnitudes (measured: 1.4e-5 of the result in the 2-norm for normally
// distributed values, 5.5e-5 for codes spread over the whole exponent range,
// at any K; the running sum keeps its 24 bits). That is far under half a step
// of a bf16 result (2e-3 in the 2-norm) or of e4m3 codes. An f32 result, and
// the hidden values on the way to one, keep f32 sums: there the codes go to the
// bf16 matrix cores, which hold them and their products exactly (1e-7; only of
// activations' blocks under 2^-115 what lies below bf16's smallest number,
// 2^-133, is lost), at half the rate.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/relpos_mhsa.h"
#include "fp8_common.hpp"
#include "fp8_kernels.hpp"
#include "quant.hpp"

namespace mhsa {
namespace {

#include "gemm_tile.hpp"

// ---------------------------------------------------------------------------
// Rounding to codes
// ---------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* x, int64_t ldx, int64_t rows, int K,
                                                            uint8_t* codes, uint8_t* scales) {
  quantize_blocks(x, ldx, rows, K, codes, scales, (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6));
}

// One workgroup per 128 x 128 block of a weight matrix.
template <typename T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* w, int N, int K, uint8_t* codes,
                                                              uint8_t* scales) {
  const int kb = (K + 127) / 128, kbp = (kb + 3) / 4 * 4, nb = (N + 127) / 128;
  const int bk = blockIdx.x, bn = blockIdx.y;
  w += (int64_t)blockIdx.z * N * K;
  codes += (int64_t)blockIdx.z * N * (kb * 128);
  scales += (int64_t)blockIdx.z * nb * kbp;
  __shared__ float part[4];
  float v[64];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int at = i * 256 + threadIdx.x, n = bn * 128 + at / 128, k = bk * 128 + at % 128;
    v[i] = n < N && k < K ? (float)w[(int64_t)n * K + k] : 0.f;
    m = fmaxf(m, fp8_mag(v[i]));
  }
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const int s = fp8_scale_byte(m);
  const float scale = fp8_scale(s);
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int at = i * 256 + threadIdx.x, n = bn * 128 + at / 128, k = bk * 128 + at % 128;
    if (n < N) codes[(int64_t)n * (kb * 128) + k] = (uint8_t)fp8_pack4_scaled(v[i], 0.f, 0.f, 0.f, scale);
  }
  if (threadIdx.x == 0) scales[bn * kbp + bk] = (uint8_t)s;
}

// Codes [rows, K] <-> [rows, Kp] and scale bytes [blocks, kb] <-> [blocks,
// kbp], 16 codes of a padded row to a thread. A scale byte of 255 says that
// its block is not a number: the block's codes then say so.
__global__ __launch_bounds__(256) void pad_weight_kernel(const uint8_t* w, const uint8_t* ws, int64_t rows, int N,
                                                         int K, bool vec, uint8_t* codes, uint8_t* scales) {
  const int kb = (K + 127) / 128, kp = kb * 128, kbp = (kb + 3) / 4 * 4, nb = (N + 127) / 128;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at < rows * (kp / 16)) {
    const int64_t n = at / (kp / 16), blk = n / N * nb + n % N / 128;
    const int k = (int)(at % (kp / 16)) * 16;
    const bool nan = ws[blk * kb + k / 128] == 255;
    uint8_t v[16];
    if (vec && !nan) {
      *reinterpret_cast<u32x4*>(v) = *reinterpret_cast<const u32x4*>(w + n * K + k);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = k + i < K ? (nan ? 0x7F : w[n * K + k + i]) : 0;
    }
    *reinterpret_cast<u32x4*>(codes + n * kp + k) = *reinterpret_cast<const u32x4*>(v);
  }
  if (at < rows / N * nb * kbp) {
    const int64_t n = at / kbp;
    const int k = (int)(at % kbp);
    const uint8_t s = k < kb ? ws[n * kb + k] : 127;
    scales[at] = s == 255 ? 127 : s;
  }
}
__global__ __launch_bounds__(256) void unpad_weight_kernel(const uint8_t* codes, const uint8_t* scales, int64_t N,
                                                           int K, int64_t nb, uint8_t* w, uint8_t* ws) {
  const int kb = (K + 127) / 128, kp = kb * 128, kbp = (kb + 3) / 4 * 4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at < N * K) w[at] = codes[at / K * kp + at % K];
  if (at < nb * kb) ws[at] = scales[at / kb * kbp + at % kb];
}

// ---------------------------------------------------------------------------
// Few rows
//
// Weights are read once and everything else is small: a workgroup computes
// 16 RC output columns of up to 16 rows, its NW waves take every NW-th block
// of 128 inputs, and their sums are added in wave order at the end. One
// 16x16x128 MFMA covers a block: lane l holds 32 inputs, 32 (l / 16) on, of
// weight row l % 16 and of activation row l % 16. The activations are rounded
// to codes in these registers (the block's maximum is one over 4 lanes), so
// there is no other launch.
// ---------------------------------------------------------------------------

// Stores one value in the output's type.
__device__ __forceinline__ void store_as(DType dt, void* out, int64_t at, float v) {
  if (dt == kBF16) reinterpret_cast<bf16*>(out)[at] = (bf16)v;
  else reinterpret_cast<float*>(out)[at] = v;
}

// Adds block b's products of RC x 16 weight rows (at wrow + off; this lane's 32
// inputs) and the lane's activation row to acc. VEC: rows of whole
// runs of 8 inputs (the code for others is several times as long, and a launch
// of a few microseconds pays for fetching it).
template <typename TX, int RC, bool EXACT, bool VEC>
__device__ __forceinline__ void few_block(const uint8_t* wrow, const int off[RC], const uint8_t* wsc, int b, const TX* xrow,
                                          int K, floatx4 acc[RC]) {
  const int c0 = b * 128 + 32 * ((threadIdx.x & 63) >> 4);
  u32x4 wf[RC][2];
#pragma unroll
  for (int c = 0; c < RC; ++c)
#pragma unroll
    for (int u = 0; u < 2; ++u) wf[c][u] = *reinterpret_cast<const u32x4*>(wrow + off[c] + b * 128 + 16 * u);
  const int sw = wsc[b];
  float v[32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (VEC) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 * i + e] = 0.f;
      if (c0 + 8 * i < K) load_run(xrow + c0 + 8 * i, v + 8 * i);
    } else {
      load8(xrow, c0 + 8 * i, K, v + 8 * i);
    }
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = fmaxf(m, fp8_mag(v[i]));
  m = fmaxf(m, __shfl_xor(m, 16, 64));
  m = fmaxf(m, __shfl_xor(m, 32, 64));
  const int s = fp8_scale_byte(m);
  const float scale = fp8_scale(s);
  i32x8 q;
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = (int)fp8_pack4_scaled(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], scale);
#pragma unroll
  for (int c = 0; c < RC; ++c) {
    if constexpr (EXACT) {
      // element group j of every lane's 32: the same inputs of both operands
      floatx4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x4 wj = wf[c][j >> 1];
        part = mma16(fp8_to_bf16(wj[2 * (j & 1)], wj[2 * (j & 1) + 1]), fp8_to_bf16(q[2 * j], q[2 * j + 1]), part);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[c][e] += __builtin_ldexpf(part[e], s + sw - 254);
    } else {
      const i32x8 a = {(int)wf[c][0][0], (int)wf[c][0][1], (int)wf[c][0][2], (int)wf[c][0][3],
                       (int)wf[c][1][0], (int)wf[c][1][1], (int)wf[c][1][2], (int)wf[c][1][3]};
      acc[c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, acc[c], 0, 0, 0, sw, 0, s);
    }
  }
}

constexpr int kScanPairs = 1024, kScanExperts = 1024;

// The pairs of the `y`-th of the chosen experts, in order, in list; returns
// their number and the expert (0 if fewer are chosen). All threads call it.
struct ExpertPairs {
  int list[kScanPairs], idx[kScanPairs];
  uint32_t used[kScanExperts / 32];
  int expert, count;
};
__device__ __forceinline__ void find_pairs(const int* idx, int pairs, int experts, int y, ExpertPairs& f) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < kScanExperts / 32) f.used[threadIdx.x] = 0;
  if (threadIdx.x == 0) f.count = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    const int e = idx[i];
    f.idx[i] = e;
    if (e >= 0 && e < experts) atomicOr(&f.used[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  // lane's 16 experts; how many are used before them
  const uint32_t mine = f.used[lane >> 1] >> (16 * (lane & 1)) & 0xFFFFu;
  int before = 0;
  for (int o = 1; o < 64; o *= 2) {
    const int n = __popc(mine) + before, t = __shfl_up(n, o, 64);
    before += lane >= o ? t : 0;
  }
  const int r = y - before;
  const uint64_t has = __ballot(r >= 0 && r < __popc(mine));
  int e = -1, n = 0;
  if (has) {
    uint32_t m = mine;
    for (int i = 0; i < min(r, 16); ++i) m &= m - 1;
    e = __shfl(16 * lane + __builtin_ctz(m | 0x10000u), __builtin_ctzll(has), 64);
    for (int i = 0; i < pairs; i += 64) {
      const bool same = i + lane < pairs && f.idx[i + lane] == e;
      const uint64_t mask = __ballot(same);
      if (same) f.list[n + __popcll(mask & (((uint64_t)1 << lane) - 1))] = i + lane;
      n += __popcll(mask);
    }
  }
  if (lane == 0) {
    f.expert = e;
    f.count = n;
  }
}

// The place of the n-th set bit of m, which has more than n.
__device__ __forceinline__ int nth_bit(uint64_t m, int n) {
  int at = 0;
#pragma unroll
  for (int w = 32; w; w /= 2) {
    const int c = __popcll(m >> at & (((uint64_t)1 << w) - 1));
    at += n >= c ? w : 0;
    n -= n >= c ? c : 0;
  }
  return at;
}

template <typename TX, int NW, int RC, bool EXACT, bool VEC>
__global__ __launch_bounds__(NW * 64) void fp8_few_kernel(Fp8Gemm p) {
  __shared__ float red[NW][RC][16][20];
  __shared__ int dst[16];
  __shared__ ExpertPairs found;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, c4 = lane >> 4;
  const int n0 = blockIdx.x * 16 * RC;
  int expert = 0, rows = p.M - blockIdx.y * 16;
  // Up to 256 pairs of up to 64 experts, four to a lane: those of the expert that
  // is the y-th of the chosen ones, found by every wave for itself. (Through LDS,
  // with two barriers and one wave's work between, the scan of 224 pairs took 3.8
  // of 18.8 us.) The experts of up to 16 pairs, or of 64 where there are more
  // experts, are gone through one by one (a frame's two: 7.0 us instead of 7.6).
  constexpr int Q = 4;
  uint64_t same[Q] = {};
  const bool masks = p.g.pairs > 16 && p.g.pairs <= 64 * Q && p.g.experts <= 64;
  const bool lanes = !p.g.tile && p.g.idx && (masks || p.g.pairs <= 64);
  if (lanes && !masks) {
    int mine = lane < p.g.pairs ? p.g.idx[lane] : -1;
    if (mine >= p.g.experts) mine = -1;
    uint64_t todo = __ballot(mine >= 0);
    for (int y = blockIdx.y;; --y) {
      if (!todo) return;
      expert = __shfl(mine, __builtin_ctzll(todo), 64);
      same[0] = __ballot(mine == expert);
      if (y == 0) break;
      todo &= ~same[0];
    }
    rows = __popcll(same[0]);
  } else if (lanes) {
    int mine[Q];
    uint32_t used[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      mine[i] = 64 * i + lane < p.g.pairs ? p.g.idx[64 * i + lane] : -1;
      const bool one = mine[i] >= 0 && mine[i] < p.g.experts;
      used[0] |= one && mine[i] < 32 ? 1u << mine[i] : 0;
      used[1] |= one && mine[i] >= 32 ? 1u << (mine[i] - 32) : 0;
    }
    auto either = [](uint32_t a, uint32_t b) { return a | b; };
    const uint64_t all = (uint64_t)wave_reduce(used[1], either) << 32 | wave_reduce(used[0], either);
    if ((int)blockIdx.y >= __popcll(all)) return;
    expert = nth_bit(all, blockIdx.y);
    rows = 0;
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      same[i] = __ballot(mine[i] == expert);
      rows += __popcll(same[i]);
    }
  } else if (p.g.tile) {
    if ((int)blockIdx.y >= *p.g.n_tiles) return;
    expert = p.g.tile[4 * blockIdx.y];
    rows = p.g.tile[4 * blockIdx.y + 2];
  } else if (p.g.idx) {
    find_pairs(p.g.idx, p.g.pairs, p.g.experts, blockIdx.y, found);
    __syncthreads();
    if (found.count == 0) return;
    expert = found.expert;
    rows = found.count;
  }
  const int kb = (p.K + 127) / 128, kbp = (kb + 3) / 4 * 4;
  const uint8_t* wrow = p.w + expert * p.w_stride + 32 * c4;
  int off[RC];  // (a matrix's codes are under 2 GiB; rows past the last repeat it, and their columns are not stored)
#pragma unroll
  for (int c = 0; c < RC; ++c) off[c] = min(n0 + 16 * c + r, p.N - 1) * (kb * 128);
  const uint8_t* wsc = p.ws + expert * p.ws_stride + (int64_t)(n0 / 128) * kbp;
  for (int first = 0; first < rows; first += 16) {  // (one pass but for an expert of many pairs)
    // row r: its output row and its source row
    int to = -1;
    if (first + r < rows) {
      if (p.g.tile) to = p.g.pair[p.g.tile[4 * blockIdx.y + 1] + r];
      else if (lanes) {
        int n = first + r, base = 0;
        uint64_t in = same[0];
#pragma unroll
        for (int i = 1; i < Q; ++i) {
          const int c = __popcll(in);
          if (base == 64 * (i - 1) && n >= c) {
            n -= c;
            base = 64 * i;
            in = same[i];
          }
        }
        to = base + nth_bit(in, n);
      }
      else if (p.g.idx) to = found.list[first + r];
      else to = blockIdx.y * 16 + r;
    }
    const int src = p.rows == Fp8Gemm::kByFrame ? to / p.g.top_k : to;
    if (threadIdx.x < 16) dst[r] = to;
    const TX* xrow = reinterpret_cast<const TX*>(p.x) + (int64_t)(to >= 0 ? src : 0) * p.ldx;
    const int K = to >= 0 ? p.K : 0;
    floatx4 acc[RC];
#pragma unroll
    for (int c = 0; c < RC; ++c) acc[c] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int b = w; b < kb; b += NW) few_block<TX, RC, EXACT, VEC>(wrow, off, wsc, b, xrow, K, acc);
    // lane: row l % 16, columns 16 c + 4 (l / 16) + [0, 4)
#pragma unroll
    for (int c = 0; c < RC; ++c) *reinterpret_cast<floatx4*>(&red[w][c][r][4 * c4]) = acc[c];
    __syncthreads();
    for (int t = threadIdx.x; t < RC * 256; t += NW * 64) {
      const int c = t >> 8, row = t >> 4 & 15, e = t & 15, n = n0 + 16 * c + e, out = dst[row];
      if (out < 0 || n >= p.N) continue;
      float v = red[0][c][row][e];
#pragma unroll
      for (int i = 1; i < NW; ++i) v += red[i][c][row][e];
      v += p.bias[(int64_t)expert * p.N + n];
      if (p.epilogue == kFp8HiddenF32) v = silu_value<float>(v);
      store_as(p.epilogue == kFp8Out ? p.out_dt : kF32, p.out, (int64_t)out * p.ldo + n, v);
    }
    if (p.g.tile || !p.g.idx) break;
    __syncthreads();
  }
}

// The second product of up to 16 pairs and their weighted sum in one: a
// workgroup's 16 waves share out the chosen experts and, for each, the blocks
// of inputs, and 16 columns of every frame are summed at the end, in the order
// of the choices. A wave's first weights are on their way while the workgroup
// rounds the hidden rows to codes in LDS.
constexpr int kSumLds = 64 * 1024;
template <typename TOut, bool EXACT>
__global__ __launch_bounds__(1024) void fp8_few_sum_kernel(Fp8Gemm p, const float* weights, const TOut* residual,
                                                           float res_scale) {
  __shared__ __attribute__((aligned(16))) uint8_t codes[kSumLds];
  __shared__ uint8_t scales[kSumLds / 128];
  __shared__ float red[16][16][20];
  __shared__ int at[16];  // pair: 16 * its expert's place + its place among the expert's pairs, or -1
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, c4 = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int kb = (p.K + 127) / 128, kbp = (kb + 3) / 4 * 4, pitch = kb * 128 + 16;
  // every wave finds the distinct experts by itself: one pair to a lane
  int mine = lane < p.g.pairs ? p.g.idx[lane] : -1;
  if (mine >= p.g.experts) mine = -1;
  const uint64_t valid = __ballot(mine >= 0);
  int groups = 0, place = -1;
  for (uint64_t todo = valid; todo; ++groups) {
    const uint64_t same = __ballot(mine == __shfl(mine, __builtin_ctzll(todo), 64));
    if (same >> lane & 1) place = 16 * groups + __popcll(same & (((uint64_t)1 << lane) - 1));
    todo &= ~same;
  }
  if (w == 0 && lane < 16) at[lane] = place;
  int share = 16;  // waves to an expert
  while (share * groups > 16) share /= 2;
  const int g = w / share, b0 = w % share;
  const int expert = g < groups ? __shfl(mine, __builtin_ctzll(__ballot(place == 16 * g)), 64) : 0;
  const uint8_t* wrow = p.w + expert * p.w_stride + (int64_t)min(n0 + r, p.N - 1) * (kb * 128) + 32 * c4;
  const uint8_t* wsc = p.ws + expert * p.ws_stride + (int64_t)(n0 / 128) * kbp;
  constexpr int D = 4;
  u32x4 wf[D][2];
  int sw[D];
  auto fetch = [&](int b, int d) {
#pragma unroll
    for (int u = 0; u < 2; ++u) wf[d][u] = *reinterpret_cast<const u32x4*>(wrow + b * 128 + 16 * u);
    sw[d] = wsc[b];
  };
  if (g < groups) {
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (b0 + d * share < kb) fetch(b0 + d * share, d);
  }
  // 16 lanes round a block of a pair's hidden row
  for (int i = threadIdx.x >> 4; i < p.g.pairs * kb; i += 64) {
    const int pr = i / kb, blk = i % kb, c = blk * 128 + 8 * (lane & 15);
    float v[8] = {};
    if (c < p.K) {
      const float* x = reinterpret_cast<const float*>(p.x) + (int64_t)pr * p.ldx + c;
#pragma unroll
      for (int u = 0; u < 2; ++u) *reinterpret_cast<floatx4*>(v + 4 * u) = *reinterpret_cast<const floatx4*>(x + 4 * u);
    }
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fp8_mag(v[e]));
#pragma unroll
    for (int o = 1; o < 16; o *= 2) m = fmaxf(m, __shfl_xor(m, o, 64));
    const int s = fp8_scale_byte(m);
    const float scale = fp8_scale(s);
    *reinterpret_cast<u32x2*>(codes + pr * pitch + c) =
        u32x2{fp8_pack4_scaled(v[0], v[1], v[2], v[3], scale), fp8_pack4_scaled(v[4], v[5], v[6], v[7], scale)};
    if ((lane & 15) == 0) scales[pr * kb + blk] = (uint8_t)s;
  }
  __syncthreads();
  if (g < groups) {
    // row r: the expert's r-th pair
    int to = -1;
    for (int i = 0; i < p.g.pairs; ++i)
      if (at[i] == 16 * g + r) to = i;
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](int b, int d) {
      u32x4 x0 = {}, x1 = {};
      int s = 127;
      if (to >= 0) {
        x0 = *reinterpret_cast<const u32x4*>(codes + to * pitch + b * 128 + 32 * c4);
        x1 = *reinterpret_cast<const u32x4*>(codes + to * pitch + b * 128 + 32 * c4 + 16);
        s = scales[to * kb + b];
      }
      if constexpr (EXACT) {
        floatx4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 wj = wf[d][j >> 1], xj = j < 2 ? x0 : x1;
          part = mma16(fp8_to_bf16(wj[2 * (j & 1)], wj[2 * (j & 1) + 1]), fp8_to_bf16(xj[2 * (j & 1)], xj[2 * (j & 1) + 1]),
                       part);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __builtin_ldexpf(part[e], s + sw[d] - 254);
      } else {
        const i32x8 a = {(int)wf[d][0][0], (int)wf[d][0][1], (int)wf[d][0][2], (int)wf[d][0][3],
                         (int)wf[d][1][0], (int)wf[d][1][1], (int)wf[d][1][2], (int)wf[d][1][3]};
        const i32x8 q = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, acc, 0, 0, 0, sw[d], 0, s);
      }
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (b0 + d * share < kb) add(b0 + d * share, d);
#pragma unroll 1
    for (int b = b0 + D * share; b < kb; b += share) {
      fetch(b, 0);
      add(b, 0);
    }
    *reinterpret_cast<floatx4*>(&red[w][r][4 * c4]) = acc;
  }
  __syncthreads();
  const int rows = p.g.pairs / p.g.top_k, row = threadIdx.x >> 4, e = threadIdx.x & 15, n = n0 + e;
  if (row >= rows || n >= p.N) return;
  float sum = 0.f;
  for (int j = 0; j < p.g.top_k; ++j) {
    const int q = row * p.g.top_k + j, a = at[q];
    if (a < 0) continue;
    float v = 0.f;
    for (int i = 0; i < share; ++i) v += red[(a >> 4) * share + i][a & 15][e];
    v += p.bias[(int64_t)p.g.idx[q] * p.N + n];
    sum = __builtin_fmaf(weights[q], v, sum);
  }
  sum *= res_scale;
  const int64_t o = (int64_t)row * p.N + n;
  if (residual) sum += (float)residual[o];
  reinterpret_cast<TOut*>(p.out)[o] = (TOut)sum;
}

// ---------------------------------------------------------------------------
// Tiles
//
// A workgroup of 4 waves (2 x 2) computes a BM x BN tile from a ring of NS LDS
// stages of 128 inputs, one block: rows of 128 bytes whose eight 16-byte
// chunks are stored XOR-permuted by (row / 2) % 8 (the 16 rows that a fragment
// read takes at a time then lie on all 64 banks), filled by direct-to-LDS
// loads of whole 128-byte lines. A 32x32x64 MFMA takes 32 bytes of each
// operand from a lane; the weight is its first operand, so a lane's
// accumulators hold four consecutive output columns of one row. A stage is two
// halves of 64 inputs. A half's fragments are read into registers between the
// MFMAs of the half before, so all of a stage has been read when its second
// half begins: there is the stage's one barrier, behind which the loads that
// refill its buffer are issued. Row scales come with the stages, 4 stages to a
// word; the weight's scale is one byte per wave and stage, read from a lane of
// a register that holds all of them.
//
// Workgroups stay and take tile after tile. A large tile has its CU to itself
// and LDS for staging its results beside the ring, so the ring runs on from
// tile to tile: the last stages' loads are the next tile's first, whose place
// in the list and rows were looked up a tile ahead (waiting for the list, the
// rows and the first lines took 3.7 us a tile). Small tiles share a CU, whose
// other workgroup computes meanwhile.
// ---------------------------------------------------------------------------

template <int BM, int BN, int NS_>
struct Fp8Cfg {
  static constexpr int NS = NS_;
  static constexpr int WM = BM / 2, WN = BN / 2, TM = WM / 32, TN = WN / 32;
  static constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
  static constexpr int NA = BM / 32, NB = BN / 32;  // 1 KB loads per wave and stage
  static constexpr int SCALES = NS * STAGE;         // a word a row (or 256 bytes) of every stage, behind the stages
  static constexpr int LOOP = SCALES + NS * BM * 4;
  // results are staged 32 rows of 128 bytes at a time and wave; behind them a
  // wave keeps its columns' bias and its rows' places
  static constexpr int OP = 128 + 16, WST = 32 * OP + 4 * (WN + WM), STG = 4 * WST, AMAX = 2 * BM * 4;
  static constexpr bool AHEAD = BM >= 192;  // staging beside the ring, else over it
  static constexpr int OUT = AHEAD ? LOOP : 0;
  static constexpr int LDS = AHEAD ? LOOP + STG : LOOP > STG + AMAX ? LOOP : STG + AMAX;
  static_assert(LDS <= 160 * 1024, "tile exceeds LDS");
  static_assert(BM >= 64 && BM <= 256 && (!AHEAD || NS == 2), "scales, stages");
};

template <int BM, int BN, int NS, bool EXACT, int EPI, typename TOut>
__device__ __forceinline__ void fp8_tile_body(const Fp8Gemm& p, char* smem) {
  using C = Fp8Cfg<BM, BN, NS>;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w >> 1, wn = w & 1;
  const int kb = (p.K + 127) / 128, kp = kb * 128, kbp = (kb + 3) / 4 * 4;

  // contiguous tile ranges per XCD, walked 8 row tiles at a time
  const bool grouped = p.g.tile != nullptr;
  const int tilesM = grouped ? *p.g.n_tiles : (p.M + BM - 1) / BM, tilesN = (p.N + BN - 1) / BN;
  const int nt = tilesM * tilesN, per = (nt + 7) / 8;
  const int T0 = (int)(blockIdx.x % 8u) * per, T1 = min(T0 + per, nt);
  int T = T0 + (int)(blockIdx.x / 8u);
  if (T >= T1) return;
  struct Tile {
    int expert, m0, rows, n0;
  };
  struct Place {  // of a tile: its row tile (of the list, if there is one) and its first column
    int tm, n0;
  };
  auto place_of = [&](int t) -> Place {
    constexpr int GM = 8;
    const int gsz = GM * tilesN, first = t / gsz * GM, gm = min(tilesM - first, GM);
    return {first + (t % gsz) % gm, (t % gsz) / gm * BN};
  };
  struct Entry {
    int expert, m0, rows;
  };
  auto entry_of = [&](int tm) -> Entry {
    if (!grouped) return {0, tm * BM, min(p.M - tm * BM, BM)};
    return {p.g.tile[4 * tm], p.g.tile[4 * tm + 1], p.g.tile[4 * tm + 2]};
  };
  auto tile_of = [&](const Entry& e, int n0) -> Tile {
    return {__builtin_amdgcn_readfirstlane(e.expert), __builtin_amdgcn_readfirstlane(e.m0),
            __builtin_amdgcn_readfirstlane(e.rows), n0};
  };

  // activations: a tile's rows, or gathered ones (rows past the tile's repeat
  // its last; their results are not stored). Row scales: a word of 4 blocks
  // to a row, or (HT) by block, bytes of consecutive slots.
  constexpr bool HT = EPI == kFp8Pair;
  const bool gather = grouped && p.rows == Fp8Gemm::kByFrame;
  __amdgpu_buffer_rsrc_t ra, rs, rb;
  int aoff[C::NA], boff[C::NB], soff;
  uint32_t wword = 0;
  const int srow = (w * 64) % BM;
#pragma unroll
  for (int g = 0; g < C::NB; ++g) {  // load g of wave w fills 8 LDS rows: lane l row l / 8, stored chunk l % 8
    const int row = (w * C::NB + g) * 8 + (lane >> 3);
    boff[g] = row * kp + 16 * ((lane & 7) ^ ((row >> 1) & 7));
  }
  auto rsrc = [](const uint8_t* base, uint32_t n) {
    // (uniform by its making, which the compiler loses over the tile loop)
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint64_t u = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32 |
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(u), (short)0, __builtin_amdgcn_readfirstlane((int)n),
                                             kRawBuffer);
  };
  // source rows of this lane's loads of tile t
  int src[C::NA + 1];
  auto look_up = [&](const Tile& t) {
    auto source = [&](int row) { return gather ? p.g.frame[t.m0 + min(row, t.rows - 1)] : min(row, t.rows - 1); };
#pragma unroll
    for (int g = 0; g < C::NA; ++g) src[g] = source((w * C::NA + g) * 8 + (lane >> 3));
    src[C::NA] = HT ? 0 : source(srow + lane);
  };
  auto aim = [&](const Tile& t) {  // the loads below are tile t's, looked up before
    const int64_t arows = gather ? p.a_rows : t.rows;
    ra = rsrc(p.a + (gather ? 0 : (int64_t)t.m0 * kp), (uint32_t)(arows * kp));
    rs = rsrc(HT ? p.as + t.m0 : p.as + (gather ? 0 : (int64_t)t.m0 * kbp), (uint32_t)(HT ? kb * p.slots - t.m0 : arows * kbp));
#pragma unroll
    for (int g = 0; g < C::NA; ++g) {
      const int row = (w * C::NA + g) * 8 + (lane >> 3);
      aoff[g] = (int)((uint32_t)src[g] * (uint32_t)kp + 16 * ((lane & 7) ^ ((row >> 1) & 7)));
    }
    soff = HT ? 4 * lane : (int)((uint32_t)src[C::NA] * (uint32_t)kbp);
    rb = rsrc(p.w + t.expert * p.w_stride + (int64_t)t.n0 * kp, (uint32_t)(min(p.N - t.n0, BN) * kp));
  };
  // the weight scales of this wave's 128-column block, a word of 4 to a lane
  auto weight_scales = [&](const Tile& t) {
    const int blk = min((t.n0 + wn * C::WN) / 128, (p.N + 127) / 128 - 1);
    return *reinterpret_cast<const uint32_t*>(p.ws + t.expert * p.ws_stride + (int64_t)blk * kbp + 4 * min(lane, kbp / 4 - 1));
  };
  constexpr int LOADS = C::NA + C::NB + 1;
  auto issue1 = [&](int g, int k, int buf) {  // load g of the aimed tile's stage k
    char* S = smem + buf * C::STAGE;
    if (g < C::NA)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void*)(S + (w * C::NA + g) * 1024), 16, aoff[g], k * 128, 0, 0);
    else if (g < C::NA + C::NB)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void*)(S + C::ABYTES + (w * C::NB + g - C::NA) * 1024), 16,
                                               boff[g - C::NA], k * 128, 0, 0);
    else if (HT)  // 256 rows' bytes, the same by every wave; past the slots: 0
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(smem + C::SCALES + buf * BM * 4), 4, soff,
                                               (int)(k * p.slots), 0, 0);
    else  // 64 rows' words, twice the same in a tile of under 256 rows
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(smem + C::SCALES + buf * BM * 4 + srow * 4), 4, soff, k & ~3, 0,
                                               0);
  };
  // everywhere: all but the last `n` memory operations issued are done, LDS reads are
  auto settled = [&](auto n) {
    constexpr int vm = decltype(n)::value;
    static_assert(vm < 64, "wait count");
    __builtin_amdgcn_s_waitcnt((vm & 15) | ((vm >> 4) << 14) | (7 << 4));  // lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
  };

  const int arow = (wm * C::WM + (lane & 31)) * 128;
  const int brow = C::ABYTES + (wn * C::WN + (lane & 31)) * 128;
  int off[2][2];  // this lane's two chunks of a row in either half
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int u = 0; u < 2; ++u) off[h][u] = 16 * ((4 * h + 2 * half + u) ^ ((lane >> 1) & 7));
  u32x4 fa[2][C::TM][2], fb[2][C::TN][2];
  int xw[C::TM];
  // read r of half h of the stage in buffer buf into set h: its fragments (the
  // weight's first, then the rows'), then the row scales
  constexpr int FRAGS = 2 * (C::TM + C::TN);
  auto rd1 = [&](int r, int buf, int h) {
    const char* S = smem + buf * C::STAGE;
    if (r < 2 * C::TN) {
      fb[h][r / 2][r % 2] = *reinterpret_cast<const u32x4*>(S + brow + off[h][r % 2] + r / 2 * 4096);
    } else if (r < FRAGS) {
      r -= 2 * C::TN;
      fa[h][r / 2][r % 2] = *reinterpret_cast<const u32x4*>(S + arow + off[h][r % 2] + r / 2 * 4096);
    } else if (HT) {
      xw[r - FRAGS] = *reinterpret_cast<const uint8_t*>(smem + C::SCALES + buf * BM * 4 + wm * C::WM + 32 * (r - FRAGS) +
                                                        (lane & 31));
    } else {
      xw[r - FRAGS] =
          *reinterpret_cast<const int*>(smem + C::SCALES + buf * BM * 4 + (wm * C::WM + 32 * (r - FRAGS) + (lane & 31)) * 4);
    }
  };
  floatx16 acc[C::TN][C::TM];

  int ws = 0, xs[C::TM];
  // Half h of stage kt, whose fragments are in set h and whose buffer is buf.
  // The reads of the next half's fragments and, behind the second half's
  // barrier, the loads that refill the buffer (stage `refill` of the aimed
  // tile) are placed between the MFMAs: issued ahead of
  // them, the reads filled the wave's queue of 15 and held the first MFMA
  // back.
  auto step = [&](int kt, int buf, int refill, auto hc) {
    constexpr int h = decltype(hc)::value;
    if constexpr (h == 0) {
      const int sh = 8 * (kt & 3);
      ws = __builtin_amdgcn_readlane((int)wword, kt >> 2) >> sh;
#pragma unroll
      for (int i = 0; i < C::TM; ++i) xs[i] = HT ? xw[i] : xw[i] >> sh;
      if constexpr (EXACT) {
        // Codes times powers of two that bf16 holds: of the weight's power what
        // lies past 2^-100 and 2^100 goes over to the rows' (from 2^120 on the
        // largest codes would pass bf16's range). What the rows then lose or
        // pass belongs to products that f32 does not hold either; below
        // infinity, so that with codes of zero these stay zero.
        const int wb = ws & 255, in = min(max(wb, 27), 227), more = wb - in;
        ws = in;
#pragma unroll
        for (int i = 0; i < C::TM; ++i) xs[i] = min(max((xs[i] & 255) + more, 0), more > 0 ? 246 : 255);
      }
    }
    const int other = buf + 1 == NS ? 0 : buf + 1;
    __builtin_amdgcn_sched_barrier(0);
    constexpr int NMF = EXACT ? 4 * C::TM * C::TN : C::TM * C::TN;
    constexpr int READS = FRAGS + (h == 1 ? C::TM : 0);
    constexpr int SLOTS = (NMF + 1) / 2;  // behind the first MFMAs the reads, behind all the loads
    constexpr int RPM = (READS + SLOTS - 1) / SLOTS;
    auto between = [&](int m) {
      if constexpr (h == 1) {
#pragma unroll
        for (int g = 0; g < LOADS; ++g)
          if (g * NMF / LOADS == m) issue1(g, refill, buf);
      }
#pragma unroll
      for (int r = m * RPM; r < (m + 1) * RPM; ++r)
        if (r < READS) rd1(r, h == 0 ? buf : other, h ^ 1);
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (!EXACT) {
#pragma unroll
      for (int m = 0; m < NMF; ++m) {
        const int j = m / C::TM, i = m % C::TM;
        auto whole = [](const u32x4* f) {
          return i32x8{(int)f[0][0], (int)f[0][1], (int)f[0][2], (int)f[0][3],
                       (int)f[1][0], (int)f[1][1], (int)f[1][2], (int)f[1][3]};
        };
        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(whole(fb[h][j]), whole(fa[h][i]), acc[j][i], 0, 0, 0,
                                                                    ws, 0, xs[i]);
        between(m);
      }
    } else {
      // Exact products and f32 sums on the bf16 cores. bf16 has f32's range, so
      // the powers of two go into the conversion of the codes.
      const float wf = fp8_scale(ws);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        bf16x8 xa[C::TM], xb[C::TN];
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
          xa[i] = fp8_to_bf16(fa[h][i][u >> 1][2 * (u & 1)], fa[h][i][u >> 1][2 * (u & 1) + 1], fp8_scale(xs[i]));
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
          xb[j] = fp8_to_bf16(fb[h][j][u >> 1][2 * (u & 1)], fb[h][j][u >> 1][2 * (u & 1) + 1], wf);
#pragma unroll
        for (int m = 0; m < C::TM * C::TN; ++m) {
          const int j = m / C::TM, i = m % C::TM;
          acc[j][i] = mma32(xb[j], xa[i], acc[j][i]);
          between(u * C::TM * C::TN + m);
        }
      }
    }
  };
  constexpr auto H0 = std::integral_constant<int, 0>{};
  constexpr auto H1 = std::integral_constant<int, 1>{};
  auto prologue = [&]() {  // the aimed tile's first NS stages
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int g = 0; g < LOADS; ++g) issue1(g, min(st, kb - 1), st);
    settled(std::integral_constant<int, (NS - 1) * LOADS>{});
  };
  // The columns' bias and the rows' places that a tile's epilogue needs, a
  // register each, then LDS (held in registers for all of the lane's columns
  // and rows, they spilled).
  constexpr int BL = (C::WN + 63) / 64, PL = EPI == kFp8Pair ? (C::WM + 63) / 64 : 0;
  float bl[BL];
  int pl[PL ? PL : 1];
  auto columns = [&](const Tile& t) {
#pragma unroll
    for (int u = 0; u < BL; ++u) {
      const int c = t.n0 + wn * C::WN + 64 * u + lane;
      bl[u] = EPI == kFp8HiddenQ && c >= p.N ? 0.f : p.bias[(int64_t)t.expert * p.N + c];
    }
#pragma unroll
    for (int u = 0; u < PL; ++u) pl[u] = p.g.pair[t.m0 + min(wm * C::WM + 64 * u + lane, t.rows - 1)];
  };

  const int stride = (int)(gridDim.x / 8u);
  Place where = place_of(T);
  Tile now = tile_of(entry_of(where.tm), where.n0), next = now;
  look_up(now);
  aim(now);
  wword = weight_scales(now);
  uint32_t wnext = 0;
  Entry after = {0, 0, 0};  // the list's entry of the tile after the next
  int after_n0 = 0, base = 0;
  // What is looked up ahead of tile T's loop, the ring's loads of which are
  // on their way: the next tile's rows and scales, the entry of the one after
  // it, and what this one's epilogue needs.
  auto look_ahead = [&]() {
    if (T + stride < T1) {
      look_up(next);
      wnext = weight_scales(next);
    }
    if (T + 2 * stride < T1) {
      const Place q = place_of(T + 2 * stride);
      after = entry_of(q.tm);
      after_n0 = q.n0;
    }
    columns(now);
  };
  if constexpr (C::AHEAD) {
    if (T + stride < T1) {
      where = place_of(T + stride);
      next = tile_of(entry_of(where.tm), where.n0);
    }
  }
  prologue();
  if constexpr (C::AHEAD) look_ahead();
  bool stored = false;  // the last epilogue's stores, a known number, are behind the ring's loads
  for (;;) {
#pragma unroll
    for (int j = 0; j < C::TN; ++j)
#pragma unroll
      for (int i = 0; i < C::TM; ++i) acc[j][i] = floatx16{};
    // (a tile's last step read these too, but held over the epilogue they spilled)
#pragma unroll
    for (int r = 0; r < FRAGS + C::TM; ++r) rd1(r, C::AHEAD ? base & 1 : 0, 0);
    const bool more = T + stride < T1;
    constexpr int STORES = C::TM * (C::WN / 32 + 1);
    if constexpr (C::AHEAD) {
      auto stage = [&](int kt, int refill) {
        const int buf = (base + kt) & 1;
        step(kt, buf, 0, H0);
        if (EPI == kFp8HiddenQ && kt == 0 && stored) settled(std::integral_constant<int, STORES>{});
        else settled(H0);
        step(kt, buf, refill, H1);
      };
      int kt = 0;
      for (; kt < kb - NS; ++kt) stage(kt, kt + NS);
      if (more) aim(next);
      for (; kt < kb; ++kt) stage(kt, more ? kt + NS - kb : kb - 1);  // (at the end: unread)
      base += kb;
    } else {
      for (int kt = 0; kt < kb; ++kt) {
        const int buf = kt % NS;
        step(kt, buf, 0, H0);
        settled(std::integral_constant<int, (NS - 2) * LOADS>{});
        step(kt, buf, min(kt + NS, kb - 1), H1);  // (past the end: the last stage again, unread)
      }
      columns(now);
      // the loads past the end still write LDS: all of them are to have landed
      // before it is used again
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }

    const Tile done = now;
    // Lane: row 32 i + lane % 32 of the wave's block, columns 32 j + 8 q +
    // 4 (lane / 32) + [0, 4).
    const int col0 = done.n0 + wn * C::WN;
    char* st = smem + C::OUT + w * C::WST;
    float* bias = reinterpret_cast<float*>(st + 32 * C::OP);
    int* place = reinterpret_cast<int*>(bias + C::WN);
#pragma unroll
    for (int u = 0; u < BL; ++u)
      if (64 * u + lane < C::WN) bias[64 * u + lane] = bl[u];
#pragma unroll
    for (int u = 0; u < PL; ++u)
      if (64 * u + lane < C::WM) place[64 * u + lane] = pl[u];
    // (keeps the sums of rows 32 i of the block in their accumulators up to
    // here: read ahead, all of them, they spilled)
    auto hold = [&](int i) {
#pragma unroll
      for (int j = 0; j < C::TN; ++j) asm volatile("" : "+a"(acc[j][i]));
    };
    auto bias4 = [&](int j, int q) { return *reinterpret_cast<const floatx4*>(bias + 32 * j + 8 * q + 4 * half); };
    T += stride;
    if (C::AHEAD && more) {
      // (ahead of the stores, which the ring's next wait leaves behind)
      now = next;
      wword = wnext;
      if (T + stride < T1) next = tile_of(after, after_n0);
      look_ahead();
      asm volatile("" ::: "memory");
      stored = true;
    }

    if constexpr (EPI == kFp8HiddenQ) {
      // silu, then codes: the block's 128 columns of a row lie in one wave
      // (both lane halves) or in the two of a row of waves
      float* amax = reinterpret_cast<float*>(smem + C::STG);
      const int np = (p.N + 127) / 128 * 128;
      constexpr int HP = C::WN + 16;
      const __amdgpu_buffer_rsrc_t rc = rsrc(p.out_codes + (int64_t)done.m0 * np, (uint32_t)(done.rows * np));
      const __amdgpu_buffer_rsrc_t rh =
          rsrc(p.out_scales + min(col0 / 128, np / 128 - 1) * p.slots + done.m0, (uint32_t)done.rows);
      // (32 rows at a time, with nothing of the next ones moved ahead: 256
      // accumulators and as many results at once spilled)
      auto hidden = [&](int i, float v[C::TN * 16]) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx4 b = bias4(j, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[16 * j + 4 * q + e] = silu_value<float>(acc[j][i][4 * q + e] + b[e]);
              top = fmaxf(top, __builtin_fabsf(v[16 * j + 4 * q + e]));
            }
          }
        if (__any(!(top < __builtin_inff()))) {  // an infinity does not count (a NaN never did): again, without
          top = 0.f;
          for (int r = 0; r < C::TN * 16; ++r) top = fmaxf(top, fp8_mag(v[r]));
        }
        return fmaxf(top, __shfl_xor(top, 32, 64));
      };
      auto store = [&](int i, const float v[C::TN * 16], float top) {
        const int s = fp8_scale_byte(top);
        const float scale = fp8_scale(s);
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* f = v + 16 * j + 4 * q;
            *reinterpret_cast<uint32_t*>(st + (lane & 31) * HP + 32 * j + 8 * q + 4 * half) =
                fp8_pack4_scaled(f[0], f[1], f[2], f[3], scale);
          }
        const int row0 = wm * C::WM + 32 * i;
        // (rows and columns that are not the tile's lie past the buffers' ends:
        // every store is issued, so that their number is known)
#pragma unroll
        for (int it = 0; it < C::WN / 32; ++it) {
          const int id = it * 64 + lane, r = id / (C::WN / 16), c = id % (C::WN / 16) * 16;
          __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const u32x4*>(st + r * HP + c), rc,
                                                 col0 + c < np ? (row0 + r) * np + col0 + c : -1, 0, 0);
        }
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)s, rh, half == 0 && col0 % 128 == 0 && col0 < np ? row0 + lane : -1, 0,
                                             0);
      };
      if constexpr (C::WN == 128) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          float v[C::TN * 16];
          hold(i);
          const float top = hidden(i, v);
          store(i, v, top);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        float v[C::TM][C::TN * 16], top[C::TM];
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          top[i] = hidden(i, v[i]);
          if (half == 0) amax[wn * BM + wm * C::WM + 32 * i + lane] = top[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
          const int r = wm * C::WM + 32 * i + (lane & 31);
          store(i, v[i], fmaxf(amax[r], amax[BM + r]));
        }
      }
    } else {
      // 32 rows of up to 128 bytes at a time through LDS, so that 8 lanes
      // store a whole line
      constexpr int V = 16 / sizeof(TOut);               // columns of a lane's store
      constexpr int JB = C::TN < V / 4 ? C::TN : V / 4;  // blocks of 32 columns staged
      constexpr int LPR = 32 * JB / V, RPI = 64 / LPR;   // lanes to a row, rows to a store
      static_assert(C::TN % JB == 0 && (EPI != kFp8Pair || RPI == 8), "blocks");
      TOut* out = reinterpret_cast<TOut*>(p.out);
#pragma unroll
      for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j0 = 0; j0 < C::TN; j0 += JB) {
          if (j0 == 0) hold(i);
#pragma unroll
          for (int j = j0; j < j0 + JB; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              TOut* to4 = reinterpret_cast<TOut*>(st + (lane & 31) * C::OP) + 32 * (j - j0) + 8 * q + 4 * half;
              const floatx4 b = bias4(j, q);
              TOut v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = (TOut)(acc[j][i][4 * q + e] + b[e]);
              if constexpr (sizeof(TOut) == 4) *reinterpret_cast<u32x4*>(to4) = *reinterpret_cast<const u32x4*>(v);
              else *reinterpret_cast<u32x2*>(to4) = *reinterpret_cast<const u32x2*>(v);
            }
          const int col = col0 + 32 * j0 + lane % LPR * V;
#pragma unroll
          for (int it = 0; it < 32 / RPI; ++it) {
            const int r = RPI * it + lane / LPR, row = wm * C::WM + 32 * i + r;
            const u32x4 raw = *reinterpret_cast<const u32x4*>(st + r * C::OP + lane % LPR * 16);
            if (row >= done.rows || col >= p.N) continue;
            TOut* to16 = out + (EPI == kFp8Pair ? (int64_t)place[32 * i + r] : (int64_t)(done.m0 + row)) * p.ldo + col;
            if (col + V <= p.N) {
              __builtin_memcpy(to16, &raw, 16);  // (at any address)
            } else {
              const TOut* v = reinterpret_cast<const TOut*>(&raw);
#pragma unroll
              for (int e = 0; e < V; ++e)
                if (col + e < p.N) to16[e] = v[e];
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (!more) {
      __builtin_amdgcn_s_waitcnt(0);  // nothing is to land in LDS that is no longer this workgroup's
      break;
    }
    if constexpr (!C::AHEAD) {
      __syncthreads();  // the staging lies over the ring
      where = place_of(T);
      now = tile_of(entry_of(where.tm), where.n0);
      look_up(now);
      aim(now);
      wword = weight_scales(now);
      prologue();
    }
  }
}

template <int BM, int BN, int NS, bool EXACT, int EPI, typename TOut>
__global__ __launch_bounds__(256, (2 * Fp8Cfg<BM, BN, NS>::LDS > 160 * 1024 ? 1 : 2)) void fp8_tile_kernel(Fp8Gemm p) {
  __shared__ __attribute__((aligned(1024))) char smem[Fp8Cfg<BM, BN, NS>::LDS];
  fp8_tile_body<BM, BN, NS, EXACT, EPI, TOut>(p, smem);
}

template <int BM, int BN, int NS, bool EXACT, int EPI, typename TOut>
hipError_t launch_tile(const Fp8Gemm& p, hipStream_t s) {
  const int64_t tm = p.g.tile ? p.g.max_tiles : (p.M + BM - 1) / BM;
  const int64_t nt = tm * ((p.N + BN - 1) / BN);
  if (p.g.tile && p.g.tile_rows != BM) return hipErrorInvalidValue;
  if (Fp8Cfg<BM, BN, NS>::AHEAD && p.K <= kFp8Block) return hipErrorInvalidValue;
  if (nt > (int64_t)1 << 28) return hipErrorInvalidValue;
  // as many workgroups as the CUs hold at a time, 8 XCDs alike
  const int64_t resident = (int64_t)device_cus() * (160 * 1024 / Fp8Cfg<BM, BN, NS>::LDS);
  const int64_t grid = (std::min(nt, resident) + 7) / 8 * 8;
  fp8_tile_kernel<BM, BN, NS, EXACT, EPI, TOut><<<(unsigned)grid, 256, 0, s>>>(p);
  return hipGetLastError();
}

// A product over experts. f32 calls are EXACT: 3000 frames to 2 of 16 experts
// of 1024 -> 4096 take 155 us so, 15001 to 4 of 64 1070. A bf16 call is not (101
// and 740): with the fp8 unit's sums 8% of its results are a bf16 step or so off,
// and their error in the 2-norm goes from 1.58e-3 to 1.61e-3. (The first product
// alone EXACT would add 30 and 180 us.)
template <bool EXACT>
hipError_t launch_experts(const Fp8Gemm& p, hipStream_t s) {
  if (p.epilogue == kFp8HiddenQ)
    return p.g.tile_rows == 256 ? launch_tile<256, 256, 2, EXACT, kFp8HiddenQ, float>(p, s)
                                : launch_tile<128, 128, 2, EXACT, kFp8HiddenQ, float>(p, s);
  if (p.epilogue != kFp8Pair) return hipErrorInvalidValue;
  // too few tiles of 256 columns to fill the CUs (the experts' last tiles
  // are half full on average): 128 columns, 3000 frames to 2 of 16 experts
  // 55 -> 46 us
  const int64_t tiles = (p.M / 256 + p.g.experts / 2) * ((p.N + 255) / 256);
  if (p.g.tile_rows == 256 && tiles <= device_cus() / 2 + device_cus() / 4)
    return launch_tile<256, 128, 2, EXACT, kFp8Pair, float>(p, s);
  return p.g.tile_rows == 256 ? launch_tile<256, 256, 2, EXACT, kFp8Pair, float>(p, s)
                              : launch_tile<128, 128, 2, EXACT, kFp8Pair, float>(p, s);
}

bool bad_gemm(const Fp8Gemm& p) {
  return p.N <= 0 || p.K <= 0 || !p.bias || p.K > kFp8MaxK || !p.w || !p.ws || (!p.out && p.epilogue != kFp8HiddenQ);
}

}  // namespace

hipError_t fp8_quantize_rows(DType dt, const void* x, int64_t ldx, int64_t rows, int K, uint8_t* codes,
                             uint8_t* scales, hipStream_t s) {
  if (rows <= 0 || K <= 0 || K > kFp8MaxK) return hipErrorInvalidValue;
  const int64_t per = fp8_kbp(K) / 4, most = ((int64_t)1 << 25) / per;  // (a grid's threads fit 32 bits)
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t m = std::min(most, rows - r);
    const unsigned grid = (unsigned)((m * per + 3) / 4);
    uint8_t *c = codes + r * fp8_kp(K), *sc = scales + r * fp8_kbp(K);
    if (dt == kBF16)
      quantize_rows_kernel<bf16><<<grid, 256, 0, s>>>(static_cast<const bf16*>(x) + r * ldx, ldx, m, K, c, sc);
    else
      quantize_rows_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(x) + r * ldx, ldx, m, K, c, sc);
  }
  return hipGetLastError();
}

hipError_t fp8_quantize_weight(int data_dtype, const void* w, int n_mats, int N, int K, uint8_t* codes,
                               uint8_t* scales, hipStream_t s) {
  if (N <= 0 || K <= 0 || n_mats <= 0 || n_mats > 65535 || (N + 127) / 128 > 65535) return hipErrorInvalidValue;
  const dim3 grid((K + 127) / 128, (N + 127) / 128, n_mats);
  switch (data_dtype) {
    case MHSA_F32: quantize_weight_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(w), N, K, codes, scales); break;
    case MHSA_BF16: quantize_weight_kernel<<<grid, 256, 0, s>>>(static_cast<const bf16*>(w), N, K, codes, scales); break;
    case MHSA_F16: quantize_weight_kernel<<<grid, 256, 0, s>>>(static_cast<const _Float16*>(w), N, K, codes, scales); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t fp8_pad_weight(const uint8_t* w, const uint8_t* ws, int n_mats, int N, int K, uint8_t* codes,
                          uint8_t* scales, hipStream_t s) {
  if (N <= 0 || K <= 0 || n_mats <= 0) return hipErrorInvalidValue;
  const int64_t rows = (int64_t)n_mats * N, nb = (int64_t)n_mats * ((N + 127) / 128);
  const int64_t grid = (std::max(rows * fp8_kp(K) / 16, nb * fp8_kbp(K)) + 255) / 256;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  const bool vec = K % 128 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  pad_weight_kernel<<<(unsigned)grid, 256, 0, s>>>(w, ws, rows, N, K, vec, codes, scales);
  return hipGetLastError();
}

hipError_t fp8_unpad_weight(const uint8_t* codes, const uint8_t* scales, int N, int K, uint8_t* w, uint8_t* ws,
                            hipStream_t s) {
  const int64_t grid = ((int64_t)N * K + 255) / 256;
  if (N <= 0 || K <= 0 || grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  unpad_weight_kernel<<<(unsigned)grid, 256, 0, s>>>(codes, scales, N, K, (N + 127) / 128, w, ws);
  return hipGetLastError();
}

// Up to 16 rows read the weights once. More read them once per 16 rows, which
// saves the second launch and the codes' way through memory while it is not
// much: with a call from Python at 128 x 1024 -> 4096 9.7 us against 12.5 and at
// 224 rows 16.9 against 13.1, at 128 x 2048 -> 2048 9.4 against 12.6 and at 160
// rows 16.8 against 12.1; 64 x 4096 -> 1024 9.0 against 14.1, 96 rows 16.0
// against 14.3 (over K > 2048 16 waves share one row group's inputs).
bool fp8_few_rows(int64_t M, int N, int K) {
  const int64_t read = (M + 15) / 16 * N * K;
  return M <= 16 || (M <= 256 && read < (K <= 2048 ? 40 : 20) << 20);
}
int fp8_scan_pairs() { return kScanPairs; }

hipError_t fp8_gemm_few(const Fp8Gemm& p, hipStream_t s) {
  if (bad_gemm(p) || !p.x) return hipErrorInvalidValue;
  if (p.g.idx && !p.g.tile && (p.g.pairs > kScanPairs || p.g.experts > kScanExperts)) return hipErrorInvalidValue;
  if (p.g.tile && p.g.tile_rows != 16) return hipErrorInvalidValue;
  const int64_t groups = p.g.tile ? p.g.max_tiles : p.g.idx ? std::min(p.g.pairs, p.g.experts) : (p.M + 15) / 16;
  if (groups <= 0 || groups > 65535) return hipErrorInvalidValue;
  const bool vec = p.K % 8 == 0;
  // (hidden values are rounded to codes next: a sum at a code's edge that is off
  // by 1e-5 gives the code beside it, and one such code of a frame's 8192 can be
  // off by as much as the frame's bf16 result is rounded)
  const bool exact = p.exact || p.epilogue == kFp8HiddenF32 || (p.epilogue == kFp8Out && p.out_dt == kF32);
  auto go = [&](auto tx, auto nw, auto rc) {
    using TX = decltype(tx);
    constexpr int NW = decltype(nw)::value, RC = decltype(rc)::value;
    const dim3 grid((p.N + 16 * RC - 1) / (16 * RC), (unsigned)groups);
    if (exact && vec) fp8_few_kernel<TX, NW, RC, true, true><<<grid, NW * 64, 0, s>>>(p);
    else if (exact) fp8_few_kernel<TX, NW, RC, true, false><<<grid, NW * 64, 0, s>>>(p);
    else if (vec) fp8_few_kernel<TX, NW, RC, false, true><<<grid, NW * 64, 0, s>>>(p);
    else fp8_few_kernel<TX, NW, RC, false, false><<<grid, NW * 64, 0, s>>>(p);
  };
  auto by_type = [&](auto nw, auto rc) {
    if (p.x_dt == kBF16) go(bf16{}, nw, rc);
    else go(float{}, nw, rc);
  };
  using std::integral_constant;
  // 64 columns where that leaves a workgroup to somewhat more than half of the
  // CUs: the rows are rounded once for all of them, and a wave has four times the
  // loads in flight (96 f32 rows x 512 -> 2048, 192 workgroups, 7.2 -> 5.6 us; 96
  // x 384 -> 1536, 144, 5.8 -> 4.5; with 128 of them 32 x 1024 -> 4096 took 6.5
  // instead of 6.0 and a frame's two experts of 1024 -> 4096 10.9 instead of 7.0)
  const bool wide = (p.N + 63) / 64 * groups >= device_cus() * 9 / 16;
  if (wide && p.K <= 1024) by_type(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (wide) by_type(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  else if (p.K > 2048) by_type(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else by_type(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  return hipGetLastError();
}

bool fp8_few_sum_ok(int64_t pairs, int K) { return pairs <= 16 && pairs * (fp8_kp(K) + 16) <= kSumLds; }

hipError_t fp8_gemm_few_sum(const Fp8Gemm& p, const float* weights, const void* residual, float res_scale, hipStream_t s) {
  if (bad_gemm(p) || !p.x || p.x_dt != kF32 || p.ldx % 4 || p.K % 8 || (reinterpret_cast<uintptr_t>(p.x) & 15) || !p.g.idx ||
      p.g.pairs <= 0 || !fp8_few_sum_ok(p.g.pairs, p.K) || p.g.top_k <= 0 || p.g.pairs % p.g.top_k || p.ldo != p.N)
    return hipErrorInvalidValue;
  const unsigned grid = (p.N + 15) / 16;
  if (p.exact != (p.out_dt == kF32)) return hipErrorInvalidValue;
  if (p.out_dt == kBF16)
    fp8_few_sum_kernel<bf16, false><<<grid, 1024, 0, s>>>(p, weights, static_cast<const bf16*>(residual), res_scale);
  else
    fp8_few_sum_kernel<float, true><<<grid, 1024, 0, s>>>(p, weights, static_cast<const float*>(residual), res_scale);
  return hipGetLastError();
}

int fp8_group_rows(int64_t pairs, int experts, int K) {
  const int64_t mean = pairs / experts;
  return mean < kFp8TileMean ? 16 : mean < kFp8LargeMean || K <= kFp8Block ? 128 : 256;  // (the large tiles' ring takes two stages)
}

hipError_t fp8_gemm_tile(const Fp8Gemm& p, hipStream_t s) {
  if (bad_gemm(p) || !p.a || !p.as) return hipErrorInvalidValue;
  if (p.g.tile) {
    if (p.a_rows * fp8_kp(p.K) > 0xFFFFFFFFll || p.slots % 16 || p.slots * (fp8_kp(p.K) / 128) > INT32_MAX)
      return hipErrorInvalidValue;
    if (p.epilogue == kFp8HiddenQ && p.N % 64) return hipErrorInvalidValue;
    return p.exact ? launch_experts<true>(p, s) : launch_experts<false>(p, s);
  }
  if (p.M <= 0 || p.epilogue != kFp8Out) return hipErrorInvalidValue;
  auto tiles = [&](int64_t bm, int64_t bn) { return (p.M + bm - 1) / bm * ((p.N + bn - 1) / bn); };
  // Large tiles from half of the CUs on, and tiles of 128 rows likewise. About
  // there either side wins, by K (us, the larger tiles against the smaller):
  // 128 large tiles of 2048 x 1024 -> 4096 23.2 and 20.1, of 2048 x 4096 -> 4096
  // 48 and 48, 188 of 3000 x 1024 -> 4096 24.8 and 27.1; 128 tiles of 128 rows of
  // 1024 x 1024 -> 2048 12.1 and 10.5, of 1000 x 4096 -> 2048 25.0 and 26.8. 192
  // rows where a CU then goes through fewer (3000 x 1024 -> 4096 24.8 against
  // 27.6, 8200 x 1024 -> 2048 37.8 against 43.8).
  const int64_t t256 = tiles(256, 256), t192 = tiles(192, 256), t128 = tiles(128, 128), cus = device_cus();
  const bool large = t256 >= cus / 2 && p.K > kFp8Block;  // (the large tiles' ring takes two stages)
  const bool fewer = (t192 + cus - 1) / cus * 192 < (t256 + cus - 1) / cus * 256;  // rows a CU goes through
  if (p.out_dt == kF32) {
    if (large && fewer) return launch_tile<192, 256, 2, true, kFp8Out, float>(p, s);
    if (large) return launch_tile<256, 256, 2, true, kFp8Out, float>(p, s);
    return t128 >= cus / 2 ? launch_tile<128, 128, 2, true, kFp8Out, float>(p, s) : launch_tile<64, 64, 4, true, kFp8Out, float>(p, s);
  }
  if (large && fewer) return launch_tile<192, 256, 2, false, kFp8Out, bf16>(p, s);
  if (large) return launch_tile<256, 256, 2, false, kFp8Out, bf16>(p, s);
  // a tile alone on its CU keeps four stages, two that share it two each
  // (3000 x 4096 -> 1024: 36.8 -> 29.7 us with the rows' codes)
  if (t128 >= cus / 2 && t128 <= cus) return launch_tile<128, 128, 4, false, kFp8Out, bf16>(p, s);
  return t128 >= cus / 2 ? launch_tile<128, 128, 2, false, kFp8Out, bf16>(p, s) : launch_tile<64, 64, 4, false, kFp8Out, bf16>(p, s);
}

}  // namespace mhsa
