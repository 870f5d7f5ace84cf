// A residual's addition with its norm, as floats or as 8-bit codes.
//
//   v = x + a d                                   (f32; sum: v rounded once)
//   rms:   y = v / sqrt(mean(v^2) + eps) * w + b
//   layer: y = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * w + b
//
// A row lies in the registers of its W waves, 8 columns to a lane and chunk, so
// that x and d are read once whatever the norm needs, the variance is taken
// around the mean itself, and results may lie over their inputs. 16 lanes hold a
// block of 128 columns: its largest magnitude is four DPP steps, and a wave's
// four blocks of a chunk are one word of scale bytes. Bound: HBM, one pass: x, delta
// and sum of 15001 x 4096 bf16 with codes, 431 MB, take 76 us (5.7 TB/s); one row of
// 1024 takes 2.5, a launch and one chain of loads and sums.
// Rows that are no whole runs of 8 pay for unaligned accesses and for putting the
// row's end in place (2^25 bf16 in rows of 2047: 42 us, of 2048: 39).
#include <algorithm>

#include "fp8_common.hpp"
#include "fp8_kernels.hpp"
#include "row_kernels.hpp"

namespace mhsa {
namespace {

// 8 values to columns [c, c + 8) of a row of D.
template <RowForm FORM, typename T>
__device__ __forceinline__ void store8(T* row, int c, int D, const float v[8]) {
  T t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
  if (c + 8 <= D) {
    __builtin_memcpy(row + c, t, sizeof t);
  } else if constexpr (FORM != kWhole) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < D) row[c + e] = t[e];
  }
}

template <typename T, int CH, int W, RowForm FORM>
__global__ __launch_bounds__(W == 1 ? 256 : W * 64) void add_norm_kernel(NormParams p) {
  __shared__ float red[2][W];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = W == 1 ? 0 : wv;
  const int64_t row = (int64_t)blockIdx.x * (W == 1 ? 4 : 1) + (W == 1 ? wv : 0);
  if (row >= p.rows) return;
  const int kb = (p.D + 127) / 128, kbp = (kb + 3) / 4 * 4;
  auto col = [&](int i) { return 8 * (64 * (wr + W * i) + lane); };
  auto in = [&](int i, int e) { return FORM == kWhole ? col(i) < p.D : col(i) + e < p.D; };
  constexpr bool HOLD = CH <= 2;  // registers for all that is read, at once
  Run<float, FORM> w[CH], b[CH];
  auto weights = [&](int i) {
    if (p.w) {
      w[i].load(p.w, col(i), p.D);
      w[i].trim(col(i), p.D);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i].u[e] = 0x3F800000u;
    }
    if (p.b) {
      b[i].load(p.b, col(i), p.D);
      b[i].trim(col(i), p.D);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) b[i].u[e] = 0;
    }
  };
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < CH; ++i) weights(i);
  }
  const float n = 1.f / (float)p.D;
  auto total = [&](float v, int which) {
    v = wave_reduce(v, [](float a, float c) { return a + c; });
    if constexpr (W > 1) {
      float* r = red[which];
      if (lane == 0) r[wr] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v += r[i];
    }
    return v;
  };
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* d = static_cast<const T*>(p.delta) + row * p.ldd;
  Run<T, FORM> tx[CH], td[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) tx[i].load(x, col(i), p.D);
  if (HOLD && p.delta) {
#pragma unroll
    for (int i = 0; i < CH; ++i) td[i].load(d, col(i), p.D);
  } else {  // (negative zeros, which leave a negative zero of x what it is)
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < Run<T, FORM>::N; ++e) td[i].u[e] = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
  }
  float v[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (!HOLD && p.delta) td[i].load(d, col(i), p.D);
    tx[i].trim(col(i), p.D);
    td[i].trim(col(i), p.D);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = __builtin_fmaf(p.scale, td[i][e], tx[i][e]);
    if constexpr (!HOLD) __builtin_amdgcn_sched_barrier(0);
  }
  if (p.sum) {
#pragma unroll
    for (int i = 0; i < CH; ++i) store8<FORM>(static_cast<T*>(p.sum) + row * p.lds, col(i), p.D, v[i]);
  }
  if (p.layer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[i][e];
    const float mean = total(s, 0) * n;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = in(i, e) ? v[i][e] - mean : 0.f;
  }
  auto squares = [&](int which) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) q = __builtin_fmaf(v[i][e], v[i][e], q);
    return total(q, which);
  };
  float m = __builtin_fmaf(squares(1), n, p.eps);
  if (m < 0x1p-100f) {  // (the same in all of the row's threads)
    // Squares near f32's end lose their bits or all of themselves, and the root's
    // instruction takes what is under 2^-126 for 0: such a row times 2^96 (its values
    // are under 2^-42), and eps times the square of that.
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= 0x1p96f;
    m = __builtin_fmaf(squares(0), n, p.eps * 0x1p96f * 0x1p96f);
  }
  const float r = __builtin_amdgcn_rsqf(m);
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if constexpr (!HOLD) weights(i);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = __builtin_fmaf(v[i][e] * r, w[i][e], b[i][e]);
    if constexpr (!HOLD) __builtin_amdgcn_sched_barrier(0);
  }
  if (p.out) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (p.out_dt == kBF16) store8<FORM>(static_cast<bf16*>(p.out) + row * p.ldo, col(i), p.D, v[i]);
      else store8<FORM>(static_cast<float*>(p.out) + row * p.ldo, col(i), p.D, v[i]);
    }
  }
  if (p.codes) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int word = wr + W * i;  // of the row's scale bytes
      if (4 * word >= kb) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = in(i, e) ? v[i][e] : 0.f;  // (a NaN of the sums reaches there too)
      const int s = fp8_scale_byte(block_max(v[i]));
      const float scale = fp8_scale(s);
      if (col(i) < kb * 128)
        *reinterpret_cast<u32x2*>(p.codes + row * ((int64_t)kb * 128) + col(i)) =
            u32x2{fp8_pack4_scaled(v[i][0], v[i][1], v[i][2], v[i][3], scale),
                  fp8_pack4_scaled(v[i][4], v[i][5], v[i][6], v[i][7], scale)};
      uint32_t bytes = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        bytes |= (uint32_t)(4 * word + j < kb ? __builtin_amdgcn_readlane(s, 16 * j) : 127) << 8 * j;
      if (lane == 0) *reinterpret_cast<uint32_t*>(p.scales + row * kbp + 4 * word) = bytes;
    }
  }
}

template <typename T, int CH, int W>
hipError_t launch(const NormParams& p, hipStream_t s) {
  if ((int64_t)512 * CH * W < p.D) return hipErrorInvalidValue;
  constexpr int64_t most = 1 << 21;  // rows of a launch: a grid's threads fit 32 bits
  static_assert(most * 64 * W < (int64_t)1 << 32, "a wave takes a row or a part of it");
  auto behind = [](auto* q, int64_t n) { return q ? q + n : q; };
  auto rows = [&](const void* q, DType dt, int64_t n) { return const_cast<char*>(behind((const char*)q, n * (dt == kBF16 ? 2 : 4))); };
  const int64_t kb = (p.D + 127) / 128, kbp = (kb + 3) / 4 * 4;
  for (int64_t r = 0; r < p.rows; r += most) {
    NormParams q = p;
    q.rows = std::min(most, p.rows - r);
    if (!p.delta) q.scale = 1.f;
    q.x = rows(p.x, p.dt, r * p.ldx);
    q.delta = rows(p.delta, p.dt, r * p.ldd);
    q.sum = rows(p.sum, p.dt, r * p.lds);
    q.out = rows(p.out, p.out_dt, r * p.ldo);
    q.codes = behind(p.codes, r * kb * 128);
    q.scales = behind(p.scales, r * kbp);
    const unsigned grid = (unsigned)(W == 1 ? (q.rows + 3) / 4 : q.rows);
    auto run = [&](auto form) { add_norm_kernel<T, CH, W, decltype(form)::value><<<grid, W == 1 ? 256 : W * 64, 0, s>>>(q); };
    const RowForm form = row_form(p.D);
    if (form == kWhole) run(std::integral_constant<RowForm, kWhole>());
    else if (form == kRagged) run(std::integral_constant<RowForm, kRagged>());
    else if constexpr (CH * W == 1) run(std::integral_constant<RowForm, kTiny>());
  }
  return hipGetLastError();
}

// As many waves as the row fills with one run of 8 a lane, up to 16: with half the
// waves and two runs a row of 1024, 4096 and 8192 bf16 takes 2.8, 3.1 and 3.7 us
// instead of 2.5, 2.9 and 3.6, 2^25 values in such rows 39.8, 40.0 and 41.0 instead
// of 38.9, 39.6 and 40.3; with twice the waves 2^25 values in rows of 512 take 45
// instead of 39. A row per wave or workgroup, no loop over rows: the compiler took
// addresses out of one and spilled (2^25 values in rows of 32768: 102 us instead of
// 48).
template <typename T>
hipError_t by_width(const NormParams& p, hipStream_t s) {
  if (p.D <= 512) return launch<T, 1, 1>(p, s);
  if (p.D <= 1024) return launch<T, 1, 2>(p, s);
  if (p.D <= 2048) return launch<T, 1, 4>(p, s);
  if (p.D <= 4096) return launch<T, 1, 8>(p, s);
  if (p.D <= 8192) return launch<T, 1, 16>(p, s);
  return p.D <= 16384 ? launch<T, 2, 16>(p, s) : launch<T, 4, 16>(p, s);
}

}  // namespace

hipError_t add_norm(const NormParams& p, hipStream_t s) {
  if (p.rows <= 0 || p.D <= 0 || p.D > kNormMaxD || !p.x || (p.codes != nullptr) != (p.scales != nullptr))
    return hipErrorInvalidValue;
  return p.dt == kBF16 ? by_width<bf16>(p, s) : by_width<float>(p, s);
}

}  // namespace mhsa
