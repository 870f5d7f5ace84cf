// Routing of frames to experts, and the bookkeeping around the experts'
// products (fp8_gemm.hip): pairs of frame and expert sorted by expert, and
// the weighted sum of a frame's experts.
#include <algorithm>
#include <type_traits>

#include "fp8_common.hpp"
#include "fp8_kernels.hpp"

namespace mhsa {
namespace {

// ---------------------------------------------------------------------------
// Routing: s_e = softmax(x)_e or sigmoid(x_e); the choice score c_e = s_e +
// bias_e; the groups with the largest sums of their two best c; in them the
// top_k experts by c, ties to the lower index; w_j = s_e / sum of the chosen
// s. Scores are formed and compared in 64 bits: two experts' scores often
// differ by less than f32 resolves, and the choice between them is then not a
// matter of the order of a sum.
//
// One wave per row, expert e in lane e % 64 (many rows: four to a wave). What
// is bound here is not the logits' bytes but the wave's instructions, half of
// them the scores' exponentials in 64 bits and half the reductions. These are
// DPP moves and lane reads, which the vector unit does itself, and a choice
// reduces one 32-bit word: a score's f32 rounding, which keeps the order. Only
// lanes that share the largest word are compared in 64 bits. (With shuffles of
// 64-bit values, which go through LDS, 30001 rows of 256 experts in 8 groups
// took 88 us, with these 44, with four rows to a wave 29.8, calls one after the
// other in a graph: 1.1 TB/s, and 423 vector instructions a row, which the unit
// issues in 70% of the time. Alone, under a profiler, a call takes 32.6.)
// ---------------------------------------------------------------------------

constexpr double kNone = -__builtin_inf();

__device__ __forceinline__ double lane_of(double v, int l) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  const i32x2 u = __builtin_bit_cast(i32x2, v);
  return __builtin_bit_cast(double, i32x2{__builtin_amdgcn_readlane(u[0], l), __builtin_amdgcn_readlane(u[1], l)});
}
// 1 / d for d >= 1 to within 2 ulp, 0 for infinity: the hardware's estimate
// and two Newton steps.
__device__ __forceinline__ double inverse(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return d < __builtin_inf() ? r : 0.0;
}
// e^x for |x| <= 800 to within 2.5 ulp: e^x = 2^k e^r, |r| <= ln 2 / 2, by the
// series up to r^12 (the rest is up to 1.5 ulp; over 10^8 values the most was
// 2.32). The range is the callers' to keep, with one instruction, and takes the
// special cases off the way: beyond it e^x is infinity or 0 in 64 bits.
__device__ __forceinline__ double exp_within(double x) {
  const double k = __builtin_rint(x * 1.4426950408889634);
  // ln 2 in two parts, the first of 32 bits, so that its product with k is exact
  double r = __builtin_fma(k, -0x1.62e42fefp-1, x);
  r = __builtin_fma(k, -0x1.473de6af278edp-34, r);
  double e = 1.0 / 479001600.0;
  constexpr double c[12] = {1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                            1.0 / 120.0,      1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
#pragma unroll
  for (int i = 0; i < 12; ++i) e = __builtin_fma(e, r, c[i]);
  return __builtin_ldexp(e, (int)k);
}
__device__ __forceinline__ double sigmoid(float v) {
  return inverse(1.0 + exp_within(-(double)__builtin_amdgcn_fmed3f(v, -800.f, 800.f)));
}
// e^(v - top), 1 also for infinities that are equal
__device__ __forceinline__ double exp_below(float v, double top) {
  const double e = exp_within(fmax((double)v - top, -800.0));
  return (double)v == top ? 1.0 : e;
}
// The order of values as unsigned words, 0 for none (-inf itself is 0x7FFFFF,
// and no value's word is 0).
__device__ __forceinline__ uint32_t rank_word(double v) {
  if (!(v > kNone)) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, (float)v);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

template <typename T, int EPL>
__global__ __launch_bounds__(256) void route_kernel(RouteParams p) {
  __shared__ double tab[4][EPL * 64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wv;
  if (row >= p.rows) return;  // (waves do not wait for each other)
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  double s[EPL], c[EPL];
  float v[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 64 * i;
    const float t = e < p.experts ? (float)x[e] : -__builtin_inff();
    v[i] = t > -__builtin_inff() ? t : -__builtin_inff();  // (a NaN is no score)
  }
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) s[i] = sigmoid(v[i]);
  } else {
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, v[i]);
    mx = wave_reduce(mx, [](float a, float b) { return fmaxf(a, b); });
    const double top = mx > -__builtin_inff() ? (double)mx : 0.0;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      s[i] = exp_below(v[i], top);
      sum += s[i];
    }
    sum = wave_reduce(sum, [](double a, double b) { return a + b; });
    const double inv = sum > 0.0 ? inverse(sum) : 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) s[i] *= inv;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 64 * i;
    const double t = p.bias && e < p.experts ? s[i] + (double)p.bias[e] : s[i];
    c[i] = v[i] > -__builtin_inff() && t > kNone ? t : kNone;
  }
  double* t = tab[wv];
  if (p.groups > 1) {
    // 64 / groups lanes (down to a power of two) to a group find its two best
    const int size = p.experts / p.groups;
    int shift = 6;
    while (p.groups << shift > 64) --shift;
    const int lanes = 1 << shift, g = lane >> shift;
    const float per = 1.f / (float)size;
#pragma unroll
    for (int i = 0; i < EPL; ++i) t[lane + 64 * i] = c[i];
    __builtin_amdgcn_wave_barrier();
    double a = kNone, b = kNone;
    if (g < p.groups)
      for (int e = lane & (lanes - 1); e < size; e += lanes) {
        const double u = t[g * size + e];
        b = fmax(b, fmin(a, u));
        a = fmax(a, u);
      }
    for (int o = 1; o < lanes; o *= 2) {
      const double a2 = __shfl_xor(a, o, 64), b2 = __shfl_xor(b, o, 64);
      b = fmax(fmin(a, a2), fmax(b, b2));
      a = fmax(a, a2);
    }
    const double best = b > kNone ? a + b : a;
    int before = 0;  // groups ahead of this lane's
    for (int o = 0; o < p.groups; ++o) {
      const double u = lane_of(best, o << shift);
      before += u > best || (u == best && o < g) ? 1 : 0;
    }
    const uint64_t kept = __ballot(g < p.groups && before < p.topk_groups);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      // (e + 0.5) / size is at least 0.5 / 512 away from a whole number
      const int e = lane + 64 * i, of = (int)(((float)e + 0.5f) * per);
      c[i] = e < p.experts && (kept >> (of << shift & 63) & 1) ? c[i] : kNone;
    }
    __builtin_amdgcn_wave_barrier();
  }
  // the scores, for the lanes that will have chosen them
#pragma unroll
  for (int i = 0; i < EPL; ++i) t[lane + 64 * i] = s[i];
  uint32_t word[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) word[i] = rank_word(c[i]);
  int idx = -1;
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t most = word[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) most = max(most, word[i]);
    most = wave_reduce(most, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    if (most == 0) break;
    // who has it: one, or several that are alike in f32, of which the larger in
    // 64 bits, and of equals the lower index
    int won = -1;
    double u = kNone;
    bool alike = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const uint64_t has = __ballot(word[i] == most);
      alike = alike || (has && (won >= 0 || (has & (has - 1))));
      if (has && won < 0) won = 64 * i + __builtin_ctzll(has);
    }
    if (alike) {
      won = -1;
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        for (uint64_t has = __ballot(word[i] == most); has; has &= has - 1) {  // (ascending indices)
          const int l = __builtin_ctzll(has);
          const double v = lane_of(c[i], l);
          if (won < 0 || v > u) {
            u = v;
            won = 64 * i + l;
          }
        }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) word[i] = lane + 64 * i == won ? 0 : word[i];
    idx = lane == j ? won : idx;
  }
  __builtin_amdgcn_wave_barrier();
  double wj = idx >= 0 ? t[idx] : 0.0;
  if (p.renormalize) {
    const double total = wave_reduce(wj, [](double a, double b) { return a + b; });
    wj = total > 0.0 ? wj / total : 0.0;
  }
  if (lane < p.top_k) {
    p.idx[row * p.top_k + lane] = idx;
    p.w[row * p.top_k + lane] = (float)(wj * (double)p.scale);
  }
}

// Many rows: four to a wave, 16 lanes each, expert e in lane e / per of them
// (per = experts / 16, rounded up). A choice's reduction then serves four rows
// and stays within 16 lanes; the lanes of a group are neighbours, so its two
// best need no exchange through LDS. For up to 256 experts, 16 choices, and
// groups that take whole lanes.
template <typename T, int EPL>
__global__ __launch_bounds__(256) void route_rows_kernel(RouteParams p) {
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15;
  const int64_t first = ((int64_t)blockIdx.x * 4 + wv) * 4;
  if (first >= p.rows) return;  // (waves do not wait for each other)
  const int64_t row = first + (lane >> 4);
  const int per = (p.experts + 15) / 16, e0 = l * per;
  const T* xr = reinterpret_cast<const T*>(p.logits) + (row < p.rows ? row : p.rows - 1) * p.ld;
  const T* x = xr + e0;
  const float none = -__builtin_inff();
  float v[EPL];
  if (p.experts == 16 * EPL) {
    T run[EPL];
    __builtin_memcpy(run, x, sizeof run);  // (rows may lie at any address)
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = (float)run[i];
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = i < per && e0 + i < p.experts ? (float)x[i] : none;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) v[i] = v[i] > none ? v[i] : none;  // (a NaN is no score)
  double c[EPL], top = 0.0, inv = 0.0;
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) c[i] = sigmoid(v[i]);
  } else {
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) mx = fmaxf(mx, v[i]);
    mx = row_reduce(mx, [](float a, float b) { return fmaxf(a, b); });
    top = mx > none ? (double)mx : 0.0;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      c[i] = exp_below(v[i], top);
      sum += c[i];
    }
    sum = row_reduce(sum, [](double a, double b) { return a + b; });
    inv = sum > 0.0 ? inverse(sum) : 0.0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) c[i] *= inv;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const double t = p.bias && i < per && e0 + i < p.experts ? c[i] + (double)p.bias[e0 + i] : c[i];
    c[i] = v[i] > none && t > kNone ? t : kNone;
  }
  bool kept = true;
  if (p.groups > 1) {
    const int lanes = 16 / p.groups, g = l / lanes;
    double a = kNone, b = kNone;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      b = fmax(b, fmin(a, c[i]));
      a = fmax(a, c[i]);
    }
    auto join = [&](auto n) {  // with the lane that the n-th step of a reduction takes
      double a2 = a, b2 = b;
      constexpr int N = decltype(n)::value;
      auto move = [](double u) {
        constexpr int C = N == 0 ? 0xB1 : N == 1 ? 0x4E : 0x141;
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        i32x2 w = __builtin_bit_cast(i32x2, u);
        w[0] = __builtin_amdgcn_update_dpp(w[0], w[0], C, 0xF, 0xF, false);
        w[1] = __builtin_amdgcn_update_dpp(w[1], w[1], C, 0xF, 0xF, false);
        return __builtin_bit_cast(double, w);
      };
      a2 = move(a);
      b2 = move(b);
      b = fmax(fmin(a, a2), fmax(b, b2));
      a = fmax(a, a2);
    };
    using std::integral_constant;
    if (lanes > 1) join(integral_constant<int, 0>{});
    if (lanes > 2) join(integral_constant<int, 1>{});
    if (lanes > 4) join(integral_constant<int, 2>{});
    const double best = b > kNone ? a + b : a;
    int before = 0;  // groups ahead of this lane's
    for (int o = 0; o < p.groups; ++o) {
      const double u = __shfl(best, (lane & 48) | o * lanes, 64);
      before += u > best || (u == best && o < g) ? 1 : 0;
    }
    kept = before < p.topk_groups;
  }
  uint32_t word[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) word[i] = kept ? rank_word(c[i]) : 0;
  constexpr uint32_t kNobody = 0xFFFFFFFF;  // (no value's word)
  uint32_t idx = kNobody;
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t most = word[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) most = max(most, word[i]);
    most = row_reduce(most, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    const int rows = __popcll(__ballot(most != 0)) / 16;
    if (rows == 0) break;
    most = most ? most : kNobody;
    // who has it: one of a row, or several that are alike in f32, of which the
    // larger in 64 bits, and of equals the lower index
    int hit = -1, hits = 0;
    bool has[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      has[i] = word[i] == most;
      hits += __popcll(__ballot(has[i]));
      hit = has[i] ? i : hit;
      word[i] = has[i] ? 0 : word[i];
    }
    uint32_t won = hit >= 0 ? (uint32_t)(e0 + hit) : kNobody;
    if (hits > rows) {
      double u = kNone;
      hit = -1;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const bool more = has[i] && c[i] > u;
        u = more ? c[i] : u;
        hit = more ? i : hit;
      }
      const double best = row_reduce(u, [](double a, double b) { return fmax(a, b); });
      won = hit >= 0 && u == best ? (uint32_t)(e0 + hit) : kNobody;
    }
    won = row_reduce(won, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
    if (hits > rows) {  // the others are still to be chosen
#pragma unroll
      for (int i = 0; i < EPL; ++i) word[i] = has[i] && won != (uint32_t)(e0 + i) ? most : word[i];
    }
    idx = l == j ? won : idx;
  }
  // the chosen expert's score again, as above: less than to keep all of them
  const float t = (float)xr[idx != kNobody ? idx : 0];
  double wj = p.sigmoid ? sigmoid(t) : exp_below(t, top) * inv;
  wj = idx != kNobody ? wj : 0.0;
  if (p.renormalize) {
    const double total = row_reduce(wj, [](double a, double b) { return a + b; });
    wj = total > 0.0 ? wj / total : 0.0;
  }
  if (l < p.top_k && row < p.rows) {
    p.idx[row * p.top_k + l] = (int)idx;
    p.w[row * p.top_k + l] = (float)(wj * (double)p.scale);
  }
}

// ---------------------------------------------------------------------------
// Pairs by expert
// ---------------------------------------------------------------------------

constexpr int kPlanThreads = 1024, kPlanPer = 8, kPlanChunk = kPlanThreads * kPlanPer;
constexpr int kPlanExperts = 1024;

struct PlanParams {
  const int* idx = nullptr;
  int pairs = 0, top_k = 1, experts = 0, tile_rows = 0, chunks = 0;
  int* hist = nullptr;  // [chunks, experts], with more than one chunk
  int *pair = nullptr, *frame = nullptr, *tile = nullptr, *n_tiles = nullptr;
};

// Counts of chunk `chunk` of the pairs per expert.
__device__ __forceinline__ void plan_count(const PlanParams& p, int chunk) {
  __shared__ int cnt[kPlanExperts];
  cnt[threadIdx.x] = 0;
  __syncthreads();
  for (int i = 0; i < kPlanPer; ++i) {
    const int q = chunk * kPlanChunk + i * kPlanThreads + threadIdx.x;
    const int e = q < p.pairs ? p.idx[q] : -1;
    if (e >= 0 && e < p.experts) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  if ((int)threadIdx.x < p.experts) p.hist[chunk * p.experts + threadIdx.x] = cnt[threadIdx.x];
}

// Slots of chunk `chunk`'s pairs (ONE: there is no other, and they are counted
// here) and, by chunk 0, the tile list. The order of an expert's pairs among
// its slots is that of the atomics and may change from call to call: no result
// depends on it, as a slot's row is computed from that row alone.
template <bool ONE>
__device__ __forceinline__ void plan_scatter(const PlanParams& p, int chunk) {
  __shared__ int cursor[kPlanExperts], part[2][16];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  int mine[kPlanPer], rank[kPlanPer];
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int q = chunk * kPlanChunk + i * kPlanThreads + t;
    mine[i] = q < p.pairs ? p.idx[q] : -1;
    if (mine[i] >= p.experts) mine[i] = -1;
  }
  int total = 0, before = 0;
  if constexpr (ONE) {
    cursor[t] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i)
      if (mine[i] >= 0) rank[i] = atomicAdd(&cursor[mine[i]], 1);
    __syncthreads();
    total = cursor[t];
  } else {
    if (t < p.experts)
      for (int c = 0; c < p.chunks; ++c) {
        const int h = p.hist[c * p.experts + t];
        total += h;
        before += c < chunk ? h : 0;
      }
  }
  const int nt = (total + p.tile_rows - 1) / p.tile_rows;
  int slots = (total + 15) / 16 * 16, tiles = nt;  // inclusive sums over the experts: in the wave, then over the waves
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int a = __shfl_up(slots, o, 64), b = __shfl_up(tiles, o, 64);
    slots += lane >= o ? a : 0;
    tiles += lane >= o ? b : 0;
  }
  if (lane == 63) {
    part[0][w] = slots;
    part[1][w] = tiles;
  }
  __syncthreads();
  for (int i = 0; i < w; ++i) {
    slots += part[0][i];
    tiles += part[1][i];
  }
  const int slot0 = slots - (total + 15) / 16 * 16, tile0 = tiles - nt;
  cursor[t] = slot0 + before;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i)
    if (mine[i] >= 0) {
      const int q = chunk * kPlanChunk + i * kPlanThreads + t;
      const int slot = ONE ? cursor[mine[i]] + rank[i] : atomicAdd(&cursor[mine[i]], 1);
      p.pair[slot] = q;
      p.frame[slot] = q / p.top_k;
    }
  if (chunk == 0) {
    if (t == kPlanThreads - 1) *p.n_tiles = tiles;
    for (int i = 0; i < nt; ++i) {
      int* e = p.tile + 4 * (tile0 + i);
      e[0] = t;
      e[1] = slot0 + i * p.tile_rows;
      e[2] = min(p.tile_rows, total - i * p.tile_rows);
      e[3] = 0;
    }
  }
}

// The frames' codes, and beside them, by the first workgroups, the list of
// pairs (ONE) or the counts for it: neither needs the other, and together they
// take as long as the longer.
template <typename T, bool ONE>
__global__ __launch_bounds__(kPlanThreads) void prepare_kernel(PlanParams p, const T* x, int64_t rows, int K, uint8_t* codes,
                                                               uint8_t* scales) {
  if ((int)blockIdx.x < p.chunks) {
    if constexpr (ONE) plan_scatter<true>(p, 0);
    else plan_count(p, blockIdx.x);
  } else {
    quantize_blocks(x, K, rows, K, codes, scales, (int64_t)(blockIdx.x - p.chunks) * 16 + (threadIdx.x >> 6));
  }
}
__global__ __launch_bounds__(kPlanThreads) void plan_scatter_kernel(PlanParams p) { plan_scatter<false>(p, blockIdx.x); }

// ---------------------------------------------------------------------------
// The experts' weighted sum, 8 columns to a thread, in the order of the
// choices.
// ---------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const float* y, const int* idx, const float* w, int64_t rows,
                                                      int top_k, int experts, int D, const T* residual,
                                                      float res_scale, T* out) {
  const int per = D / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= rows * per) return;
  const int64_t row = id / per;
  const int col = (int)(id % per) * 8;
  float f[8] = {};
  for (int j = 0; j < top_k; ++j) {
    const int e = idx[row * top_k + j];
    if (e < 0 || e >= experts) continue;
    const float wj = w[row * top_k + j];
    const floatx4* src = reinterpret_cast<const floatx4*>(y + (row * top_k + j) * D + col);
    const floatx4 a = src[0], b = src[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __builtin_fmaf(wj, a[i], f[i]);
      f[i + 4] = __builtin_fmaf(wj, b[i], f[i + 4]);
    }
  }
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= res_scale;
  if (residual) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<u32x4*>(v)[i] = reinterpret_cast<const u32x4*>(residual + row * D + col)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += (float)v[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)f[i];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    reinterpret_cast<u32x4*>(out + row * D + col)[i] = reinterpret_cast<const u32x4*>(v)[i];
}

}  // namespace

hipError_t route(const RouteParams& p, hipStream_t s) {
  if (p.rows <= 0 || p.experts <= 0 || p.experts > kRouteMaxExperts || p.top_k <= 0 || p.top_k > kRouteMaxK ||
      p.top_k > p.experts || p.groups <= 0 || p.groups > kRouteMaxGroups || p.experts % p.groups ||
      p.topk_groups <= 0 || p.topk_groups > p.groups)
    return hipErrorInvalidValue;
  const int64_t grid = (p.rows + 3) / 4;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  // Four rows to a wave where there are enough of them: 8000 rows of 256 experts
  // in 8 groups 15.3 -> 12.3 us, 30001 44.4 -> 29.8; of 64 experts 4.8 -> 4.4 and
  // 12.6 -> 9.2 (in a graph, as all of these). Of fewer rows a wave's longer way
  // weighs more (3000: 9.0 against 10.0 and 3.2 against 3.9).
  const bool many = p.rows >= 6144 && p.experts <= 256 && p.top_k <= 16 &&
                    (p.groups == 1 || (16 % p.groups == 0 && p.experts % 16 == 0));
  auto go = [&](auto t) {
    using T = decltype(t);
    if (many && p.experts <= 64) route_rows_kernel<T, 4><<<(unsigned)((p.rows + 15) / 16), 256, 0, s>>>(p);
    else if (many && p.experts <= 128) route_rows_kernel<T, 8><<<(unsigned)((p.rows + 15) / 16), 256, 0, s>>>(p);
    else if (many) route_rows_kernel<T, 16><<<(unsigned)((p.rows + 15) / 16), 256, 0, s>>>(p);
    else if (p.experts <= 64) route_kernel<T, 1><<<(unsigned)grid, 256, 0, s>>>(p);
    else if (p.experts <= 128) route_kernel<T, 2><<<(unsigned)grid, 256, 0, s>>>(p);
    else if (p.experts <= 256) route_kernel<T, 4><<<(unsigned)grid, 256, 0, s>>>(p);
    else route_kernel<T, 8><<<(unsigned)grid, 256, 0, s>>>(p);
  };
  if (p.dt == kBF16) go(bf16{});
  else go(float{});
  return hipGetLastError();
}

int64_t plan_scratch_ints(int64_t pairs, int experts) { return (pairs + kPlanChunk - 1) / kPlanChunk * experts; }

hipError_t experts_prepare(const int* idx, int pairs, int top_k, int experts, int tile_rows, int* pair, int* frame, int* tile,
                           int* n_tiles, int* scratch, DType dt, const void* x, int64_t rows, int K, uint8_t* codes,
                           uint8_t* scales, hipStream_t s) {
  if (pairs <= 0 || top_k <= 0 || experts <= 0 || experts > kPlanExperts || tile_rows <= 0 || rows < 0 || K <= 0 || K % 8 ||
      (reinterpret_cast<uintptr_t>(x) & 15))
    return hipErrorInvalidValue;
  PlanParams p;
  p.idx = idx;
  p.pairs = pairs;
  p.top_k = top_k;
  p.experts = experts;
  p.tile_rows = tile_rows;
  p.chunks = (pairs + kPlanChunk - 1) / kPlanChunk;
  p.hist = scratch;
  p.pair = pair;
  p.frame = frame;
  p.tile = tile;
  p.n_tiles = n_tiles;
  const int64_t items = codes ? rows * (fp8_kbp(K) / 4) : 0, grid = p.chunks + (items + 15) / 16;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  auto go = [&](auto t) {
    using T = decltype(t);
    const T* xt = static_cast<const T*>(x);
    if (p.chunks == 1) prepare_kernel<T, true><<<(unsigned)grid, kPlanThreads, 0, s>>>(p, xt, rows, K, codes, scales);
    else prepare_kernel<T, false><<<(unsigned)grid, kPlanThreads, 0, s>>>(p, xt, rows, K, codes, scales);
  };
  if (dt == kBF16) go(bf16{});
  else go(float{});
  if (p.chunks > 1) plan_scatter_kernel<<<p.chunks, kPlanThreads, 0, s>>>(p);
  return hipGetLastError();
}

hipError_t experts_combine(DType dt, const float* y, const int* idx, const float* w, int64_t rows, int top_k,
                           int experts, int D, const void* residual, float res_scale, void* out, hipStream_t s) {
  const int64_t grid = (rows * (D / 8) + 255) / 256;
  if (rows <= 0 || D <= 0 || D % 8 || grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  if (dt == kBF16)
    combine_kernel<bf16><<<(unsigned)grid, 256, 0, s>>>(y, idx, w, rows, top_k, experts, D,
                                                        static_cast<const bf16*>(residual), res_scale, static_cast<bf16*>(out));
  else
    combine_kernel<float><<<(unsigned)grid, 256, 0, s>>>(y, idx, w, rows, top_k, experts, D,
                                                         static_cast<const float*>(residual), res_scale, static_cast<float*>(out));
  return hipGetLastError();
}

}  // namespace mhsa
