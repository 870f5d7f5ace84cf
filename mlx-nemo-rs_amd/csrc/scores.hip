// Log probabilities of given tokens, entropy and the likeliest tokens of rows of
// logits x [V], at z = x / T:
//
//   M = max x, d = (x - M) c, c = log2(e) / T, S = sum 2^d, U = sum 2^d d
//   log p(t) = (x_t - M) / T - log2 S ln 2,  H = (log2 S - U / S) ln 2
//
// One pass: each lane keeps M, S and U of what it has seen and rescales them when
// M grows (chunk by chunk of 16 or 32 values), lanes, waves and parts of a long
// row are joined in the same way. x - M is taken before the factor, so that
// logits of the type's lowest value do not overflow, and d is held at -200 where
// it is multiplied by 2^d = 0 (a masked logit of -inf).
//
// The k best: a wave keeps a list of candidates in LDS and a border that k of
// them reach; a chunk whose maximum does not reach it (nearly every one, after
// the first) costs one comparison. The border starts from the lanes' maxima of
// the first chunk. Keys are 64 bits, the value's bits in their order above the
// complement of the index, so that no two are alike and ties go to the lower
// index; candidates of all waves that reach the highest border are ranked by
// counting the larger ones.
#include <algorithm>

#include "fp8_common.hpp"
#include "row_kernels.hpp"

namespace mhsa {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kLoads = 4;  // of 16 bytes, of a lane and chunk

template <typename T> constexpr int kPer = 16 / (int)sizeof(T);            // values of a load
template <typename T> constexpr int kChunk = 64 * kLoads * kPer<T>;       // values of a wave's chunk

// The order of floats as that of unsigned integers; -0 counts as 0.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t key_of(float v, int i) { return (uint64_t)ordered(v) << 32 | (uint32_t)~i; }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

struct Stats {
  float m = kLowest, s = 0.f, u = 0.f;
  // brings the sums to maximum M
  __device__ __forceinline__ void to(float M, float c) {
    const float d = (m - M) * c, f = __builtin_amdgcn_exp2f(d);
    u = f * __builtin_fmaf(s, fmaxf(d, -200.f), u);
    s *= f;
    m = M;
  }
};

__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }

__device__ __forceinline__ Stats wave_stats(Stats a, float c) {
  a.to(wave_reduce(a.m, larger), c);
  a.s = wave_reduce(a.s, add);
  a.u = wave_reduce(a.u, add);
  return a;
}

// The largest number with the low `skip` bits clear that k of the wave's 64 R
// numbers reach (0 if fewer than k are not 0).
template <int R>
__device__ __forceinline__ uint32_t kth(const uint32_t o[R], int k, int skip) {
  uint32_t t = 0;
  for (int bit = 31; bit >= skip; --bit) {
    const uint32_t at = t | 1u << bit;
    int n = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) n += __popcll(__ballot(o[r] >= at));
    if (n >= k) t = at;
  }
  return t;
}

constexpr int kList = 128;  // up to 64 candidates, and 64 more

// A wave's candidates and border: values above `low`, or equal to it and of an
// index below `before`.
struct Best {
  uint64_t* list;
  int n, k;
  float low;
  int before;
  __device__ __forceinline__ bool in(float v, int i) const { return v > low || (v == low && i < before); }
};

// The k best of the list's n > k candidates stay.
__device__ __forceinline__ void shrink(Best& b) {
  const int lane = threadIdx.x & 63;
  uint64_t key[2];
  uint32_t hi[2], lo[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    key[r] = 64 * r + lane < b.n ? b.list[64 * r + lane] : 0;
    hi[r] = (uint32_t)(key[r] >> 32);
  }
  const uint32_t t = kth<2>(hi, b.k, 0);
  int above = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    above += __popcll(__ballot(hi[r] > t));
    lo[r] = hi[r] == t ? (uint32_t)key[r] : 0;
  }
  const uint32_t l = kth<2>(lo, b.k - above, 0);  // (complements of indices are not 0)
  int n = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const bool keep = hi[r] > t || (hi[r] == t && lo[r] >= l);
    const uint64_t mask = __ballot(keep);
    if (keep) b.list[n + __popcll(mask & (((uint64_t)1 << lane) - 1))] = key[r];
    n += __popcll(mask);
  }
  b.n = n;
  b.low = value_of(t);
  b.before = (int)~l;
}

// Ranks n keys in LDS and gives the best min(n, k) to `put(rank, key)`; `put`
// gets key 0 for ranks past n. All of `threads` threads take part.
template <typename F>
__device__ __forceinline__ void rank_keys(const uint64_t* list, int n, int k, int at, int threads, F put) {
  for (int i = at; i < n; i += threads) {
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < k) put(rank, key);
  }
  for (int i = n + at; i < k; i += threads) put(i, (uint64_t)0);
}

template <typename T>
__device__ __forceinline__ float value_at(const T* x, int i) { return (float)x[i]; }

// A row's results from its statistics (the same in all threads).
struct RowOut {
  float m, inv_t, ls;  // ls: log2 S
  bool empty;          // no logit above -inf: no token has a probability
  __device__ __forceinline__ RowOut(const Stats& a, float inv_t_)
      : m(a.m), inv_t(inv_t_), ls(__builtin_amdgcn_logf(a.s)), empty(a.s == 0.f) {}
  // (not through c: a logit of the type's lowest value stays a float)
  __device__ __forceinline__ float log_prob(float v) const {
    return empty ? -__builtin_inff() : __builtin_fmaf(v - m, inv_t, -ls * kLn2);
  }
  __device__ __forceinline__ float entropy(const Stats& a) const {
    const float h = (ls - a.u / a.s) * kLn2;
    return empty || h < 0.f ? 0.f : h;  // (a NaN stays)
  }
};

template <typename T>
__device__ __forceinline__ void write_row(const ScoresParams& p, int64_t row, const Stats& a, int at, int threads) {
  const RowOut o(a, p.inv_t);
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  if (at == 0 && p.entropy) p.entropy[row] = o.entropy(a);
  for (int i = at; i < p.nt; i += threads) {
    const int t = p.tokens[row * p.nt + i];
    p.log_probs[row * p.nt + i] = t >= 0 && t < p.V ? o.log_prob(value_at(x, t)) : 0.f;
  }
}
__device__ __forceinline__ void write_top(const ScoresParams& p, int64_t row, const RowOut& o, int rank, uint64_t key) {
  p.top[row * p.k + rank] = key ? index_of(key) : -1;
  p.top_lp[row * p.k + rank] = key ? o.log_prob(value_of((uint32_t)(key >> 32))) : -__builtin_inff();
}

// Part `part` of a row's partial results.
struct Partial {
  float m, s, u, pad;
};
__device__ __host__ inline int64_t partial_bytes(int k) { return (int64_t)sizeof(Partial) + 8 * (int64_t)k; }

// NW waves to a row, or to each of its `parts` parts; one wave: four rows to a
// workgroup.
template <typename T, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void scores_kernel(ScoresParams p, int parts, int per) {
  constexpr int WAVES = NW == 1 ? 4 : NW, E = kPer<T>, G = kLoads * E;
  __shared__ uint64_t lists[WAVES][kList];
  __shared__ uint64_t all[NW == 1 ? 1 : NW * 64];
  __shared__ float stats[WAVES][3];
  __shared__ uint32_t border[WAVES];
  __shared__ int total;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, wr = NW == 1 ? 0 : w;
  const float c = kLog2e * p.inv_t;
  const int64_t items = p.rows * parts;
  for (int64_t item = NW == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x; item < items;
       item += (int64_t)gridDim.x * (NW == 1 ? 4 : 1)) {
    const int64_t row = item / parts;
    const int part = (int)(item % parts), v0 = part * per, v1 = min(p.V, v0 + per);
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    Stats a;
    Best b{lists[w], 0, p.k, -__builtin_inff(), 0};
    bool first = true;
#pragma unroll 1
    for (int base = v0 + wr * kChunk<T>; base < v1; base += NW * kChunk<T>) {
      float v[G];
      if (base + kChunk<T> <= v1) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          T t[E];
          __builtin_memcpy(t, x + base + (u * 64 + lane) * E, sizeof t);
#pragma unroll
          for (int e = 0; e < E; ++e) v[u * E + e] = (float)t[e];
        }
      } else {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          const int at = base + (u * 64 + lane) * E;
          if (at + E <= v1) {
            T t[E];
            __builtin_memcpy(t, x + at, sizeof t);
#pragma unroll
            for (int e = 0; e < E; ++e) v[u * E + e] = (float)t[e];
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[u * E + e] = at + e < v1 ? (float)x[at + e] : -__builtin_inff();
          }
        }
      }
      float top = v[0];
#pragma unroll
      for (int i = 1; i < G; ++i) top = fmaxf(top, v[i]);
      a.to(fmaxf(a.m, top), c);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const float d = (v[i] - a.m) * c, e = __builtin_amdgcn_exp2f(d);
        a.s += e;
        a.u = __builtin_fmaf(e, fmaxf(d, -200.f), a.u);
      }
      if (p.k == 0) continue;
      if (!(top > -__builtin_inff())) top = -__builtin_inff();  // (all of them NaN)
      if (first) {
        // 16 bits are enough of a border, and any lower one is right
        const uint32_t o[1] = {ordered(top)};
        const float t = value_of(kth<1>(o, p.k, 16));
        if (t > -__builtin_inff()) b.low = t, b.before = 0x7FFFFFFF;
        first = false;
      }
      if (__ballot(b.in(top, base + lane * E)) == 0) continue;
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < G; ++i)
        bits |= b.in(v[i], base + (i / E * 64 + lane) * E + i % E) ? 1u << i : 0;
      while (__ballot(bits != 0)) {
        const int i = __builtin_ctz(bits | 1u << 31), at = base + (i / E * 64 + lane) * E + i % E;
        // (read again: registers have no index)
        const float vi = bits ? value_at(x, at) : -__builtin_inff();
        const bool in = bits && b.in(vi, at);
        const uint64_t mask = __ballot(in);
        if (in) b.list[b.n + __popcll(mask & (((uint64_t)1 << lane) - 1))] = key_of(vi, at);
        b.n += __popcll(mask);
        bits &= bits - 1;
        if (b.n > 64) shrink(b);
      }
    }
    a = wave_stats(a, c);
    if constexpr (NW == 1) {
      write_row<T>(p, row, a, lane, 64);
      if (p.k) {
        const RowOut o(a, p.inv_t);
        rank_keys(b.list, b.n, p.k, lane, 64, [&](int rank, uint64_t key) { write_top(p, row, o, rank, key); });
      }
    } else {
      if (p.k) {
        const uint64_t mine = lane < b.n ? b.list[lane] : 0;
        const uint32_t o[1] = {(uint32_t)(mine >> 32)};
        const uint32_t t = kth<1>(o, p.k, 16);
        if (lane == 0) border[w] = t;
      }
      if (lane == 0) stats[w][0] = a.m, stats[w][1] = a.s, stats[w][2] = a.u;
      if (threadIdx.x == 0) total = 0;
      __syncthreads();
      Stats r;
      if (lane < NW) r.m = stats[lane][0], r.s = stats[lane][1], r.u = stats[lane][2];
      r = wave_stats(r, c);
      if (p.k) {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) t = max(t, border[i]);
        const uint64_t mine = lane < b.n ? b.list[lane] : 0;
        const bool in = mine != 0 && (uint32_t)(mine >> 32) >= t;
        const uint64_t mask = __ballot(in);
        int at = 0;
        if (lane == 0 && mask) at = atomicAdd(&total, __popcll(mask));
        at = __builtin_amdgcn_readfirstlane(at);
        if (in) all[at + __popcll(mask & (((uint64_t)1 << lane) - 1))] = mine;
        __syncthreads();
      }
      if (parts == 1) {
        write_row<T>(p, row, r, threadIdx.x, NW * 64);
        if (p.k) {
          const RowOut o(r, p.inv_t);
          rank_keys(all, total, p.k, threadIdx.x, NW * 64, [&](int rank, uint64_t key) { write_top(p, row, o, rank, key); });
        }
      } else {
        char* to = static_cast<char*>(p.ws) + item * partial_bytes(p.k);
        if (threadIdx.x == 0) *reinterpret_cast<Partial*>(to) = Partial{r.m, r.s, r.u, 0.f};
        uint64_t* keys = reinterpret_cast<uint64_t*>(to + sizeof(Partial));
        if (p.k) rank_keys(all, total, p.k, threadIdx.x, NW * 64, [&](int rank, uint64_t key) { keys[rank] = key; });
      }
      __syncthreads();
    }
  }
}

constexpr int kMaxParts = 16;

// The parts of long rows joined, a wave to a row.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(ScoresParams p, int parts) {
  __shared__ uint64_t lists[4][kMaxParts * kScoresMaxK];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const float c = kLog2e * p.inv_t;
  for (int64_t row = (int64_t)blockIdx.x * 4 + w; row < p.rows; row += (int64_t)gridDim.x * 4) {
    const int64_t pb = partial_bytes(p.k);
    const char* from = static_cast<const char*>(p.ws) + row * parts * pb;
    Stats a;
    if (lane < parts) {
      const Partial q = *reinterpret_cast<const Partial*>(from + lane * pb);
      a.m = q.m, a.s = q.s, a.u = q.u;
    }
    a = wave_stats(a, c);
    write_row<T>(p, row, a, lane, 64);
    if (p.k) {
      auto key = [&](int part, int i) { return reinterpret_cast<const uint64_t*>(from + part * pb + sizeof(Partial))[i]; };
      // the highest of the parts' k-th best
      uint32_t t = lane < parts ? (uint32_t)(key(lane, p.k - 1) >> 32) : 0;
      t = wave_reduce(t, [](uint32_t x, uint32_t y) { return max(x, y); });
      int n = 0;
      for (int i = lane; i < (parts * p.k + 63) / 64 * 64; i += 64) {
        const uint64_t mine = i < parts * p.k ? key(i / p.k, i % p.k) : 0;
        const bool in = mine != 0 && (uint32_t)(mine >> 32) >= t;
        const uint64_t mask = __ballot(in);
        if (in) lists[w][n + __popcll(mask & (((uint64_t)1 << lane) - 1))] = mine;
        n += __popcll(mask);
      }
      const RowOut o(a, p.inv_t);
      rank_keys(lists[w], n, p.k, lane, 64, [&](int rank, uint64_t k) { write_top(p, row, o, rank, k); });
    }
  }
}

struct Plan {
  int waves = 1, parts = 1, per = 0;
};

int64_t max_parts(int V) { return std::clamp<int64_t>(V / 16384, 1, kMaxParts); }

Plan plan_of(int64_t rows, int V) {
  Plan q;
  q.per = V;
  if (V <= 4096) return q;
  q.waves = 8;
  // parts of 16384 values or more while there are fewer of them than 2 to a CU
  const int64_t most = max_parts(V);
  while (q.parts < most && rows * q.parts < 2 * device_cus()) ++q.parts;
  q.per = ((V + q.parts - 1) / q.parts + 63) / 64 * 64;
  return q;
}

template <typename T>
hipError_t go(const ScoresParams& p, hipStream_t s) {
  const Plan q = plan_of(p.rows, p.V);
  if (q.parts > 1 && !p.ws) return hipErrorInvalidValue;
  if (q.waves == 1) {
    const unsigned grid = (unsigned)std::min<int64_t>((p.rows + 3) / 4, 1 << 20);
    scores_kernel<T, 1><<<grid, 256, 0, s>>>(p, 1, p.V);
  } else {
    const unsigned grid = (unsigned)std::min<int64_t>(p.rows * q.parts, 1 << 20);
    scores_kernel<T, 8><<<grid, 512, 0, s>>>(p, q.parts, q.per);
    if (q.parts > 1) join_kernel<T><<<(unsigned)((p.rows + 3) / 4), 256, 0, s>>>(p, q.parts);
  }
  return hipGetLastError();
}

}  // namespace

// (for any number of rows up to `rows`: r rows in p parts have r p < 2 CUs + r
// and p <= most, and none have parts from 2 CUs on)
int64_t scores_workspace(int64_t rows, int V, int k) {
  const int64_t most = max_parts(V), want = 2 * device_cus(), r = std::min(rows, want - 1);
  return most > 1 ? std::min(r * most, want - 1 + r) * partial_bytes(k) : 0;
}

hipError_t token_scores(const ScoresParams& p, hipStream_t s) {
  if (p.rows <= 0 || p.V <= 0 || p.V > kScoresMaxV || p.k < 0 || p.k > kScoresMaxK || p.k > p.V || p.nt < 0 || !p.x ||
      (p.nt && (!p.tokens || !p.log_probs)) || (p.k && (!p.top || !p.top_lp)))
    return hipErrorInvalidValue;
  return p.dt == kBF16 ? go<bf16>(p, s) : go<float>(p, s);
}

}  // namespace mhsa
