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
// The k best. Keys are 64 bits, a value's bits in their order above the
// complement of its index, so that no two are alike and ties go to the lower
// index. Each of NW waves keeps a list of candidates in LDS, and in LDS for all to
// see a key that q = ceil(k / NW) of its values reach; k of the row then reach the
// ceil(k / q)-th largest of these keys, and a value below it is none of the k
// best. A chunk whose maximum is below costs one comparison. The keys start from
// the lanes' maxima of the first chunk and rise with the lists; they are read
// without a barrier, for an old one is only lower. (With a border of each wave's
// own there were three times as many candidates, 140 of 16384 values for 20 best,
// and ranking them took longer than reading the row.) At the end the candidates that reach the border, and
// then those of a long row's parts, are ranked by counting the larger ones. Rows
// of up to 8 loads to a lane stay in one wave's registers as a single chunk.
//
// Bound: HBM over long rows of many (4001 x 50001 f32, 5 best: 146 us, 5.5 TB/s),
// else the vector unit (15 instructions a value there, 27 in short rows) and the
// candidates' bookkeeping, some 500 of a wave and one chain of LDS reads:
// 3000 x 9848 f32 take 21 us without the k best (5.6 TB/s), 29 with 5, 34 with 20;
// 64 x 128000 bf16, 20 best, 16.5, of which the join of the parts is 5.
#include <algorithm>

#include "fp8_common.hpp"
#include "row_kernels.hpp"

namespace mhsa {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kLoads = 4;  // of 16 bytes, of a lane and chunk

template <typename T> constexpr int kPer = 16 / (int)sizeof(T);  // values of a load

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
// numbers reach (0 if fewer than k are not 0), two bits at a time.
template <int R>
__device__ __forceinline__ uint32_t kth(const uint32_t o[R], int k, int skip) {
  uint32_t t = 0;
  for (int bit = 30; bit >= skip; bit -= 2) {
    int n[3] = {0, 0, 0};
#pragma unroll
    for (uint32_t q = 1; q < 4; ++q)
#pragma unroll
      for (int r = 0; r < R; ++r) n[q - 1] += __popcll(__ballot(o[r] >= (t | q << bit)));
    t |= (uint32_t)((n[0] >= k) + (n[1] >= k) + (n[2] >= k)) << bit;
  }
  return t;
}

constexpr int kList = 128;  // up to 64 candidates, and 64 more

// A wave's candidates, and its border: keys below it are not looked at. A border
// of no index (kAnyIndex) takes all values that are equal to its own.
constexpr uint32_t kAnyIndex = 0x80000000u;
struct Best {
  uint64_t* list;
  int k = 0, n = 0;
  float low = -__builtin_inff();  // values above it, or equal and of an index under `before`
  int before = 0;
  uint64_t key = 0;
  __device__ __forceinline__ void raise(uint64_t to) {
    if (to <= key) return;
    key = to;
    const uint32_t hi = (uint32_t)(to >> 32), lo = (uint32_t)to;
    if (hi <= ordered(-__builtin_inff())) return;  // (logits of -inf are none)
    low = value_of(hi);
    before = lo == kAnyIndex ? 0x7FFFFFFF : (int)~lo + 1;
  }
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
  const uint64_t least = (uint64_t)t << 32 | l;
  int n = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const bool keep = key[r] >= least;
    const uint64_t mask = __ballot(keep);
    if (keep) b.list[n + __popcll(mask & (((uint64_t)1 << lane) - 1))] = key[r];
    n += __popcll(mask);
  }
  b.n = n;
  b.raise(least);
}

// A key that `nth` of the list's up to 64 candidates reach, 0 if there are not so
// many: 16 bits of a value are enough, and the last index of that very value.
__device__ __forceinline__ uint64_t reached(const Best& b, int nth) {
  const int lane = threadIdx.x & 63;
  if (b.n < nth) return 0;
  const uint64_t key = lane < b.n ? b.list[lane] : 0;
  const uint32_t hi[1] = {(uint32_t)(key >> 32)};
  const uint32_t t = kth<1>(hi, nth, 16);
  const uint32_t lo = wave_reduce(hi[0] == t ? (uint32_t)key : ~0u, [](uint32_t x, uint32_t y) { return min(x, y); });
  return (uint64_t)t << 32 | lo;
}

// Value i of the words that a lane has loaded.
template <typename T>
__device__ __forceinline__ float unpack(const uint32_t* raw, int i) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, raw[i]);
  else return __builtin_bit_cast(float, i % 2 ? raw[i / 2] & 0xFFFF0000u : raw[i / 2] << 16);
}
// The place-th largest (from 1) of the keys of lanes 0 to N - 1, of which equal
// ones count as one behind the other.
template <int N>
__device__ __forceinline__ uint64_t nth_largest(uint64_t key, int place) {
  const int lane = threadIdx.x & 63, lo = (int)(uint32_t)key, hi = (int)(key >> 32);
  int rank = 1;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, j) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, j);
    rank += other > key || (other == key && j < lane);
  }
  const int at = __builtin_ctzll(__ballot(lane < N && rank == place));
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, at) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, at);
}

// Ranks the n keys in LDS and gives the best min(n, k) to `put(rank, key)`, and
// key 0 for the ranks past n. One wave.
template <typename F>
__device__ __forceinline__ void rank_keys(const uint64_t* list, int n, int k, F put) {
  const int lane = threadIdx.x & 63;
  if (n <= 64) {
    const uint64_t key = lane < n ? list[lane] : 0;
    const int lo = (int)(uint32_t)key, hi = (int)(key >> 32);
    int rank = 0;
    for (int j = 0; j < n; ++j) {
      const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, j) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, j);
      rank += other > key;
    }
    if (lane < n && rank < k) put(rank, key);
  } else {
    for (int i = lane; i < n; i += 64) {
      const uint64_t key = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[j] > key;
      if (rank < k) put(rank, key);
    }
  }
  if (n + lane < k) put(n + lane, (uint64_t)0);
}

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

// A wave's log probabilities of given tokens and the entropy. The first 64 tokens'
// logits are on their way from the beginning.
template <typename T> struct Given {
  int t = -1;
  float v = 0.f;
  __device__ __forceinline__ void fetch(const ScoresParams& p, int64_t row, int i) {
    t = i < p.nt ? p.tokens[row * p.nt + i] : -1;
    if (t >= p.V) t = -1;
    v = (float)(static_cast<const T*>(p.x) + row * p.ld)[max(t, 0)];
  }
};
template <typename T>
__device__ __forceinline__ void write_row(const ScoresParams& p, int64_t row, const Stats& a, Given<T> g) {
  const RowOut o(a, p.inv_t);
  const int lane = threadIdx.x & 63;
  if (lane == 0 && p.entropy) p.entropy[row] = o.entropy(a);
  for (int i = lane; i < p.nt; i += 64) {
    if (i >= 64) g.fetch(p, row, i);
    p.log_probs[row * p.nt + i] = g.t >= 0 ? o.log_prob(g.v) : 0.f;
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

// L loads of a lane from x + base on (values up to v1, the first FULL loads of all
// lanes below it) as they lie in memory, into the statistics; the largest value.
// A lane whose load would pass the end of the row (of V >= kPer values, or TINY)
// loads the row's last values, and what is not its own, or past v1, is -inf: no
// branch keeps a load waiting for another.
template <typename T, int L, int FULL, bool TINY = false>
__device__ __forceinline__ float load_chunk(const T* x, int base, int v1, int V, float c, uint32_t raw[4 * L], Stats& a) {
  constexpr int E = kPer<T>;
  const int lane = threadIdx.x & 63;
  if constexpr (TINY) {
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = x[min(base + lane * E + e, V - 1)];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (base + lane * E + e >= V) t[e] = (T)-__builtin_inff();
    __builtin_memcpy(raw, t, 16);
  } else {
#pragma unroll
    for (int u = 0; u < L; ++u) {
      const int at = base + (u * 64 + lane) * E;
      __builtin_memcpy(raw + 4 * u, x + (u < FULL ? at : min(at, V - E)), 16);
    }
#pragma unroll
    for (int u = FULL; u < L; ++u) {
      const int from = base + (u * 64 + lane + 1) * E - v1;  // values that are not its own, if positive
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t& r = raw[4 * u + i];
        if constexpr (sizeof(T) == 4) r = from > i ? 0xFF800000u : r;
        else r = from > 2 * i + 1 ? 0xFF80FF80u : from > 2 * i ? (r & 0xFFFF0000u) | 0xFF80u : r;
      }
    }
  }
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < L * E; ++i) top = fmaxf(top, unpack<T>(raw, i));  // (a NaN does not count)
  a.to(fmaxf(a.m, top), c);
#pragma unroll
  for (int i = 0; i < L * E; ++i) {
    const float d = (unpack<T>(raw, i) - a.m) * c, e = __builtin_amdgcn_exp2f(d);
    a.s += e;
    a.u = __builtin_fmaf(e, fmaxf(d, -200.f), a.u);
  }
  return top;
}

// Whether a chunk may have candidates.
template <typename T>
__device__ __forceinline__ bool any_candidate(const Best& b, int base, float top) {
  return __ballot(top > b.low || (top == b.low && base + (int)(threadIdx.x & 63) * kPer<T> < b.before)) != 0;
}

// Those that the border lets through join the list, one of each lane at a time;
// `stash` (LDS of the wave) takes the chunk, for registers have no index. `last`:
// where the row's last load begins.
template <typename T, int L>
__device__ __forceinline__ void collect(Best& b, int base, int last, const uint32_t raw[4 * L], T* stash) {
  constexpr int E = kPer<T>, G = L * E;
  const int lane = threadIdx.x & 63;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  const float low = fmaxf(b.low, kLowest);  // (-inf is never one)
  typedef std::conditional_t<(G > 32), uint64_t, uint32_t> Bits;
  Bits bits = 0;
#pragma unroll
  for (int i = G - 1; i >= 0; --i) bits = bits + bits + (unpack<T>(raw, i) >= low);
#pragma unroll
  for (int u = 0; u < L; ++u)
    *reinterpret_cast<u32x4*>(stash + (u * 64 + lane) * E) = u32x4{raw[4 * u], raw[4 * u + 1], raw[4 * u + 2], raw[4 * u + 3]};
  while (__ballot(bits != 0)) {
    const int i = bits ? __builtin_ctzll((uint64_t)bits) : 0, load = (i / E * 64 + lane) * E;
    const float v = (float)stash[load + i % E];
    const int at = min(base + load, last) + i % E;
    const bool in = bits && (v > b.low || (v == b.low && at < b.before));
    const uint64_t mask = __ballot(in);
    if (in) b.list[b.n + __popcll(mask & below)] = key_of(v, at);
    b.n += __popcll(mask);
    bits &= bits - 1;
    if (b.n > 64) shrink(b);
  }
}

// The border that k values of the wave's lanes' largest ones reach.
__device__ __forceinline__ uint64_t lanes_border(float top, int k) {
  const uint32_t o[1] = {ordered(top)};
  const uint32_t t = kth<1>(o, k, 16);  // (16 bits are enough, and any lower one is right)
  return t > ordered(-__builtin_inff()) ? (uint64_t)t << 32 | kAnyIndex : 0;
}

// Rows of L loads to a lane, a wave to each. (bf16 rows of 6 to 8 loads take 132 to
// 172 registers, values unpacked, and run 3 and 2 waves a SIMD.)
template <typename T, int L>
__global__ __launch_bounds__(256) void scores_small_kernel(ScoresParams p) {
  __shared__ uint64_t lists[4][kList];
  __shared__ __attribute__((aligned(16))) T stash[4][64 * L * kPer<T>];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float c = kLog2e * p.inv_t;
  const int64_t row = (int64_t)blockIdx.x * 4 + w;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  Given<T> given;
  given.fetch(p, row, lane);
  Stats a;
  uint32_t raw[4 * L];
  const bool tiny = L == 1 && p.V < kPer<T>;
  const float top = tiny ? load_chunk<T, 1, 0, true>(x, 0, p.V, p.V, c, raw, a) : load_chunk<T, L, L - 1>(x, 0, p.V, p.V, c, raw, a);
  a = wave_stats(a, c);
  write_row(p, row, a, given);
  if (p.k == 0) return;
  Best b{lists[w]};
  b.k = p.k;
  b.raise(lanes_border(top, p.k));
  if (any_candidate<T>(b, 0, top)) collect<T, L>(b, 0, tiny ? 0 : p.V - kPer<T>, raw, stash[w]);
  const RowOut o(a, p.inv_t);
  rank_keys(b.list, b.n, p.k, [&](int rank, uint64_t key) { write_top(p, row, o, rank, key); });
}

// NW waves to a row, or to each of its `parts` parts of `per` values. Registers for 6
// waves a SIMD, which costs one of bf16 a place in scratch (30000 rows of 5000, 5
// best: 104 us; with 100 registers, 4 waves a SIMD, 122, and without the k best of
// 4001 x 50001 89 instead of 97).
template <typename T, int NW>
__global__ __launch_bounds__(NW * 64, 6) void scores_kernel(ScoresParams p, int parts, int per) {
  constexpr int E = kPer<T>, L = kLoads, CHUNK = 64 * L * E;
  static_assert(L == 4, "the parts of a chunk");
  __shared__ uint64_t lists[NW][kList];
  __shared__ uint64_t all[NW * 64];
  __shared__ __attribute__((aligned(16))) T stash[NW][CHUNK];
  __shared__ float stats[NW][3];
  __shared__ int found[NW];
  __shared__ uint64_t border[NW];  // of each wave
  __shared__ int total;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float c = kLog2e * p.inv_t;
  const int nth = (p.k + NW - 1) / NW, place = p.k ? (p.k + nth - 1) / nth : 0;
  const int64_t item = blockIdx.x;
  const int64_t row = item / parts;
  // a wave's values, as many as another's: with chunks dealt out in turn the last
  // wave's few values gave a border far too low (128 rows x 50000 bf16, 20 best, by
  // eight waves: 37 us instead of 13)
  const int p0 = (int)(item % parts) * per, p1 = min(p.V, p0 + per), each = ((p1 - p0 + NW - 1) / NW + E - 1) / E * E;
  const int v0 = min(p1, p0 + w * each), v1 = min(p1, v0 + each);
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  Given<T> given;
  if (parts == 1 && w == NW - 1) given.fetch(p, row, lane);
  Stats a;
  Best b{lists[w]};
  b.k = p.k;
  auto common = [&]() {
    const uint64_t mine =
        lane < NW ? __hip_atomic_load(&border[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : (uint64_t)0;
    return nth_largest<NW>(mine, place);
  };
  auto publish = [&]() {
    const uint64_t key = reached(b, nth);
    if (lane == 0 && key > border[w]) __hip_atomic_store(&border[w], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  int known = 0;  // candidates when the wave's border was last made
  bool first = true;
#pragma unroll 1
  for (int base = v0; base < v1; base += CHUNK) {
    uint32_t raw[4 * L];
    float top;
    auto part = [&](auto loads) {
      constexpr int M = decltype(loads)::value;
#pragma unroll
      for (int i = 4 * M; i < 4 * L; ++i) raw[i] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
      top = load_chunk<T, M, M - 1>(x, base, v1, p.V, c, raw, a);
    };
    if (base + CHUNK <= v1) top = load_chunk<T, L, L>(x, base, v1, p.V, c, raw, a);
    else if (base + 3 * 64 * E < v1) part(std::integral_constant<int, 4>());
    else if (base + 2 * 64 * E < v1) part(std::integral_constant<int, 3>());
    else if (base + 64 * E < v1) part(std::integral_constant<int, 2>());
    else part(std::integral_constant<int, 1>());
    if (p.k == 0) continue;
    uint64_t key = 0;
    if (first) {  // (every wave has values)
      // the wave's own border where another's values do not reach one, as in a mask
      // that leaves one stretch (3000 x 9848 f32, 7 of 8 ruled out: 42 -> 24 us)
#pragma unroll 1
      for (int turn = 0; turn < 2 && key == 0; ++turn) {
        key = lanes_border(top, turn ? p.k : nth);
        if (turn) break;
        if (lane == 0) border[w] = key;
        __syncthreads();
        key = common();
      }
    } else {
      if (!any_candidate<T>(b, base, top)) continue;
      key = common();
    }
    b.raise(key);
    if (any_candidate<T>(b, base, top)) {
      collect<T, L>(b, base, p.V - E, raw, stash[w]);
      if (first) {
        known = b.n;
      } else if (b.n < known || 2 * b.n >= 3 * known + 2) {  // (a new border costs more than a candidate)
        if (base + CHUNK < v1) publish();
        known = b.n;
      }
    }
    first = false;
  }

  a = wave_stats(a, c);
  if (lane == 0) stats[w][0] = a.m, stats[w][1] = a.s, stats[w][2] = a.u, found[w] = b.n;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  Stats r;
  if (lane < NW) r.m = stats[lane][0], r.s = stats[lane][1], r.u = stats[lane][2];
  r = wave_stats(r, c);
  int n = 0;
  if (p.k) {
    const uint64_t mine = lane < b.n ? b.list[lane] : 0;
    int before = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      before += i < w ? found[i] : 0;
      n += found[i];
    }
    if (n <= 64) {
      if (mine) all[before + lane] = mine;
    } else {  // more than a wave ranks at once: those that reach the border
      publish();
      __syncthreads();
      const uint64_t least = common();
      const bool in = mine != 0 && ((uint32_t)least == kAnyIndex ? mine >> 32 >= least >> 32 : mine >= least);
      const uint64_t mask = __ballot(in);
      int at = 0;
      if (lane == 0 && mask) at = atomicAdd(&total, __popcll(mask));
      at = __builtin_amdgcn_readfirstlane(at);
      if (in) all[at + __popcll(mask & (((uint64_t)1 << lane) - 1))] = mine;
    }
    __syncthreads();
    if (n > 64) n = total;
  }
  if (parts == 1) {
    if (w == NW - 1) write_row(p, row, r, given);
    if (p.k && w == 0) {
      const RowOut o(r, p.inv_t);
      rank_keys(all, n, p.k, [&](int rank, uint64_t key) { write_top(p, row, o, rank, key); });
    }
  } else {
    char* to = static_cast<char*>(p.ws) + item * partial_bytes(p.k);
    if (threadIdx.x == 0) *reinterpret_cast<Partial*>(to) = Partial{r.m, r.s, r.u, 0.f};
    uint64_t* keys = reinterpret_cast<uint64_t*>(to + sizeof(Partial));
    if (p.k && w == 0) rank_keys(all, n, p.k, [&](int rank, uint64_t key) { keys[rank] = key; });
  }
}

constexpr int kMaxParts = 16;

// The parts of long rows joined, a wave to a row; everything is read at once.
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(ScoresParams p, int parts) {
  constexpr int PER = kMaxParts * kScoresMaxK / 64;
  __shared__ uint64_t list[kMaxParts * kScoresMaxK];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x, pb = partial_bytes(p.k);
  const char* from = static_cast<const char*>(p.ws) + row * parts * pb;
  Given<T> given;
  given.fetch(p, row, lane);
  Stats a;
  uint64_t key[PER];
  if (lane < parts) {
    const Partial q = *reinterpret_cast<const Partial*>(from + lane * pb);
    a.m = q.m, a.s = q.s, a.u = q.u;
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = 64 * u + lane;
    key[u] = 0;
    if (64 * u < parts * p.k && i < parts * p.k)
      key[u] = reinterpret_cast<const uint64_t*>(from + i / p.k * pb + sizeof(Partial))[i % p.k];
  }
  // the parts' borders (a part's keys are in order)
  const int nth = p.k ? (p.k + parts - 1) / parts : 1, place = (p.k + nth - 1) / nth;
  const uint64_t best = p.k && lane < parts ? reinterpret_cast<const uint64_t*>(from + lane * pb + sizeof(Partial))[nth - 1] : 0;
  a = wave_stats(a, kLog2e * p.inv_t);
  write_row(p, row, a, given);
  if (p.k == 0) return;
  const uint64_t least = nth_largest<kMaxParts>(best, place);
  int n = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const bool in = key[u] != 0 && key[u] >= least;
    const uint64_t mask = __ballot(in);
    if (in) list[n + __popcll(mask & (((uint64_t)1 << lane) - 1))] = key[u];
    n += __popcll(mask);
  }
  const RowOut o(a, p.inv_t);
  rank_keys(list, n, p.k, [&](int rank, uint64_t k) { write_top(p, row, o, rank, k); });
}

int64_t max_parts(int V) { return std::clamp<int64_t>(V / 4096, 1, kMaxParts); }

// Fewer rows than 2 to a CU are cut into parts of 4096 values or more, of which
// there are about 4 to a CU: with 2 to a CU 400 rows of 100000 f32, 20 best, take 44
// us instead of 40 and 300 of 30000 bf16 18.3 instead of 16.7 (64 of 128000 alike).
// Eight waves to a part instead of four, 2 to a CU: 48, 18.9.
int64_t parts_of(int64_t rows, int V) {
  const int64_t cus = device_cus();
  return rows >= 2 * cus ? 1 : std::clamp<int64_t>((4 * cus + rows - 1) / rows, 1, max_parts(V));
}

template <typename T>
hipError_t go(const ScoresParams& p, hipStream_t s) {
  const int loads = (p.V + 64 * kPer<T> - 1) / (64 * kPer<T>);
  if (loads <= 8) {
    const unsigned grid = (unsigned)((p.rows + 3) / 4);
    auto run = [&](auto l) { scores_small_kernel<T, decltype(l)::value><<<grid, 256, 0, s>>>(p); };
    using std::integral_constant;
    switch (loads) {
      case 1: run(integral_constant<int, 1>()); break;
      case 2: run(integral_constant<int, 2>()); break;
      case 3: run(integral_constant<int, 3>()); break;
      case 4: run(integral_constant<int, 4>()); break;
      case 5: run(integral_constant<int, 5>()); break;
      case 6: run(integral_constant<int, 6>()); break;
      case 7: run(integral_constant<int, 7>()); break;
      default: run(integral_constant<int, 8>()); break;
    }
    return hipGetLastError();
  }
  const int parts = (int)parts_of(p.rows, p.V), per = ((p.V + parts - 1) / parts + 63) / 64 * 64;
  // every wave has values (they take a multiple of kPer each, the last what is left)
  if (p.V - (parts - 1) * per <= 16 * kPer<T>) return hipErrorInvalidValue;
  if (parts > 1) {
    if (!p.ws) return hipErrorInvalidValue;
    scores_kernel<T, 4><<<(unsigned)(p.rows * parts), 256, 0, s>>>(p, parts, per);
    join_kernel<T><<<(unsigned)p.rows, 64, 0, s>>>(p, parts);
    return hipGetLastError();
  }
  // Waves by the vocabulary alone: two up to 32 loads a lane, four beyond. 30000
  // rows of 5000 bf16, 20 best, took 132 us with two waves, 172 with four, 407 with
  // eight; 4001 of 50001 f32, 5 best, 154, 145 and 144; 771 of 20000 f32, 20 best,
  // 28, 21, 27. Rows that are not cut into parts so have the same bits however many
  // come with them; those of fewer than 2 to a CU, of 8192 values or more, are summed
  // in as many parts as their number gives.
  constexpr int64_t most = 1 << 22;  // rows of a launch: a grid's threads fit 32 bits
  for (int64_t r = 0; r < p.rows; r += most) {
    ScoresParams q = p;
    q.rows = std::min(most, p.rows - r);
    q.x = static_cast<const T*>(p.x) + r * p.ld;
    q.tokens = p.tokens ? p.tokens + r * p.nt : nullptr;
    q.log_probs = p.log_probs ? p.log_probs + r * p.nt : nullptr;
    q.entropy = p.entropy ? p.entropy + r : nullptr;
    q.top = p.top ? p.top + r * p.k : nullptr;
    q.top_lp = p.top_lp ? p.top_lp + r * p.k : nullptr;
    if (loads <= 32) scores_kernel<T, 2><<<(unsigned)q.rows, 128, 0, s>>>(q, 1, per);
    else scores_kernel<T, 4><<<(unsigned)q.rows, 256, 0, s>>>(q, 1, per);
  }
  return hipGetLastError();
}

}  // namespace

// (for any number of rows up to `rows`: r rows in p parts have r p < 4 CUs + r
// and p <= most, and none have parts from 2 CUs on)
int64_t scores_workspace(int64_t rows, int V, int k) {
  const int64_t most = max_parts(V), cus = device_cus(), r = std::min(rows, 2 * cus - 1);
  return most > 1 ? std::min(r * most, 4 * cus - 1 + r) * partial_bytes(k) : 0;
}

hipError_t token_scores(const ScoresParams& p, hipStream_t s) {
  if (p.rows <= 0 || p.V <= 0 || p.V > kScoresMaxV || p.k < 0 || p.k > kScoresMaxK || p.k > p.V || p.nt < 0 || !p.x ||
      (p.nt && (!p.tokens || !p.log_probs)) || (p.k && (!p.top || !p.top_lp)))
    return hipErrorInvalidValue;
  return p.dt == kBF16 ? go<bf16>(p, s) : go<float>(p, s);
}

}  // namespace mhsa
