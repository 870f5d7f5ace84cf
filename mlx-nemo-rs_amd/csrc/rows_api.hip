// C ABI of the operators on rows: a residual's addition with its norm, and the
// log probabilities of tokens. Neither has a handle; what they need beside
// their tensors the caller passes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "api_common.hpp"
#include "fp8_kernels.hpp"
#include "row_kernels.hpp"

namespace {

// Rows of n elements of es bytes, ld elements apart.
struct Rows {
  const void* p;
  int64_t n, ld, es;
  int64_t bytes(int64_t rows) const { return p ? ((rows - 1) * ld + n) * es : 0; }
};
bool share(const Rows& a, const Rows& b, int64_t rows) {
  return a.p && b.p && rows_overlap(a.p, a.n * a.es, a.ld * a.es, b.p, b.n * b.es, b.ld * b.es, rows);
}
// The same rows: an element is read before it is written, by one thread.
bool same(const Rows& a, const Rows& b) { return a.p == b.p && a.ld == b.ld && a.es == b.es; }
bool misaligned(const void* p, int64_t es) { return reinterpret_cast<uintptr_t>(p) % es != 0; }

}  // namespace

extern "C" int32_t mhsa_add_norm(const void* x, int32_t dtype, int32_t rows, int32_t dim, int64_t x_stride, const void* delta,
                                 int64_t delta_stride, float delta_scale, void* sum, int64_t sum_stride, int32_t kind,
                                 const float* weight, const float* bias, float eps, void* out, int32_t out_dtype,
                                 int64_t out_stride, uint8_t* codes, uint8_t* scales, void* hs) {
  mhsa::NormParams p;
  if (!act_dtype(dtype, &p.dt)) return fail(MHSA_ENOTSUP, "dtype %d not supported (f32, bf16)", dtype);
  if (out && !act_dtype(out_dtype, &p.out_dt)) return fail(MHSA_ENOTSUP, "dtype %d not supported (f32, bf16)", out_dtype);
  if (kind != MHSA_NORM_RMS && kind != MHSA_NORM_LAYER) return fail(MHSA_ENOTSUP, "norm %d not supported (rms, layer)", kind);
  if (rows < 0 || dim <= 0) return fail(MHSA_EINVAL, "bad shape: %d rows of %d", rows, dim);
  if (dim > mhsa::kNormMaxD) return fail(MHSA_ENOTSUP, "dim %d exceeds %d", dim, mhsa::kNormMaxD);
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(MHSA_EINVAL, "eps must be finite and not negative");
  if (!std::isfinite(delta_scale)) return fail(MHSA_EINVAL, "delta_scale must be finite");
  if (rows == 0) return MHSA_OK;
  if (!x || (!sum && !out && !codes)) return fail(MHSA_EINVAL, "null tensor pointer");
  if (!codes != !scales) return fail(MHSA_EINVAL, "codes and scales are to be given together");
  if (rows > kMaxRows) return fail(MHSA_ENOTSUP, "%d rows exceed %d", rows, kMaxRows);
  const int64_t es = mhsa::dtype_size(p.dt), os = out ? mhsa::dtype_size(p.out_dt) : 4;
  const Rows tx{x, dim, x_stride, es}, td{delta, dim, delta_stride, es}, ts{sum, dim, sum_stride, es}, to{out, dim, out_stride, os};
  for (const Rows& t : {tx, td, ts, to}) {
    if (!t.p) continue;
    if (t.ld < dim) return fail(MHSA_EINVAL, "row stride %lld is shorter than a row (%d)", (long long)t.ld, dim);
    if (t.ld > kMaxStride) return fail(MHSA_ENOTSUP, "row stride %lld exceeds 2^30", (long long)t.ld);
    if (misaligned(t.p, t.es)) return fail(MHSA_EINVAL, "device tensors must be aligned to their elements");
  }
  if (misaligned(weight, 4) || misaligned(bias, 4)) return fail(MHSA_EINVAL, "weight and bias must be aligned to their elements");
  if (misaligned(codes, 16) || misaligned(scales, 16)) return fail(MHSA_EINVAL, "codes and scales must be 16-byte aligned");
  const int64_t nc = codes ? rows * mhsa::fp8_kp(dim) : 0, ns = codes ? rows * mhsa::fp8_kbp(dim) : 0;
  bool bad = share(ts, to, rows);
  for (const Rows& in : {tx, td}) {
    bad |= share(ts, in, rows) && !same(ts, in);
    bad |= share(to, in, rows) && !same(to, in);
  }
  bad |= overlap(codes, nc, scales, ns);
  for (const Rows& t : {tx, td, ts, to})
    bad |= t.p && (overlap(codes, nc, t.p, t.bytes(rows)) || overlap(scales, ns, t.p, t.bytes(rows)));
  for (const float* t : {weight, bias}) {
    const int64_t n = t ? dim * 4 : 0;
    bad |= overlap(codes, nc, t, n) || overlap(scales, ns, t, n) || overlap(sum, ts.bytes(rows), t, n) ||
           overlap(out, to.bytes(rows), t, n);
  }
  if (bad) return fail(MHSA_EINVAL, "results must not overlap another tensor, but sum and out may be x or delta");
  p.x = x;
  p.ldx = x_stride;
  p.delta = delta;
  p.ldd = delta_stride;
  p.scale = delta_scale;
  p.sum = sum;
  p.lds = sum_stride;
  p.rows = rows;
  p.D = dim;
  p.layer = kind == MHSA_NORM_LAYER;
  p.w = weight;
  p.b = bias;
  p.eps = eps;
  p.out = out;
  p.ldo = out_stride;
  p.codes = codes;
  p.scales = scales;
  HIPCHK(mhsa::add_norm(p, static_cast<hipStream_t>(hs)));
  return MHSA_OK;
}

extern "C" int64_t mhsa_token_log_probs_workspace(int32_t rows, int32_t vocab, int32_t top_k) {
  if (rows < 0 || rows > kMaxRows || vocab <= 0 || vocab > mhsa::kScoresMaxV || top_k < 0 || top_k > mhsa::kScoresMaxK) return -1;
  return rows == 0 ? 0 : mhsa::scores_workspace(rows, vocab, top_k);
}

extern "C" int32_t mhsa_token_log_probs(const void* logits, int32_t dtype, int32_t rows, int32_t vocab, int64_t stride,
                                        float temperature, const int32_t* tokens, int32_t n_tokens, float* log_probs,
                                        float* entropy, int32_t top_k, int32_t* top_indices, float* top_log_probs,
                                        void* workspace, int64_t workspace_bytes, void* hs) {
  mhsa::ScoresParams p;
  if (!act_dtype(dtype, &p.dt)) return fail(MHSA_ENOTSUP, "dtype %d not supported (f32, bf16)", dtype);
  if (rows < 0 || vocab <= 0) return fail(MHSA_EINVAL, "bad shape: %d rows of %d", rows, vocab);
  if (vocab > mhsa::kScoresMaxV) return fail(MHSA_ENOTSUP, "a vocabulary of %d exceeds %d", vocab, mhsa::kScoresMaxV);
  // (down to 0.01 distances of up to 2^120, times log2 e / T, are floats; farther ones
  // are infinite there, and their exponential 0 all the same)
  if (!(temperature >= 0.01f) || !(temperature <= 100.f)) return fail(MHSA_EINVAL, "temperature is to be in [0.01, 100]");
  if (top_k < 0 || top_k > vocab) return fail(MHSA_EINVAL, "top_k %d is not in [0, %d]", top_k, vocab);
  if (top_k > mhsa::kScoresMaxK) return fail(MHSA_ENOTSUP, "top_k %d exceeds %d", top_k, mhsa::kScoresMaxK);
  if (n_tokens < 0) return fail(MHSA_EINVAL, "n_tokens must not be negative (got %d)", n_tokens);
  if (n_tokens > mhsa::kScoresMaxTokens) return fail(MHSA_ENOTSUP, "%d tokens a row exceed %d", n_tokens, mhsa::kScoresMaxTokens);
  if (rows == 0) return MHSA_OK;
  if (!logits || (n_tokens && (!tokens || !log_probs)) || (top_k && (!top_indices || !top_log_probs)))
    return fail(MHSA_EINVAL, "null tensor pointer");
  const int es = mhsa::dtype_size(p.dt);
  if (misaligned(logits, es) || misaligned(tokens, 4) || misaligned(log_probs, 4) || misaligned(entropy, 4) ||
      misaligned(top_indices, 4) || misaligned(top_log_probs, 4))
    return fail(MHSA_EINVAL, "device tensors must be aligned to their elements");
  if (stride < vocab) return fail(MHSA_EINVAL, "row stride %lld is shorter than a row", (long long)stride);
  if (rows > kMaxRows || stride > kMaxStride)
    return fail(MHSA_ENOTSUP, "%d rows, %lld apart, exceed %d and 2^30", rows, (long long)stride, kMaxRows);
  const int64_t need = mhsa::scores_workspace(rows, vocab, top_k);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(MHSA_EINVAL, "%d rows need a 16-byte aligned workspace of %lld bytes", rows, (long long)need);
  const struct {
    const void* p;
    int64_t n;
    bool written;
  } t[] = {{logits, ((rows - 1) * stride + vocab) * es, false},
           {tokens, n_tokens ? (int64_t)rows * n_tokens * 4 : 0, false},
           {log_probs, n_tokens ? (int64_t)rows * n_tokens * 4 : 0, true},
           {entropy, entropy ? (int64_t)rows * 4 : 0, true},
           {top_indices, (int64_t)rows * top_k * 4, true},
           {top_log_probs, (int64_t)rows * top_k * 4, true},
           {workspace, need, true}};
  for (const auto& a : t)
    for (const auto& b : t)
      if (&a != &b && a.written && overlap(a.p, a.n, b.p, b.n))
        return fail(MHSA_EINVAL, "results and the workspace must not overlap another tensor");
  p.x = logits;
  p.ld = stride;
  p.rows = rows;
  p.V = vocab;
  p.inv_t = 1.f / temperature;
  p.tokens = tokens;
  p.nt = n_tokens;
  p.log_probs = log_probs;
  p.entropy = entropy;
  p.k = top_k;
  p.top = top_indices;
  p.top_lp = top_log_probs;
  p.ws = workspace;
  HIPCHK(mhsa::token_scores(p, static_cast<hipStream_t>(hs)));
  return MHSA_OK;
}
