// C ABI of the 8-bit block-scaled projection, the routing of frames to
// experts and the experts' FeedForward. The handles hold weights alone, laid
// out once at loading; a forward call takes its scratch memory from the
// caller, so calls on one handle may run at once on different streams, and
// captured graphs share nothing.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <new>
#include <vector>

#include "fp8_kernels.hpp"
#include "host_common.hpp"
#include "kernels.hpp"

using mhsa::DType;

namespace {

// Bounds under which no size or offset below leaves 63 bits and no grid has
// 2^32 threads along one axis.
constexpr int32_t kMaxRows = 1 << 25, kMaxOut = 1 << 22;
constexpr int64_t kMaxStride = 1 << 30;

// n weight matrices [N, K] in the kernels' format.
struct Fp8Weights {
  int n = 0, N = 0, K = 0;
  int device = -1;  // where the buffers are
  bool use_bias = false, loaded = false;
  DevBuf codes, scales, bias;
  int64_t stride() const { return (int64_t)N * mhsa::fp8_kp(K); }
  int64_t scale_stride() const { return (int64_t)((N + 127) / 128) * mhsa::fp8_kbp(K); }
  int64_t scale_in() const { return (int64_t)((N + 127) / 128) * ((K + 127) / 128); }
};

// Whether p is memory of the current GPU (true) or host memory (false).
int32_t on_device(const void* p, bool* yes) {
  hipPointerAttribute_t a{};
  *yes = false;
  if (hipPointerGetAttributes(&a, p) != hipSuccess) {
    (void)hipGetLastError();  // memory that HIP does not know: the host's
    return MHSA_OK;
  }
  if (a.type != hipMemoryTypeDevice) return MHSA_OK;
  int dev = 0;
  HIPCHK(hipGetDevice(&dev));
  if (a.device != dev) return fail(MHSA_EINVAL, "the tensor is on GPU %d, the current GPU is %d", a.device, dev);
  *yes = true;
  return MHSA_OK;
}

// The bias, or zeros without one, and zeros behind it.
int32_t load_bias(Fp8Weights& w, int data_dtype, const void* bias) {
  const size_t n = (size_t)w.n * w.N, es = data_dtype == MHSA_F32 ? 4 : 2;
  std::vector<float> f(n + mhsa::kFp8BiasTail, 0.f);
  if (w.use_bias) {
    std::vector<char> raw(n * es);
    HIPCHK(hipMemcpy(raw.data(), bias, raw.size(), hipMemcpyDefault));
    for (size_t i = 0; i < n; ++i) f[i] = load_host(data_dtype, raw.data(), i);
  }
  HIPCHK(w.bias.ensure(f.size() * 4));
  HIPCHK(hipMemcpy(w.bias.p, f.data(), f.size() * 4, hipMemcpyHostToDevice));
  return MHSA_OK;
}

// From floats (codes null) or from codes and scale bytes; host or device
// memory. Everything queued on the GPU comes first: a forward may still read
// the old weights, and device tensors may still be being written.
int32_t load_weights(Fp8Weights& w, int data_dtype, const void* weight, const uint8_t* codes, const uint8_t* scales,
                     const void* bias) try {
  if (codes ? !scales : !weight) return fail(MHSA_EINVAL, "null weight pointer");
  if (w.use_bias != (bias != nullptr))
    return fail(MHSA_EINVAL, w.use_bias ? "a bias is expected" : "the layer was created without a bias");
  if (!codes && !float_dtype(data_dtype)) return fail(MHSA_ENOTSUP, "weight dtype %d not supported (f32, bf16, f16)", data_dtype);
  bool dev = false, sdev = false;
  if (int32_t rc = on_device(codes ? codes : weight, &dev)) return rc;
  if (codes)
    if (int32_t rc = on_device(scales, &sdev)) return rc;
  if (codes && dev != sdev) return fail(MHSA_EINVAL, "codes and scales are to be both on the host or both on the GPU");
  int now = 0;
  HIPCHK(hipGetDevice(&now));
  if (w.device >= 0 && now != w.device)
    return fail(MHSA_EINVAL, "the weights are on GPU %d, the current GPU is %d", w.device, now);
  HIPCHK(hipDeviceSynchronize());
  w.loaded = false;
  w.device = now;
  HIPCHK(w.codes.ensure(w.n * w.stride()));
  HIPCHK(w.scales.ensure(w.n * w.scale_stride()));
  const int64_t es = codes ? 1 : data_dtype == MHSA_F32 ? 4 : 2, mat = (int64_t)w.N * w.K * es;
  uint8_t* dc = static_cast<uint8_t*>(w.codes.p);
  uint8_t* ds = static_cast<uint8_t*>(w.scales.p);
  const uint8_t* src = codes ? codes : static_cast<const uint8_t*>(weight);
  DevBuf stage, sstage;
  if (!dev) {
    HIPCHK(stage.ensure(mat));
    if (codes) HIPCHK(sstage.ensure(w.scale_in()));
  }
  // device tensors: as many matrices to a launch as its grid takes (a matrix
  // has up to 2 GiB of codes); host ones one by one through the staging buffer
  const int step = dev ? (int)std::clamp<int64_t>(((int64_t)1 << 32) / w.stride(), 1, 1024) : 1;
  for (int i = 0; i < w.n; i += step) {
    const int m = std::min(step, w.n - i);
    const uint8_t* from = src + i * mat;
    const uint8_t* sfrom = codes ? scales + i * w.scale_in() : nullptr;
    if (!dev) {
      HIPCHK(hipMemcpy(stage.p, from, mat, hipMemcpyHostToDevice));
      from = static_cast<const uint8_t*>(stage.p);
      if (codes) {
        HIPCHK(hipMemcpy(sstage.p, sfrom, w.scale_in(), hipMemcpyHostToDevice));
        sfrom = static_cast<const uint8_t*>(sstage.p);
      }
    }
    if (codes)
      HIPCHK(mhsa::fp8_pad_weight(from, sfrom, m, w.N, w.K, dc + i * w.stride(), ds + i * w.scale_stride(), nullptr));
    else
      HIPCHK(mhsa::fp8_quantize_weight(data_dtype, from, m, w.N, w.K, dc + i * w.stride(), ds + i * w.scale_stride(), nullptr));
    HIPCHK(hipStreamSynchronize(nullptr));
  }
  if (int32_t rc = load_bias(w, codes ? MHSA_F32 : data_dtype, bias)) return rc;
  w.loaded = true;
  return MHSA_OK;
} catch (const std::bad_alloc&) {
  return fail(MHSA_ENOMEM, "out of host memory");
}

// Weights are where they were loaded.
int32_t check_device(int device) {
  int dev = 0;
  HIPCHK(hipGetDevice(&dev));
  if (dev != device) return fail(MHSA_EINVAL, "the weights are on GPU %d, the current GPU is %d", device, dev);
  return MHSA_OK;
}

bool act_dtype(int32_t d, DType* out) {
  *out = d == MHSA_BF16 ? mhsa::kBF16 : mhsa::kF32;
  return d == MHSA_F32 || d == MHSA_BF16;
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// Whether rows of na bytes from a on, pa bytes apart, and rows of nb bytes from
// b on share bytes. Rows of two tensors in one buffer side by side (the same
// distance, none within the other's) do not; of two that are interleaved in any
// other way it is taken that they do.
bool rows_overlap(const void* a, int64_t na, int64_t pa, const void* b, int64_t nb, int64_t pb, int64_t rows) {
  if (!overlap(a, (rows - 1) * pa + na, b, (rows - 1) * pb + nb)) return false;
  if (pa != pb) return true;
  const int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));
  const int64_t at = (off % pa + pa) % pa;  // of b's rows within a's distance
  return at < na || at + nb > pa;
}

// Hands out 256-byte aligned pieces of a workspace (or only adds them up).
struct Arena {
  char* base;
  int64_t used = 0;
  explicit Arena(void* p) : base(static_cast<char*>(p)) {}
  template <typename T> T* take(int64_t n) {
    T* p = reinterpret_cast<T*>(base + used);
    used = align_up(used + n * (int64_t)sizeof(T), 256);
    return p;
  }
};

}  // namespace

// ---------------------------------------------------------------------------
// The projection
// ---------------------------------------------------------------------------

struct mhsa_fp8_linear {
  Fp8Weights w;
};

namespace {

struct LinearPlan {
  bool few = false;
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  int64_t bytes = 0;
};

LinearPlan linear_plan(const Fp8Weights& w, int64_t rows, void* ws) {
  LinearPlan p;
  p.few = mhsa::fp8_few_rows(rows, w.N, w.K);
  if (p.few) return p;
  Arena a(ws);
  p.codes = a.take<uint8_t>(rows * mhsa::fp8_kp(w.K));
  p.scales = a.take<uint8_t>(rows * mhsa::fp8_kbp(w.K));
  p.bytes = a.used;
  return p;
}

}  // namespace

extern "C" {

int32_t mhsa_fp8_linear_create(int32_t in_dim, int32_t out_dim, int32_t use_bias, mhsa_fp8_linear** out) {
  if (!out) return fail(MHSA_EINVAL, "null output pointer");
  *out = nullptr;
  if (in_dim <= 0 || out_dim <= 0) return fail(MHSA_EINVAL, "in_dim %d and out_dim %d must be positive", in_dim, out_dim);
  if (in_dim > mhsa::kFp8MaxK) return fail(MHSA_ENOTSUP, "in_dim %d exceeds %d", in_dim, mhsa::kFp8MaxK);
  if ((int64_t)out_dim * mhsa::fp8_kp(in_dim) > INT32_MAX)
    return fail(MHSA_ENOTSUP, "a weight of %d x %d exceeds 2 GiB", out_dim, in_dim);
  if (out_dim > kMaxOut) return fail(MHSA_ENOTSUP, "out_dim %d exceeds %d", out_dim, kMaxOut);
  mhsa_fp8_linear* h = new (std::nothrow) mhsa_fp8_linear();
  if (!h) return fail(MHSA_ENOMEM, "out of host memory");
  h->w.n = 1;
  h->w.N = out_dim;
  h->w.K = in_dim;
  h->w.use_bias = use_bias != 0;
  *out = h;
  return MHSA_OK;
}

void mhsa_fp8_linear_destroy(mhsa_fp8_linear* h) { delete h; }

int32_t mhsa_fp8_linear_load(mhsa_fp8_linear* h, int32_t data_dtype, const void* weight, const void* bias) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  return load_weights(h->w, data_dtype, weight, nullptr, nullptr, bias);
}

int32_t mhsa_fp8_linear_load_codes(mhsa_fp8_linear* h, const uint8_t* codes, const uint8_t* scales, const float* bias) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  if (!codes) return fail(MHSA_EINVAL, "null weight pointer");
  return load_weights(h->w, MHSA_F32, nullptr, codes, scales, bias);
}

int32_t mhsa_fp8_linear_read_codes(const mhsa_fp8_linear* h, uint8_t* codes, uint8_t* scales) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  if (!codes || !scales) return fail(MHSA_EINVAL, "null output pointer");
  if (!h->w.loaded) return fail(MHSA_EINVAL, "no weights are loaded");
  if (int32_t rc = check_device(h->w.device)) return rc;
  DevBuf c, s;
  const int64_t n = (int64_t)h->w.N * h->w.K;
  HIPCHK(c.ensure(n));
  HIPCHK(s.ensure(h->w.scale_in()));
  HIPCHK(mhsa::fp8_unpad_weight(static_cast<const uint8_t*>(h->w.codes.p), static_cast<const uint8_t*>(h->w.scales.p),
                                h->w.N, h->w.K, static_cast<uint8_t*>(c.p), static_cast<uint8_t*>(s.p), nullptr));
  HIPCHK(hipStreamSynchronize(nullptr));
  HIPCHK(hipMemcpy(codes, c.p, n, hipMemcpyDefault));
  HIPCHK(hipMemcpy(scales, s.p, h->w.scale_in(), hipMemcpyDefault));
  return MHSA_OK;
}

int64_t mhsa_fp8_linear_workspace(const mhsa_fp8_linear* h, int32_t rows) {
  if (!h || rows < 0 || rows > kMaxRows) return -1;
  return rows == 0 ? 0 : linear_plan(h->w, rows, nullptr).bytes;
}

int32_t mhsa_fp8_linear_forward(const mhsa_fp8_linear* h, const void* x, int32_t x_dtype, int32_t rows,
                                int64_t x_stride, void* out, int32_t out_dtype, int64_t out_stride, void* workspace,
                                int64_t workspace_bytes, void* hs) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  const Fp8Weights& w = h->w;
  DType xd, od;
  if (!act_dtype(x_dtype, &xd) || !act_dtype(out_dtype, &od))
    return fail(MHSA_ENOTSUP, "dtypes %d and %d not supported (f32, bf16)", x_dtype, out_dtype);
  if (rows < 0) return fail(MHSA_EINVAL, "rows must not be negative (got %d)", rows);
  if (rows > kMaxRows) return fail(MHSA_ENOTSUP, "%d rows exceed %d", rows, kMaxRows);
  if (rows == 0) return MHSA_OK;
  if (!x || !out) return fail(MHSA_EINVAL, "null tensor pointer");
  const int xs = mhsa::dtype_size(xd), os = mhsa::dtype_size(od);
  if (reinterpret_cast<uintptr_t>(x) % xs || reinterpret_cast<uintptr_t>(out) % os)
    return fail(MHSA_EINVAL, "device tensors must be aligned to their elements");
  if (x_stride < w.K || out_stride < w.N)
    return fail(MHSA_EINVAL, "row strides %lld and %lld are shorter than the rows (%d, %d)", (long long)x_stride,
                (long long)out_stride, w.K, w.N);
  if (x_stride > kMaxStride || out_stride > kMaxStride)
    return fail(MHSA_ENOTSUP, "row strides %lld and %lld exceed 2^30", (long long)x_stride, (long long)out_stride);
  if (!w.loaded) return fail(MHSA_EINVAL, "no weights are loaded");
  const LinearPlan plan = linear_plan(w, rows, workspace);
  if (plan.bytes > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < plan.bytes))
    return fail(MHSA_EINVAL, "%d rows need a 16-byte aligned workspace of %lld bytes", rows, (long long)plan.bytes);
  const int64_t xn = ((rows - 1) * x_stride + w.K) * xs, on = ((rows - 1) * out_stride + w.N) * os;
  if (rows_overlap(x, w.K * xs, x_stride * xs, out, w.N * os, out_stride * os, rows) || overlap(workspace, plan.bytes, x, xn) || overlap(workspace, plan.bytes, out, on))
    return fail(MHSA_EINVAL, "x, out and the workspace must not overlap");
  if (int32_t rc = check_device(w.device)) return rc;
  hipStream_t s = static_cast<hipStream_t>(hs);
  mhsa::Fp8Gemm p;
  p.w = static_cast<const uint8_t*>(w.codes.p);
  p.ws = static_cast<const uint8_t*>(w.scales.p);
  p.bias = static_cast<const float*>(w.bias.p);
  p.M = rows;
  p.N = w.N;
  p.K = w.K;
  p.out = out;
  p.out_dt = od;
  p.ldo = out_stride;
  if (plan.few) {
    p.x = x;
    p.x_dt = xd;
    p.ldx = x_stride;
    HIPCHK(mhsa::fp8_gemm_few(p, s));
    return MHSA_OK;
  }
  HIPCHK(mhsa::fp8_quantize_rows(xd, x, x_stride, rows, w.K, plan.codes, plan.scales, s));
  p.a = plan.codes;
  p.as = plan.scales;
  p.a_rows = rows;
  HIPCHK(mhsa::fp8_gemm_tile(p, s));
  return MHSA_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Routing
// ---------------------------------------------------------------------------

extern "C" int32_t mhsa_route(const void* logits, int32_t dtype, int32_t rows, int32_t n_experts, int64_t stride,
                              int32_t score, const float* bias, int32_t n_groups, int32_t topk_groups, int32_t top_k,
                              int32_t renormalize, float scale, int32_t* indices, float* weights, void* hs) {
  mhsa::RouteParams p;
  if (!act_dtype(dtype, &p.dt)) return fail(MHSA_ENOTSUP, "dtype %d not supported (f32, bf16)", dtype);
  if (score != MHSA_ROUTE_SOFTMAX && score != MHSA_ROUTE_SIGMOID)
    return fail(MHSA_ENOTSUP, "score %d not supported (softmax, sigmoid)", score);
  if (rows < 0 || n_experts <= 0) return fail(MHSA_EINVAL, "bad shape: %d rows, %d experts", rows, n_experts);
  if (n_experts > mhsa::kRouteMaxExperts) return fail(MHSA_ENOTSUP, "%d experts exceed %d", n_experts, mhsa::kRouteMaxExperts);
  if (n_groups <= 0 || n_experts % n_groups)
    return fail(MHSA_EINVAL, "%d experts do not divide into %d groups", n_experts, n_groups);
  if (n_groups > mhsa::kRouteMaxGroups) return fail(MHSA_ENOTSUP, "%d groups exceed %d", n_groups, mhsa::kRouteMaxGroups);
  if (topk_groups <= 0 || topk_groups > n_groups)
    return fail(MHSA_EINVAL, "topk_groups %d is not in [1, %d]", topk_groups, n_groups);
  if (top_k <= 0 || top_k > topk_groups * (n_experts / n_groups))
    return fail(MHSA_EINVAL, "top_k %d is not in [1, %d], the experts of %d groups", top_k,
                topk_groups * (n_experts / n_groups), topk_groups);
  if (top_k > mhsa::kRouteMaxK) return fail(MHSA_ENOTSUP, "top_k %d exceeds %d", top_k, mhsa::kRouteMaxK);
  if (stride < n_experts) return fail(MHSA_EINVAL, "row stride %lld is shorter than a row", (long long)stride);
  if (!std::isfinite(scale)) return fail(MHSA_EINVAL, "scale must be finite");
  if (rows == 0) return MHSA_OK;
  if (!logits || !indices || !weights) return fail(MHSA_EINVAL, "null tensor pointer");
  if (reinterpret_cast<uintptr_t>(logits) % mhsa::dtype_size(p.dt) || reinterpret_cast<uintptr_t>(indices) % 4 ||
      reinterpret_cast<uintptr_t>(weights) % 4 || reinterpret_cast<uintptr_t>(bias) % 4)
    return fail(MHSA_EINVAL, "device tensors must be aligned to their elements");
  if (rows > kMaxRows || stride > kMaxStride) return fail(MHSA_ENOTSUP, "%d rows, %lld apart, exceed %d and 2^30", rows, (long long)stride, kMaxRows);
  const int64_t ln = ((rows - 1) * stride + n_experts) * mhsa::dtype_size(p.dt), kn = (int64_t)rows * top_k * 4;
  if (overlap(indices, kn, logits, ln) || overlap(weights, kn, logits, ln) || overlap(indices, kn, weights, kn) ||
      overlap(indices, kn, bias, bias ? n_experts * 4 : 0) || overlap(weights, kn, bias, bias ? n_experts * 4 : 0))
    return fail(MHSA_EINVAL, "indices and weights must not overlap another tensor");
  p.logits = logits;
  p.ld = stride;
  p.rows = rows;
  p.experts = n_experts;
  p.top_k = top_k;
  p.sigmoid = score == MHSA_ROUTE_SIGMOID;
  p.groups = n_groups;
  p.topk_groups = topk_groups;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  p.bias = bias;
  p.idx = indices;
  p.w = weights;
  HIPCHK(mhsa::route(p, static_cast<hipStream_t>(hs)));
  return MHSA_OK;
}

// ---------------------------------------------------------------------------
// The experts' FeedForward
// ---------------------------------------------------------------------------

struct mhsa_experts {
  Fp8Weights lin[2];  // linear1 [E, F, D], linear2 [E, D, F]
  int E = 0, D = 0, F = 0;
};

namespace {

constexpr int kMaxExperts = 1024, kMaxTopK = 32;
constexpr int64_t kMaxPairs = 1 << 18, kListPairs = 256;

// How a call runs, and its pieces of the workspace. Rows go in runs of
// `step`, each through the same buffers, which bounds them.
struct ExpertsPlan {
  int64_t step = 0;
  int tile_rows = 0;  // 0: no list; 16: few-row kernel; else tiles
  int max_tiles = 0;
  int64_t slots = 0;
  int *pair = nullptr, *frame = nullptr, *tile = nullptr, *n_tiles = nullptr, *scratch = nullptr;
  uint8_t *xc = nullptr, *xs = nullptr, *hc = nullptr, *hsc = nullptr;
  float *h = nullptr, *y = nullptr;
  int64_t bytes = 0;
};

ExpertsPlan experts_layout(const mhsa_experts* e, int64_t rows, int top_k, void* ws) {
  ExpertsPlan p;
  const int64_t dp = mhsa::fp8_kp(e->D), fp = mhsa::fp8_kp(e->F);
  const int64_t most = std::min({kMaxPairs / top_k, INT32_MAX / (fp * top_k), INT32_MAX / dp});
  p.step = std::min(rows, most);
  const int64_t pairs = p.step * top_k;
  Arena a(ws);
  // A list costs a launch; without one every workgroup scans the indices, and an
  // expert's pairs go by 16 at a time, each time with its weights. Up to 256 pairs
  // there is none, whatever their experts: 32 pairs of one expert of 1024 -> 4096
  // take 33.3 us (36.7 with a list and tiles), 64 of four 38.5 (37.8), but 256 of
  // one 215 (57), of four 107 (42) and of eight 96 (42).
  p.tile_rows = mhsa::fp8_group_rows(pairs, e->E, std::min(e->D, e->F));
  if (rows * top_k <= kListPairs || (p.tile_rows == 16 && rows * top_k <= mhsa::fp8_scan_pairs())) p.tile_rows = 0;
  if (p.tile_rows) {
    p.max_tiles = (int)(pairs / p.tile_rows + std::min<int64_t>(pairs, e->E));
    p.pair = a.take<int>(mhsa::expert_slots(pairs, e->E));
    p.frame = a.take<int>(mhsa::expert_slots(pairs, e->E));
    p.tile = a.take<int>(4 * (int64_t)p.max_tiles);
    p.n_tiles = a.take<int>(1);
    p.scratch = a.take<int>(mhsa::plan_scratch_ints(pairs, e->E));
  }
  if (p.tile_rows > 16) {
    p.xc = a.take<uint8_t>(p.step * dp);
    p.xs = a.take<uint8_t>(p.step * mhsa::fp8_kbp(e->D));
    p.slots = mhsa::expert_slots(pairs, e->E);
    p.hc = a.take<uint8_t>(p.slots * fp);
    p.hsc = a.take<uint8_t>(p.slots * (fp / 128));
  } else {
    p.h = a.take<float>(pairs * e->F);
  }
  p.y = a.take<float>(pairs * e->D);
  p.bytes = a.used;
  return p;
}

// Bytes of a workspace that serves `rows` rows and any fewer: a call's kernels
// change with its number of pairs, and those of fewer keep hidden rows in f32,
// which takes more than the next ones' codes. Within a range the bytes grow with
// the rows, so the most are those of `rows` or of the end of a range before it.
int64_t experts_bytes(const mhsa_experts* e, int64_t rows, int top_k) {
  int64_t most = experts_layout(e, rows, top_k, nullptr).bytes;
  for (const int64_t pairs : {kListPairs, (int64_t)mhsa::fp8_scan_pairs(), (int64_t)mhsa::kFp8TileMean * e->E - 1,
                              (int64_t)mhsa::kFp8LargeMean * e->E - 1})
    if (const int64_t r = pairs / top_k; r > 0 && r < rows) most = std::max(most, experts_layout(e, r, top_k, nullptr).bytes);
  return most;
}

int32_t experts_run(const mhsa_experts* e, const ExpertsPlan& plan, const void* x, DType dt, int64_t rows,
                    const int32_t* idx, const float* weights, int top_k, const void* residual, float res_scale,
                    void* out, hipStream_t s) {
  const int pairs = (int)(rows * top_k);
  mhsa::Fp8Gemm g[2];
  for (int i = 0; i < 2; ++i) {
    const Fp8Weights& w = e->lin[i];
    g[i].w = static_cast<const uint8_t*>(w.codes.p);
    g[i].ws = static_cast<const uint8_t*>(w.scales.p);
    g[i].w_stride = w.stride();
    g[i].ws_stride = w.scale_stride();
    g[i].bias = static_cast<const float*>(w.bias.p);
    g[i].N = w.N;
    g[i].K = w.K;
    g[i].M = pairs;
    g[i].ldo = w.N;
    g[i].exact = dt == mhsa::kF32;
    g[i].g.top_k = top_k;
    g[i].g.experts = e->E;
    g[i].g.pairs = pairs;
    if (plan.tile_rows) {
      g[i].g.tile = plan.tile;
      g[i].g.n_tiles = plan.n_tiles;
      g[i].g.max_tiles = (int)(pairs / plan.tile_rows + std::min(pairs, e->E));
      g[i].g.tile_rows = plan.tile_rows;
      g[i].g.pair = plan.pair;
      g[i].g.frame = plan.frame;
    } else {
      g[i].g.idx = idx;
    }
  }
  g[1].epilogue = mhsa::kFp8Pair;
  g[1].out = plan.y;
  if (plan.tile_rows)
    HIPCHK(mhsa::experts_prepare(idx, pairs, top_k, e->E, plan.tile_rows, plan.pair, plan.frame, plan.tile, plan.n_tiles,
                                 plan.scratch, dt, x, rows, e->D, plan.xc, plan.xs, s));
  if (plan.tile_rows > 16) {
    g[0].a = plan.xc;
    g[0].as = plan.xs;
    g[0].a_rows = rows;
    g[0].rows = mhsa::Fp8Gemm::kByFrame;
    g[0].epilogue = mhsa::kFp8HiddenQ;
    g[0].out_codes = plan.hc;
    g[0].out_scales = plan.hsc;
    g[0].slots = g[1].slots = plan.slots;
    HIPCHK(mhsa::fp8_gemm_tile(g[0], s));
    g[1].a = plan.hc;
    g[1].as = plan.hsc;
    HIPCHK(mhsa::fp8_gemm_tile(g[1], s));
  } else {
    g[0].x = x;
    g[0].x_dt = dt;
    g[0].ldx = e->D;
    g[0].rows = mhsa::Fp8Gemm::kByFrame;
    g[0].epilogue = mhsa::kFp8HiddenF32;
    g[0].out = plan.h;
    HIPCHK(mhsa::fp8_gemm_few(g[0], s));
    g[1].x = plan.h;
    g[1].x_dt = mhsa::kF32;
    g[1].ldx = e->F;
    g[1].rows = mhsa::Fp8Gemm::kByPair;
    if (!plan.tile_rows && mhsa::fp8_few_sum_ok(pairs, e->F)) {
      g[1].out = out;
      g[1].out_dt = dt;
      HIPCHK(mhsa::fp8_gemm_few_sum(g[1], weights, residual, res_scale, s));
      return MHSA_OK;
    }
    HIPCHK(mhsa::fp8_gemm_few(g[1], s));
  }
  HIPCHK(mhsa::experts_combine(dt, plan.y, idx, weights, rows, top_k, e->E, e->D, residual, res_scale, out, s));
  return MHSA_OK;
}

// Both matrices or none: a load that fails halfway leaves no mixture behind.
int32_t experts_load(mhsa_experts* h, int data_dtype, const void* const weight[2], const uint8_t* const codes[2],
                     const uint8_t* const scales[2], const void* const bias[2]) {
  for (int i = 0; i < 2; ++i)
    if (int32_t rc = load_weights(h->lin[i], data_dtype, weight[i], codes[i], scales[i], bias[i])) {
      if (i == 1) h->lin[0].loaded = false;
      return rc;
    }
  return MHSA_OK;
}

}  // namespace

extern "C" {

int32_t mhsa_experts_create(int32_t n_experts, int32_t d_model, int32_t ff_dim, int32_t use_bias, mhsa_experts** out) {
  if (!out) return fail(MHSA_EINVAL, "null output pointer");
  *out = nullptr;
  if (n_experts <= 0 || d_model <= 0 || ff_dim <= 0 || d_model % 64 || ff_dim % 64)
    return fail(MHSA_EINVAL, "n_experts %d must be positive, d_model %d and ff_dim %d positive multiples of 64", n_experts,
                d_model, ff_dim);
  if (n_experts > kMaxExperts || d_model > mhsa::kFp8MaxK || ff_dim > mhsa::kFp8MaxK)
    return fail(MHSA_ENOTSUP, "n_experts %d, d_model %d, ff_dim %d exceed %d, %d, %d", n_experts, d_model, ff_dim,
                kMaxExperts, mhsa::kFp8MaxK, mhsa::kFp8MaxK);
  mhsa_experts* h = new (std::nothrow) mhsa_experts();
  if (!h) return fail(MHSA_ENOMEM, "out of host memory");
  h->E = n_experts;
  h->D = d_model;
  h->F = ff_dim;
  for (int i = 0; i < 2; ++i) {
    h->lin[i].n = n_experts;
    h->lin[i].N = i == 0 ? ff_dim : d_model;
    h->lin[i].K = i == 0 ? d_model : ff_dim;
    h->lin[i].use_bias = use_bias != 0;
  }
  *out = h;
  return MHSA_OK;
}

void mhsa_experts_destroy(mhsa_experts* h) { delete h; }

int32_t mhsa_experts_load(mhsa_experts* h, int32_t data_dtype, const void* weight1, const void* bias1,
                          const void* weight2, const void* bias2) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  if (!weight1 || !weight2) return fail(MHSA_EINVAL, "null weight pointer");
  const void *weight[2] = {weight1, weight2}, *bias[2] = {bias1, bias2};
  const uint8_t* none[2] = {};
  return experts_load(h, data_dtype, weight, none, none, bias);
}

int32_t mhsa_experts_load_codes(mhsa_experts* h, const uint8_t* codes1, const uint8_t* scales1, const float* bias1,
                                const uint8_t* codes2, const uint8_t* scales2, const float* bias2) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  if (!codes1 || !codes2) return fail(MHSA_EINVAL, "null weight pointer");
  const void *none[2] = {}, *bias[2] = {bias1, bias2};
  const uint8_t *codes[2] = {codes1, codes2}, *scales[2] = {scales1, scales2};
  return experts_load(h, MHSA_F32, none, codes, scales, bias);
}

int64_t mhsa_experts_workspace(const mhsa_experts* h, int32_t rows, int32_t top_k) {
  if (!h || rows < 0 || rows > kMaxRows || top_k <= 0 || top_k > kMaxTopK) return -1;
  return rows == 0 ? 0 : experts_bytes(h, rows, top_k);
}

int32_t mhsa_experts_forward(const mhsa_experts* h, const void* x, int32_t dtype, int32_t rows, const int32_t* indices,
                             const float* weights, int32_t top_k, const void* residual, float res_scale, void* out,
                             void* workspace, int64_t workspace_bytes, void* hs) {
  if (!h) return fail(MHSA_EINVAL, "null handle");
  DType dt;
  if (!act_dtype(dtype, &dt)) return fail(MHSA_ENOTSUP, "dtype %d not supported (f32, bf16)", dtype);
  if (rows < 0) return fail(MHSA_EINVAL, "rows must not be negative (got %d)", rows);
  if (rows > kMaxRows) return fail(MHSA_ENOTSUP, "%d rows exceed %d", rows, kMaxRows);
  if (top_k <= 0 || top_k > kMaxTopK) return fail(MHSA_EINVAL, "top_k %d is not in [1, %d]", top_k, kMaxTopK);
  if (rows == 0) return MHSA_OK;
  if (!x || !indices || !weights || !out) return fail(MHSA_EINVAL, "null tensor pointer");
  if (!aligned16(x) || !aligned16(out) || !aligned16(residual))
    return fail(MHSA_EINVAL, "device tensors must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(indices) % 4 || reinterpret_cast<uintptr_t>(weights) % 4)
    return fail(MHSA_EINVAL, "indices and weights must be aligned to their elements");
  if (!h->lin[0].loaded || !h->lin[1].loaded) return fail(MHSA_EINVAL, "no weights are loaded");
  const ExpertsPlan plan = experts_layout(h, rows, top_k, workspace);
  const int64_t need = experts_bytes(h, rows, top_k);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need)
    return fail(MHSA_EINVAL, "%d rows of %d experts need a 16-byte aligned workspace of %lld bytes", rows, top_k,
                (long long)need);
  const int64_t es = mhsa::dtype_size(dt), n = (int64_t)rows * h->D * es, np = (int64_t)rows * top_k * 4;
  if (overlap(x, n, out, n) || (residual && residual != out && overlap(residual, n, out, n)) ||
      overlap(indices, np, out, n) || overlap(weights, np, out, n))
    return fail(MHSA_EINVAL, "out must not overlap another tensor, but may be the residual");
  for (const void* t : {x, static_cast<const void*>(out), residual})
    if (t && overlap(workspace, plan.bytes, t, n)) return fail(MHSA_EINVAL, "the workspace must not overlap a tensor");
  if (overlap(workspace, plan.bytes, indices, np) || overlap(workspace, plan.bytes, weights, np))
    return fail(MHSA_EINVAL, "the workspace must not overlap a tensor");
  if (int32_t rc = check_device(h->lin[0].device)) return rc;
  for (int64_t r = 0; r < rows; r += plan.step) {
    const int64_t m = std::min<int64_t>(plan.step, rows - r), at = r * h->D * es;
    const int32_t rc = experts_run(h, plan, static_cast<const char*>(x) + at, dt, m, indices + r * top_k,
                                   weights + r * top_k, top_k, residual ? static_cast<const char*>(residual) + at : nullptr,
                                   res_scale, static_cast<char*>(out) + at, static_cast<hipStream_t>(hs));
    if (rc) return rc;
  }
  return MHSA_OK;
}

}  // extern "C"
