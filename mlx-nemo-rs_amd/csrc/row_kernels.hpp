// Launch interface of the operators on rows (norm.hip, scores.hip), used by
// rows_api.hip. Every launcher checks the shape assumptions its kernels rely on
// and returns a hipError_t (hipErrorInvalidValue when a shape does not fit).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.hpp"

namespace mhsa {

// v = x + scale * delta; sum = v; y = norm(v) * w + b as floats and / or codes
// (fp8_kernels.hpp has their format).
struct NormParams {
  const void* x = nullptr;
  DType dt = kF32;
  int64_t ldx = 0;
  const void* delta = nullptr;  // like x, or null
  int64_t ldd = 0;
  float scale = 1.f;
  void* sum = nullptr;  // like x, or null; may be x or delta
  int64_t lds = 0;
  int64_t rows = 0;
  int D = 0;
  bool layer = false;
  const float* w = nullptr;  // null: ones
  const float* b = nullptr;  // null: zeros
  float eps = 0.f;
  void* out = nullptr;  // or null; may be x
  DType out_dt = kF32;
  int64_t ldo = 0;
  uint8_t* codes = nullptr;  // or null: [rows, Kp] and [rows, kbp]
  uint8_t* scales = nullptr;
};
constexpr int kNormMaxD = 32768;
hipError_t add_norm(const NormParams& p, hipStream_t s);

struct ScoresParams {
  const void* x = nullptr;  // logits
  DType dt = kF32;
  int64_t ld = 0, rows = 0;
  int V = 0;
  float inv_t = 1.f;
  const int* tokens = nullptr;  // [rows, nt]
  int nt = 0;
  float* log_probs = nullptr;
  float* entropy = nullptr;  // or null
  int k = 0;
  int* top = nullptr;
  float* top_lp = nullptr;
  void* ws = nullptr;  // scores_workspace bytes
};
constexpr int kScoresMaxV = 1 << 24, kScoresMaxK = 32, kScoresMaxTokens = 1024;
int64_t scores_workspace(int64_t rows, int V, int k);
hipError_t token_scores(const ScoresParams& p, hipStream_t s);

}  // namespace mhsa
