// Argument checks, workspace layout and device look-ups shared by the C-ABI
// sources of the operators beside the attention path (fp8_api.hip,
// rows_api.hip).
#pragma once

#include <climits>

#include "host_common.hpp"
#include "kernels.hpp"

namespace {

using mhsa::DType;

// Bounds under which no size or offset below leaves 63 bits and no grid has
// 2^32 threads along one axis.
constexpr int32_t kMaxRows = 1 << 25, kMaxOut = 1 << 22;
constexpr int64_t kMaxStride = 1 << 30;

// Whether p is memory of the current GPU (true) or host memory (false).
inline int32_t on_device(const void* p, bool* yes) {
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

// Weights are where they were loaded.
inline int32_t check_device(int device) {
  int dev = 0;
  HIPCHK(hipGetDevice(&dev));
  if (dev != device) return fail(MHSA_EINVAL, "the weights are on GPU %d, the current GPU is %d", device, dev);
  return MHSA_OK;
}

inline bool act_dtype(int32_t d, DType* out) {
  *out = d == MHSA_BF16 ? mhsa::kBF16 : mhsa::kF32;
  return d == MHSA_F32 || d == MHSA_BF16;
}

inline bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// Whether rows of na bytes from a on, pa bytes apart, and rows of nb bytes from
// b on share bytes. Rows of two tensors in one buffer side by side (the same
// distance, none within the other's) do not; of two that are interleaved in any
// other way it is taken that they do.
inline bool rows_overlap(const void* a, int64_t na, int64_t pa, const void* b, int64_t nb, int64_t pb, int64_t rows) {
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
