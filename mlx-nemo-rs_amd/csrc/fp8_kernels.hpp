// Launch interface of the 8-bit block-scaled products, the routing of frames
// to experts and the experts' FeedForward (fp8_gemm.hip, experts.hip), used
// by fp8_api.hip. Every launcher checks the shape assumptions its kernels
// rely on and returns a hipError_t (hipErrorInvalidValue when a shape does not
// fit).
//
// Formats. Values are OCP e4m3 codes (1 sign, 4 exponent, 3 mantissa bits,
// largest 448, 0x7F and 0xFF NaN). A block of 128 of them shares a power of
// two 2^(s - 127), s one byte: for activations 128 inputs of one row, for
// weights 128 x 128. A matrix [rows, K] is held as codes [rows, Kp], Kp = K
// rounded up to 128 and the columns past K zero, beside scale bytes
// [rows or blocks of 128 rows, kbp], kbp = Kp / 128 rounded up to 4. The
// experts' hidden rows have their scale bytes by block instead,
// [Kp / 128, slots]: a tile writes the bytes of its rows for one or two blocks,
// and single bytes of lines that other tiles write too cost the first product
// 20 of 440 us (15001 frames to 4 of 64 experts).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.hpp"

namespace mhsa {

constexpr int kFp8Block = 128;
// A wave holds one row block's weight scales across its lanes, 4 to a word.
constexpr int kFp8MaxK = 64 * 4 * kFp8Block;

constexpr int kFp8BiasTail = 256;  // tiles read whole blocks of columns of the bias

inline int64_t fp8_kp(int64_t k) { return (k + kFp8Block - 1) / kFp8Block * kFp8Block; }
inline int64_t fp8_kbp(int64_t k) { return (fp8_kp(k) / kFp8Block + 3) / 4 * 4; }

// codes and scales of x [rows, K] (row stride ldx, f32 or bf16)
hipError_t fp8_quantize_rows(DType dt, const void* x, int64_t ldx, int64_t rows, int K, uint8_t* codes,
                             uint8_t* scales, hipStream_t s);

// Codes and scales of `n_mats` weight matrices [N, K] back to back, from
// floats (host dtype codes MHSA_F32, MHSA_BF16, MHSA_F16) or from codes
// [n_mats, N, K] and scale bytes [n_mats, N / 128, K / 128] (rounded up).
hipError_t fp8_quantize_weight(int data_dtype, const void* w, int n_mats, int N, int K, uint8_t* codes,
                               uint8_t* scales, hipStream_t s);
hipError_t fp8_pad_weight(const uint8_t* w, const uint8_t* ws, int n_mats, int N, int K, uint8_t* codes,
                          uint8_t* scales, hipStream_t s);
// The way back: codes [N, K] and scales [N / 128, K / 128].
hipError_t fp8_unpad_weight(const uint8_t* codes, const uint8_t* scales, int N, int K, uint8_t* w, uint8_t* ws,
                            hipStream_t s);

// Where the rows of a product over experts come from (null `tile`: one dense
// product). tile[t] = {expert, first slot, slots}, t < *n_tiles <= max_tiles;
// slot s stands for pair[s], which is frame pair[s] / top_k's choice number
// pair[s] % top_k. An expert's slots begin at a multiple of 16.
struct Fp8Groups {
  const int* tile = nullptr;  // [max_tiles, 4]
  const int* n_tiles = nullptr;
  int max_tiles = 0, tile_rows = 0;
  const int* pair = nullptr;
  const int* frame = nullptr;  // pair / top_k
  int top_k = 1;
  // up to fp8_scan_pairs() pairs: no tile list; workgroup column y looks for
  // the y-th of the experts that idx names
  const int* idx = nullptr;
  int pairs = 0, experts = 0;
};

// Low-rank adapters beside a dense product (null `which`: none): out row r gets
// B_a t_r, a = which[r], nothing for a outside [0, n). t_r = s_a A_a x_r comes
// as `parts` bf16 numbers that add up to it, [rows, parts * rank], from
// adapter_rows. Three hold f32, for an f32 result. Two are off by 2^-15 at most,
// 1/128 of a bf16 result's own rounding and under what the fp8 matrix unit drops
// of the projection's sums beside them. (One, off by 2^-8, would add as much as
// the store does: results 1.2e-3 in the 2-norm from f32 sums stored once instead of
// 2.6e-4, which the fp8 unit's sums leave. 3000 x 1024 -> 4096, rank 32, takes
// 29.7, 32.3 and 34.3 us with one, two and three, 15001 x 4096 -> 1024, rank 64,
// 126, 133 and 140.) B_a [N, rank] bf16.
struct Fp8Adapted {
  const int* which = nullptr;
  int n = 0, rank = 0, parts = 2;  // rank 16, 32, 64 or 128
  const uint16_t* t = nullptr;  // null: formed in the few-row kernel (fp8_few_inner) from
  const uint16_t* a = nullptr;  // A and the scales, as AdapterRows has them
  const float* scale = nullptr;
  const uint16_t* b = nullptr;  // [n, N, rank]
};

enum Fp8Epilogue {
  kFp8Out = 0,     // out [M, N] = acc + bias, in out_dt
  kFp8HiddenQ,     // silu(acc + bias) as codes [slots, Np] and scales
  kFp8HiddenF32,   // silu(acc + bias) in f32 [pairs, N], by pair
  kFp8Pair,        // acc + bias in f32 [pairs, N], by pair
};

struct Fp8Gemm {
  // activations: codes and scales (a, as), or, for the few-row kernel, x (of
  // dense products also codes, x null)
  const uint8_t* a = nullptr;
  const uint8_t* as = nullptr;
  const void* x = nullptr;
  DType x_dt = kF32;
  int64_t ldx = 0;
  // gathered rows: x or a by frame (pair / top_k), by pair, or by slot
  enum Rows { kBySlot = 0, kByFrame, kByPair } rows = kBySlot;
  int64_t a_rows = 0;  // rows of a (or x) there are
  const uint8_t* w = nullptr;
  const uint8_t* ws = nullptr;
  // [N] or [experts, N] (zeros, if there is none) with kFp8BiasTail floats
  // behind it
  const float* bias = nullptr;
  int64_t w_stride = 0, ws_stride = 0;  // bytes between experts
  int M = 0, N = 0, K = 0;
  int epilogue = kFp8Out;
  // products over experts: exact products and f32 sums, as a dense product with
  // f32 out always has
  bool exact = false;
  void* out = nullptr;
  DType out_dt = kF32;
  int64_t ldo = 0;
  uint8_t* out_codes = nullptr;
  uint8_t* out_scales = nullptr;
  int64_t slots = 0;  // of the hidden rows' scales
  Fp8Groups g;
  Fp8Adapted ad;
};
// Whether the few-row kernel (activations rounded inside it) takes M rows.
bool fp8_few_rows(int64_t M, int N, int K);
// Whether it forms the adapters' inner products as well.
bool fp8_few_inner(int64_t M, int K, int rank);
hipError_t fp8_gemm_few(const Fp8Gemm& p, hipStream_t s);
int fp8_scan_pairs();
// The second product over few pairs (fp8_few_sum_ok) with the weighted sum:
// out [pairs / top_k, N] in out_dt = residual (or null, or out) + res_scale *
// sum_j weights_j (acc + bias); x [pairs, K] f32, by pair.
bool fp8_few_sum_ok(int64_t pairs, int K);
hipError_t fp8_gemm_few_sum(const Fp8Gemm& p, const float* weights, const void* residual, float res_scale, hipStream_t s);
// Tile kernel on codes; a dense product with f32 out and an `exact` one over
// experts sum on the bf16 matrix cores (exact products), every other on the fp8
// ones.
hipError_t fp8_gemm_tile(const Fp8Gemm& p, hipStream_t s);
// Rows of a tile for `pairs` pairs over `experts` experts (16: the few-row
// kernel's groups), by the pairs an expert has in the mean; K: the smaller of the
// two products'.
constexpr int kFp8TileMean = 24, kFp8LargeMean = 192;
int fp8_group_rows(int64_t pairs, int experts, int K);

// Slots that `pairs` pairs take at most, a multiple of 16.
inline int64_t expert_slots(int64_t pairs, int experts) {
  return (pairs + 15 * (pairs < experts ? pairs : experts) + 15) / 16 * 16;
}
// Experts' bookkeeping: pairs sorted by expert and their frames (pair and
// frame [expert_slots]), and the tile list of tile_rows slots. scratch: plan_scratch_ints(pairs, experts) ints.
int64_t plan_scratch_ints(int64_t pairs, int experts);
// The same launch rounds x [rows, K] (contiguous, 16-byte aligned, K a multiple
// of 8) to codes, unless `codes` is null.
hipError_t experts_prepare(const int* idx, int pairs, int top_k, int experts, int tile_rows, int* pair, int* frame, int* tile,
                           int* n_tiles, int* scratch, DType dt, const void* x, int64_t rows, int K, uint8_t* codes,
                           uint8_t* scales, hipStream_t s);
// out = residual + res_scale * sum_j w[r, j] y[r * top_k + j] over the chosen
// experts in [0, experts); residual may be null or out.
hipError_t experts_combine(DType dt, const float* y, const int* idx, const float* w, int64_t rows, int top_k,
                           int experts, int D, const void* residual, float res_scale, void* out, hipStream_t s);

// t of Fp8Adapted for x [rows, K] (f32, bf16 or, x null, codes and scales): a
// [n, rank, Kp] bf16, each adapter's as adapter_weights leaves it in fragments,
// scale [n] f32. With q_codes, the rows' codes
// and scales are written there in the same launch (x given).
struct AdapterRows {
  const void* x = nullptr;
  DType x_dt = kF32;
  int64_t ldx = 0, rows = 0;
  int K = 0;
  const uint8_t* codes = nullptr;
  const uint8_t* scales = nullptr;
  const int* which = nullptr;
  int n = 0, rank = 0, parts = 2;
  const uint16_t* a = nullptr;
  const float* scale = nullptr;
  uint16_t* t = nullptr;
  uint8_t* q_codes = nullptr;
  uint8_t* q_scales = nullptr;
};
hipError_t adapter_rows(const AdapterRows& p, hipStream_t s);
// A is held in fragments: step of 32 inputs, block of 16 ranks, lane, 8 values;
// lane l has rank l % 16 and inputs 32 step + 8 (l / 16) on.
__device__ __host__ inline int64_t adapter_fragment(int step, int block, int rank) {
  return ((int64_t)step * (rank / 16) + block) * 512;
}
// [rows, cols] floats (host dtype codes) to bf16 [rows_to, cols_to], zeros
// behind, in rows or in the fragments that adapter_rows reads; *bad is set to 1
// if one is not finite as bf16 (to null: only that).
hipError_t adapter_weights(int data_dtype, const void* from, int rows, int cols, uint16_t* to, int rows_to, int cols_to,
                           bool fragments, int* bad, hipStream_t s);

struct RouteParams {
  const void* logits = nullptr;
  DType dt = kF32;
  int64_t ld = 0, rows = 0;
  int experts = 0, top_k = 0, sigmoid = 0, groups = 1, topk_groups = 1, renormalize = 0;
  float scale = 1.f;
  const float* bias = nullptr;
  int* idx = nullptr;
  float* w = nullptr;
};
constexpr int kRouteMaxExperts = 512, kRouteMaxK = 32, kRouteMaxGroups = 64;
hipError_t route(const RouteParams& p, hipStream_t s);

}  // namespace mhsa
