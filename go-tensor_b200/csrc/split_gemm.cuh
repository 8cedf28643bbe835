// float32 products of operands kept as two halves (float16 planes): the GEMMs
// of the large-vocabulary loss (linear_xent.cu).
#pragma once
#include <cuda_fp16.h>

#include "gt_common.cuh"

namespace gt {

// A float32 matrix (rows x cols) as two float16 planes, hi = half(x s) and
// lo = half(x s - hi) with s a power of two per row (or, for G, per row or
// column of a group): base[plane * plane_elems + row * pitch + col]. pitch and
// plane_elems are multiples of 8 and the base is 16-byte aligned (TMA).
// grouped: 128 columns of a row lie together, hi before lo: base[row * pitch +
// col / 128 * 256 + plane * 128 + col % 128]; the pitch is a multiple of 256 and
// what lies behind cols in the last group is zero.
struct HalfPlanes {
  const __half* base = nullptr;
  int64_t rows = 0, cols = 0, pitch = 0, plane_elems = 0;
  bool grouped = false;
};

// Values of K that share a scale of A in dx and dw, and classes per strip.
constexpr int kSplitGroup = 128;

// C (M x N) = A (M x K) B (K x N). A is stored with rows M and columns K, or
// with rows K and columns M (a_mn); B with rows N and columns K, or with rows
// K and columns N (b_mn). The logits: both K-major; dx: A K-major and grouped, B
// N-major; dw: both M/N-major.
struct SplitGemm {
  int64_t M = 0, N = 0, K = 0;
  // The rows (a_mn: the K) that there really are, known on the device only:
  // min(M or K, max(0, *kept - kept_from)); NULL: all. What lies behind them, up
  // to a multiple of 32 of K, is zero.
  const int64_t* kept = nullptr;
  int64_t kept_from = 0;
  const int32_t* row_index = nullptr;  // row m of C goes to row row_index[m] of out
  HalfPlanes a, b;
  bool a_mn = false, b_mn = false;
  // dx, dw: C = scale * sum over the groups of kSplitGroup values of K of group_scale[group *
  // group_ld + row] * (the group's products). Both on the device.
  const float* scale = nullptr;
  const float* group_scale = nullptr;
  int64_t group_ld = 0;
  float* out = nullptr;               // row-major, pitch ldc; logits: may be NULL
  int64_t ldc = 0;
  bool accumulate = false;  // out += instead of out =
  int64_t partial_bytes = 0;  // the most that the partial sums of K-splits may take
  // The logits (strips set): C = row_scale[row] * col_scale[col] * products
  // (powers of two), out = C + bias, and for every row and
  // strip of kStripCols columns the maximum of C + bias and the sum of exp(. -
  // maximum), at strips[strip * strip_rows + row]; the label's logit goes to
  // picked[row].
  // Up to a multiple of 256 columns, col_scale is 1 and bias -infinity behind the last.
  const float *row_scale = nullptr, *col_scale = nullptr, *bias = nullptr;
  const int32_t* labels = nullptr;
  float2* strips = nullptr;
  int64_t strip_rows = 0;
  float* picked = nullptr;
};

constexpr int kStripCols = 128;

char* split_gemm(gt_ctx* ctx, const SplitGemm& g);

// Reports (and clears) a pipeline wait of split_gemm's kernel that ran out.
char* split_gemm_check_errors();

// The bounded waits' limit and the test hook of gt_debug_tc_withhold_arrive (taken once), gemm_tc.cu.
uint64_t tc_wait_limit_ns();
int tc_take_withhold();

}  // namespace gt
