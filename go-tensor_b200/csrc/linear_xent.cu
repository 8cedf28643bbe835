// Softmax cross-entropy of a Linear over a large vocabulary, with all
// gradients, without keeping the logits.
//
//   z_iv  = sum_k x_ik w_vk + b_v
//   lse_i = max_v z_iv + log sum_v exp(z_iv - max)
//   row_i = lse_i - z_i,y(i)                      (0 for an ignored row)
//   loss  = sum_i row_i / n                       (n: the rows that count)
//   G_iv  = (exp(z_iv - lse_i) - [v = y(i)]) / n  (0 for an ignored row)
//   dx = G w,  dw = G^T x,  db_v = sum_i G_iv
//
// The rows are taken in pieces: the logits of one piece live in workspace,
// become the gradient in place and are overwritten by the next piece, so
// memory does not grow with the number of rows.
#include <algorithm>
#include <cmath>

#include "gemm.cuh"

namespace gt {

__device__ __forceinline__ float exp_t(float x) { return expf(x); }
__device__ __forceinline__ double exp_t(double x) { return exp(x); }
__device__ __forceinline__ float log_t(float x) { return logf(x); }
__device__ __forceinline__ double log_t(double x) { return log(x); }

// counts[0] = rows that count (label != ignore); a label outside [0, V) sets *bad.
__global__ void __launch_bounds__(1024) label_count_kernel(const int32_t* __restrict__ labels, int64_t M, int64_t V,
                                                           int32_t ignore, int64_t* counts, int32_t* bad) {
  __shared__ int64_t ws[32];
  int64_t n = 0;
  bool outside = false;
  for (int64_t i = threadIdx.x; i < M; i += blockDim.x) {
    const int32_t y = labels[i];
    if (y != ignore) {
      n++;
      outside |= y < 0 || y >= V;
    }
  }
  if (outside && bad) *bad = 1;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (int w = 0; w < 32; w++) n += ws[w];
    counts[0] = n;
  }
}

// out = x with the ignored rows zeroed (padding may hold anything).
template <typename T>
__global__ void keep_rows_kernel(const T* __restrict__ x, const int32_t* __restrict__ labels, int64_t rows, int64_t K,
                                 int32_t ignore, T* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * K; i += (int64_t)gridDim.x * blockDim.x)
    out[i] = labels[i / K] == ignore ? (T)0 : x[i];
}

// Joins two running (maximum, sum of exp(z - maximum)) pairs.
template <typename T>
__device__ __forceinline__ void join(T& m, T& s, T m2, T s2) {
  const T top = go_max(m, m2);
  s = (m == top ? s : s * exp_t(m - top)) + (m2 == top ? s2 : s2 * exp_t(m2 - top));
  m = top;
}

// A block per row: the running maximum and sum in one pass over the row, then
// the gradient in place.
template <typename T>
__global__ void __launch_bounds__(256) xent_piece_kernel(T* __restrict__ z, const int32_t* __restrict__ labels,
                                                         int64_t rows, int64_t V, int32_t ignore,
                                                         const int64_t* __restrict__ counts, T* __restrict__ row_loss,
                                                         bool grad) {
  __shared__ T wm[8], wsum[8];
  const T inv = (T)(1.0 / (double)counts[0]);
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    T* zr = z + i * V;
    const int32_t y = labels[i];
    if (y == ignore) {
      if (threadIdx.x == 0) row_loss[i] = (T)0;
      if (grad)
        for (int64_t j = threadIdx.x; j < V; j += blockDim.x) zr[j] = (T)0;
      continue;
    }
    T m = (T)(-INFINITY), s = (T)0;
    for (int64_t j = threadIdx.x; j < V; j += blockDim.x) {
      const T v = zr[j];
      if (v > m) {
        s = s * exp_t(m - v) + (T)1;
        m = v;
      } else if (v != (T)(-INFINITY)) {  // (a NaN comes here too)
        s += exp_t(v - m);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const T m2 = __shfl_xor_sync(0xffffffffu, m, off), s2 = __shfl_xor_sync(0xffffffffu, s, off);
      join(m, s, m2, s2);
    }
    if ((threadIdx.x & 31) == 0) wm[threadIdx.x >> 5] = m, wsum[threadIdx.x >> 5] = s;
    __syncthreads();
    m = wm[0], s = wsum[0];
    for (int w = 1; w < 8; w++) join(m, s, wm[w], wsum[w]);
    const bool bad = y < 0 || y >= V;
    if (threadIdx.x == 0) row_loss[i] = bad ? (T)NAN : log_t(s) + (m - zr[y]);
    __syncthreads();  // the label's logit is read, and wm / wsum are free
    if (grad)
      // (not exp(z - lse): the logarithm would vanish beside a maximum that is
      // a mask's lowest value)
      for (int64_t j = threadIdx.x; j < V; j += blockDim.x) {
        const T e = exp_t(zr[j] - m) / s * inv;
        zr[j] = j == y ? e - inv : e;
      }
  }
}

// loss = sum of the rows' losses / n, in float64, one block, a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) mean_rows_kernel(const T* __restrict__ rows, int64_t M,
                                                         const int64_t* __restrict__ counts, T* __restrict__ loss) {
  __shared__ double part[32];
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < M; i += blockDim.x) acc += (double)rows[i];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    acc = 0.0;
    for (int w = 0; w < 32; w++) acc += part[w];
    *loss = (T)(acc / (double)counts[0]);
  }
}

// db (+)= column sums of a piece's gradient, rows in order.
template <typename T>
__global__ void piece_columns_kernel(const T* __restrict__ g, int64_t rows, int64_t V, bool first, T* __restrict__ db) {
  for (int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; j < V; j += (int64_t)gridDim.x * blockDim.x) {
    double acc = first ? 0.0 : (double)db[j];
    for (int64_t i = 0; i < rows; i++) acc += (double)g[i * V + j];
    db[j] = (T)acc;
  }
}

template <typename T>
__global__ void add_kernel(T* __restrict__ out, const T* __restrict__ x, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    out[i] = out[i] + x[i];
}

template <typename T>
struct XentCall {
  const T *x, *w, *bias;
  const int32_t* labels;
  int64_t M, K, V;
  int32_t ignore;
  int64_t workspace;
  T *loss, *rows, *dx, *dw, *db;
  int32_t* bad;
};

// float32 products on the FP32 pipe: the 3xTF32 path loses subnormal operands.
static char* product(gt_ctx* ctx, const GemmShape& s, const float* A, const float* B, const Epi<float>& e) {
  return gemm_simt<float>(ctx, s, A, B, e);
}
static char* product(gt_ctx* ctx, const GemmShape& s, const double* A, const double* B, const Epi<double>& e) {
  return gemm<double>(ctx, s, A, B, e);
}

// Pieces of rows over the GEMM entry points: one piece's logits in workspace.
template <typename T>
static char* linear_xent_pieces(gt_ctx* ctx, const XentCall<T>& c, void** held) {
  const bool grad = c.dx || c.dw || c.db;
  int64_t R = std::max<int64_t>(1, c.workspace / (int64_t)(c.V * sizeof(T)));
  R = std::min(c.M, R >= 128 ? R / 128 * 128 : 128);
  const int64_t pieces = ceil_div(c.M, R);
  T *z, *xk, *more = nullptr, *rows = c.rows;
  int64_t* counts;
  GT_TRY(scratch(ctx, (size_t)R * c.V * sizeof(T), &held[0]));
  GT_TRY(scratch(ctx, (size_t)R * c.K * sizeof(T), &held[1]));
  GT_TRY(scratch(ctx, 64, &held[2]));
  if (!rows) {
    GT_TRY(scratch(ctx, (size_t)c.M * sizeof(T), &held[3]));
    rows = (T*)held[3];
  }
  if (c.dw && pieces > 1) {
    GT_TRY(scratch(ctx, (size_t)c.V * c.K * sizeof(T), &held[4]));
    more = (T*)held[4];
  }
  z = (T*)held[0], xk = (T*)held[1], counts = (int64_t*)held[2];
  label_count_kernel<<<1, 1024, 0, ctx->stream>>>(c.labels, c.M, c.V, c.ignore, counts, c.bad);
  GT_LAUNCH_CHECK();
  for (int64_t r0 = 0; r0 < c.M; r0 += R) {
    const int64_t r = std::min(R, c.M - r0);
    keep_rows_kernel<T><<<grid_for(ctx, r * c.K, 256), 256, 0, ctx->stream>>>(c.x + r0 * c.K, c.labels + r0, r, c.K,
                                                                               c.ignore, xk);
    GT_LAUNCH_CHECK();
    Epi<T> e;
    e.out = z, e.ldc = c.V, e.bias = c.bias;
    GT_TRY(product(ctx, GemmShape{r, c.V, c.K, false, true, c.K, c.K}, xk, c.w, e));
    xent_piece_kernel<T><<<(unsigned)std::min<int64_t>(r, (int64_t)ctx->sm_count * 8), 256, 0, ctx->stream>>>(
        z, c.labels + r0, r, c.V, c.ignore, counts, rows + r0, grad);
    GT_LAUNCH_CHECK();
    if (c.dx) {
      Epi<T> d;
      d.out = c.dx + r0 * c.K, d.ldc = c.K;
      GT_TRY(product(ctx, GemmShape{r, c.K, c.V, false, false, c.V, c.K}, z, c.w, d));
    }
    if (c.dw) {
      Epi<T> d;
      d.out = r0 ? more : c.dw, d.ldc = c.K;
      GT_TRY(product(ctx, GemmShape{c.V, c.K, r, true, false, c.V, c.K}, z, xk, d));
      if (r0) {
        add_kernel<T><<<grid_for(ctx, c.V * c.K, 256), 256, 0, ctx->stream>>>(c.dw, more, c.V * c.K);
        GT_LAUNCH_CHECK();
      }
    }
    if (c.db) {
      piece_columns_kernel<T><<<grid_for(ctx, c.V, 64), 64, 0, ctx->stream>>>(z, r, c.V, r0 == 0, c.db);
      GT_LAUNCH_CHECK();
    }
  }
  mean_rows_kernel<T><<<1, 1024, 0, ctx->stream>>>(rows, c.M, counts, c.loss);
  GT_LAUNCH_CHECK();
  return nullptr;
}

struct Range {
  const void* p;
  int64_t bytes;
};

static bool overlap(const Range& a, const Range& b) {
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes &&
         (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
}

}  // namespace gt

using namespace gt;

extern "C" char* gt_linear_xent_fwd_bwd(gt_ctx* ctx, int dtype, const void* x, const void* w, const void* bias,
                                        const int32_t* labels, int64_t M, int64_t K, int64_t V, int32_t ignore_label,
                                        int64_t workspace_bytes, void* loss, void* row_loss, void* dx, void* dw,
                                        void* db, int32_t* bad_label) {
  GT_CHECK_DTYPE(dtype);
  if (!x || !w || !labels || !loss) return errorf("gt_linear_xent_fwd_bwd: null argument");
  if (M <= 0 || K <= 0 || V <= 0) return errorf("gt_linear_xent_fwd_bwd: M, K and V must be positive");
  if (M > INT32_MAX / 2 || K > INT32_MAX / 2 || V > INT32_MAX / 2)
    return errorf("gt_linear_xent_fwd_bwd: M, K and V must stay below 2^30");
  if (workspace_bytes < 0) return errorf("gt_linear_xent_fwd_bwd: negative workspace");
  const int64_t es = dtype == GT_FLOAT64 ? 8 : 4;
  if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)loss | (uintptr_t)row_loss | (uintptr_t)dx |
        (uintptr_t)dw | (uintptr_t)db) & (es - 1)) || (((uintptr_t)labels | (uintptr_t)bad_label) & 3))
    return errorf("gt_linear_xent_fwd_bwd: a pointer is not aligned to its elements");
  const Range in[] = {{x, M * K * es}, {w, V * K * es}, {bias, V * es}, {labels, M * 4}};
  const Range out[] = {{loss, es}, {row_loss, M * es}, {dx, M * K * es}, {dw, V * K * es}, {db, V * es}, {bad_label, 4}};
  for (const Range& o : out) {
    for (const Range& i : in)
      if (overlap(o, i)) return errorf("gt_linear_xent_fwd_bwd: an output overlaps an input");
    for (const Range& p : out)
      if (&p != &o && overlap(o, p)) return errorf("gt_linear_xent_fwd_bwd: two outputs overlap");
  }
  GT_ENTER(ctx);
  if (workspace_bytes == 0) workspace_bytes = (int64_t)1 << 30;
  void* held[5] = {};
  char* err = nullptr;
  GT_DISPATCH(dtype, {
    const XentCall<T> c{(const T*)x, (const T*)w, (const T*)bias, labels, M, K, V, ignore_label, workspace_bytes,
                        (T*)loss, (T*)row_loss, (T*)dx, (T*)dw, (T*)db, bad_label};
    err = linear_xent_pieces<T>(ctx, c, held);
  });
  for (void* h : held) release(ctx, h);
  return err;
}
