// What the paths of the large-vocabulary loss share.
#pragma once
#include "gt_common.cuh"

namespace gt {

// One call of gt_linear_xent_fwd_bwd (outputs that are not wanted are NULL).
template <typename T>
struct XentCall {
  const T *x, *w, *bias;
  const int32_t* labels;
  int64_t M, K, V;
  int32_t ignore;
  int64_t workspace;
  T *loss, *rows, *dx, *dw, *db;
  int32_t* bad;
  const double* over;  // what the sums are divided by; NULL: the number of rows that count
};

// The most that the partial sums of a product's K-splits take. They have a sixteenth of the workspace
// (at most this), and what the pieces leave of it.
constexpr int64_t kPartialBytes = (int64_t)128 << 20;

// The pointers of one workspace block.
struct Carver {
  char* base;
  int64_t used = 0;
  template <typename U>
  U* take(int64_t n) {
    U* p = base ? (U*)(base + used) : nullptr;
    used += ceil_div(n * (int64_t)sizeof(U), 256) * 256;
    return p;
  }
};

// The kernels of one call run one after another; each is launched while the one
// before it still runs, does what needs no input, and waits here until that
// one is done and its writes are visible (so every kernel before it is done
// too). It hides the launches' latency: 128 x 256 x 4000 takes 90 us without and 73 so.
// What an earlier kernel of the call writes is read through pointers that are
// not `const __restrict__` and without __ldg: those loads are taken as
// invariant and may be moved above the wait.
__device__ __forceinline__ void after_predecessor() {
  asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
inline cudaError_t launch_overlapped(gt_ctx* ctx, void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                                     A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// exp(d) for d <= 0 as the hardware's power of two: relative error about 2^-22
// and 2^-24 |d| of the rounded exponent.
__device__ __forceinline__ float exp_below(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
  return r;
}

// Joins two (maximum, sum of exponentials) pairs; one without a finite or
// infinite value has the maximum -infinity and the sum 0.
__device__ __forceinline__ void join(float2& a, const float2 b) {
  const float top = fmaxf(a.x, b.x), from = top == -INFINITY ? 0.0f : top;
  a.y = a.y * expf(a.x - from) + b.y * expf(b.x - from);
  a.x = top;
}

// loss = sum of the rows' losses / *n, in float64, one block, a fixed order; listed: only
// that many rows are there.
template <typename T>
__global__ void __launch_bounds__(1024) mean_rows_kernel(const T* rows, int64_t M, const int64_t* listed,
                                                         const double* n, T* loss) {
  after_predecessor();
  __shared__ double part[32];
  double acc = 0.0;
  if (listed) M = *listed;
  for (int64_t i = threadIdx.x; i < M; i += blockDim.x) acc += (double)rows[i];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    acc = 0.0;
    for (int w = 0; w < 32; w++) acc += part[w];
    *loss = (T)(acc / *n);
  }
}

// Calls of few rows (linear_xent_few.cu, at most 64): all with at most 8 rows,
// and those whose products stay below 2^27 terms, where the tensor-core path's
// dozen launches and mostly empty tiles cost more. (Its grid holds 2^25 classes.)
inline bool few_rows(int64_t M, int64_t K, int64_t V) {
  return V <= (int64_t)1 << 25 && (M <= 8 || (M <= 64 && (double)M * (double)K * (double)V <= 134217728.0));
}
char* linear_xent_few(gt_ctx* ctx, const XentCall<float>& c, void** held);

char* linear_xent(gt_ctx* ctx, const XentCall<double>& c, void** held);  // linear_xent_f64.cu

}  // namespace gt
