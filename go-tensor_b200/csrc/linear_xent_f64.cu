// The large-vocabulary loss in float64 (see linear_xent.cu for the formulas):
// pieces of rows, each through three products on the FP64 tensor pipe with one
// piece's logits in workspace.
//
//   label_count_kernel    the rows that count
//   per piece:
//     keep_rows_kernel    x with the ignored rows zeroed, its pitch even
//     f64_tile_kernel     z = x w^T + b
//     xent_segment_kernel, xent_scale_kernel  the rows' losses, G in place of z
//     f64_tile_kernel     dx = G w, dw (+)= G^T x
//     piece_columns_kernel  db
//   mean_rows_kernel      the loss
//
// The products range from one row to thousands and from K = 16 up, where the
// 128 x 128 tiles of the general FP64 GEMM are mostly padding and
// its small-shape kernels stay far from both peaks (4 x 1000 x 50000 took 3124 us
// through them). So they have tiles of their own, chosen by the least padding, two to
// four blocks to an SM, and K split over whatever SMs are left.
#include <algorithm>

#include "linear_xent.cuh"

namespace gt {

// *divisor = rows that count (label != ignore), or *over; a label outside [0, V) sets *bad.
__global__ void __launch_bounds__(1024) label_count_kernel(const int32_t* __restrict__ labels, int64_t M, int64_t V,
                                                           int32_t ignore, const double* over, double* divisor,
                                                           int32_t* bad) {
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
    *divisor = over ? *over : (double)n;
  }
}

// out = x with the ignored rows zeroed (padding may hold anything), a warp per
// 256 values of a row.
__global__ void __launch_bounds__(256) keep_rows_kernel(const double* __restrict__ x, const int32_t* __restrict__ labels,
                                                        int64_t rows, int64_t K, int64_t Kp, int32_t ignore,
                                                        double* out) {
  after_predecessor();
  const int64_t across = (K + 255) / 256;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < rows * across; u += (int64_t)gridDim.x * 8) {
    const int64_t i = u / across, k0 = (u - i * across) * 256 + (threadIdx.x & 31);
    const bool keep = labels[i] != ignore;
    double v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = keep && k0 + 32 * j < K ? x[i * K + k0 + 32 * j] : 0.0;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (k0 + 32 * j < K) out[i * Kp + k0 + 32 * j] = v[j];
  }
}

__device__ __forceinline__ double block_reduce(double v, double* ws, bool sum) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const double o = __shfl_xor_sync(0xffffffffu, v, off);
    v = sum ? v + o : go_max(v, o);
  }
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  v = ws[0];
  for (int w = 1; w < 8; w++) v = sum ? v + ws[w] : go_max(v, ws[w]);
  __syncthreads();
  return v;
}

// A block per segment of 4096 classes of a row, in registers: the segment's
// maximum and sum of exponentials. A row of one segment is finished here (z read
// once, G written once: 8000 x 3000 took 215 us in three passes over a row);
// of more, e = exp(z - the segment's maximum) is left in place of z for
// xent_scale_kernel.
constexpr int kSegment = 4096;
__global__ void __launch_bounds__(256) xent_segment_kernel(double* z, const int32_t* __restrict__ labels, int64_t V,
                                                           int64_t Vp, int64_t segments, int32_t ignore,
                                                           const double* divisor, double2* pairs, double* picked,
                                                           double* row_loss, bool grad) {
  after_predecessor();
  __shared__ double ws[8];
  const int64_t i = blockIdx.x / segments, seg = blockIdx.x - i * segments;
  const int32_t y = labels[i];
  const int64_t n = min((int64_t)kSegment, V - seg * kSegment), at = (int64_t)y - seg * kSegment;
  double* zr = z + i * Vp + seg * kSegment;
  auto put = [&](const double(&e)[16]) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int c = 2 * (threadIdx.x + 256 * j);
      if (c < n) *reinterpret_cast<double2*>(zr + c) = make_double2(e[2 * j], e[2 * j + 1]);  // (the pitch is even)
    }
  };
  double e[16];
  if (y == ignore) {
    if (seg == 0 && threadIdx.x == 0) row_loss[i] = 0.0;
#pragma unroll
    for (int j = 0; j < 16; j++) e[j] = 0.0;
    if (grad) put(e);
    return;
  }
  double m = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int c = 2 * (threadIdx.x + 256 * j);
    double2 v = make_double2(-INFINITY, -INFINITY);
    if (c < n) v = *reinterpret_cast<const double2*>(zr + c);
    e[2 * j] = v.x, e[2 * j + 1] = c + 1 < n ? v.y : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 16; j++) m = go_max(m, e[j]);
  m = block_reduce(m, ws, false);
  const bool outside = y < 0 || y >= V;
  const double label_z = at >= 0 && at < n && !outside ? zr[at] : (double)NAN;
  // (from 0 where nothing is above -infinity: the sum is then 0, not NaN)
  const double from = segments > 1 && m == -INFINITY ? 0.0 : m;
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    // (not exp(z - lse): the logarithm would vanish beside a maximum that is a
    // mask's lowest value)
    const int c = 2 * (threadIdx.x + 256 * (j >> 1)) + (j & 1);
    e[j] = c < n ? exp(e[j] - from) : 0.0;
    s += e[j];
  }
  s = block_reduce(s, ws, true);  // (every thread has read label_z by now)
  if (segments > 1) {
    if (threadIdx.x == 0) {
      pairs[i * segments + seg] = make_double2(m, s);
      if (at >= 0 && at < n) picked[i] = label_z;
    }
  } else {
    if (threadIdx.x == 0) row_loss[i] = log(s) + (m - label_z);
    const double inv = 1.0 / *divisor, f = inv / s;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const int c = 2 * (threadIdx.x + 256 * (j >> 1)) + (j & 1);
      e[j] = c == at ? e[j] * f - inv : e[j] * f;
    }
  }
  if (grad) put(e);
}

// Rows of several segments: the pairs joined (by every block of the row), the
// row's loss, and e -> G.
__global__ void __launch_bounds__(256) xent_scale_kernel(double* z, const int32_t* __restrict__ labels, int64_t V,
                                                         int64_t Vp, int64_t segments, int64_t blocks, int32_t ignore,
                                                         const double* divisor, const double2* pairs,
                                                         const double* picked, double* row_loss, bool grad) {
  after_predecessor();
  __shared__ double ws[8];
  const int64_t i = blockIdx.x / blocks, seg = blockIdx.x - i * blocks;
  const int32_t y = labels[i];
  if (y == ignore) return;  // done
  double m = -INFINITY, s = 0.0;
  for (int64_t g = threadIdx.x; g < segments; g += 256) m = go_max(m, pairs[i * segments + g].x);
  m = block_reduce(m, ws, false);
  const double from = m == -INFINITY ? 0.0 : m;
  for (int64_t g = threadIdx.x; g < segments; g += 256) {
    const double2 p = pairs[i * segments + g];
    s += p.y * exp(p.x - from);
  }
  s = block_reduce(s, ws, true);
  if (seg == 0 && threadIdx.x == 0) row_loss[i] = y < 0 || y >= V ? (double)NAN : log(s) + (m - picked[i]);
  if (!grad) return;
  const double inv = 1.0 / *divisor;
  const double f = exp(pairs[i * segments + seg].x - from) * (inv / s);
  const int64_t n = min((int64_t)kSegment, V - seg * kSegment), at = (int64_t)y - seg * kSegment;
  double* zr = z + i * Vp + seg * kSegment;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int c = 2 * (threadIdx.x + 256 * j);
    if (c >= n) continue;
    double2 v = *reinterpret_cast<const double2*>(zr + c);
    v.x = c == at ? v.x * f - inv : v.x * f;
    v.y = c + 1 == at ? v.y * f - inv : v.y * f;
    *reinterpret_cast<double2*>(zr + c) = v;
  }
}

// C (M, N) = sum_k A(m, k) B(k, n), with C's columns offset by bias, its rows with
// an ignored label set to 0 (0 times an infinity in w is not), or C added to.
struct F64Product {
  int64_t M, N, K;
  const double* a;  // (m, k) at m lda + k, or k lda + m when transposed
  int64_t lda;
  const double* b;  // (k, n) at n ldb + k when transposed, or k ldb + n
  int64_t ldb;
  double* out;
  int64_t ldc;
  const double* bias = nullptr;
  const int32_t* labels = nullptr;
  int32_t ignore = 0;
  bool accumulate = false;
  int64_t partial_bytes = 0;  // the most that the partial sums of K-splits may take
};

// Units 0 .. whole - 1 are tiles; each further tile is `splits` units over
// ranges of k_per, whose partial tiles are added in the order of K.
struct F64Plan {
  int64_t gx = 1, tiles = 0, whole = 0, splits = 1, k_per = 0;
};

constexpr int kF64Depth = 16;  // K per stage

// BM x BN per block, WM x 32 per warp.
template <int BM_, int BN_, int WM_, int STAGES_, int CTAS_>
struct F64Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, STAGES = STAGES_, CTAS = CTAS_;
  static constexpr int WARPS = (BM / WM) * (BN / 32), THREADS = 32 * WARPS;
};

// An operand stays in its memory order in shared memory: [row][k] in rows of
// 20 doubles where K is contiguous, else [k][row] in rows of R + 4. In both, a
// fragment (thread t: k = t % 4, row t / 4) falls in distinct banks.
template <int R, bool KC>
struct F64Stage {
  static constexpr int PITCH = KC ? kF64Depth + 4 : R + 4, SIZE = KC ? R * PITCH : kF64Depth * PITCH;
  static __device__ __forceinline__ int at(int k, int r) { return KC ? r * PITCH + k : k * PITCH + r; }

  // The slice [k0, k0 + 16) x [r0, r0 + R); what lies behind k_end or rows is
  // zero and not read. V16: two elements a copy.
  template <int THREADS, bool V16>
  static __device__ __forceinline__ void copy(double* dst, const double* src, int64_t ld, int64_t k0, int64_t k_end,
                                              int64_t r0, int64_t rows) {
    constexpr int W = V16 ? 2 : 1, N = R * kF64Depth / (W * THREADS);
    static_assert(N * W * THREADS == R * kF64Depth);
#pragma unroll
    for (int q = 0; q < N; q++) {
      const int e = threadIdx.x + THREADS * q;
      const int k = KC ? W * (e % (kF64Depth / W)) : e / (R / W), r = KC ? e / (kF64Depth / W) : W * (e % (R / W));
      const int64_t gk = k0 + k, gr = r0 + r, left = KC ? k_end - gk : rows - gr;
      const int n = (KC ? gr < rows : gk < k_end) ? (int)max((int64_t)0, min((int64_t)W, left)) : 0;
      const double* from = n ? src + (KC ? gr * ld + gk : gk * ld + gr) : src;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst + at(k, r));
      if constexpr (V16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(8 * n) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(8 * n) : "memory");
    }
  }
};

__device__ __forceinline__ double f64_finish(const F64Product& p, int64_t m, int64_t n, double v) {
  if (p.bias) v += p.bias[n];
  if (p.labels && p.labels[m] == p.ignore) v = 0.0;
  return v;
}

// KA, KB: K is contiguous in A, in B. 512 x 512 x 8192: z 177 us, dx 155, dw 174 (24 to 28 of 37
// TFLOP/s, bound by the FP64 tensor pipe and, at 512 tiles on 296 places, by
// rounds); 4 x 1000 x 50000: 78, 73 and 113 us against 62 each for w's bytes.
template <typename T, bool KA, bool KB, bool VA, bool VB>
__global__ void __launch_bounds__(T::THREADS, T::CTAS) f64_tile_kernel(const F64Product p, const F64Plan plan,
                                                                       double* ws) {
  after_predecessor();
  using SA = F64Stage<T::BM, KA>;
  using SB = F64Stage<T::BN, KB>;
  constexpr int MI = T::WM / 8, STAGE = SA::SIZE + SB::SIZE;
  extern __shared__ __align__(16) double f64_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wm = T::WM * (warp / (T::BN / 32)), wn = 32 * (warp % (T::BN / 32));
  int64_t tile = blockIdx.x, k_begin = 0, k_end = p.K;
  double* part = nullptr;
  if (tile >= plan.whole) {
    const int64_t unit = tile - plan.whole;
    tile = plan.whole + unit / plan.splits;
    k_begin = unit % plan.splits * plan.k_per;
    k_end = min(k_begin + plan.k_per, p.K);
    if (plan.splits > 1) part = ws + unit * (T::BM * T::BN);
  }
  const int64_t m0 = tile / plan.gx * T::BM, n0 = tile % plan.gx * T::BN;
  const int64_t slices = (k_end - k_begin + kF64Depth - 1) / kF64Depth;
  auto load = [&](int64_t slice) {
    if (slice < slices) {
      double* s = f64_smem + slice % T::STAGES * STAGE;
      const int64_t k0 = k_begin + slice * kF64Depth;
      SA::template copy<T::THREADS, VA>(s, p.a, p.lda, k0, k_end, m0, p.M);
      SB::template copy<T::THREADS, VB>(s + SA::SIZE, p.b, p.ldb, k0, k_end, n0, p.N);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  double acc[MI][4][2];
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j][0] = acc[i][j][1] = 0.0;
  const int fk = lane & 3, fr = lane >> 2;
#pragma unroll
  for (int s = 0; s < T::STAGES - 1; s++) load(s);
  for (int64_t t = 0; t < slices; t++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(T::STAGES - 2) : "memory");
    __syncthreads();  // slice t is there for all, and the stage of slice t - 1 is free
    load(t + T::STAGES - 1);
    const double* as = f64_smem + t % T::STAGES * STAGE + SA::at(fk, wm + fr);
    const double* bs = f64_smem + t % T::STAGES * STAGE + SA::SIZE + SB::at(fk, wn + fr);
    const int64_t left = k_end - k_begin - t * kF64Depth;
#pragma unroll
    for (int k = 0; k < kF64Depth; k += 4) {
      if (k >= left) break;  // dw of a few rows
      double a[MI], b[4];
#pragma unroll
      for (int i = 0; i < MI; i++) a[i] = as[SA::at(k, 8 * i)];
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = bs[SB::at(k, 8 * j)];
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
                       : "+d"(acc[i][j][0]), "+d"(acc[i][j][1])
                       : "d"(a[i]), "d"(b[j]));
    }
  }
  // A thread holds C(8 i + lane / 4, 8 j + 2 (lane % 4) + {0, 1}) of the warp's tile.
  const bool pairs = ((p.ldc & 1) | ((uintptr_t)p.out & 15)) == 0;
#pragma unroll
  for (int i = 0; i < MI; i++) {
    const int64_t m = m0 + wm + 8 * i + fr;
    if (m >= p.M) continue;
    const int64_t n = n0 + wn + 2 * fk;
    if (part) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        *reinterpret_cast<double2*>(part + (m - m0) * T::BN + wn + 8 * j + 2 * fk) =
            make_double2(acc[i][j][0], acc[i][j][1]);
      continue;
    }
    double* o = p.out + m * p.ldc + n;
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        if (n + 8 * j + h < p.N) {
          acc[i][j][h] = f64_finish(p, m, n + 8 * j + h, acc[i][j][h]);
          if (p.accumulate) acc[i][j][h] = o[8 * j + h] + acc[i][j][h];
        }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (pairs && n + 8 * j + 1 < p.N) {
        *reinterpret_cast<double2*>(o + 8 * j) = make_double2(acc[i][j][0], acc[i][j][1]);
      } else {
#pragma unroll
        for (int h = 0; h < 2; h++)
          if (n + 8 * j + h < p.N) o[8 * j + h] = acc[i][j][h];
      }
    }
  }
}

// The split tiles, their partials in the order of K.
__global__ void __launch_bounds__(256) f64_parts_kernel(const F64Product p, const F64Plan plan, int bm, int bn,
                                                        const double* ws) {
  after_predecessor();
  const int64_t area = (int64_t)bm * bn, total = (plan.tiles - plan.whole) * area;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / area, e = i - r * area, tile = plan.whole + r;
    const int64_t m = tile / plan.gx * bm + e / bn, n = tile % plan.gx * bn + e % bn;
    if (m >= p.M || n >= p.N) continue;
    const double* q = ws + r * plan.splits * area + e;
    double v = q[0];
#pragma unroll 8
    for (int64_t s = 1; s < plan.splits; s++) v += q[s * area];
    v = f64_finish(p, m, n, v);
    double* o = p.out + m * p.ldc + n;
    *o = p.accumulate ? *o + v : v;
  }
}

// Whole tiles for as many rounds as fill every SM; the rest in the number of
// ranges of K (at least 64 deep) that costs least: rounds of units, by flops or
// bytes, plus the partials' way through memory and one more launch.
template <typename T>
static F64Plan f64_plan(const gt_ctx* ctx, const F64Product& p) {
  F64Plan best;
  best.gx = ceil_div(p.N, T::BN), best.tiles = best.gx * ceil_div(p.M, T::BM);
  best.whole = best.tiles, best.k_per = p.K;
  const int64_t slots = (int64_t)ctx->sm_count * T::CTAS, rest = best.tiles % slots;
  if (rest == 0) return best;
  const double rows = (double)std::min<int64_t>(p.M, T::BM), cols = (double)std::min<int64_t>(p.N, T::BN);
  const double tile_s = (double)p.K * (double)slots *
                        std::max(2.0 * T::BM * T::BN / 30e12, 8.0 * (rows + cols) / 5e12);
  auto cost = [&](int64_t k_per, int64_t splits) {
    const int64_t units = rest * splits;
    const double traffic = splits > 1 ? 3e-6 + 16.0 * (double)units * rows * cols / 5e12 : 0.0;
    return (double)ceil_div(units, slots) * tile_s * ((double)k_per / (double)p.K) + traffic;
  };
  double least = cost(p.K, 1);
  for (int64_t s = 2; s <= 256 && p.K / s >= 64 && rest * s <= 4 * slots; s++) {
    const int64_t k_per = ceil_div(ceil_div(p.K, s), kF64Depth) * kF64Depth, splits = ceil_div(p.K, k_per);
    if (rest * splits * T::BM * T::BN * 8 > p.partial_bytes) break;
    const double c = cost(k_per, splits);
    if (c < 0.97 * least) least = c, best.k_per = k_per, best.splits = splits, best.whole = best.tiles - rest;
  }
  return best;
}

template <typename T, bool KA, bool KB, bool VA, bool VB>
static char* f64_run(gt_ctx* ctx, const F64Product& p, double* ws, int64_t* need) {
  constexpr size_t smem = T::STAGES * (F64Stage<T::BM, KA>::SIZE + F64Stage<T::BN, KB>::SIZE) * sizeof(double);
  const F64Plan plan = f64_plan<T>(ctx, p);
  const int64_t parts = (plan.tiles - plan.whole) * plan.splits, units = plan.whole + parts;
  if (units > INT32_MAX) return errorf("gt_linear_xent_fwd_bwd: %lld tiles of a product", (long long)units);
  if (need) {
    if (plan.splits > 1) *need = std::max(*need, parts * T::BM * T::BN);
    return nullptr;
  }
  auto kernel = f64_tile_kernel<T, KA, KB, VA, VB>;
  static bool configured[64] = {};
  if (ctx->device < 0 || ctx->device >= 64 || !configured[ctx->device]) {
    GT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (ctx->device >= 0 && ctx->device < 64) configured[ctx->device] = true;
  }
  GT_CUDA(launch_overlapped(ctx, kernel, (unsigned)units, T::THREADS, smem, p, plan, ws));
  if (plan.splits > 1)
    GT_CUDA(launch_overlapped(ctx, f64_parts_kernel, grid_for(ctx, (plan.tiles - plan.whole) * T::BM * T::BN, 256), 256,
                              0, p, plan, (int)T::BM, (int)T::BN, ws));
  return nullptr;
}

// The tile with the least padded work, the smaller ones charged for what they
// read more often per product. With `need`, only the doubles of ws that the product
// wants (at least *need). A has an even pitch and an aligned base (it and, for
// dw, B are workspace); B may be the caller's.
template <bool KA, bool KB>
static char* f64_product(gt_ctx* ctx, const F64Product& p, double* ws, int64_t* need) {
  const bool vb = ((p.ldb & 1) | ((uintptr_t)p.b & 15)) == 0;
  auto area = [&](int bm, int bn) { return (double)(ceil_div(p.M, bm) * bm) * (double)(ceil_div(p.N, bn) * bn); };
  const double cost[5] = {area(64, 128), area(128, 64), 1.15 * area(32, 128), 1.15 * area(128, 32), 1.4 * area(16, 128)};
  const int t = (int)(std::min_element(cost, cost + 5) - cost);
#define GT_F64_RUN(...) \
  (vb ? f64_run<F64Tile<__VA_ARGS__>, KA, KB, true, true>(ctx, p, ws, need) : f64_run<F64Tile<__VA_ARGS__>, KA, KB, true, false>(ctx, p, ws, need))
  if (t == 0) return GT_F64_RUN(64, 128, 32, 3, 2);
  if (t == 1) return GT_F64_RUN(128, 64, 32, 3, 2);
  if (t == 2) return GT_F64_RUN(32, 128, 32, 2, 4);
  if (t == 3) return GT_F64_RUN(128, 32, 32, 2, 4);
  return GT_F64_RUN(16, 128, 16, 2, 4);
#undef GT_F64_RUN
}

// db (+)= column sums of a piece's gradient: 32 columns per block, warp w adds
// the rows w, w + 32, ... in order, then the warps' sums in order.
__global__ void __launch_bounds__(1024) piece_columns_kernel(const double* g, int64_t rows, int64_t V,
                                                             int64_t Vp, bool first, double* db) {
  after_predecessor();
  __shared__ double ws[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  double acc = 0.0;
  if (c < V) {
#pragma unroll 8
    for (int64_t i = warp; i < rows; i += 32) acc += g[i * Vp + c];
  }
  ws[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || c >= V) return;
  for (int i = 1; i < 32; i++) acc += ws[i][lane];
  db[c] = first ? acc : db[c] + acc;
}

char* linear_xent(gt_ctx* ctx, const XentCall<double>& c, void** held) {
  const bool grad = c.dx || c.dw || c.db;
  const int64_t Kp = ceil_div(c.K, 2) * 2, Vp = ceil_div(c.V, 2) * 2;  // even: 16-byte copies
  const int64_t segments = ceil_div(c.V, kSegment);
  // Rows per piece: as many as the workspace holds beside the products' partial sums.
  const int64_t per_row = 8 * Vp + 8 * Kp + (segments > 1 ? 16 * segments + 8 : 0);
  int64_t R = (c.workspace - std::min(c.workspace / 16, kPartialBytes)) / per_row;
  R = std::min(c.M, R >= 128 ? R / 128 * 128 : 128);
  const int64_t partial_bytes = std::min(kPartialBytes, std::max<int64_t>(0, c.workspace - R * per_row));
  struct {
    double *divisor, *z, *x, *rows, *parts, *picked;
    double2* pairs;
  } ws{};
  // The products of the piece of r rows at r0, one kind at a time.
  auto logits = [&](int64_t r, int64_t* need) {
    F64Product p{r, c.V, c.K, ws.x, Kp, c.w, c.K, ws.z, Vp};
    p.bias = c.bias, p.partial_bytes = partial_bytes;
    return f64_product<true, true>(ctx, p, ws.parts, need);
  };
  auto dx = [&](int64_t r0, int64_t r, int64_t* need) {
    F64Product p{r, c.K, c.V, ws.z, Vp, c.w, c.K, c.dx + r0 * c.K, c.K};
    p.labels = c.labels + r0, p.ignore = c.ignore, p.partial_bytes = partial_bytes;
    return f64_product<true, false>(ctx, p, ws.parts, need);
  };
  auto dw = [&](int64_t r0, int64_t r, int64_t* need) {
    F64Product p{c.V, c.K, r, ws.z, Vp, ws.x, Kp, c.dw, c.K};
    p.accumulate = r0 > 0, p.partial_bytes = partial_bytes;
    return f64_product<false, false>(ctx, p, ws.parts, need);
  };
  int64_t need = 0;
  for (const int64_t r : {R, c.M - (c.M - 1) / R * R}) {  // a full piece, the last one
    GT_TRY(logits(r, &need));
    if (c.dx) GT_TRY(dx(0, r, &need));
    if (c.dw) GT_TRY(dw(0, r, &need));
  }
  auto carve = [&](Carver& k) {
    ws.divisor = k.take<double>(1);
    ws.z = k.take<double>(R * Vp);
    ws.x = k.take<double>(R * Kp);
    ws.rows = k.take<double>(c.rows ? 0 : c.M);
    ws.parts = k.take<double>(need);
    ws.pairs = k.take<double2>(segments > 1 ? R * segments : 0);
    ws.picked = k.take<double>(segments > 1 ? R : 0);
  };
  Carver size{nullptr};
  carve(size);
  GT_TRY(scratch(ctx, (size_t)size.used, &held[0]));
  Carver at{(char*)held[0]};
  carve(at);
  double* rows = c.rows ? c.rows : ws.rows;
  label_count_kernel<<<1, 1024, 0, ctx->stream>>>(c.labels, c.M, c.V, c.ignore, c.over, ws.divisor, c.bad);
  GT_LAUNCH_CHECK();
  for (int64_t r0 = 0; r0 < c.M; r0 += R) {
    const int64_t r = std::min(R, c.M - r0);
    const int32_t* labels = c.labels + r0;
    GT_CUDA(launch_overlapped(ctx, keep_rows_kernel, grid_for(ctx, r * ceil_div(c.K, 256), 8), 256, 0, c.x + r0 * c.K, labels, r, c.K, Kp,
                              c.ignore, ws.x));
    GT_TRY(logits(r, nullptr));
    GT_CUDA(launch_overlapped(ctx, xent_segment_kernel, (unsigned)(r * segments), 256, 0, ws.z, labels, c.V, Vp, segments,
                              c.ignore, ws.divisor, ws.pairs, ws.picked, rows + r0, grad));
    if (segments > 1) {
      const int64_t blocks = grad ? segments : 1;
      GT_CUDA(launch_overlapped(ctx, xent_scale_kernel, (unsigned)(r * blocks), 256, 0, ws.z, labels, c.V, Vp, segments,
                                blocks, c.ignore, ws.divisor, ws.pairs, ws.picked, rows + r0, grad));
    }
    if (c.dx) GT_TRY(dx(r0, r, nullptr));
    if (c.dw) GT_TRY(dw(r0, r, nullptr));
    if (c.db)
      GT_CUDA(launch_overlapped(ctx, piece_columns_kernel, (unsigned)ceil_div(c.V, 32), 1024, 0, ws.z, r, c.V, Vp,
                                r0 == 0, c.db));
  }
  GT_CUDA(launch_overlapped(ctx, mean_rows_kernel<double>, 1, 1024, 0, rows, c.M, nullptr, ws.divisor, c.loss));
  return nullptr;
}

}  // namespace gt
