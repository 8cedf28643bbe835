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
// become the gradient and are overwritten by the next piece, so memory does
// not grow with the number of rows. float32 runs on the tensor cores
// (split_gemm.cu):
//
//   row_count_kernel     the rows that count
//   operand_split_kernel w and the rows of x that count, which are listed: only
//                        they go through the products, as two float16 planes each,
//                        every row with a power of two of its own
//   per piece of these rows:
//     split_gemm         z, and per strip of 128 classes of a row its maximum
//                        and sum of exponentials, from the registers of the
//                        product; a forward pass alone never writes z
//     strip_join_kernel  the strips' pairs joined: lse, the rows' losses
//     grad_planes_kernel z -> n G as two float16 planes, once for dx and once for
//                        dw, its column sums
//     split_gemm         dx = G w, dw (+)= G^T x
//   mean_rows_kernel     the loss
//
// float64: linear_xent_f64.cu.
#include <algorithm>
#include <cmath>

#include "linear_xent.cuh"
#include "split_gemm.cuh"

namespace gt {

// What the kernels of one float32 call share: how many rows count, n (their
// number, or what the caller gave), the smallest up_to >= 0 with n <= 2^up_to (at
// most 31), and 2^up_to / n (0 when no row counts).
struct XentMeta {
  int64_t count;
  double n;
  int up_to;
  float share;
};

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

__device__ __forceinline__ uint32_t finite_bits4(float4 v) {
  return max(max(finite_bits(v.x), finite_bits(v.y)), max(finite_bits(v.z), finite_bits(v.w)));
}

constexpr int kCompactRows = 1024;  // rows per block of the compaction

// How many of each 1024 rows count; a label outside [0, V) sets *bad.
__global__ void __launch_bounds__(256) row_count_kernel(const int32_t* __restrict__ labels, int64_t M, int64_t V,
                                                        int32_t ignore, int32_t* counts, int32_t* bad) {
  int kept = 0;
  for (int i = threadIdx.x; i < kCompactRows; i += 256) {
    const int64_t m = (int64_t)blockIdx.x * kCompactRows + i;
    const int32_t y = m < M ? labels[m] : ignore;
    if (y != ignore && bad && (y < 0 || y >= V)) *bad = 1;
    kept += __syncthreads_count(y != ignore);
  }
  if (threadIdx.x == 0) counts[blockIdx.x] = kept;
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent e that puts a largest magnitude at 2^14 .. 2^15 when
// multiplied by 2^e: -113 .. 126. (2^126 is enough for any: what a plane then
// loses is below 2^-150, half of the smallest float32.) A row of zeros has 126
// too, so that G weighted with 2^-e counts it for nothing beside others.
__device__ __forceinline__ int plane_exponent(uint32_t top) {
  if (top == 0) return 126;
  return min(126, 14 - (top < 0x800000u ? 31 - __clz((int)top) - 149 : (int)(top >> 23) - 127));
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  const float back = __half2float(hi);
  lo = __float2half_rn(isfinite(back) ? __fsub_rn(v, back) : 0.0f);  // an infinity stays one
}

// w and the rows of x that count, in their order, as planes of pitch Kp, a warp
// per row: index[j] = the j-th such row, y[j] its label, xs[j] and ws[v] what the
// rows' values in the planes are to be multiplied by, wb[v] the class' bias; an
// ignored row's dx and loss are 0. A row's first 1024 values stay in registers, the
// rest is read twice, the second time from cache (its largest magnitude is wanted
// first): 34000 rows of 1024 in 42 us, 51000 of 1111, value by value, in 107.
// Behind the last row of x come zeros up to a multiple of 32
// rows (dw's products read that far). A row's place is the number of rows that
// count before it: the counts of the 1024-row blocks before its own, and a
// ballot over the labels of its own (a kernel of its own for this took 4 us more).
__global__ void __launch_bounds__(256, 4)
    operand_split_kernel(const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ bias,
                         const int32_t* __restrict__ labels, int64_t M, int64_t K, int64_t V, int64_t Kp,
                         int32_t ignore, const int32_t* counts, XentMeta* meta, int32_t* index, int32_t* y, float* xs,
                         float* ws, float* wb, __half* __restrict__ xp, __half* __restrict__ wp,
                         float* __restrict__ dx, float* rows, const double* over) {
  after_predecessor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the rows that count before row `end`
  auto count_before = [&](int64_t end) {
    const int64_t full = end / kCompactRows;
    int64_t n = 0;
    for (int64_t b = lane; b < full; b += 32) n += counts[b];
#pragma unroll 4
    for (int64_t m = full * kCompactRows + lane; m < end; m += 32) n += labels[m] != ignore;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
    return n;
  };
  if (blockIdx.x == 0 && warp == 0) {
    const int64_t count = count_before(M);
    if (lane == 0) {
      const double n = over ? *over : (double)count;
      int up_to = 0;
      while (up_to < 31 && n > (double)((int64_t)1 << up_to)) up_to++;
      meta->count = count;
      meta->n = n;
      meta->up_to = up_to;
      meta->share = count ? (float)((double)((int64_t)1 << up_to) / n) : 0.0f;
    }
  }
  for (int64_t v = V + (int64_t)blockIdx.x * 256 + threadIdx.x; v < (V + 255) / 256 * 256; v += (int64_t)gridDim.x * 256)
    ws[v] = 1.0f, wb[v] = -INFINITY;
  for (int64_t i = (int64_t)blockIdx.x * 8 + warp; i < V + M + 32; i += (int64_t)gridDim.x * 8) {
    const bool is_x = i >= V;
    bool keep = true;
    int64_t row = is_x ? i - V : i, to = row;
    if (is_x && row < M) {
      const int32_t label = labels[row];
      if (label == ignore) {
        if (rows && lane == 0) rows[row] = 0.0f;
        if (dx)
          for (int64_t k = lane; k < K; k += 32) dx[row * K + k] = 0.0f;
        continue;
      }
      to = count_before(row);
      if (lane == 0) index[to] = (int32_t)row, y[to] = label;
    } else if (is_x) {  // the zeros behind the last row
      const int64_t count = count_before(M);
      to = count + (row - M);
      if (to >= M || to >= (count + 31) / 32 * 32) continue;
      keep = false, row = 0;
    }
    const float* src = (is_x ? x : w) + row * K;
    __half* hi = (is_x ? xp : wp) + to * Kp;
    __half* lo = hi + (is_x ? M : V) * Kp;
    const bool vec = (K & 7) == 0 && ((uintptr_t)src & 15) == 0;
    auto load8 = [&](int64_t k, float (&v)[8]) {
      const float4 a = reinterpret_cast<const float4*>(src)[2 * k], b = reinterpret_cast<const float4*>(src)[2 * k + 1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    };
    float held[4][8];  // the row's first 1024 values
    uint32_t top = 0;
    if (vec) {
#pragma unroll
      for (int u = 0; u < 4; u++) {
#pragma unroll
        for (int j = 0; j < 8; j++) held[u][j] = 0.0f;
        if (keep && lane + 32 * u < K / 8) load8(lane + 32 * u, held[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, finite_bits(held[u][j]));
      if (keep) {
#pragma unroll 4
        for (int64_t k = 256 + lane; k < K / 4; k += 32)
          top = max(top, finite_bits4(reinterpret_cast<const float4*>(src)[k]));
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int64_t k = lane + 32 * (8 * u + j);
          held[u][j] = keep && k < K ? src[k] : 0.0f;
        }
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, finite_bits(held[u][j]));
      if (keep) {
#pragma unroll 8
        for (int64_t k = 1024 + lane; k < K; k += 32) top = max(top, finite_bits(src[k]));
      }
    }
    const int e = plane_exponent(__reduce_max_sync(0xffffffffu, top));
    const float f = exp2_int(e);
    if (lane == 0) (is_x ? xs : ws)[to] = exp2_int(-e);
    if (lane == 0 && !is_x) wb[to] = bias ? bias[to] : 0.0f;
    if (vec) {
      auto store8 = [&](int64_t k, const float (&v)[8]) {
        __align__(16) __half h[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; j++) split_half(__fmul_rn(v[j], f), h[j], l[j]);
        reinterpret_cast<uint4*>(hi)[k] = *reinterpret_cast<uint4*>(h);
        reinterpret_cast<uint4*>(lo)[k] = *reinterpret_cast<uint4*>(l);
      };
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (lane + 32 * u < K / 8) store8(lane + 32 * u, held[u]);
      for (int64_t k = 128 + lane; k < K / 8; k += 32) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (keep) load8(k, v);
        store8(k, v);
      }
    } else {
      auto store1 = [&](int64_t k, const float (&v)[8]) {  // values k, k + 32, ...
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (k + 32 * j < K) split_half(__fmul_rn(v[j], f), hi[k + 32 * j], lo[k + 32 * j]);
      };
#pragma unroll
      for (int u = 0; u < 4; u++) store1(lane + 256 * u, held[u]);
      for (int64_t k = 1024 + lane; k < K; k += 256) {  // eight loads in flight
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = keep && k + 32 * j < K ? src[k + 32 * j] : 0.0f;
        store1(k, v);
      }
    }
  }
}

// The rows of the piece at r0 that there are.
__device__ __forceinline__ int64_t rows_here(const XentMeta* meta, int64_t r0, int64_t R) {
  return max((int64_t)0, min(R, meta->count - r0));
}

// Per row: the strips' pairs joined (32 rows per block; a warp takes every
// 32nd strip, then the warps' pairs are joined in order), the row's loss (also
// at its place in the caller's rows), and (maximum, 1 / sum) for the gradient.
__global__ void __launch_bounds__(1024) strip_join_kernel(const float2* strips, int64_t R, int n, const int32_t* y,
                                                          const int32_t* index, const XentMeta* meta, int64_t r0,
                                                          int64_t V, const float* picked, float2* stat,
                                                          float* losses, float* rows) {
  after_predecessor();
  __shared__ float2 ws[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t m = (int64_t)blockIdx.x * 32 + lane, here = rows_here(meta, r0, R);
  if ((int64_t)blockIdx.x * 32 >= here) return;
  float2 a = make_float2(-INFINITY, 0.0f);
  if (m < here) {
#pragma unroll 4
    for (int i = warp; i < n; i += 32) join(a, strips[(int64_t)i * R + m]);
  }
  ws[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && m < here) {
    for (int i = 1; i < 32; i++) join(a, ws[i][lane]);
    const int32_t label = y[r0 + m];
    stat[m] = make_float2(a.x, __fdiv_rn(1.0f, a.y));
    const float loss = label < 0 || label >= V ? NAN : logf(a.y) + (a.x - picked[m]);
    losses[r0 + m] = loss;
    if (rows) rows[index[r0 + m]] = loss;
  }
}

// n G = exp(z - maximum) / sum - [label] for 128 rows of 128 columns, as two
// float16 planes for each of the products that it goes into, and, for db, summed over the rows.
//
// dx = G w sums over classes, whose rows of w have scales of their own, and dw = G^T x over
// rows of x. So the planes for dx hold q 2^T with q = n G ws[v] (and, where the tile's largest ws
// is below 1, a factor 2^-base that makes it 1: q stays a normal number), T of the row and
// the tile such that the largest |q| lands at 2^14 .. 2^15; those for dw the same with xs of
// the tile's rows and a T of the column. A class that is far from
// likely so keeps its digits in dw beside those that are likely, as does a
// row of small gradients in dx. What undoes it goes to dx_scale and dw_scale, with
// 2^-up_to, whose rest, share, the products multiply by at the end (no sum
// exceeds the result's own range so).
//
// A block has a tile of 128 x 128 in registers, since a column's T is known
// only when all its rows are; a warp has every 16th row, a lane four columns. The planes for
// dx take z's place: a row's 128 columns are as many bytes, and are read before they are written.
// 2048 x 32000: 136 us, 12 bytes per logit at 5.8 TB/s (one set of planes with one scale for all of G took 87 us).
constexpr int kGradTile = 128;
static_assert(kGradTile == kSplitGroup && kGradTile == kStripCols, "a tile is one group of K of either product");

// exp(d) for d <= 0, -infinity and NaN included (0): the exponent's rounding error is put back
// to first order, so the relative error is that of the hardware's power of two, about 2^-22, whatever d is.
__device__ __forceinline__ float exp_exact(float d) {
  constexpr float kLog2e = 1.4426950408889634f, kRest = (float)(1.4426950408889634 - (double)kLog2e);
  d = fmaxf(d, -200.0f);
  const float t = __fmul_rn(d, kLog2e);
  const float r = fmaf(d, kRest, fmaf(d, kLog2e, -t));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return fmaf(e, __fmul_rn(r, 0.6931471805599453f), e);
}

__device__ __forceinline__ void split_store(__half* hi, __half* lo, const float (&v)[4]) {
  const __half2 h[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
  const float2 a = __half22float2(h[0]), b = __half22float2(h[1]);
  const __half2 l[2] = {__floats2half2_rn(__fsub_rn(v[0], a.x), __fsub_rn(v[1], a.y)),
                        __floats2half2_rn(__fsub_rn(v[2], b.x), __fsub_rn(v[3], b.y))};
  *reinterpret_cast<uint2*>(hi) = *reinterpret_cast<const uint2*>(h);
  *reinterpret_cast<uint2*>(lo) = *reinterpret_cast<const uint2*>(l);
}

// The exponent of a power of two, or of a value's magnitude (a subnormal's as if it were 2^-127).
__device__ __forceinline__ int exponent_of(float v) { return (int)((__float_as_uint(v) >> 23) & 0xffu) - 127; }

// T for a largest |q| of `top` whose q already lacks a factor 2^base: such that
// neither 2^T nor 2^-(T - base + up_to) leaves the normal numbers.
__device__ __forceinline__ int tile_shift(float top, int base, int up_to) {
  return min(min(14 - exponent_of(top), 127), 126 - up_to + base);
}

template <bool DX, bool DW, bool DB>
__global__ void __launch_bounds__(512, 2) grad_planes_kernel(float* z, const float2* stat, const int32_t* y,
                                                             const float* xs, const float* ws, const XentMeta* meta,
                                                             int64_t r0, int64_t R, int64_t V, int64_t Vp, int across,
                                                             __half* g, int64_t plane, float* dx_scale,
                                                             float* dw_scale, float* part) {
  after_predecessor();
  __shared__ float tops[16][kGradTile], sums[16][kGradTile];
  __shared__ float4 about[kGradTile];  // per row: maximum, 1 / sum, xs, and the label's place in the tile
  __shared__ int shift[kGradTile];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rb = blockIdx.x / across, cb = blockIdx.x - rb * across;
  const int64_t m0 = rb * kGradTile, c = cb * kGradTile + 4 * lane, here = rows_here(meta, r0, R);
  // behind the last row come zeros up to a multiple of 32 rows (dw's products read that far)
  const int64_t end = min(R, (here + 31) / 32 * 32);
  if (m0 >= end) return;
  const int rows = (int)max((int64_t)0, min((int64_t)kGradTile, here - m0)), zeroed = (int)min((int64_t)kGradTile, end - m0);
  const int cols = (int)min((int64_t)4, max((int64_t)0, V - c));  // of this lane's four
  const int up_to = meta->up_to;
  float* zr = z + (m0 + warp) * Vp + c;
  float p[8][4];
#pragma unroll
  for (int u = 0; u < 8; u++) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (warp + 16 * u < rows) v = *reinterpret_cast<const float4*>(zr + (int64_t)(16 * u) * Vp);
    p[u][0] = v.x, p[u][1] = v.y, p[u][2] = v.z, p[u][3] = v.w;
  }
  if (threadIdx.x < rows) {
    const int64_t m = m0 + threadIdx.x;
    const float2 s = stat[m];
    const int64_t at = (int64_t)y[r0 + m] - cb * kGradTile;
    about[threadIdx.x] = make_float4(s.x, s.y, xs[r0 + m], __int_as_float(at >= 0 && at < kGradTile ? (int)at : -4));
  }
  __syncthreads();
  // ws and xs relative to the tile's largest where that is below 1
  float wf[4] = {0.f, 0.f, 0.f, 0.f};
  int w_base = 0, x_base = 0;
  if (DX) {
    const float4 f = *reinterpret_cast<const float4*>(ws + c);
    wf[0] = f.x, wf[1] = f.y, wf[2] = f.z, wf[3] = f.w;
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (j >= cols) wf[j] = 0.0f;
      top = fmaxf(top, wf[j]);
    }
    w_base = min(0, exponent_of(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)))));
#pragma unroll
    for (int j = 0; j < 4; j++) wf[j] *= exp2_int(-w_base);
  }
  if (DW) {
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (lane + 32 * u < rows) top = fmaxf(top, about[lane + 32 * u].z);
    x_base = min(0, exponent_of(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)))));
  }
  const float x_unit = exp2_int(-x_base);
  float top[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 8; u++) {
    const int row = warp + 16 * u;
    if (row >= rows) {
#pragma unroll
      for (int j = 0; j < 4; j++) p[u][j] = 0.0f;
      continue;
    }
    const float4 s = about[row];
#pragma unroll
    for (int j = 0; j < 4; j++) p[u][j] = exp_exact(p[u][j] - s.x) * s.y;
    const int at = __float_as_int(s.w) - 4 * lane;
    if ((unsigned)at < 4u) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (at == j) p[u][j] -= 1.0f;
    }
    if (cols < 4) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j >= cols) p[u][j] = 0.0f;
    }
    if (DX) {
      float q[4], row_top = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) q[j] = p[u][j] * wf[j], row_top = fmaxf(row_top, fabsf(q[j]));
      row_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(row_top)));
      const int t = tile_shift(row_top, w_base, up_to);
      const float f = exp2_int(t);
#pragma unroll
      for (int j = 0; j < 4; j++) q[j] *= f;
      __half* o = reinterpret_cast<__half*>(zr + (int64_t)(16 * u) * Vp - 4 * lane) + 4 * lane;
      split_store(o, o + kGradTile, q);
      if (lane == 0) dx_scale[cb * R + m0 + row] = exp2_int(-(t - w_base + up_to));
    }
    const float xf = s.z * x_unit;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (DB) sum[j] += p[u][j];
      if (DW) p[u][j] *= xf, top[j] = fmaxf(top[j], fabsf(p[u][j]));
    }
  }
  if constexpr (DW || DB) {
    if (DW) *reinterpret_cast<float4*>(&tops[warp][4 * lane]) = make_float4(top[0], top[1], top[2], top[3]);
    if (DB) *reinterpret_cast<float4*>(&sums[warp][4 * lane]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (threadIdx.x < kGradTile) {
      const int64_t col = cb * kGradTile + threadIdx.x;
      float most = 0.0f, s = 0.0f;
#pragma unroll
      for (int u = 0; u < 16; u++) {
        if (DW) most = fmaxf(most, tops[u][threadIdx.x]);
        if (DB) s += sums[u][threadIdx.x];
      }
      const int t = tile_shift(most, x_base, up_to);
      if (DW) shift[threadIdx.x] = t;
      if (DW && col < V) dw_scale[rb * V + col] = exp2_int(-(t - x_base + up_to));
      if (DB && col < V) part[rb * V + col] = s;
    }
  }
  if constexpr (DW) {
    __syncthreads();
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = exp2_int(shift[4 * lane + j]);
    __half* o = g + (m0 + warp) * Vp + c;
#pragma unroll
    for (int u = 0; u < 8; u++) {
      if (warp + 16 * u >= zeroed) break;
      const float q[4] = {p[u][0] * f[0], p[u][1] * f[1], p[u][2] * f[2], p[u][3] * f[3]};
      split_store(o + (int64_t)(16 * u) * Vp, o + (int64_t)(16 * u) * Vp + plane, q);
    }
  }
}

// db (+)= the column sums of the tiles' rows, / n: 32 columns per block,
// warp w adds the rows w, w + 8, ... in order, then the warps' sums in order.
__global__ void __launch_bounds__(256) db_kernel(const float* part, int64_t r0, int64_t R, int64_t V,
                                                 const XentMeta* meta, float* db) {
  after_predecessor();
  __shared__ double ws[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, blocks = (rows_here(meta, r0, R) + kGradTile - 1) / kGradTile;
  double acc = 0.0;
  if (c < V) {
#pragma unroll 8
    for (int64_t i = warp; i < blocks; i += 8) acc += (double)part[i * V + c];
  }
  ws[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || c >= V) return;
  for (int i = 1; i < 8; i++) acc += ws[i][lane];
  const float d = (float)(meta->count ? acc / meta->n : 0.0);
  db[c] = r0 == 0 ? d : db[c] + d;
}

// float32: see the top of the file.
static char* linear_xent(gt_ctx* ctx, const XentCall<float>& c, void** held) {
  if (few_rows(c.M, c.K, c.V)) return linear_xent_few(ctx, c, held);
  const bool grad = c.dx || c.dw || c.db;
  const int64_t Kp = ceil_div(c.K, 8) * 8, Vp = ceil_div(c.V, kGradTile) * kGradTile, groups = Vp / kGradTile;
  // Rows per piece: as many as the workspace holds beside the products' partial sums, in multiples of the tiles'
  // 256 rows, and the pieces of equal size. A row takes 4 bytes per logit for z and 4 for dw's
  // planes of G, and per 128 logits its strip and the scales and sums of G.
  const int64_t per_row = (grad ? 4 * Vp : 0) + (c.dw ? 4 * Vp : 0) + 24 * groups + 12;
  const int64_t rest = c.workspace - std::min(c.workspace / 16, kPartialBytes);
  int64_t R = std::max<int64_t>(1, rest / per_row / 256) * 256;
  R = std::min(c.M, ceil_div(ceil_div(c.M, ceil_div(c.M, R)), 256) * 256);
  const int64_t partial_bytes = std::min(kPartialBytes, std::max<int64_t>(0, c.workspace - R * per_row));
  const int64_t row_blocks = ceil_div(c.M, kCompactRows), tiles = ceil_div(R, kGradTile);
  struct {
    XentMeta* meta;
    __half *x, *w, *g;
    float *xs, *ws, *wb, *z, *losses, *picked, *part, *dx_scale, *dw_scale;
    float2 *strips, *stat;
    int32_t *counts, *index, *y;
  } ws;
  auto carve = [&](Carver& k) {
    ws.meta = k.take<XentMeta>(1);
    ws.x = k.take<__half>(2 * c.M * Kp);
    ws.w = k.take<__half>(2 * c.V * Kp);
    ws.xs = k.take<float>(c.M);
    ws.ws = k.take<float>(ceil_div(c.V, 256) * 256);
    ws.wb = k.take<float>(ceil_div(c.V, 256) * 256);
    ws.g = k.take<__half>(c.dw ? 2 * R * Vp : 0);
    ws.z = k.take<float>(grad ? R * Vp : 0);
    ws.losses = k.take<float>(c.M);
    ws.picked = k.take<float>(R);
    ws.part = k.take<float>(c.db ? tiles * c.V : 0);
    ws.dx_scale = k.take<float>(c.dx ? groups * R : 0);
    ws.dw_scale = k.take<float>(c.dw ? tiles * c.V : 0);
    ws.strips = k.take<float2>(groups * R);
    ws.stat = k.take<float2>(R);
    ws.counts = k.take<int32_t>(row_blocks);
    ws.index = k.take<int32_t>(c.M);
    ws.y = k.take<int32_t>(c.M);
  };
  Carver size{nullptr};
  carve(size);
  GT_TRY(scratch(ctx, (size_t)size.used, &held[0]));
  Carver at{(char*)held[0]};
  carve(at);

  row_count_kernel<<<(unsigned)row_blocks, 256, 0, ctx->stream>>>(c.labels, c.M, c.V, c.ignore, ws.counts, c.bad);
  GT_LAUNCH_CHECK();
  const int sb = (int)std::min<int64_t>(ceil_div(c.M + c.V + 32, 8), (int64_t)ctx->sm_count * 32);
  GT_CUDA(launch_overlapped(ctx, operand_split_kernel, sb, 256, 0, c.x, c.w, c.bias, c.labels, c.M, c.K, c.V, Kp,
                            c.ignore, ws.counts, ws.meta, ws.index, ws.y, ws.xs, ws.ws, ws.wb, ws.x, ws.w, c.dx, c.rows,
                            c.over));
  const HalfPlanes w{ws.w, c.V, c.K, Kp, c.V * Kp};
  for (int64_t r0 = 0; r0 < c.M; r0 += R) {
    // As many pieces as all rows would need; those behind the rows that count find nothing to do.
    const int64_t r = std::min(R, c.M - r0);
    const HalfPlanes x{ws.x + r0 * Kp, r, c.K, Kp, c.M * Kp};
    SplitGemm f;
    f.M = r, f.N = c.V, f.K = c.K, f.kept = &ws.meta->count, f.kept_from = r0, f.a = x, f.b = w;
    f.row_scale = ws.xs + r0, f.col_scale = ws.ws;
    f.out = grad ? ws.z : nullptr, f.ldc = Vp, f.bias = ws.wb, f.labels = ws.y + r0;
    f.strips = ws.strips, f.strip_rows = R, f.picked = ws.picked;
    GT_TRY(split_gemm(ctx, f));
    GT_CUDA(launch_overlapped(ctx, strip_join_kernel, (unsigned)ceil_div(r, 32), 1024, 0, ws.strips, R,
                              (int)ceil_div(c.V, kStripCols), ws.y, ws.index, ws.meta, r0, c.V, ws.picked, ws.stat,
                              ws.losses, c.rows));
    if (!grad) continue;
    const decltype(&grad_planes_kernel<false, false, true>) planes[8] = {
        nullptr, grad_planes_kernel<false, false, true>,
        grad_planes_kernel<false, true, false>, grad_planes_kernel<false, true, true>,
        grad_planes_kernel<true, false, false>, grad_planes_kernel<true, false, true>,
        grad_planes_kernel<true, true, false>, grad_planes_kernel<true, true, true>};
    GT_CUDA(launch_overlapped(ctx, planes[(c.dx ? 4 : 0) + (c.dw ? 2 : 0) + (c.db ? 1 : 0)],
                              (unsigned)(groups * ceil_div(r, kGradTile)), 512, 0, ws.z, ws.stat, ws.y, ws.xs, ws.ws,
                              ws.meta, r0, r, c.V, Vp, (int)groups, ws.g, R * Vp, ws.dx_scale, ws.dw_scale, ws.part));
    if (c.dx) {
      SplitGemm d;
      d.M = r, d.N = c.K, d.K = c.V, d.kept = &ws.meta->count, d.kept_from = r0, d.b = w, d.b_mn = true;
      d.a = HalfPlanes{reinterpret_cast<const __half*>(ws.z), r, c.V, 2 * Vp, 0, true};
      d.scale = &ws.meta->share, d.group_scale = ws.dx_scale, d.group_ld = r;
      d.out = c.dx, d.ldc = c.K, d.row_index = ws.index + r0, d.partial_bytes = partial_bytes;
      GT_TRY(split_gemm(ctx, d));
    }
    if (c.dw) {
      SplitGemm d;
      d.M = c.V, d.N = c.K, d.K = r, d.kept = &ws.meta->count, d.kept_from = r0, d.a_mn = true, d.b = x;
      d.a = HalfPlanes{ws.g, r, c.V, Vp, R * Vp}, d.b_mn = true;
      d.scale = &ws.meta->share, d.group_scale = ws.dw_scale, d.group_ld = c.V;
      d.out = c.dw, d.ldc = c.K, d.accumulate = r0 > 0, d.partial_bytes = partial_bytes;
      GT_TRY(split_gemm(ctx, d));
    }
    if (c.db)
      GT_CUDA(launch_overlapped(ctx, db_kernel, (unsigned)ceil_div(c.V, 32), 256, 0, ws.part, r0, r, c.V, ws.meta,
                                c.db));
  }
  GT_CUDA(launch_overlapped(ctx, mean_rows_kernel<float>, 1, 1024, 0, ws.losses, c.M, &ws.meta->count, &ws.meta->n,
                            c.loss));
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

static char* head_call(const char* who, gt_ctx* ctx, int dtype, const void* x, const void* w, const void* bias,
                       const int32_t* labels, int64_t M, int64_t K, int64_t V, int32_t ignore_label,
                       int64_t workspace_bytes, void* loss, void* row_loss, void* dx, void* dw, void* db,
                       int32_t* bad_label, const double* over) {
  GT_CHECK_DTYPE(dtype);
  if (!x || !w || !labels || !loss) return errorf("%s: null argument", who);
  if (M <= 0 || K <= 0 || V <= 0) return errorf("%s: M, K and V must be positive", who);
  if (M > INT32_MAX / 2 || K > INT32_MAX / 2 || V > INT32_MAX / 2)
    return errorf("%s: M, K and V must stay below 2^30", who);
  if ((double)M * (double)K > 0x1p56 || (double)V * (double)K > 0x1p56)
    return errorf("%s: x and w must stay below 2^56 elements", who);
  if (workspace_bytes < 0) return errorf("%s: negative workspace", who);
  const int64_t es = dtype == GT_FLOAT64 ? 8 : 4;
  if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)loss | (uintptr_t)row_loss | (uintptr_t)dx |
        (uintptr_t)dw | (uintptr_t)db) & (es - 1)) || (((uintptr_t)labels | (uintptr_t)bad_label) & 3) ||
      ((uintptr_t)over & 7))
    return errorf("%s: a pointer is not aligned to its elements", who);
  const Range in[] = {{x, M * K * es}, {w, V * K * es}, {bias, V * es}, {labels, M * 4}, {over, 8}};
  const Range out[] = {{loss, es}, {row_loss, M * es}, {dx, M * K * es}, {dw, V * K * es}, {db, V * es}, {bad_label, 4}};
  for (const Range& o : out) {
    for (const Range& i : in)
      if (overlap(o, i)) return errorf("%s: an output overlaps an input", who);
    for (const Range& p : out)
      if (&p != &o && overlap(o, p)) return errorf("%s: two outputs overlap", who);
  }
  GT_ENTER(ctx);
  if (workspace_bytes == 0) workspace_bytes = (int64_t)2 << 30;
  void* held[5] = {};
  char* err = nullptr;
  GT_DISPATCH(dtype, {
    const XentCall<T> c{(const T*)x, (const T*)w, (const T*)bias, labels, M, K, V, ignore_label, workspace_bytes,
                        (T*)loss, (T*)row_loss, (T*)dx, (T*)dw, (T*)db, bad_label, over};
    err = linear_xent(ctx, c, held);
  });
  for (void* h : held) release(ctx, h);
  return err;
}

// The number of labels that are not ignore, one block.
__global__ void __launch_bounds__(1024) count_labels_kernel(const int32_t* __restrict__ labels, int64_t n,
                                                            int32_t ignore, double* count) {
  __shared__ int64_t ws[32];
  int64_t kept = 0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) kept += labels[i] != ignore;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, off);
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = kept;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; w++) kept += ws[w];
    *count = (double)kept;
  }
}

extern "C" {

char* gt_linear_xent_fwd_bwd(gt_ctx* ctx, int dtype, const void* x, const void* w, const void* bias,
                             const int32_t* labels, int64_t M, int64_t K, int64_t V, int32_t ignore_label,
                             int64_t workspace_bytes, void* loss, void* row_loss, void* dx, void* dw, void* db,
                             int32_t* bad_label) {
  return head_call("gt_linear_xent_fwd_bwd", ctx, dtype, x, w, bias, labels, M, K, V, ignore_label, workspace_bytes,
                   loss, row_loss, dx, dw, db, bad_label, nullptr);
}

char* gt_linear_xent_fwd_bwd_over(gt_ctx* ctx, int dtype, const void* x, const void* w, const void* bias,
                                  const int32_t* labels, int64_t M, int64_t K, int64_t V, int32_t ignore_label,
                                  int64_t workspace_bytes, const double* over, void* loss, void* row_loss, void* dx,
                                  void* dw, void* db, int32_t* bad_label) {
  if (!over) return errorf("gt_linear_xent_fwd_bwd_over: null argument");
  return head_call("gt_linear_xent_fwd_bwd_over", ctx, dtype, x, w, bias, labels, M, K, V, ignore_label,
                   workspace_bytes, loss, row_loss, dx, dw, db, bad_label, over);
}

char* gt_count_labels(gt_ctx* ctx, const int32_t* labels, int64_t n, int32_t ignore_label, double* count) {
  if (!labels || !count) return errorf("gt_count_labels: null argument");
  if (n < 0) return errorf("gt_count_labels: negative length");
  if (((uintptr_t)labels & 3) || ((uintptr_t)count & 7))
    return errorf("gt_count_labels: a pointer is not aligned to its elements");
  GT_ENTER(ctx);
  count_labels_kernel<<<1, 1024, 0, ctx->stream>>>(labels, n, ignore_label, count);
  GT_LAUNCH_CHECK();
  return nullptr;
}

}  // extern "C"
