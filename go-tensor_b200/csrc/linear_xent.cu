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
//   operand_top_kernel   largest magnitudes of x and w, the rows that count
//   operand_split_kernel w and the rows of x that count, which are listed: only
//                        they go through the products, as two float16 planes each
//   per piece of these rows:
//     split_gemm         z, and per strip of 128 classes of a row its maximum
//                        and sum of exponentials, from the registers of the
//                        product; a forward pass alone never writes z
//     strip_join_kernel  the strips' pairs joined: lse, the rows' losses
//     grad_planes_kernel z -> n G as two float16 planes, its column sums
//     split_gemm         dx = G w, dw (+)= G^T x
//   mean_rows_kernel     the loss
//
// float64: linear_xent_f64.cu.
#include <algorithm>
#include <cmath>

#include "linear_xent.cuh"
#include "split_gemm.cuh"

namespace gt {

// What the kernels of one float32 call share: the operands' largest finite
// magnitudes (as ordered words), the rows that count, and the products' factors.
struct XentMeta {
  uint32_t x_top, w_top;
  int64_t count;
  SplitScale logits, dx, dw;
};

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

__device__ __forceinline__ uint32_t finite_bits4(float4 v) {
  return max(max(finite_bits(v.x), finite_bits(v.y)), max(finite_bits(v.z), finite_bits(v.w)));
}

constexpr int kCompactRows = 1024;  // rows per block of the compaction

// The largest magnitudes of w (blocks 0 .. w_blocks - 1) and of the rows of x
// that count (the next x_blocks, a warp per row), and how many of each 1024 rows
// count (the others); a label outside [0, V) sets *bad.
__global__ void __launch_bounds__(256) operand_top_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                          const int32_t* __restrict__ labels, int64_t M, int64_t K,
                                                          int64_t V, int32_t ignore, int w_blocks, int x_blocks,
                                                          XentMeta* meta, int32_t* counts, int32_t* bad) {
  __shared__ uint32_t tops[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t top = 0;
  if ((int)blockIdx.x >= w_blocks + x_blocks) {
    const int64_t b = blockIdx.x - w_blocks - x_blocks;
    int kept = 0;
    for (int i = threadIdx.x; i < kCompactRows; i += 256) {
      const int64_t m = b * kCompactRows + i;
      kept += __syncthreads_count(m < M && labels[m] != ignore);
    }
    if (threadIdx.x == 0) counts[b] = kept;
    return;
  }
  if ((int)blockIdx.x < w_blocks) {
    const int64_t n = V * K, stride = (int64_t)w_blocks * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t n4 = ((uintptr_t)w & 15) == 0 ? n / 4 : 0;
    const float4* w4 = reinterpret_cast<const float4*>(w);
    for (int64_t i = at; i < n4; i += 4 * stride) {  // four loads in flight
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; u++) v[u] = i + u * stride < n4 ? w4[i + u * stride] : float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 4; u++) top = max(top, finite_bits4(v[u]));
    }
    for (int64_t i = n4 * 4 + at; i < n; i += stride) top = max(top, finite_bits(w[i]));
  } else {
    for (int64_t m = (int64_t)(blockIdx.x - w_blocks) * 8 + warp; m < M; m += (int64_t)x_blocks * 8) {
      const int32_t y = labels[m];
      if (y == ignore) continue;
      if (lane == 0 && bad && (y < 0 || y >= V)) *bad = 1;
      const float* r = x + m * K;
      const int64_t k4 = ((K & 3) | ((uintptr_t)x & 15)) == 0 ? K / 4 : 0;
      for (int64_t k = lane; k < k4; k += 128) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
          v[u] = k + 32 * u < k4 ? reinterpret_cast<const float4*>(r)[k + 32 * u] : float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 4; u++) top = max(top, finite_bits4(v[u]));
      }
#pragma unroll 4
      for (int64_t k = 4 * k4 + lane; k < K; k += 32) top = max(top, finite_bits(r[k]));
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; i++) top = max(top, tops[i]);
    if (top) atomicMax((int)blockIdx.x < w_blocks ? &meta->w_top : &meta->x_top, top);
  }
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent e that puts a largest magnitude at 2^14 .. 2^15 when
// multiplied by 2^e: -113 .. 163.
__device__ __forceinline__ int plane_exponent(uint32_t top) {
  if (top == 0) return 0;
  return 14 - (top < 0x800000u ? 31 - __clz((int)top) - 149 : (int)(top >> 23) - 127);
}

// 2^-e times f (at most 1), as one factor, or as two halves of the power where one
// would not be a normal number (beyond 2^-252 nothing is left of an accumulator anyway).
__device__ __forceinline__ SplitScale undo(int e, float f) {
  e = min(e, 252);
  if (e >= -126 && e <= 64) return {__fmul_rn(exp2_int(-e), f), 1.0f};
  return {exp2_int(-e / 2), __fmul_rn(exp2_int(-e - (-e / 2)), f)};
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  const float back = __half2float(hi);
  lo = __float2half_rn(isfinite(back) ? __fsub_rn(v, back) : 0.0f);  // an infinity stays one
}

constexpr int kGradExponent = 15;  // n G lies in [-1, 1]

// w and the rows of x that count, in their order, as planes of pitch Kp, a warp
// per row: index[j] = the j-th such row, y[j] its label; an ignored row's dx
// and loss are 0. Behind the last row of x come zeros up to a multiple of 32
// rows (dw's products read that far). A row's place is the number of rows that
// count before it: the counts of the 1024-row blocks before its own, and a
// ballot over the labels of its own (a kernel of its own for this took 4 us more).
__global__ void __launch_bounds__(256) operand_split_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                            const int32_t* __restrict__ labels, int64_t M, int64_t K,
                                                            int64_t V, int64_t Kp, int32_t ignore,
                                                            const int32_t* counts, XentMeta* meta, int32_t* index,
                                                            int32_t* y, __half* __restrict__ xp,
                                                            __half* __restrict__ wp, float* __restrict__ dx,
                                                            float* rows) {
  after_predecessor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ex = plane_exponent(meta->x_top), ew = plane_exponent(meta->w_top);
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
      const float inv = (float)(1.0 / (double)count);
      meta->count = count;
      meta->logits = undo(ex + ew, 1.0f);
      meta->dx = undo(ew + kGradExponent, inv);
      meta->dw = undo(ex + kGradExponent, inv);
      if (count == 0)  // no row counts: the gradients are 0
        meta->dx.c1 = meta->dw.c1 = meta->dx.c2 = meta->dw.c2 = 0.0f;
    }
  }
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
    const int e = is_x ? ex : ew;
    const float f1 = exp2_int(e / 2), f2 = exp2_int(e - e / 2);
    if ((K & 7) == 0 && ((uintptr_t)src & 15) == 0) {
      for (int64_t k = lane; k < K / 8; k += 32) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        if (keep) a = reinterpret_cast<const float4*>(src)[2 * k], b = reinterpret_cast<const float4*>(src)[2 * k + 1];
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        __align__(16) __half h[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; j++) split_half(__fmul_rn(__fmul_rn(v[j], f1), f2), h[j], l[j]);
        reinterpret_cast<uint4*>(hi)[k] = *reinterpret_cast<uint4*>(h);
        reinterpret_cast<uint4*>(lo)[k] = *reinterpret_cast<uint4*>(l);
      }
    } else {
      for (int64_t k = lane; k < K; k += 256) {  // eight loads in flight
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = keep && k + 32 * j < K ? src[k + 32 * j] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (k + 32 * j < K) split_half(__fmul_rn(__fmul_rn(v[j], f1), f2), hi[k + 32 * j], lo[k + 32 * j]);
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

// n G = exp(z - maximum) / sum - [label] for up to 32 rows of 1024 columns (4 per
// thread), as two float16 planes of n G 2^15 and, for db, summed over the rows.
constexpr int kGradCols = 1024;
// Rows per block: 32, or 8 when that leaves SMs idle (15 us against 4 at 128 x 4000).
static int grad_rows(const gt_ctx* ctx, int64_t rows, int64_t V) {
  return ceil_div(rows, 32) * ceil_div(V, kGradCols) >= 2 * (int64_t)ctx->sm_count ? 32 : 8;
}
template <bool DB>
__global__ void __launch_bounds__(256) grad_planes_kernel(const float* z, const float2* stat, const int32_t* y,
                                                          const XentMeta* meta, int64_t r0, int64_t R, int64_t V,
                                                          int64_t Vp, int across, int rpb, __half* g, int64_t plane,
                                                          float* part) {
  after_predecessor();
  __shared__ float2 st[32];
  __shared__ int32_t ys[32];
  const int64_t rb = blockIdx.x / across, cb = blockIdx.x - rb * across;
  const int64_t m0 = rb * rpb, c = cb * kGradCols + 4 * threadIdx.x, here = rows_here(meta, r0, R);
  // behind the last row come zeros up to a multiple of 32 rows (dw's products read that far)
  const int n = (int)min((int64_t)rpb, min(R, (here + 31) / 32 * 32) - m0);
  if (n <= 0) return;
  if (threadIdx.x < n) {
    const bool row = m0 + threadIdx.x < here;
    st[threadIdx.x] = row ? stat[m0 + threadIdx.x] : make_float2(0.0f, 0.0f);
    ys[threadIdx.x] = row ? y[r0 + m0 + threadIdx.x] : -1;
  }
  __syncthreads();
  if (c >= V) return;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < n; i++) {
    const float4 v = *reinterpret_cast<const float4*>(z + (m0 + i) * Vp + c);
    const float2 s = st[i];
    const int64_t at = (int64_t)ys[i] - c;
    float p[4] = {v.x, v.y, v.z, v.w};
    __align__(8) __half hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      p[j] = s.y == 0.0f ? 0.0f : expf(p[j] - s.x) * s.y - (at == j ? 1.0f : 0.0f);
      if (DB) sum[j] += p[j];
      split_half(p[j] * (float)(1 << kGradExponent), hi[j], lo[j]);
    }
    __half* o = g + (m0 + i) * Vp + c;
    *reinterpret_cast<uint2*>(o) = *reinterpret_cast<uint2*>(hi);
    *reinterpret_cast<uint2*>(o + plane) = *reinterpret_cast<uint2*>(lo);
  }
  if (DB) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (c + j < V) part[rb * V + c + j] = sum[j];
  }
}

// db (+)= the column sums of the blocks of rows, / n: 32 columns per block,
// warp w adds the rows w, w + 8, ... in order, then the warps' sums in order.
__global__ void __launch_bounds__(256) db_kernel(const float* part, int rpb, int64_t r0, int64_t R, int64_t V, const XentMeta* meta,
                                                 float* db) {
  after_predecessor();
  __shared__ double ws[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, blocks = (rows_here(meta, r0, R) + rpb - 1) / rpb;
  double acc = 0.0;
  if (c < V) {
#pragma unroll 8
    for (int64_t i = warp; i < blocks; i += 8) acc += (double)part[i * V + c];
  }
  ws[warp][lane] = acc;
  __syncthreads();
  if (warp != 0 || c >= V) return;
  for (int i = 1; i < 8; i++) acc += ws[i][lane];
  const float d = (float)(meta->count ? acc / (double)meta->count : 0.0);
  db[c] = r0 == 0 ? d : db[c] + d;
}

// float32: see the top of the file.
static char* linear_xent(gt_ctx* ctx, const XentCall<float>& c, void** held) {
  if (few_rows(c.M, c.K, c.V)) return linear_xent_few(ctx, c, held);
  const bool grad = c.dx || c.dw || c.db;
  const int64_t Kp = ceil_div(c.K, 8) * 8, Vp = ceil_div(c.V, 8) * 8, strips = ceil_div(c.V, kStripCols);
  // Rows per piece: as many as the workspace holds (z and the two planes of G
  // take 8 bytes per logit, the strips 8 per 128), in multiples of the tiles'
  // 256 rows, and the pieces of equal size.
  const int64_t per_row = (grad ? 8 * Vp : 0) + 8 * strips;
  int64_t R = std::max<int64_t>(1, c.workspace / per_row / 256) * 256;
  R = std::min(c.M, ceil_div(ceil_div(c.M, ceil_div(c.M, R)), 256) * 256);
  const int rpb = grad_rows(ctx, R, c.V);
  const int64_t row_blocks = ceil_div(c.M, kCompactRows);
  struct {
    XentMeta* meta;
    __half *x, *w, *g;
    float *z, *losses, *picked, *part;
    float2 *strips, *stat;
    int32_t *counts, *index, *y;
  } ws;
  auto carve = [&](Carver& k) {
    ws.meta = k.take<XentMeta>(1);
    ws.x = k.take<__half>(2 * c.M * Kp);
    ws.w = k.take<__half>(2 * c.V * Kp);
    ws.g = k.take<__half>(grad ? 2 * R * Vp : 0);
    ws.z = k.take<float>(grad ? R * Vp : 0);
    ws.losses = k.take<float>(c.M);
    ws.picked = k.take<float>(R);
    ws.part = k.take<float>(c.db ? ceil_div(R, rpb) * c.V : 0);
    ws.strips = k.take<float2>(strips * R);
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

  GT_CUDA(cudaMemsetAsync(ws.meta, 0, sizeof(XentMeta), ctx->stream));
  const int most = 8 * ctx->sm_count;  // resident blocks: one round each
  const int wb = std::min(most, grid_for(ctx, c.V * c.K, 256, 16)), xb = std::min(most, grid_for(ctx, c.M * c.K, 256, 16));
  operand_top_kernel<<<(unsigned)(wb + xb + row_blocks), 256, 0, ctx->stream>>>(
      c.x, c.w, c.labels, c.M, c.K, c.V, c.ignore, wb, xb, ws.meta, ws.counts, c.bad);
  GT_LAUNCH_CHECK();
  const int sb = (int)std::min<int64_t>(ceil_div(c.M + c.V + 32, 8), (int64_t)ctx->sm_count * 32);
  GT_CUDA(launch_overlapped(ctx, operand_split_kernel, sb, 256, 0, c.x, c.w, c.labels, c.M, c.K, c.V, Kp, c.ignore,
                            ws.counts, ws.meta, ws.index, ws.y, ws.x, ws.w, c.dx, c.rows));
  const HalfPlanes w{ws.w, c.V, c.K, Kp, c.V * Kp};
  for (int64_t r0 = 0; r0 < c.M; r0 += R) {
    // As many pieces as all rows would need; those behind the rows that count find nothing to do.
    const int64_t r = std::min(R, c.M - r0);
    const HalfPlanes x{ws.x + r0 * Kp, r, c.K, Kp, c.M * Kp}, g{ws.g, r, c.V, Vp, R * Vp};
    SplitGemm f;
    f.M = r, f.N = c.V, f.K = c.K, f.kept = &ws.meta->count, f.kept_from = r0, f.a = x, f.b = w;
    f.scale = &ws.meta->logits;
    f.out = grad ? ws.z : nullptr, f.ldc = Vp, f.bias = c.bias, f.labels = ws.y + r0;
    f.strips = ws.strips, f.strip_rows = R, f.picked = ws.picked;
    GT_TRY(split_gemm(ctx, f));
    GT_CUDA(launch_overlapped(ctx, strip_join_kernel, (unsigned)ceil_div(r, 32), 1024, 0, ws.strips, R, (int)strips,
                              ws.y, ws.index, ws.meta, r0, c.V, ws.picked, ws.stat, ws.losses, c.rows));
    if (!grad) continue;
    const int64_t across = ceil_div(c.V, kGradCols);
    GT_CUDA(launch_overlapped(ctx, c.db ? grad_planes_kernel<true> : grad_planes_kernel<false>,
                              (unsigned)(across * ceil_div(r, rpb)), 256, 0, ws.z, ws.stat, ws.y, ws.meta, r0, r, c.V,
                              Vp, (int)across, rpb, ws.g, R * Vp, ws.part));
    if (c.dx) {
      SplitGemm d;
      d.M = r, d.N = c.K, d.K = c.V, d.kept = &ws.meta->count, d.kept_from = r0, d.a = g, d.b = w, d.b_mn = true;
      d.scale = &ws.meta->dx;
      d.out = c.dx, d.ldc = c.K, d.row_index = ws.index + r0;
      GT_TRY(split_gemm(ctx, d));
    }
    if (c.dw) {
      SplitGemm d;
      d.M = c.V, d.N = c.K, d.K = r, d.kept = &ws.meta->count, d.kept_from = r0, d.a = g, d.a_mn = true, d.b = x;
      d.b_mn = true, d.scale = &ws.meta->dw;
      d.out = c.dw, d.ldc = c.K, d.accumulate = r0 > 0;
      GT_TRY(split_gemm(ctx, d));
    }
    if (c.db)
      GT_CUDA(launch_overlapped(ctx, db_kernel, (unsigned)ceil_div(c.V, 32), 256, 0, ws.part, rpb, r0, r, c.V, ws.meta,
                                c.db));
  }
  GT_CUDA(launch_overlapped(ctx, mean_rows_kernel<float>, 1, 1024, 0, ws.losses, c.M, true, &ws.meta->count, c.loss));
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
  if ((double)M * (double)K > 0x1p56 || (double)V * (double)K > 0x1p56)
    return errorf("gt_linear_xent_fwd_bwd: x and w must stay below 2^56 elements");
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
  if (workspace_bytes == 0) workspace_bytes = (int64_t)2 << 30;
  void* held[5] = {};
  char* err = nullptr;
  GT_DISPATCH(dtype, {
    const XentCall<T> c{(const T*)x, (const T*)w, (const T*)bias, labels, M, K, V, ignore_label, workspace_bytes,
                        (T*)loss, (T*)row_loss, (T*)dx, (T*)dw, (T*)db, bad_label};
    err = linear_xent(ctx, c, held);
  });
  for (void* h : held) release(ctx, h);
  return err;
}
