// The large-vocabulary loss for at most 64 rows, float32 (see linear_xent.cu for
// the formulas).
//
// With so few rows the call is bound by latency when w is small, by reading w
// twice and writing dw once when it is large; splitting w into planes first, as the
// tensor-core path does, moves 8 more bytes per value, and its 256-row tiles
// are mostly empty. So the products run on the FP32 pipe from w as it is:
//
//   few_logits_kernel  a block per strip of classes: z for all rows, the strip's
//                      maximum and sum of exponentials per row
//   few_join_kernel    one block: the strips joined, the rows' losses, the loss
//   few_grad_kernel    a block per columns of w and run of classes: G from
//                      z on the fly, dw (finished: all rows are here), a
//                      partial dx, and db
//   few_dx_kernel      the partial dx of the runs, added up
// (few8_logits_kernel and few8_grad_kernel for at most 8 rows)
//
// Sums are float32 in runs of at most 256 (logits) or 1024 (dx) terms of a thread
// that are then added up, so they stay as exact as the tensor-core path's.
//
// Measured (the tensor-core path in brackets): 7 x 96 x 517 17 us (54), 64 x 128 x
// 1000 37 us (65), 64 x 512 x 5000 94 us (73), 8 x 2048 x 50000 393 us (503; w read
// twice and dw written once take 190 at HBM rate), 16 x 2048 x 50000 660 us (494): it
// is bound by shared-memory reads there, so the choice goes by the products'
// size (few_rows).
#include <algorithm>

#include "f32x2.cuh"
#include "linear_xent.cuh"

namespace gt {

constexpr int kFewStrip = 64;   // classes per block of the logits
constexpr int kFewChunk = 32;   // K per shared-memory stage of the logits
constexpr int kFewPitch = 36;   // floats per staged row: 16-byte reads of 8 rows are free of bank conflicts
constexpr int kFewCols = 128;   // columns of w per block of the gradient
constexpr int kFewClasses = 32; // classes per step of the gradient

struct FewMeta {
  float inv_n;  // 0 when no row counts
};

// At most 8 rows. A warp has 4 classes, whose rows of w go straight to its
// registers one step of K ahead, its lanes sharing out K; x comes from shared
// memory once for the 4 classes. (From tiles of both in shared memory, as below,
// its reads bounded the call: 216 us at 8 x 2048 x 50000.)
constexpr int kEight = 8;
constexpr int kEightStrip = 32;    // classes per block
constexpr int kEightChunk = 1024;  // K per stage of x
constexpr int kEightRun = 8;       // stages per run: 256 terms of a lane
__global__ void __launch_bounds__(256, 2) few8_logits_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                             const float* __restrict__ bias,
                                                             const int32_t* __restrict__ labels, int M, int64_t K,
                                                             int64_t V, int32_t ignore, float* __restrict__ z,
                                                             int64_t Vp, float2* __restrict__ strips,
                                                             float* __restrict__ picked) {
  __shared__ __align__(16) float xs[kEight][kEightChunk];
  __shared__ float zs[kEight][kEightStrip + 1];
  __shared__ bool keep[kEight];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t v0 = (int64_t)blockIdx.x * kEightStrip, mine = v0 + 4 * warp;
  if (tid < kEight) keep[tid] = tid < M && labels[tid] != ignore;
  // A lane's four values of a step: 4 lane .. + 3 where rows of w are 16-byte
  // aligned, else lane + 32 j.
  const bool vec = ((K & 3) | ((uintptr_t)w & 15)) == 0;
  const float* row[4];
#pragma unroll
  for (int c = 0; c < 4; c++) row[c] = w + min(mine + c, V - 1) * K;
  float4 next[4];
  auto fetch = [&](int64_t k) {  // the step at k
#pragma unroll
    for (int c = 0; c < 4; c++) {
      next[c] = float4{0.f, 0.f, 0.f, 0.f};
      if (vec) {
        if (k + 4 * lane < K) next[c] = __ldg(reinterpret_cast<const float4*>(row[c] + k + 4 * lane));
      } else {
        if (k + lane < K) next[c].x = __ldg(row[c] + k + lane);
        if (k + lane + 32 < K) next[c].y = __ldg(row[c] + k + lane + 32);
        if (k + lane + 64 < K) next[c].z = __ldg(row[c] + k + lane + 64);
        if (k + lane + 96 < K) next[c].w = __ldg(row[c] + k + lane + 96);
      }
    }
  };
  float acc[32], total = 0.0f;  // [class][row]; the sums of earlier runs
#pragma unroll
  for (int i = 0; i < 32; i++) acc[i] = 0.0f;
  fetch(0);
  for (int64_t k0 = 0; k0 < K; k0 += kEightChunk) {
    __syncthreads();
    for (int i = tid; i < kEight * kEightChunk; i += 256) {
      const int m = i / kEightChunk, k = i % kEightChunk;
      xs[m][k] = keep[m] && k0 + k < K ? __ldg(x + m * K + k0 + k) : 0.0f;
    }
    __syncthreads();
    const int left = (int)min((int64_t)kEightChunk, K - k0);
#pragma unroll 1
    for (int k = 0; k < left; k += 128) {
      float4 a[4];
#pragma unroll
      for (int c = 0; c < 4; c++) a[c] = next[c];
      fetch(k0 + k + 128);
#pragma unroll
      for (int m = 0; m < kEight; m++) {
        float4 b;
        if (vec)
          b = *reinterpret_cast<const float4*>(&xs[m][k + 4 * lane]);
        else
          b = make_float4(xs[m][k + lane], xs[m][k + lane + 32], xs[m][k + lane + 64], xs[m][k + lane + 96]);
#pragma unroll
        for (int c = 0; c < 4; c++)
          acc[c * kEight + m] =
              fmaf(a[c].w, b.w, fmaf(a[c].z, b.z, fmaf(a[c].y, b.y, fmaf(a[c].x, b.x, acc[c * kEight + m]))));
      }
    }
    if (k0 / kEightChunk % kEightRun != kEightRun - 1 && k0 + kEightChunk < K) continue;
    // The 32 sums over the lanes by halving exchanges: lane l ends with sum l.
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const bool up = lane & off;
#pragma unroll
      for (int j = 0; j < off; j++) {
        const float keep_v = up ? acc[j + off] : acc[j], send = up ? acc[j] : acc[j + off];
        acc[j] = keep_v + __shfl_xor_sync(0xffffffffu, send, off);
      }
    }
    total += acc[0];
#pragma unroll
    for (int i = 0; i < 32; i++) acc[i] = 0.0f;
  }
  {
    const int c = lane / kEight, m = lane % kEight;
    const int64_t v = mine + c;
    zs[m][4 * warp + c] = v < V ? total + (bias ? __ldg(bias + v) : 0.0f) : -INFINITY;
  }
  __syncthreads();
  if (warp < M) {
    const int m = warp;
    const float a = zs[m][lane];
    float top = a;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float sum = expf(a - (top == -INFINITY ? 0.0f : top));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      strips[(int64_t)blockIdx.x * kEight + m] = make_float2(top, sum);
      const int64_t at = (int64_t)labels[m] - v0;
      if (at >= 0 && at < kEightStrip && v0 + at < V) picked[m] = zs[m][at];
    }
    if (z && v0 + lane < V) z[m * Vp + v0 + lane] = a;
  }
}

// More rows (MT: rounded up to 16, 32 or 64). A thread has the classes tv + TV i
// and the rows tm + TM j.
template <int MT>
__global__ void __launch_bounds__(256) few_logits_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                         const float* __restrict__ bias,
                                                         const int32_t* __restrict__ labels, int M, int64_t K,
                                                         int64_t V, int32_t ignore, float* __restrict__ z, int64_t Vp,
                                                         float2* __restrict__ strips, float* __restrict__ picked) {
  constexpr int TV = 16, TM = 16, VI = kFewStrip / TV, MJ = MT / TM;
  __shared__ __align__(16) float buf[2 * (kFewStrip + MT) * kFewPitch];
  auto ws = reinterpret_cast<float (*)[kFewStrip][kFewPitch]>(buf);
  auto xs = reinterpret_cast<float (*)[MT][kFewPitch]>(buf + 2 * kFewStrip * kFewPitch);
  auto zs = reinterpret_cast<float (*)[kFewStrip + 1]>(buf);  // after the products
  const int tid = threadIdx.x, tv = tid % TV, tm = tid / TV, lane = tid & 31, warp = tid >> 5;
  const int64_t v0 = (int64_t)blockIdx.x * kFewStrip;
  float wr[8], xr[MT / 8];
  bool keep[MT / 8];
#pragma unroll
  for (int i = 0; i < MT / 8; i++) keep[i] = warp + 8 * i < M && labels[warp + 8 * i] != ignore;
  auto fetch = [&](int64_t k0) {  // a warp reads 32 consecutive values of a row
    const int64_t k = k0 + lane;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t v = v0 + warp + 8 * i;
      wr[i] = k < K && v < V ? __ldg(w + v * K + k) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < MT / 8; i++) xr[i] = k < K && keep[i] ? __ldg(x + (int64_t)(warp + 8 * i) * K + k) : 0.0f;
  };
  auto stage = [&](int b) {
#pragma unroll
    for (int i = 0; i < 8; i++) ws[b][warp + 8 * i][lane] = wr[i];
#pragma unroll
    for (int i = 0; i < MT / 8; i++) xs[b][warp + 8 * i][lane] = xr[i];
  };
  float acc[VI][MJ], tot[VI][MJ];
#pragma unroll
  for (int i = 0; i < VI; i++)
#pragma unroll
    for (int j = 0; j < MJ; j++) acc[i][j] = tot[i][j] = 0.0f;
  fetch(0);
  int c = 0;
  for (int64_t k0 = 0; k0 < K; k0 += kFewChunk, c++) {
    stage(c & 1);
    __syncthreads();  // (the other buffer's readers are a barrier behind by now)
    if (k0 + kFewChunk < K) fetch(k0 + kFewChunk);
#pragma unroll
    for (int kk = 0; kk < kFewChunk; kk += 4) {
      float4 a[VI], b[MJ];
#pragma unroll
      for (int i = 0; i < VI; i++) a[i] = *reinterpret_cast<const float4*>(&ws[c & 1][tv + TV * i][kk]);
#pragma unroll
      for (int j = 0; j < MJ; j++) b[j] = *reinterpret_cast<const float4*>(&xs[c & 1][tm + TM * j][kk]);
#pragma unroll
      for (int i = 0; i < VI; i++)
#pragma unroll
        for (int j = 0; j < MJ; j++)
          acc[i][j] = fmaf(a[i].w, b[j].w, fmaf(a[i].z, b[j].z, fmaf(a[i].y, b[j].y, fmaf(a[i].x, b[j].x, acc[i][j]))));
    }
    if ((c & 7) == 7 || k0 + kFewChunk >= K) {  // runs of 256 terms
#pragma unroll
      for (int i = 0; i < VI; i++)
#pragma unroll
        for (int j = 0; j < MJ; j++) tot[i][j] += acc[i][j], acc[i][j] = 0.0f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VI; i++) {
    const int64_t v = v0 + tv + TV * i;
    const float add = bias && v < V ? __ldg(bias + v) : 0.0f;
#pragma unroll
    for (int j = 0; j < MJ; j++) zs[tm + TM * j][tv + TV * i] = v < V ? tot[i][j] + add : -INFINITY;
  }
  __syncthreads();
  for (int m = warp; m < M; m += 8) {  // a warp per row: two values per lane
    const float a = zs[m][lane], b = zs[m][lane + 32];
    float top = fmaxf(a, b);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = expf(a - from) + expf(b - from);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) {
      strips[(int64_t)blockIdx.x * MT + m] = make_float2(top, sum);
      const int64_t at = (int64_t)labels[m] - v0;
      if (at >= 0 && at < kFewStrip && v0 + at < V) picked[m] = zs[m][at];
    }
    if (z) {
      if (v0 + lane < V) z[m * Vp + v0 + lane] = a;
      if (v0 + lane + 32 < V) z[m * Vp + v0 + lane + 32] = b;
    }
  }
}

// One block of 32 warps, 32 / MT of them (at least one) per row: the strips
// joined, the rows' losses, the loss. stat[m] = (maximum, 1 / sum), the latter 0
// for an ignored row.
template <int MT>
__global__ void __launch_bounds__(1024) few_join_kernel(const float2* strips, int n, int M,
                                                        const int32_t* __restrict__ labels, int64_t V, int32_t ignore,
                                                        const float* picked, float2* stat,
                                                        float* rows, float* loss, const double* over,
                                                        FewMeta* meta, int32_t* bad) {
  after_predecessor();
  constexpr int PARTS = MT >= 32 ? 1 : 32 / MT;
  __shared__ float2 pair[PARTS][MT];
  __shared__ float row_loss[MT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp / (32 / PARTS);
  for (int m = warp % (32 / PARTS); m < M; m += 32 / PARTS) {
    float2 a = make_float2(-INFINITY, 0.0f);
#pragma unroll 4
    for (int i = lane + 32 * part; i < n; i += 32 * PARTS) join(a, strips[(int64_t)i * MT + m]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float2 b = make_float2(__shfl_xor_sync(0xffffffffu, a.x, off), __shfl_xor_sync(0xffffffffu, a.y, off));
      join(a, b);
    }
    if (lane == 0) pair[part][m] = a;
  }
  __syncthreads();
  const int m = threadIdx.x;
  int kept = 0;
  if (m < M) {
    const int32_t y = labels[m];
    float2 a = pair[0][m];
    for (int i = 1; i < PARTS; i++) join(a, pair[i][m]);
    kept = y != ignore;
    const bool outside = kept && (y < 0 || y >= V);
    const float r = !kept ? 0.0f : outside ? NAN : logf(a.y) + (a.x - picked[m]);
    stat[m] = kept ? make_float2(a.x, __fdiv_rn(1.0f, a.y)) : make_float2(0.0f, 0.0f);
    row_loss[m] = r;
    if (rows) rows[m] = r;
    if (outside && bad) *bad = 1;
  }
  const int count = __syncthreads_count(kept);
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < M; i++) sum += (double)row_loss[i];
    const double n = over ? *over : (double)count;
    *loss = (float)(sum / n);
    meta->inv_n = count ? (float)(1.0 / n) : 0.0f;
  }
}

// At most 8 rows: block (kb, run) has the columns 64 kb .. and the classes [run *
// per, + per). A warp has 8 classes of a step of 64, a lane the columns lane and
// lane + 32 of all of them, packed: x and the warp's part of dx stay in
// registers, a value of w goes from memory to a register that both products
// use and that is refilled for the next step at once, and only n G (twice, as a
// pair) comes from shared memory, one address for the whole warp.
constexpr int kEightCols = 64, kEightStep = 64;
__global__ void __launch_bounds__(256, 2) few8_grad_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                           const float* z, int64_t Vp, const float2* stat,
                                                           const int32_t* __restrict__ labels, int M, int64_t K,
                                                           int64_t V, int32_t ignore, int64_t per, const FewMeta* meta,
                                                           float* dw, float* db, float* dx_part) {
  after_predecessor();
  __shared__ __align__(16) F2 gs[2][kEightStep][kEight];
  __shared__ float parts[8][kEight][kEightCols];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t k0 = (int64_t)blockIdx.x * kEightCols + lane;
  const bool in0 = k0 < K, in1 = k0 + 32 < K;
  const int64_t va = (int64_t)blockIdx.y * per;
  const int n = (int)(min(va + per, V) - va);  // classes of the run
  const float inv_n = meta->inv_n;
  F2 xr[kEight], acc[kEight];
  float w0[8], w1[8];
#pragma unroll
  for (int m = 0; m < kEight; m++) {
    const bool keep = m < M && labels[m] != ignore;
    xr[m] = f2(keep && in0 ? __ldg(x + m * K + k0) : 0.0f, keep && in1 ? __ldg(x + m * K + k0 + 32) : 0.0f);
    acc[m] = both(0.0f);
  }
  const float* wp = w + (va + 8 * warp) * K + k0;
  float* dp = dw ? dw + (va + 8 * warp) * K + k0 : nullptr;
  auto fetch = [&](int at, int c) {  // class c of the warp's in the step at `at`
    const bool live = dx_part && at + 8 * warp + c < n;
    const float* r = wp + (int64_t)(at + c) * K;
    w0[c] = live && in0 ? __ldg(r) : 0.0f, w1[c] = live && in1 ? __ldg(r + 32) : 0.0f;
  };
  // n G: a thread has the class zc of a step for the rows zm and zm + 4
  const int zc = tid & 63, zm = tid >> 6;
  float zr[2], top[2], inv[2];
  int y[2];
  auto fetch_z = [&](int at) {
#pragma unroll
    for (int u = 0; u < 2; u++) zr[u] = zm + 4 * u < M && at + zc < n ? z[(zm + 4 * u) * Vp + va + at + zc] : 0.0f;
  };
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int m = zm + 4 * u;
    const float2 s = m < M ? stat[m] : make_float2(0.0f, 0.0f);
    top[u] = s.x, inv[u] = s.y;
    const int64_t label = m < M ? (int64_t)labels[m] - va : -1;
    y[u] = label >= 0 && label < n ? (int)label : -1;  // in the run
  }
#pragma unroll
  for (int c = 0; c < 8; c++) fetch(0, c);
  fetch_z(0);
  int b = 0;
#pragma unroll 1
  for (int at = 0; at < n; at += kEightStep, b ^= 1) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float g = 0.0f;
      if (inv[u] != 0.0f && at + zc < n) g = expf(zr[u] - top[u]) * inv[u] - (y[u] == at + zc ? 1.0f : 0.0f);
      gs[b][zc][zm + 4 * u] = both(g);
    }
    fetch_z(at + kEightStep);
    __syncthreads();  // (the other buffer's readers are a barrier behind by now)
#pragma unroll
    for (int c = 0; c < 8; c++) {
      F2 d = both(0.0f);
      const F2 wv = f2(w0[c], w1[c]);
      float sum = 0.0f;
#pragma unroll
      for (int m = 0; m < kEight; m++) {
        const F2 g = gs[b][8 * warp + c][m];
        d = fma2(g, xr[m], d);
        acc[m] = fma2(g, wv, acc[m]);
        if (db && blockIdx.x == 0) {
          float lo, hi;
          unpack(g, lo, hi);
          sum += lo;
        }
      }
      const int v = at + 8 * warp + c;
      fetch(at + kEightStep, c);  // on its way while the others are computed
      if (v >= n) continue;
      if (dp) {
        float lo, hi;
        unpack(d * both(inv_n), lo, hi);
        float* o = dp + (int64_t)(at + c) * K;
        if (in0) o[0] = lo;
        if (in1) o[32] = hi;
      }
      if (db && blockIdx.x == 0 && lane == 0) db[va + v] = sum * inv_n;
    }
  }
  if (!dx_part) return;
#pragma unroll
  for (int m = 0; m < kEight; m++) {
    float lo, hi;
    unpack(acc[m], lo, hi);
    parts[warp][m][lane] = lo, parts[warp][m][lane + 32] = hi;
  }
  __syncthreads();
  for (int i = tid; i < kEight * kEightCols; i += 256) {
    const int m = i / kEightCols, c = i % kEightCols;
    const int64_t k = (int64_t)blockIdx.x * kEightCols + c;
    if (m >= M || k >= K) continue;
    float s = parts[0][m][c];
#pragma unroll
    for (int u = 1; u < 8; u++) s += parts[u][m][c];
    dx_part[((int64_t)blockIdx.y * M + m) * K + k] = s;
  }
}

template <int MT>
struct FewShared {
  float w[kFewClasses][kFewCols];
  float x[MT][kFewCols];
  float gm[MT][kFewClasses + 4];  // n G, [row][class]
  float gv[kFewClasses][MT + 1];  // [class][row]
  float2 stat[MT];
  int32_t label[MT];
};

// Block (kb, run): columns 128 kb .. of w, classes [run * per, + per). A thread
// has the columns 4 (tid % 32) .. + 3; of dw the classes 4 (tid / 32) .. + 3 of a
// step, of dx the rows (tid / 32) MT / 8 ....
template <int MT>
__global__ void __launch_bounds__(256) few_grad_kernel(const float* __restrict__ x, const float* __restrict__ w,
                                                       const float* z, int64_t Vp,
                                                       const float2* stat,
                                                       const int32_t* __restrict__ labels, int M, int64_t K, int64_t V,
                                                       int32_t ignore, int64_t per, const FewMeta* meta,
                                                       float* dw, float* db,
                                                       float* dx_part, int dw_vec) {
  after_predecessor();
  constexpr int R = MT / 8;  // rows of dx per thread
  extern __shared__ __align__(16) uint8_t few_smem[];
  FewShared<MT>& sh = *reinterpret_cast<FewShared<MT>*>(few_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t k0 = (int64_t)blockIdx.x * kFewCols, va = (int64_t)blockIdx.y * per, vb = min(va + per, V);
  const float inv_n = meta->inv_n;
  for (int i = tid; i < MT; i += 256) {
    sh.stat[i] = i < M ? stat[i] : make_float2(0.0f, 0.0f);
    sh.label[i] = i < M ? labels[i] : ignore;
  }
  __syncthreads();
  for (int i = tid; i < MT * kFewCols; i += 256) {
    const int m = i / kFewCols, c = i % kFewCols;
    sh.x[m][c] = m < M && sh.stat[m].y != 0.0f && k0 + c < K ? __ldg(x + m * K + k0 + c) : 0.0f;
  }
  float wr[16];
  auto fetch = [&](int64_t v0) {  // 32 classes x 128 columns, a warp 4 classes
    if (!dx_part) return;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int64_t v = v0 + warp * 4 + i / 4, k = k0 + lane + 32 * (i % 4);
      wr[i] = v < vb && k < K ? __ldg(w + v * K + k) : 0.0f;
    }
  };
  float acc[R][4];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[r][j] = 0.0f;
  fetch(va);
  for (int64_t v0 = va; v0 < vb; v0 += kFewClasses) {
    // n G of the step's classes: a warp takes a row's 32 classes at a time
    for (int m = warp; m < MT; m += 8) {
      const float2 s = sh.stat[m];
      float g = 0.0f;
      if (s.y != 0.0f && v0 + lane < vb)
        g = expf(z[m * Vp + v0 + lane] - s.x) * s.y - (sh.label[m] == v0 + lane ? 1.0f : 0.0f);
      sh.gm[m][lane] = g;
      sh.gv[lane][m] = g;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) sh.w[warp * 4 + i / 4][lane + 32 * (i % 4)] = wr[i];
    __syncthreads();
    if (v0 + kFewClasses < vb) fetch(v0 + kFewClasses);
    if (dx_part) {
#pragma unroll 4
      for (int v = 0; v < kFewClasses; v++) {
        const float4 a = *reinterpret_cast<const float4*>(&sh.w[v][4 * lane]);
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float g = sh.gv[v][warp * R + r];
          acc[r][0] = fmaf(g, a.x, acc[r][0]), acc[r][1] = fmaf(g, a.y, acc[r][1]);
          acc[r][2] = fmaf(g, a.z, acc[r][2]), acc[r][3] = fmaf(g, a.w, acc[r][3]);
        }
      }
    }
    if (dw) {
      float d[4][4];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) d[i][j] = 0.0f;
#pragma unroll 4
      for (int m = 0; m < MT; m++) {
        const float4 a = *reinterpret_cast<const float4*>(&sh.x[m][4 * lane]);
        const float4 g = *reinterpret_cast<const float4*>(&sh.gm[m][4 * warp]);
        const float gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          d[i][0] = fmaf(gs[i], a.x, d[i][0]), d[i][1] = fmaf(gs[i], a.y, d[i][1]);
          d[i][2] = fmaf(gs[i], a.z, d[i][2]), d[i][3] = fmaf(gs[i], a.w, d[i][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int64_t v = v0 + 4 * warp + i, k = k0 + 4 * lane;
        if (v >= vb || k >= K) continue;
        float* o = dw + v * K + k;
        if (dw_vec) {
          *reinterpret_cast<float4*>(o) = make_float4(d[i][0] * inv_n, d[i][1] * inv_n, d[i][2] * inv_n, d[i][3] * inv_n);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (k + j < K) o[j] = d[i][j] * inv_n;
        }
      }
    }
    if (db && blockIdx.x == 0 && warp == 0 && v0 + lane < vb) {
      float s = 0.0f;
      for (int m = 0; m < MT; m++) s += sh.gm[m][lane];
      db[v0 + lane] = s * inv_n;
    }
    __syncthreads();
  }
  if (dx_part) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int m = warp * R + r;
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (k0 + 4 * lane + j < K) dx_part[((int64_t)blockIdx.y * M + m) * K + k0 + 4 * lane + j] = acc[r][j];
    }
  }
}

// dx = the runs' partials, added by 8 warps (warp w the runs w, w + 8, ... in
// order, then the warps' sums in order), 32 values per block. An ignored row's
// is 0 whatever w holds (0 times an infinity in the partials is not).
__global__ void __launch_bounds__(256) few_dx_kernel(const float* part, int runs, int64_t n, int64_t K,
                                                     const float2* stat, const FewMeta* meta, float* dx) {
  after_predecessor();
  __shared__ float ws[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int r = warp; r < runs; r += 8) s += part[r * n + i];
  }
  ws[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || i >= n) return;
#pragma unroll
  for (int u = 1; u < 8; u++) s += ws[u][lane];
  dx[i] = stat[i / K].y == 0.0f ? 0.0f : s * meta->inv_n;
}

template <int MT>
static char* few_run(gt_ctx* ctx, const XentCall<float>& c, void** held) {
  const bool grad = c.dx || c.dw || c.db;
  const int64_t strips = ceil_div(c.V, MT == kEight ? kEightStrip : kFewStrip), Vp = ceil_div(c.V, 8) * 8;
  // Runs of classes: whole rounds of blocks (2 or more are resident on every SM), at most 1024 classes
  // (the longest plain sum of dx; 4096 where a warp adds an eighth of them).
  constexpr bool eight = MT == kEight;
  const int64_t kb = c.dx || c.dw ? ceil_div(c.K, eight ? kEightCols : kFewCols) : 1;
  const int64_t step = eight ? kEightStep : kFewClasses, steps = ceil_div(c.V, step);
  const int64_t runs0 = std::min(steps, std::max<int64_t>((eight ? 6 : 4) * (int64_t)ctx->sm_count / kb,
                                                          std::max<int64_t>(1, ceil_div(c.V, eight ? 4096 : 1024))));
  const int64_t per = ceil_div(steps, runs0) * step, runs = ceil_div(c.V, per);
  struct {
    FewMeta* meta;
    float *z, *picked, *part;
    float2 *strips, *stat;
  } ws;
  auto carve = [&](Carver& k) {
    ws.meta = k.take<FewMeta>(1);
    ws.picked = k.take<float>(MT);
    ws.stat = k.take<float2>(MT);
    ws.strips = k.take<float2>(strips * MT);
    ws.z = k.take<float>(grad ? c.M * Vp : 0);
    ws.part = k.take<float>(c.dx ? runs * c.M * c.K : 0);
  };
  Carver size{nullptr};
  carve(size);
  GT_TRY(scratch(ctx, (size_t)size.used, &held[0]));
  Carver at{(char*)held[0]};
  carve(at);
  if constexpr (eight)
    few8_logits_kernel<<<(unsigned)strips, 256, 0, ctx->stream>>>(c.x, c.w, c.bias, c.labels, (int)c.M, c.K, c.V,
                                                                  c.ignore, grad ? ws.z : nullptr, Vp, ws.strips,
                                                                  ws.picked);
  else
    few_logits_kernel<MT><<<(unsigned)strips, 256, 0, ctx->stream>>>(c.x, c.w, c.bias, c.labels, (int)c.M, c.K, c.V,
                                                                       c.ignore, grad ? ws.z : nullptr, Vp, ws.strips,
                                                                       ws.picked);
  GT_LAUNCH_CHECK();
  GT_CUDA(launch_overlapped(ctx, few_join_kernel<MT>, 1, 1024, 0, ws.strips, (int)strips, (int)c.M, c.labels, c.V,
                            c.ignore, ws.picked, ws.stat, c.rows, c.loss, c.over, ws.meta, c.bad));
  if (!grad) return nullptr;
  const dim3 grid((unsigned)kb, (unsigned)runs);
  if constexpr (eight) {
    GT_CUDA(launch_overlapped(ctx, few8_grad_kernel, grid, 256, 0, c.x, c.w, ws.z, Vp, ws.stat, c.labels, (int)c.M, c.K,
                              c.V, c.ignore, per, ws.meta, c.dw, c.db, c.dx ? ws.part : nullptr));
  } else {
    static bool configured[64] = {};
    if (ctx->device < 0 || ctx->device >= 64 || !configured[ctx->device]) {
      GT_CUDA(cudaFuncSetAttribute(few_grad_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)sizeof(FewShared<MT>)));
      if (ctx->device >= 0 && ctx->device < 64) configured[ctx->device] = true;
    }
    GT_CUDA(launch_overlapped(ctx, few_grad_kernel<MT>, grid, 256, sizeof(FewShared<MT>),
                              c.x, c.w, ws.z, Vp, ws.stat, c.labels, (int)c.M, c.K, c.V, c.ignore, per, ws.meta, c.dw,
                              c.db, c.dx ? ws.part : nullptr, ((c.K & 3) | ((uintptr_t)c.dw & 15)) == 0));
  }
  if (c.dx)
    GT_CUDA(launch_overlapped(ctx, few_dx_kernel, (unsigned)ceil_div(c.M * c.K, 32), 256, 0, ws.part, (int)runs,
                              c.M * c.K, c.K, ws.stat, ws.meta, c.dx));
  return nullptr;
}

char* linear_xent_few(gt_ctx* ctx, const XentCall<float>& c, void** held) {
  if (c.M <= 8) return few_run<8>(ctx, c, held);
  if (c.M <= 16) return few_run<16>(ctx, c, held);
  if (c.M <= 32) return few_run<32>(ctx, c, held);
  return few_run<64>(ctx, c, held);
}

}  // namespace gt
