// tcgen05 GEMM of float32 operands held as two float16 planes, for sm_100a.
//
// Precision. x s = hi + lo with hi = half(x s), lo = half(x s - hi), s a power of
// two that puts the largest magnitude that shares it at 2^14 .. 2^15: 22 bits
// of every value down to 2^-16 of that largest, and an error of at most 2^-39 of
// it below. What shares a scale is what stands in one sum anyway: a row of x
// and a row of w in the logits, whose epilogue undoes both; in dx and dw, whose
// sums run over rows of w and of x with scales of their own, those scales are
// folded into G, which is scaled again per group of 128 values of K and row of
// the result, undone as the group's partial sum is added. (One scale per
// operand cost a product's other rows 2^-39 of the largest row's, and what G had
// below 2^-39.) A product is
//   a b ~= hi(a) hi(b) + hi(a) lo(b) + lo(a) hi(b)          (lo lo dropped, 2^-22)
// the same three products and the same mantissas as 3xTF32 (gemm_tc.cu), but
// kind::f16 runs at twice the rate of kind::tf32 and a plane takes half the
// bytes. The range that float16 lacks is in the scales, which are powers of
// two. The operands arrive split (each is used by two GEMMs), so
// no warp splits them here.
// Tensor-core accumulation truncates, so, as there, the MMAs accumulate 128
// values of K into one of two partial buffers in tensor memory and promoter
// warps add each partial to a total in registers with rounded adds.
//
// Work split. A CTA pair (cta_group::2) computes 256 x 256 outputs: each CTA
// stages 128 rows of A and of B, both planes, 32 values of K per stage (32
// KB), six stages. Warp roles of the 12 warps: warp 0 TMA producer, warp 1 MMA
// issuer (leader), warp 2 relays "my half of the stage has landed" to the
// leader, warps 4-11 promoters and epilogue. Persistent over units (tiles, or
// K-splits of tiles when the tiles do not fill the SM pairs).
// The operand with more rows is walked in the outer loop, so that it is read
// from HBM once while the other stays in L2.
//
// Every barrier wait is bounded, with the same exit as gemm_tc.cu's kernel.
#include "split_gemm.cuh"

#include <algorithm>
#include <cmath>

#include "linear_xent.cuh"
#include "tc_pipe.cuh"

namespace gt {
namespace tc {

constexpr int SBM = 128;                         // rows of A and of B per CTA
constexpr int SBK = 32;                          // K per stage
constexpr int SSTAGES = 6;
// Stages per promotion: 128 of K, the values that share a scale in dx and dw.
// The sum of a partial is truncated at every MMA, by up to 2^-23 of what it holds
// by then, always towards zero, so short groups are more exact and long ones leave the
// epilogue more time under the next tile's first two groups. With 256, sums of positive
// products came out 13.7 * 2^-23 too small on average, with 128 half of that;
// dx at V = 517 was off by 1.3e-6 of the result (0.6e-6), dw at 1880 x 1118 x 544 by
// 1.01e-6 (0.67e-6, where plain float32 sums have 0.59e-6), the loss at 4096 x 1024 x 65536 by 2.7e-7
// (1.4e-7; plain 1.0e-7). At 2048 x 1024 x 32000 with z stored through registers: logits 329 us
// against 299 with 256, dw 276 against 260, dx 277 either way.
constexpr int SGROUP = kSplitGroup / SBK;
constexpr int SMIN_SPLIT = 16;                   // stages that a K-split has at least
constexpr int STHREADS = 384;
constexpr uint32_t PLANE_BYTES = SBM * SBK * 2;  // one plane of one operand, 8 KB
constexpr uint32_t OPER_BYTES = 2 * PLANE_BYTES;
constexpr uint32_t SSTAGE_BYTES = 2 * OPER_BYTES;
constexpr int SPROMOTERS = 8;                    // warps
constexpr int STILE = 256;
constexpr uint32_t SEPI_OFFSET = SSTAGES * SSTAGE_BYTES;  // (1024-byte aligned: the 128-byte swizzle)
constexpr uint32_t SBAR_OFFSET = SEPI_OFFSET + SPROMOTERS * 32 * 32 * 4;
constexpr uint32_t SSMEM_BYTES = SBAR_OFFSET + 512 + 1024;
static_assert(SSMEM_BYTES <= 232448, "shared memory budget");
constexpr int64_t STILE_ELEMS = (int64_t)STILE * STILE;
// The launch gives every thread 65536 / 384 = 170, rounded down to 168: 4
// warps with 64 and 8 with 216 stay within 12 * 168.
constexpr int SREGS_LOW = 64, SREGS_HIGH = 216;
static_assert(128 * SREGS_LOW + 256 * SREGS_HIGH <= STHREADS * 168, "register split exceeds the launch's registers");

struct SplitUnits {
  int whole = 0, splits = 1;  // tiles computed whole; K-splits of the others
  int pairs = 1;              // SM pairs
  float* ws = nullptr;        // [splits][tiles - whole][256 * 256]
  uint64_t wait_limit_ns = kTimeoutNs;
  int withhold = 0;  // test hook: the peer's relay withholds its first arrival
};

struct SplitShared {
  uint64_t full[SSTAGES];   // TMA -> local relay (and the leader's MMA)
  uint64_t ready[SSTAGES];  // the peer's relay -> the leader's MMA
  uint64_t empty[SSTAGES];  // MMA -> producers of both CTAs
  uint64_t pfull[2], pempty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int failed;
};

struct SplitArgs {
  int64_t M, N, K;
  const int64_t* kept;
  int64_t kept_from;
  int kept_k;  // the rows that there are limit K, not M
  const int32_t* row_index;
  const float *scale, *group_scale;
  int64_t group_ld;
  float* out;
  int64_t ldc;
  int accumulate;
  int vec;     // out's rows are 16-byte aligned
  int m_fast;  // consecutive tiles share their columns of C, else their rows
  const float *row_scale, *col_scale, *bias;
  const int32_t* labels;
  float2* strips;
  int64_t strip_rows;
  float* picked;
};

// The sizes that there really are (SplitGemm::kept), and the units for them: the
// host planned for all rows. Whole tiles stay whole and tiles that were all
// split stay split S ways; where only the last round's tiles were, the new
// last round's are split as far as the pairs go round (so the workspace, one
// partial tile per pair, holds them).
struct SplitSizes {
  int M, K;  // (below 2^30)
  int whole, splits;
};
__device__ __forceinline__ SplitSizes actual_sizes(const SplitArgs& s, const SplitUnits& su) {
  SplitSizes z{(int)s.M, (int)s.K, su.whole, su.splits};
  if (!s.kept) return z;
  const int host = s.kept_k ? z.K : z.M, n = (int)max((int64_t)0, min((int64_t)host, *s.kept - s.kept_from));
  if (n == host) return z;
  if (s.kept_k) {
    z.K = n;
    if (n == 0 && s.accumulate) z = {0, 0, 0, 1};  // nothing to add
    return z;
  }
  z.M = n;
  const int tiles = (z.M + STILE - 1) / STILE * (int)((s.N + STILE - 1) / STILE);
  if (su.splits > 1 && su.whole > 0) {
    z.whole = tiles / su.pairs * su.pairs;
    const int rest = tiles - z.whole;
    z.splits = rest ? max(1, min(min(su.pairs / rest, 64), (z.K + SBK - 1) / SBK / SMIN_SPLIT)) : 1;
  }
  if (z.splits == 1) z.whole = tiles;
  return z;
}

// Unit u: tile (mt, nt) over the stages [kb, ke), kb at a group's first; the split index or -1.
__device__ __forceinline__ int split_unit(int u, int m_tiles, int n_tiles, int m_fast, const SplitSizes& su, int num_k,
                                          int& t, int& mt, int& nt, int& kb, int& ke) {
  const int tiles = m_tiles * n_tiles;
  int sidx = -1;
  t = u, kb = 0, ke = num_k;
  if (u >= su.whole) {
    const int rest = tiles - su.whole, v = u - su.whole;
    sidx = v / rest;
    t = su.whole + (v - sidx * rest);
    const int groups = (num_k + SGROUP - 1) / SGROUP;
    kb = min(num_k, (int)((int64_t)sidx * groups / su.splits) * SGROUP);
    ke = min(num_k, (int)((int64_t)(sidx + 1) * groups / su.splits) * SGROUP);
  }
  if (m_fast)
    nt = t / m_tiles, mt = t - nt * m_tiles;
  else
    mt = t / n_tiles, nt = t - mt * n_tiles;
  return sidx;
}

// Descriptors of an operand's first K step of 16 in stage 0's hi plane. K-major:
// 64-byte rows, 64-byte swizzle, 8-row groups 512 bytes apart; a K step is +32
// bytes, the lo plane + PLANE_BYTES. M/N-major: 128-byte rows of 64 values,
// one per k, 128-byte swizzle, 8-k groups 1024 bytes apart; 64-value groups
// (each its hi and lo planes, 4 KB both) 8 KB apart; a K step is + 2048 bytes,
// the lo plane + 4 KB.
template <bool MN>
__device__ __forceinline__ uint64_t split_desc(uint32_t base) {
  return MN ? smem_desc(base, 8192, 1024, 2) : smem_desc(base, 16, 512, 4);
}
template <bool MN>
constexpr uint32_t kstep_units() { return (MN ? 2048 : 32) >> 4; }
template <bool MN>
constexpr uint32_t lo_units() { return (MN ? 4096 : PLANE_BYTES) >> 4; }

// kind::f16, both operands float16, float32 accumulator, 256 x 256.
template <bool A_MN, bool B_MN>
__device__ __forceinline__ uint32_t split_idesc() {
  return 1u << 4 | (A_MN ? 1u : 0u) << 15 | (B_MN ? 1u : 0u) << 16 | (uint32_t)(STILE >> 3) << 17 |
         (uint32_t)(STILE >> 4) << 24;
}

__device__ __forceinline__ void mma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One operand's stage: both planes. K-major: one box {32, 128, 2}, or, grouped,
// a box {32, 1, 1, 128} per plane; M/N-major: a box {64, 32, 2} per 64 values.
template <bool MN, bool GROUPED>
__device__ __forceinline__ void split_load(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int k0) {
  if (GROUPED) {
    tma_load_4d(dst, map, bar, k0 % kSplitGroup, 0, k0 / kSplitGroup, row);
    tma_load_4d(dst + PLANE_BYTES, map, bar, k0 % kSplitGroup, 1, k0 / kSplitGroup, row);
  } else if (MN) {
    tma_load_3d(dst, map, bar, row, k0, 0);
    tma_load_3d(dst + PLANE_BYTES, map, bar, row + 64, k0, 0);
  } else {
    tma_load_3d(dst, map, bar, k0, row, 0);
  }
}

// A 32 x 32 block in a warp's transpose buffer: 16-byte chunk c of row r at
// chunk c ^ (r % 8), so that 8 rows' same chunk and one row's 8 chunks are both
// free of bank conflicts.
__device__ __forceinline__ float4* block_chunk(float* xpose, int r, int c) {
  return reinterpret_cast<float4*>(xpose) + r * 8 + (c ^ (r & 7));
}
__device__ __forceinline__ float& block_at(float* xpose, int r, int c) {
  return xpose[r * 32 + ((((c >> 2) ^ (r & 7)) << 2) | (c & 3))];
}

// tcgen05.ld of 32 columns without waiting, and the wait for all loads before.
__device__ __forceinline__ void tmem_issue32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// The registers pass through the wait, so nothing reads them before it.
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}

template <bool A_MN, bool B_MN, bool LOGITS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(STHREADS, 1)
    split_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmOut, const SplitArgs s, const SplitUnits su) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  SplitShared* sh = (SplitShared*)(smem + SBAR_OFFSET);
  constexpr bool INDEXED = !A_MN && !LOGITS;  // dx: A is grouped, the rows of C are scattered
  volatile int* failed = &sh->failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair = (int)cluster_id(), pairs = (int)num_clusters();

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmB)) : "memory");
    for (int i = 0; i < SSTAGES; i++) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->ready[i], 1);
      mbar_init(&sh->empty[i], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&sh->pfull[b], 1);
      mbar_init(&sh->pempty[b], 2 * SPROMOTERS);
    }
    mbar_init(&sh->mma_done, 1);
    sh->failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  after_predecessor();
  const SplitSizes sz = actual_sizes(s, su);
  const int num_k = (sz.K + SBK - 1) / SBK;
  const int m_tiles = (sz.M + STILE - 1) / STILE, n_tiles = (int)((s.N + STILE - 1) / STILE);
  const int tiles = m_tiles * n_tiles;
  const int units = sz.whole + (tiles - sz.whole) * sz.splits;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SREGS_LOW));
    if (warp == 0) {  // ---- TMA producer
      const bool issuer = elect_one();
      int it = 0, issued_to = 0;
      for (int u = pair; u < units && !__shfl_sync(0xffffffffu, *failed, 0); u += pairs) {
        int t, mt, nt, kb, ke;
        split_unit(u, m_tiles, n_tiles, s.m_fast, sz, num_k, t, mt, nt, kb, ke);
        const int a_row = mt * STILE + (int)rank * SBM, b_row = nt * STILE + (int)rank * SBM;
        for (int kt = kb; kt < ke; kt++, it++) {
          const int st = it % SSTAGES;
          if (!__all_sync(0xffffffffu, mbar_wait(&sh->empty[st], ((it / SSTAGES) & 1) ^ 1, 1, su.wait_limit_ns))) {
            if (lane == 0) *failed = 1;
            break;
          }
          if (issuer) {
            uint64_t* bar = &sh->full[st];
            uint8_t* stage = smem + st * SSTAGE_BYTES;
            mbar_expect_tx(bar, SSTAGE_BYTES);
            split_load<A_MN, INDEXED>(stage, &tmA, bar, a_row, kt * SBK);
            split_load<B_MN, false>(stage + OPER_BYTES, &tmB, bar, b_row, kt * SBK);
          }
          __syncwarp();
          issued_to = it + 1;
        }
      }
      if (__shfl_sync(0xffffffffu, *failed, 0)) {  // let copies in flight land before the CTA tears down
        for (int i = issued_to > SSTAGES ? issued_to - SSTAGES : 0; i < issued_to; i++)
          mbar_wait(&sh->full[i % SSTAGES], (i / SSTAGES) & 1, 5, kTimeoutNs);
      }
    } else if (warp == 1) {
      if (leader) {  // ---- MMA issuer
        const bool issuer = elect_one();
        const uint32_t idesc = split_idesc<A_MN, B_MN>();
        const uint64_t adesc0 = split_desc<A_MN>(smem_u32(smem)), bdesc0 = split_desc<B_MN>(smem_u32(smem) + OPER_BYTES);
        int it = 0, group = 0;
        bool stop = false;
        for (int u = pair; u < units && !stop; u += pairs) {
          int t, mt, nt, kb, ke;
          split_unit(u, m_tiles, n_tiles, s.m_fast, sz, num_k, t, mt, nt, kb, ke);
          for (int kt = kb; kt < ke; kt++, it++) {
            const int st = it % SSTAGES;
            const uint32_t phase = (it / SSTAGES) & 1;
            const bool start = (kt - kb) % SGROUP == 0;
            const uint32_t buf = (uint32_t)(group & 1);
            bool ok = mbar_wait(&sh->full[st], phase, 3, su.wait_limit_ns);
            ok = ok && mbar_wait(&sh->ready[st], phase, 4, su.wait_limit_ns);
            if (start) ok = ok && mbar_wait(&sh->pempty[buf], ((group >> 1) & 1) ^ 1, 2, su.wait_limit_ns);
            if (!__all_sync(0xffffffffu, ok)) {
              stop = true;
              break;
            }
            tc_fence_after();
            const uint64_t slot = (uint64_t)((st * SSTAGE_BYTES) >> 4);
            const uint32_t d = tmem + buf * 256;
            uint64_t ah[2], bh[2];
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
              ah[kk] = adesc0 + slot + kk * kstep_units<A_MN>();
              bh[kk] = bdesc0 + slot + kk * kstep_units<B_MN>();
            }
            if (issuer) {
#pragma unroll
              for (int kk = 0; kk < 2; kk++) {
                mma_f16_pair(d, ah[kk] + lo_units<A_MN>(), bh[kk], idesc, start && kk == 0 ? 0u : 1u);
                mma_f16_pair(d, ah[kk], bh[kk] + lo_units<B_MN>(), idesc, 1u);
                mma_f16_pair(d, ah[kk], bh[kk], idesc, 1u);
              }
              mma_commit_pair(&sh->empty[st]);
            }
            __syncwarp();
            if ((kt - kb) % SGROUP == SGROUP - 1 || kt == ke - 1) {
              if (issuer) mma_commit_pair(&sh->pfull[buf]);
              __syncwarp();
              group++;
            }
          }
        }
        if (stop && lane == 0) *failed = 1;
        if (issuer)
          asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                           smem_u32(&sh->mma_done))
                       : "memory");
        __syncwarp();
        mbar_wait(&sh->mma_done, 0, 6, kTimeoutNs);
      }
    } else if (warp == 2 && !leader) {  // ---- the peer's half of each stage has landed
      int it = 0;
      bool stop = false;
      for (int u = pair; u < units && !stop; u += pairs) {
        int t, mt, nt, kb, ke;
        split_unit(u, m_tiles, n_tiles, s.m_fast, sz, num_k, t, mt, nt, kb, ke);
        for (int kt = kb; kt < ke; kt++, it++) {
          const int st = it % SSTAGES;
          if (__shfl_sync(0xffffffffu, *failed, 0) ||
              !__all_sync(0xffffffffu, mbar_wait(&sh->full[st], (it / SSTAGES) & 1, 8, su.wait_limit_ns))) {
            if (lane == 0) *failed = 1;
            stop = true;
            break;
          }
          if (lane == 0 && !(su.withhold && it == 0)) mbar_arrive_rank(&sh->ready[st], 0);
          __syncwarp();
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SREGS_HIGH));
    // ---- promoters and epilogue: warp quarter q has TMEM lanes 32 q .. (its
    // rows), half h the columns 128 h .. 128 h + 127.
    const int q = warp & 3, h = (warp - 4) >> 2;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16) + 128 * h;
    float* xpose = (float*)(smem + SEPI_OFFSET) + (warp - 4) * 32 * 32;
    const float sc = LOGITS ? 1.0f : *s.scale;
    int group = 0;
    for (int u = pair; u < units && !__shfl_sync(0xffffffffu, *failed, 0); u += pairs) {
      int t, mt, nt, kb, ke;
      const int sidx = split_unit(u, m_tiles, n_tiles, s.m_fast, sz, num_k, t, mt, nt, kb, ke);
      const int groups = (ke - kb + SGROUP - 1) / SGROUP;
      const int m0 = mt * STILE + (int)rank * SBM + 32 * q, n0 = nt * STILE + 128 * h;  // (sizes stay below 2^30)
      const int rows = max(0, min(32, sz.M - m0));
      // What the epilogue reads besides, fetched while the products run: row m0 +
      // r of C in out (lane r holds it; without an index, and in the
      // workspace, the r-th), the row's label, the columns' scales and biases.
      int32_t my_row = lane;
      if constexpr (INDEXED) {
        if (sidx < 0 && lane < rows) my_row = s.row_index[m0 + lane] - m0;
      }
      const int32_t label = LOGITS && lane < rows ? s.labels[m0 + lane] : -1;
      // the row's scale as a factor of at most 1 and one of at least 1, on either side of the
      // column's, so that no product on the way leaves the range that the last one is in
      float down = 1.0f, up_again = 1.0f;
      if constexpr (LOGITS) {
        const float r = lane < rows ? s.row_scale[m0 + lane] : 1.0f;
        down = fminf(r, 1.0f), up_again = fmaxf(r, 1.0f);
        if (lane < 8)
          asm volatile("prefetch.global.L1 [%0];" ::"l"((lane < 4 ? s.col_scale : s.bias) + n0 + 32 * (lane & 3)));
      }
      float tot[128];
#pragma unroll
      for (int i = 0; i < 128; i++) tot[i] = 0.0f;
      bool ok = true;
      for (int g = 0; g < groups; g++, group++) {
        const uint32_t buf = (uint32_t)(group & 1);
        float gs = 1.0f;  // the group's scale of this lane's row, on its way during the wait
        if constexpr (!LOGITS) {
          if (lane < rows) gs = s.group_scale[(int64_t)(kb / SGROUP + g) * s.group_ld + m0 + lane];
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&sh->pfull[buf], (group >> 1) & 1, 7, su.wait_limit_ns))) {
          *failed = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        {
          uint32_t p[2][32];
          tmem_issue32(lane_base + buf * 256, p[0]);
          tmem_wait32(p[0]);
#pragma unroll
          for (int j = 0; j < 4; j++) {  // the next chunk's load runs under this one's adds
            if (j < 3) tmem_issue32(lane_base + buf * 256 + 32 * (j + 1), p[(j + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 32; i++) {
              const float v = __uint_as_float(p[j & 1][i]);
              tot[32 * j + i] = LOGITS ? __fadd_rn(tot[32 * j + i], v) : __fmaf_rn(v, gs, tot[32 * j + i]);
            }
            if (j < 3) tmem_wait32(p[(j + 1) & 1]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_rank(&sh->pempty[buf], 0);
      }
      if (!ok) break;
      float* part = sidx < 0 ? nullptr
                             : su.ws + ((int64_t)sidx * (tiles - sz.whole) + (t - sz.whole)) * STILE_ELEMS +
                                   (int64_t)(rank * SBM + 32 * q) * STILE + 128 * h;
      float* dst = part ? part : s.out ? s.out + (int64_t)m0 * s.ldc + n0 : nullptr;
      const int64_t ld = part ? STILE : s.ldc;
      const bool vec = part || s.vec;
      float top = -INFINITY, sum = 0.0f;  // LOGITS: this lane's row over the strip
      // 32 x 32 blocks, what is stored through the per-warp buffer
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float z[32];
#pragma unroll
        for (int i = 0; i < 32; i++) z[i] = tot[32 * j + i];
        const int nb = n0 + 32 * j, cols = part ? 32 : max(0, min(32, (int)s.N - nb));
        if constexpr (LOGITS) {
          // (the same addresses for all lanes; the scales' products are exact, so one rounding, the bias')
          const float4 *cs = reinterpret_cast<const float4*>(s.col_scale + nb),
                       *cb = reinterpret_cast<const float4*>(s.bias + nb);
#pragma unroll
          for (int c = 0; c < 8; c++) {
            const float4 f = cs[c], b = cb[c];
            z[4 * c] = __fmaf_rn(__fmul_rn(__fmul_rn(z[4 * c], down), f.x), up_again, b.x);
            z[4 * c + 1] = __fmaf_rn(__fmul_rn(__fmul_rn(z[4 * c + 1], down), f.y), up_again, b.y);
            z[4 * c + 2] = __fmaf_rn(__fmul_rn(__fmul_rn(z[4 * c + 2], down), f.z), up_again, b.z);
            z[4 * c + 3] = __fmaf_rn(__fmul_rn(__fmul_rn(z[4 * c + 3], down), f.w), up_again, b.w);
          }
        } else if (!part) {
#pragma unroll
          for (int i = 0; i < 32; i++) z[i] = __fmul_rn(z[i], sc);
        }
        if (dst) {
          if constexpr (LOGITS) {  // the buffer's last copy has been read
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int c = 0; c < 8; c++)
            *block_chunk(xpose, lane, c) = make_float4(z[4 * c], z[4 * c + 1], z[4 * c + 2], z[4 * c + 3]);
          if constexpr (LOGITS) {
            // z goes out by TMA, which leaves these warps to the statistics (its pitch is a multiple of 32); through
            // registers, 4 rows x 128 bytes at a time, 2048 x 1024 x 32000 took 333 us instead of 302
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && rows > 0 && nb < s.ldc) {
              tma_store_2d(&tmOut, xpose, nb, m0);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            __syncwarp();
          }
          if constexpr (LOGITS) {
          } else if (vec && cols == 32) {  // 4 rows x 128 bytes per access
            const int r0 = lane >> 3, c = lane & 7;
            float* o = dst + (INDEXED ? 0 : (int64_t)r0 * ld) + 32 * j + 4 * c;
            if (A_MN && s.accumulate && !part) {
              // the old values of all rows before any is written: a load per
              // row behind the store before it made the kernel three times as
              // slow
              float4 was[8];
#pragma unroll
              for (int k = 0; k < 8; k++)
                was[k] = r0 + 4 * k < rows ? *reinterpret_cast<const float4*>(o + 4 * k * ld) : float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int k = 0; k < 8; k++) {
                const float4 v = *block_chunk(xpose, r0 + 4 * k, c);
                if (r0 + 4 * k < rows)
                  *reinterpret_cast<float4*>(o + 4 * k * ld) =
                      make_float4(__fadd_rn(was[k].x, v.x), __fadd_rn(was[k].y, v.y), __fadd_rn(was[k].z, v.z),
                                  __fadd_rn(was[k].w, v.w));
              }
            } else {
#pragma unroll
              for (int k = 0; k < 8; k++) {
                const int64_t row = INDEXED ? __shfl_sync(0xffffffffu, my_row, r0 + 4 * k) : 4 * k;
                if (part || r0 + 4 * k < rows)
                  *reinterpret_cast<float4*>(o + row * ld) = *block_chunk(xpose, r0 + 4 * k, c);
              }
            }
          } else if constexpr (INDEXED) {  // (every lane: the rows come by shuffle)
            float* o = dst + 32 * j + lane;
#pragma unroll 8
            for (int r = 0; r < rows; r++) {
              const int64_t row = __shfl_sync(0xffffffffu, my_row, r);
              if (lane < cols) o[row * ld] = block_at(xpose, r, lane);
            }
          } else if (lane < cols) {
            float* o = dst + 32 * j + lane;
            if (A_MN && s.accumulate) {
#pragma unroll 1
              for (int r0 = 0; r0 < 32; r0 += 16) {
                float was[16];
#pragma unroll
                for (int r = 0; r < 16; r++) was[r] = r0 + r < rows ? o[(r0 + r) * ld] : 0.0f;
#pragma unroll
                for (int r = 0; r < 16; r++)
                  if (r0 + r < rows) o[(r0 + r) * ld] = __fadd_rn(was[r], block_at(xpose, r0 + r, lane));
              }
            } else {
#pragma unroll 8
              for (int r = 0; r < rows; r++) o[r * ld] = block_at(xpose, r, lane);
            }
          }
        }
        if constexpr (LOGITS) {
          // the running maximum and sum; a maximum of -infinity sums to 0, a
          // NaN (which fmaxf passes over) reaches the sum
          float block_top = z[0];
#pragma unroll
          for (int i = 1; i < 32; i++) block_top = fmaxf(block_top, z[i]);
          const float up = fmaxf(top, block_top), from = up == -INFINITY ? 0.0f : up;
          float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 32; i++) add[i & 3] += exp_below(z[i] - from);
          sum = sum * exp_below(top - from) + ((add[0] + add[1]) + (add[2] + add[3]));
          top = up;
          if (label >= nb && label < nb + cols) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (label - nb == i) s.picked[m0 + lane] = z[i];
          }
        }
        __syncwarp();
      }
      if constexpr (LOGITS) {
        if (!part && lane < rows && n0 < s.N)
          s.strips[(int64_t)(n0 / kStripCols) * s.strip_rows + m0 + lane] = make_float2(top, sum);
      }
    }
    if (LOGITS && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// The split tiles: their partials added in split order, then the epilogue.
__global__ void split_reduce_kernel(SplitUnits su, SplitArgs s) {
  after_predecessor();
  const SplitSizes sz = actual_sizes(s, su);
  const int m_tiles = (sz.M + STILE - 1) / STILE, n_tiles = (int)((s.N + STILE - 1) / STILE);
  const int rest = m_tiles * n_tiles - sz.whole;
  const int64_t total = (int64_t)rest * STILE_ELEMS;
  const float sc = *s.scale;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int r = (int)(i / STILE_ELEMS), e = (int)(i - (int64_t)r * STILE_ELEMS), t = sz.whole + r;
    const int mt = s.m_fast ? t % m_tiles : t / n_tiles, nt = s.m_fast ? t / m_tiles : t % n_tiles;
    const int64_t m = (int64_t)mt * STILE + e / STILE, n = (int64_t)nt * STILE + e % STILE;
    if (m >= sz.M || n >= s.N) continue;
    float acc = su.ws[i];
    for (int k = 1; k < sz.splits; k++) acc = __fadd_rn(acc, su.ws[(int64_t)k * total + i]);
    float* o = s.out + (s.row_index ? (int64_t)s.row_index[m] : m) * s.ldc + n;
    acc = __fmul_rn(acc, sc);
    *o = s.accumulate ? __fadd_rn(*o, acc) : acc;
  }
}

// float32 rows x cols of pitch `ld`, stored from 32 x 32 blocks in the 128-byte swizzle (block_chunk).
static char* out_map(gt_ctx* ctx, CUtensorMap* map, float* out, int64_t rows, int64_t ld) {
  auto encode = (EncodeTiledFn)ctx->encode_tiled;
  if (!encode) return errorf("split_gemm: cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)ld, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 4};
  cuuint32_t box[2] = {32, 32}, estr[2] = {1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, (void*)out, dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return errorf("split_gemm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return nullptr;
}

static char* split_map(gt_ctx* ctx, CUtensorMap* map, const HalfPlanes& p, bool mn) {
  auto encode = (EncodeTiledFn)ctx->encode_tiled;
  if (!encode) return errorf("split_gemm: cuTensorMapEncodeTiled is unavailable");
  if (p.grouped) {
    cuuint64_t dims[4] = {kSplitGroup, 2, (cuuint64_t)(p.pitch / (2 * kSplitGroup)), (cuuint64_t)p.rows};
    cuuint64_t strides[3] = {kSplitGroup * 2, kSplitGroup * 4, (cuuint64_t)p.pitch * 2};
    cuuint32_t box[4] = {(cuuint32_t)SBK, 1, 1, (cuuint32_t)SBM}, estr[4] = {1, 1, 1, 1};
    CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, (void*)p.base, dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return errorf("split_gemm: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return nullptr;
  }
  cuuint64_t dims[3] = {(cuuint64_t)p.cols, (cuuint64_t)p.rows, 2};
  cuuint64_t strides[2] = {(cuuint64_t)p.pitch * 2, (cuuint64_t)p.plane_elems * 2};
  cuuint32_t box[3] = {mn ? 64u : (cuuint32_t)SBK, mn ? (cuuint32_t)SBK : (cuuint32_t)SBM, 2};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)p.base, dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, mn ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return errorf("split_gemm: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return nullptr;
}

// K-splits: whole tiles, every tile split S ways, or only the tiles of the
// last round, whichever the cost model finds cheapest. In units of a stage on
// a pair (768 clocks of MMA, 0.42 us): rounds of (stages + a fixed overhead per
// unit), plus the partials' trip through memory at about 5 TB/s. The partials
// stay within max_bytes (the last round's may be up to one per pair, see actual_sizes).
static SplitUnits split_plan(int64_t tiles, int64_t pairs, int64_t num_k, int64_t max_bytes) {
  constexpr double kOverhead = 12.0;
  SplitUnits best;
  best.whole = (int)tiles;
  auto rounds = [&](int64_t units) { return std::ceil((double)units / pairs); };
  auto traffic = [&](int64_t t, int S) { return (S + 1) * (double)t * STILE_ELEMS * 4.0 / 5e6 / 0.42; };
  const double base = rounds(tiles) * (num_k + kOverhead);
  double cost = base;
  for (int S = 2; S <= 64 && num_k / S >= SMIN_SPLIT; S++) {
    const double per = std::ceil((double)num_k / S) + kOverhead;
    if ((double)S * tiles * STILE_ELEMS * 4 <= (double)max_bytes) {
      const double c = rounds(tiles * S) * per + traffic(tiles, S);
      if (c < cost) cost = c, best.whole = 0, best.splits = S;
    }
    const int64_t full = tiles / pairs * pairs, rest = tiles - full;
    if (full > 0 && rest > 0 && rest * S <= pairs && pairs * STILE_ELEMS * 4 <= max_bytes) {
      const double c = (double)(tiles / pairs) * (num_k + kOverhead) + per + traffic(rest, S);
      if (c < cost) cost = c, best.whole = (int)full, best.splits = S;
    }
  }
  if (cost > 0.95 * base) best.whole = (int)tiles, best.splits = 1;
  return best;
}

template <bool A_MN, bool B_MN, bool LOGITS>
static char* split_launch(gt_ctx* ctx, const SplitGemm& g) {
  auto kern = split_gemm_kernel<A_MN, B_MN, LOGITS>;
  static bool configured[64] = {};
  if (ctx->device < 0 || ctx->device >= 64 || !configured[ctx->device]) {
    GT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SSMEM_BYTES));
    if (ctx->device >= 0 && ctx->device < 64) configured[ctx->device] = true;
  }
  CUtensorMap ta, tb, tout{};
  GT_TRY(split_map(ctx, &ta, g.a, A_MN));
  GT_TRY(split_map(ctx, &tb, g.b, B_MN));
  if (LOGITS && g.out) GT_TRY(out_map(ctx, &tout, g.out, g.M, g.ldc));
  const int64_t m_tiles = ceil_div(g.M, STILE), n_tiles = ceil_div(g.N, STILE), tiles = m_tiles * n_tiles;
  if (tiles > INT32_MAX / 64) return errorf("split_gemm: too many tiles");
  const int64_t free_sms = (int64_t)ctx->sm_count - ctx->gemm_sm_reserve, avail = free_sms >= 2 ? free_sms / 2 : 1;
  SplitUnits su;
  if (LOGITS)  // its epilogue needs whole rows of a tile
    su.whole = (int)tiles;
  else
    su = split_plan(tiles, avail, ceil_div(g.K, SBK), g.partial_bytes);
  su.pairs = (int)avail;
  su.wait_limit_ns = tc_wait_limit_ns();
  su.withhold = tc_take_withhold();
  const int vec = (((uintptr_t)g.out & 15) | (g.ldc & 3)) == 0;
  SplitArgs s{g.M,    g.N,        g.K,     g.kept,      g.kept_from, A_MN,        g.row_index, g.scale,  g.group_scale,
              g.group_ld, g.out,  g.ldc,   g.accumulate, vec,        g.N > g.M,   g.row_scale, g.col_scale, g.bias,
              g.labels, g.strips, g.strip_rows, g.picked};
  void* ws = nullptr;
  if (su.splits > 1) {
    // (with fewer rows than planned, the tiles split in the last round may be up to one per pair)
    const int64_t parts = su.whole > 0 ? avail : su.splits * tiles;
    GT_TRY(scratch(ctx, (size_t)parts * STILE_ELEMS * sizeof(float), &ws));
    su.ws = (float*)ws;
  }
  const int64_t units = su.whole + (tiles - su.whole) * su.splits;
  cudaError_t e = launch_overlapped(ctx, kern, (unsigned)(2 * std::min(units, avail)), STHREADS, SSMEM_BYTES, ta, tb, tout,
                                    s, su);
  if (e == cudaSuccess && su.splits > 1)
    e = launch_overlapped(ctx, split_reduce_kernel, grid_for(ctx, (tiles - su.whole) * STILE_ELEMS, 256), 256, 0, su, s);
  if (e == cudaSuccess) e = cudaGetLastError();
  release(ctx, ws);
  if (e != cudaSuccess) return cuda_error(e, "split_gemm launch", __FILE__, __LINE__);
  return nullptr;
}

}  // namespace tc

static bool g_split_used = false;

char* split_gemm(gt_ctx* ctx, const SplitGemm& g) {
  if (ctx->sm_count < 2) return errorf("split_gemm: needs a pair of SMs");
  g_split_used = true;
  if (g.strips) {
    if (g.a_mn || g.b_mn || g.a.grouped) return errorf("split_gemm: the logits' operands are K-major");
    if (g.ldc % 32 || ((uintptr_t)g.out & 15)) return errorf("split_gemm: the logits' rows come in blocks of 32");
    if (!g.row_scale || !g.col_scale || !g.bias) return errorf("split_gemm: the logits' scales or biases are missing");
    return tc::split_launch<false, false, true>(ctx, g);
  }
  if (g.a_mn ? g.row_index != nullptr : !g.row_index || g.accumulate)
    return errorf("split_gemm: an index of rows goes with K-major A and no accumulation");
  if (g.a_mn == g.a.grouped || !g.scale || !g.group_scale)
    return errorf("split_gemm: K-major A comes in groups, and every group has its scales");
  if (!g.a_mn && g.b_mn) return tc::split_launch<false, true, false>(ctx, g);
  if (g.a_mn && g.b_mn) return tc::split_launch<true, true, false>(ctx, g);
  return errorf("split_gemm: layout not built");
}

char* split_gemm_check_errors() {
  if (!g_split_used) return nullptr;
  int e = 0;
  GT_CUDA(cudaMemcpyFromSymbol(&e, g_tc_error, sizeof e));
  if (e) {
    int zero = 0;
    cudaMemcpyToSymbol(g_tc_error, &zero, sizeof zero);
    return errorf("tcgen05 split GEMM: a pipeline wait timed out (site %d); results are invalid", e);
  }
  return nullptr;
}

}  // namespace gt
