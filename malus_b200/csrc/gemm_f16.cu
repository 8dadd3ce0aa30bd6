// f32 GEMM on the half-precision tensor pipe.
//
// Each operand row is scaled by a power of two and split into two halves, hi =
// half_rn(x), lo = half_rn(x - hi): 22 bits of every element within 2^-16 of its
// row's largest, and an error of at most 2^-38 of that largest for smaller ones
// (the largest is brought to 2^13 or more, where half's grid of 2^-24 rounds by
// 2^-25).  An operand may have a scale per 256 of K and row instead, applied as each
// accumulator is added to the sums: then "its row's largest" is that of the 256.
// The product keeps hi*lo + lo*hi + hi*hi (the dropped lo*lo is below
// 2^-22 of a term).  Against three tf32 products of the same 22 bits this takes
// half the tensor time and half the operand bytes.
//
// The tensor core truncates when it adds into its f32 accumulator (measured
// with products of known sums: a chain of n additions loses about n * 2e-8 of
// the magnitude, all in one direction; K = 50304 as one chain is off by 8e-5).
// So a chain is kept short: within a 64-deep stage the small cross products come
// first, then the four hi*hi additions, and after every fourth stage (K = 256; every
// second in short units) the epilogue warps take the accumulator out of tensor memory and add it,
// rounding to nearest, to sums in their registers, while the tensor core fills
// the other accumulator.
//
// Work: 2-CTA clusters, each unit a 256 x 256 tile (one tcgen05.mma of M = 256
// per k-step, cta_group::2) over all of K or a slice of it.  Each CTA loads its
// 128 rows of A and 128 of B, both planes, 64 deep: 64 KB a stage, three stages,
// so an SM takes in 64 KB per 1536 cycles of tensor time.  A single CTA's 128 x
// 256 tile would take 96 KB per the same time, more than L2 delivers.
// Warp 0 issues the TMA loads, warp 1 (of rank 0) the MMAs, warps 4-11 hold the
// sums (128 columns of a row per thread) and store by TMA.
#include "gemm_f16.cuh"
#include "tc_common.cuh"

#include <vector>

namespace malus {
namespace {
using namespace malus::tc;

constexpr int BM = 128, BN = 256, BK = 64, STAGES = 3;
constexpr int kTile = 128 * BK * 2;                 // one plane's 128 rows, 64 deep
constexpr int kStageBytes = 4 * kTile;              // A hi, A lo, B hi, B lo
// Stages per accumulator, and for units short enough that the pipeline's latency
// and not its rate decides (one unit of at most kShortUnit stages per pair).
constexpr int kChunk = 4, kShortChunk = 2, kShortUnit = 16;
constexpr int kEpiWarps = 8, kThreads = 128 + 32 * kEpiWarps;
constexpr int kCols = BN * 4 / kEpiWarps;           // columns of a row that an epilogue thread holds
// Registers per thread: 168 at launch; the warpgroup of the TMA and MMA warps
// gives up all but 40, the two epilogue warpgroups take 232 (128 sums, 32 in
// flight from tensor memory).  128 * 40 + 256 * 232 = 384 * 168.
constexpr int kRegsLaunch = 168, kRegsIo = 40, kRegsEpi = 232;
static_assert(128 * kRegsIo + 32 * kEpiWarps * kRegsEpi <= kThreads * kRegsLaunch, "registers");
constexpr int kStaging = 32 * 32 * 4;               // per epilogue warp: 32 rows x 32 columns
constexpr int kSmem = STAGES * kStageBytes + 1024 + 256 + kEpiWarps * kStaging;
static_assert(kSmem <= 232448 && kCols == 128, "shared memory; a warp's lanes hold four column scales each");

struct Params {
  int M, N, K, tiles_m, tiles_n, nst, splits;
  int chunk;           // stages per accumulator
  int align;           // K slices start at multiples of so many stages
  int a_mn, b_mn, a_grouped;
  int64_t a_k0, b_k0;
  const float *a_inv, *b_inv;
  const float* block_inv;   // of A (kByM) or of B (kByN)
  int64_t block_pitch;
  float inv_all;
  int accumulate;
  const int* count;
  int inner_m;         // consecutive units walk M (else N)
  float2* part;
  float* at;
  const void* target;
  int tdt;
  int32_t* err;
};

struct Unit { int m0, n0, st_lo, st_hi, split; };
__device__ __forceinline__ Unit unit_at(const Params& p, int u) {
  Unit r;
  const int tile = u / p.splits;
  r.split = u % p.splits;
  const int i = p.inner_m ? tile % p.tiles_m : tile / p.tiles_n;
  const int j = p.inner_m ? tile / p.tiles_m : tile % p.tiles_n;
  r.m0 = i * 2 * BM;
  r.n0 = j * BN;
  const int64_t steps = (p.nst + p.align - 1) / p.align;
  r.st_lo = (int)(r.split * steps / p.splits) * p.align;
  r.st_hi = min((int)((r.split + 1) * steps / p.splits) * p.align, p.nst);
  return r;
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc));
}
// half x half -> f32, M = 256 over the pair, N = 256
__device__ __forceinline__ uint32_t idesc_f16(bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
         ((uint32_t)((2 * BM) >> 4) << 24);
}
// 128-byte swizzle.  K-major: rows of 64 halves, 8-row groups 1 KB apart; a step
// of 16 in K is 32 bytes.  MN-major: columns in chunks of 64 (8 KB each: 64 rows
// of K), groups of 8 K rows 1 KB apart; a step of 16 in K is 2 KB.
__device__ __forceinline__ uint64_t desc_of(uint32_t tile, bool mn) {
  return mn ? umma_desc(tile, BK * 128, 1024, 2) : umma_desc(tile, 16, 1024, 2);
}

// What becomes of the sums: stored; row statistics; both; stored, with A's or B's
// scales (which change from chunk to chunk) applied to each chunk as it is added.
enum Mode : int { kStore = 0, kLse = 1, kBoth = 2, kByM = 3, kByN = 4 };

// v times the row's scale and those of four columns, which lane `from` holds.  The
// scales meet first: each alone may take a sum past the largest float.
__device__ __forceinline__ float4 scale4(float4 v, float sa, float4 sb4, int from) {
  v.x *= sa * __shfl_sync(0xffffffffu, sb4.x, from);
  v.y *= sa * __shfl_sync(0xffffffffu, sb4.y, from);
  v.z *= sa * __shfl_sync(0xffffffffu, sb4.z, from);
  v.w *= sa * __shfl_sync(0xffffffffu, sb4.w, from);
  return v;
}

// The sums acc of 32 rows from m0 (one per lane, scale sa), columns n0 .. n0 +
// kCols - 1 (lane i holds the scales of columns 4 i .. 4 i + 3 of them):
// scaled and sent to the output 32 columns at a time through the warp's staging
// block, which a TMA store (or, accumulating, a TMA add: one per element and
// launch, so the order is fixed) takes from there.  The copy drops what lies
// past M or N.  SCALED: acc has its scales already.
template <bool SCALED>
__device__ __forceinline__ void finish_store(const Params& p, const CUtensorMap* mOut, const Unit& un,
                                             float (&acc)[kCols], int m0, int n0, float sa, float4 sb4, uint8_t* stage) {
  const int lane = threadIdx.x & 31;
  if (m0 >= p.M) return;   // uniform over the warp
  float4* mine = reinterpret_cast<float4*>(stage + lane * 128);
#pragma unroll
  for (int c = 0; c < kCols; c += 32) {
    if (n0 + c >= p.N) break;
    if (lane == 0) bulk_wait_read<0>();   // the block's last copy has left it
    __syncwarp();
#pragma unroll
    for (int g = 0; g < 8; ++g) {   // 16-byte granule g of row r lies at g ^ (r & 7): the map's swizzle
      const float4 v = make_float4(acc[c + 4 * g], acc[c + 4 * g + 1], acc[c + 4 * g + 2], acc[c + 4 * g + 3]);
      mine[g ^ (lane & 7)] = SCALED ? v : scale4(v, sa, sb4, c / 4 + g);
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (p.accumulate) tma_add_3d(mOut, smem_u32(stage), n0 + c, m0, un.split);
      else tma_store_3d(mOut, smem_u32(stage), n0 + c, m0, un.split);
      bulk_commit();
    }
  }
}

// The sums of a row into its maximum, sum of exponentials and target value; acc is
// scaled after it (-inf past N).
__device__ __forceinline__ void finish_lse(const Params& p, float (&acc)[kCols], int m, int n0, float sa, float4 sb4) {
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < kCols; j += 4) {
    const float4 v = scale4(make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]), sa, sb4, j / 4);
    acc[j] = n0 + j < p.N ? v.x : -INFINITY;
    acc[j + 1] = n0 + j + 1 < p.N ? v.y : -INFINITY;
    acc[j + 2] = n0 + j + 2 < p.N ? v.z : -INFINITY;
    acc[j + 3] = n0 + j + 3 < p.N ? v.w : -INFINITY;
    mx = fmaxf(mx, fmaxf(fmaxf(acc[j], acc[j + 1]), fmaxf(acc[j + 2], acc[j + 3])));
  }
  if (m >= p.M) return;
  float s = 0.0f;
  const float mm = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
  for (int j = 0; j < kCols; ++j) s += exp2_hw((acc[j] - mm) * kLog2e);
  p.part[(int64_t)m * (BN / kCols * p.tiles_n) + n0 / kCols] = make_float2(mx, s);
  const int64_t t = p.tdt == MALUS_I64 ? ((const int64_t*)p.target)[m] : (int64_t)((const int32_t*)p.target)[m];
  if (t >= n0 && t < n0 + kCols && t < p.N) {
    const int o = (int)(t - n0);
    float zt = 0.0f;
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (j == o) zt = acc[j];
    p.at[m] = zt;
  }
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
k_gemm_f16(const __grid_constant__ CUtensorMap mAh, const __grid_constant__ CUtensorMap mAl,
           const __grid_constant__ CUtensorMap mBh, const __grid_constant__ CUtensorMap mBl,
           const __grid_constant__ CUtensorMap mOut, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + STAGES * kStageBytes + kEpiWarps * kStaging);
  uint64_t* empty = full + STAGES;
  uint64_t* accf = empty + STAGES;
  uint64_t* acce = accf + 2;
  uint64_t* drain = acce + 2;
  uint64_t* done = drain + 1;   // every epilogue warp finished reading tensor memory
  uint32_t* tmem_slot = (uint32_t*)(done + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int grp = (int)(blockIdx.x >> 1), ngrp = (int)(gridDim.x >> 1);
  const int total = p.tiles_m * p.tiles_n * p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&accf[b]), 1);
      mbar_init(smem_u32(&acce[b]), 2 * kEpiWarps);   // both CTAs' epilogues
    }
    mbar_init(smem_u32(drain), 1);
    mbar_init(smem_u32(done), kEpiWarps);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers exist before either signals the other
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIo));
  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int u = grp; u < total && ok; u += ngrp) {
        const Unit un = unit_at(p, u);
        const int m0 = un.m0 + (int)rank * BM, n0 = un.n0 + (int)rank * 128;   // this CTA's rows of A and of B
        for (int st = un.st_lo; st < un.st_hi; ++st, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES && !mbar_wait(smem_u32(&empty[s]), ((it / STAGES) & 1) ^ 1, abort_flag, p.err, 41)) {
            ok = false;
            break;
          }
          uint8_t* sp = smem + s * kStageBytes;
          uint32_t fb = smem_u32(&full[s]);
          if (rank == 0) mbar_expect_tx(fb, 2 * kStageBytes);   // this CTA's and rank 1's copies
          fb = cluster_addr(fb, 0);
          const int ka = (int)p.a_k0 + st * BK, kb = (int)p.b_k0 + st * BK;
          // K-major boxes are 64 (K) x 128 rows, grouped ones 64 x 1 group x 128 rows; MN-major
          // boxes 64 columns x 64 (K) x 2 column chunks
          const int a0 = p.a_mn || p.a_grouped ? 0 : ka;
          const int a1 = p.a_mn ? ka : p.a_grouped ? ka >> 6 : m0;
          const int a2 = p.a_mn ? m0 >> 6 : p.a_grouped ? m0 : 0;
          const int b0 = p.b_mn ? 0 : kb, b1 = p.b_mn ? kb : n0, b2 = p.b_mn ? n0 >> 6 : 0;
          tma_load_3d_pair(smem_u32(sp), &mAh, fb, a0, a1, a2);
          tma_load_3d_pair(smem_u32(sp + kTile), &mAl, fb, a0, a1, a2);
          tma_load_3d_pair(smem_u32(sp + 2 * kTile), &mBh, fb, b0, b1, b2);
          tma_load_3d_pair(smem_u32(sp + 3 * kTile), &mBl, fb, b0, b1, b2);
        }
      }
      if (*abort_flag) {
        // Every issued copy must land before the CTA exits.  The pair's copies
        // count on rank 0's barriers: rank 0 waits for its stages (bounded),
        // rank 1, which cannot observe its own, waits a fixed 200 us.
        const uint64_t t0 = gtimer();
        if (rank != 0) {
          while (gtimer() - t0 < 200000ull) {}
        } else {
          for (uint32_t q = it > (uint32_t)STAGES ? it - STAGES : 0; q < it; ++q)
            while (!mbar_try(smem_u32(&full[q % STAGES]), (q / STAGES) & 1) && gtimer() - t0 < kWaitNs) {}
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (rank 0) ----------------
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_f16(p.a_mn, p.b_mn);
      const uint32_t s0 = smem_u32(smem);
      // descriptors of stage 0; a stage or k-step adds (bytes / 16) to the address field
      const uint64_t da0 = desc_of(s0, p.a_mn), db0 = desc_of(s0 + 2 * kTile, p.b_mn);
      const uint32_t ka = p.a_mn ? 2048 / 16 : 32 / 16, kb = p.b_mn ? 2048 / 16 : 32 / 16;
      constexpr uint32_t kLo = kTile / 16, kStage16 = kStageBytes / 16;
      uint32_t it = 0, chunk = 0;
      bool ok = true, issued = false;
      for (int u = grp; u < total && ok; u += ngrp) {
        const Unit un = unit_at(p, u);
        for (int st = un.st_lo; st < un.st_hi && ok; st += p.chunk, ++chunk) {
          const uint32_t b = chunk & 1, v = chunk >> 1;
          if (v >= 1 && !mbar_wait_cluster(smem_u32(&acce[b]), (v - 1) & 1, abort_flag, p.err, 44)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t dacc = tmem + b * BN;
          const int end = min(st + p.chunk, un.st_hi);
          for (int q = st; q < end; ++q, ++it) {
            const int s = it % STAGES;
            if (!mbar_wait(smem_u32(&full[s]), (it / STAGES) & 1, abort_flag, p.err, 42)) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t ah = da0 + (uint64_t)(s * kStage16), bh = db0 + (uint64_t)(s * kStage16);
            const uint64_t al = ah + kLo, bl = bh + kLo;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              mma_f16_pair(dacc, al + k * ka, bh + k * kb, idesc, q > st || k > 0 ? 1u : 0u);
              mma_f16_pair(dacc, ah + k * ka, bl + k * kb, idesc, 1u);
            }
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) mma_f16_pair(dacc, ah + k * ka, bh + k * kb, idesc, 1u);
            issued = true;
            mma_commit_pair_both(smem_u32(&empty[s]));   // frees the stage in both CTAs
          }
          if (ok) mma_commit_pair_both(smem_u32(&accf[b]));
        }
      }
      if (issued) {
        // no MMA or commit of this pair may be in flight past the closing cluster barrier
        mma_commit_pair(smem_u32(drain));
        const uint64_t t0 = gtimer();
        while (!mbar_try(smem_u32(drain), 0) && gtimer() - t0 < kWaitNs) {}
      }
      if (!ok) *abort_flag = 1;
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // ---------------- epilogue ----------------
    // Warp w owns lane quarter w % 4 (32 rows, one per lane) and kCols of the
    // tile's columns.
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part * kCols);
    uint8_t* stage = smem + STAGES * kStageBytes + (warp - 4) * kStaging;
    const float alpha = p.inv_all * (p.count ? 1.0f / (float)max(1, *p.count) : 1.0f);
    uint32_t chunk = 0;
    bool ok = true;
    for (int u = grp; u < total && ok; u += ngrp) {
      const Unit un = unit_at(p, u);
      const int m0 = un.m0 + (int)rank * BM + quarter * 32, n0 = un.n0 + part * kCols;
      // the scales, on their way while the sums come in (b's are padded to whole tiles)
      const float sa = alpha * (p.a_inv && m0 + lane < p.M ? p.a_inv[m0 + lane] : 1.0f);
      const float4 sb4 = p.b_inv ? *reinterpret_cast<const float4*>(p.b_inv + n0 + 4 * lane)
                                 : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      float acc[kCols];
      for (int st = un.st_lo; st < un.st_hi; st += p.chunk, ++chunk) {
        const uint32_t b = chunk & 1;
        // the chunk's scales, on their way while its sums come in
        const float* block = MODE == kByM || MODE == kByN
                                 ? p.block_inv + (int64_t)(st / (kF16Block / BK)) * p.block_pitch : nullptr;
        const float bm = MODE == kByM ? block[m0 + lane] : 1.0f;
        const float4 bn = MODE == kByN ? *reinterpret_cast<const float4*>(block + n0 + 4 * lane)
                                       : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (!mbar_wait(smem_u32(&accf[b]), (chunk >> 1) & 1, abort_flag, p.err, 43)) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const bool first = st == un.st_lo;
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
          uint32_t r[32];
          tmem_ld32(tbase + b * BN + c, r);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            float4 s = make_float4(bm, bm, bm, bm);
            if (MODE == kByN) s = scale4(make_float4(1.0f, 1.0f, 1.0f, 1.0f), 1.0f, bn, (c + j) / 4);
            float* a = acc + c + j;
            a[0] = fmaf(__uint_as_float(r[j]), s.x, first ? 0.0f : a[0]);
            a[1] = fmaf(__uint_as_float(r[j + 1]), s.y, first ? 0.0f : a[1]);
            a[2] = fmaf(__uint_as_float(r[j + 2]), s.z, first ? 0.0f : a[2]);
            a[3] = fmaf(__uint_as_float(r[j + 3]), s.w, first ? 0.0f : a[3]);
          }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_u32(&acce[b]), 0));
      }
      if (!ok) break;
      if (MODE == kLse || MODE == kBoth) finish_lse(p, acc, m0 + lane, n0, sa, sb4);
      if (MODE == kBoth) __syncwarp();
      if (MODE != kLse) finish_store<MODE == kBoth>(p, &mOut, un, acc, m0, n0, sa, sb4, stage);
      __syncwarp();   // rows past M return early: the next tensor memory load needs the whole warp
    }
    if (MODE != kLse && lane == 0) bulk_wait<0>();   // every copy is done before the CTA exits
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(done));
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  __syncthreads();
  // rank 0 has drained its MMAs and both CTAs' epilogues and copies are done
  // before either frees its tensor memory or exits
  cluster_sync_all();
  if (warp == 1) {
    mbar_wait_bounded(smem_u32(done), 0);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// out = sum over the K slices, in slice order, of ws[s][m][n] (row pitch ldw, a
// multiple of 4); a block takes 1024 columns of a row
template <bool VEC>
__global__ void __launch_bounds__(256) k_f16_join(const float* __restrict__ ws, int splits, int64_t sstride, int N,
                                                  int64_t ldw, float* __restrict__ out, int64_t ldo, int accumulate) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= N) return;
  const float* p = ws + (int64_t)blockIdx.y * ldw + n;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(p + k * sstride);
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  float* o = out + (int64_t)blockIdx.y * ldo + n;
  if (VEC && n + 4 <= N) {
    float4* q = reinterpret_cast<float4*>(o);
    if (accumulate) {
      const float4 w = *q;
      s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
    }
    *q = s;
    return;
  }
  const float x[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < N) o[i] = accumulate ? o[i] + x[i] : x[i];
}

// ------------------------------------------------------------------ planes
// One row per group of G threads (a warp, or a block of 512).
template <int G, bool VEC>
__global__ void __launch_bounds__(G == 32 ? 256 : G) k_split_rows(const float* __restrict__ src, int64_t R, int64_t C,
                                                                  int64_t Cp, __half* __restrict__ hi,
                                                                  __half* __restrict__ lo, float* __restrict__ inv) {
  __shared__ uint32_t sh[G / 32];
  constexpr int PER = G == 32 ? 8 : 1;
  const int t = threadIdx.x % G;
  for (int64_t r = (int64_t)blockIdx.x * PER + threadIdx.x / G; r < R; r += (int64_t)gridDim.x * PER) {
    const float* s = src + r * C;
    uint32_t m = 0;
    if (VEC) {
      for (int64_t c = 4 * t; c < C; c += 4 * G) {
        const float4 v = *reinterpret_cast<const float4*>(s + c);
        m = max(m, max(max(f16_finite_bits(v.x), f16_finite_bits(v.y)), max(f16_finite_bits(v.z), f16_finite_bits(v.w))));
      }
    } else {
      for (int64_t c = t; c < C; c += G) m = max(m, f16_finite_bits(s[c]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (G > 32) {
      if ((t & 31) == 0) sh[t >> 5] = m;
      __syncthreads();
      for (int i = 0; i < G / 32; ++i) m = max(m, sh[i]);
      __syncthreads();
    }
    float up, iv;
    f16_scale(m, &up, &iv);
    if (t == 0) inv[r] = iv;
    __half *hr = hi + r * Cp, *lr = lo + r * Cp;
    for (int64_t c = 4 * t; c < Cp; c += 4 * G) {
      float v[4];
      if (VEC && c < C) {
        const float4 q = *reinterpret_cast<const float4*>(s + c);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < C ? s[c + j] : 0.0f;
      }
      __align__(8) __half h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f16_split(v[j] * up, &h[j], &l[j]);
      *reinterpret_cast<uint2*>(hr + c) = *reinterpret_cast<uint2*>(h);
      *reinterpret_cast<uint2*>(lr + c) = *reinterpret_cast<uint2*>(l);
    }
  }
}

// Whether row r is kept; loaded beside the row, not before it.  err: where to report
// an id at or past the limit.
__device__ __forceinline__ bool kept(const void* keep, int dt, int64_t limit, int64_t r, int32_t* err = nullptr) {
  if (!keep) return true;
  const int64_t t = dt == MALUS_I64 ? ((const int64_t*)keep)[r] : (int64_t)((const int32_t*)keep)[r];
  if (err && t >= limit) atomicExch(err, 4);
  return t >= 0 && t < limit;
}

// Up to two matrices of C columns split in one launch: their blocks follow one another.
struct SplitJobs {
  F16Split j[2];
  uint32_t* bits[2];
  int blocks[2];
  int* count;       // kept rows of the first (null: not wanted)
  int32_t* err;
};

// Rows of up to 1024 columns (C a multiple of 4, aligned), a warp each, held in
// registers: their planes and, for the planes of the columns, the columns' largest
// finite magnitudes over the kept rows (as bits, zeroed before), in the same pass.
template <int NV>
__global__ void __launch_bounds__(512, 1) k_split_rows_max(const SplitJobs jobs, int C, int Cp) {
  extern __shared__ uint32_t sh[];   // [16][128 NV]
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int which = (int)blockIdx.x >= jobs.blocks[0], block = (int)blockIdx.x - (which ? jobs.blocks[0] : 0);
  const F16Split& job = jobs.j[which];
  const float* __restrict__ src = job.src;
  const int64_t R = job.R, limit = job.limit;
  __half* __restrict__ hi = job.rhi;
  __half* __restrict__ lo = job.rlo;
  float* __restrict__ inv = job.rinv;
  uint32_t* __restrict__ bits = jobs.bits[which];
  const void* keep = job.keep;
  const int kdt = job.keep_dtype;
  int rows_kept = 0;
  uint32_t cm[4 * NV] = {};
  float4 next[NV];
  bool next_in = false;
  auto fetch = [&](int64_t r) {   // a row ahead
    const float4* p = reinterpret_cast<const float4*>(src + r * C);
#pragma unroll
    for (int k = 0; k < NV; ++k) next[k] = 4 * (k * 32 + lane) < C ? p[k * 32 + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    next_in = kept(keep, kdt, limit, r, lane == 0 ? jobs.err : nullptr);
  };
  const int64_t step = (int64_t)jobs.blocks[which] * 16;
  int64_t r = (int64_t)block * 16 + g;
  if (r < R) fetch(r);
  for (; r < R; r += step) {
    rows_kept += next_in;
    float v[4 * NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      v[4 * k] = next[k].x; v[4 * k + 1] = next[k].y; v[4 * k + 2] = next[k].z; v[4 * k + 3] = next[k].w;
    }
    const bool in = next_in;
    if (r + step < R) fetch(r + step);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4 * NV; ++k) {
      const uint32_t b = f16_finite_bits(v[k]);
      m = max(m, b);
      cm[k] = max(cm[k], in ? b : 0u);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    float up, iv;
    f16_scale(m, &up, &iv);
    if (lane == 0) inv[r] = iv;
    __half *hr = hi + r * Cp, *lr = lo + r * Cp;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = 4 * (k * 32 + lane);
      if (i < Cp) {
        __align__(8) __half h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f16_split(v[4 * k + j] * up, &h[j], &l[j]);
        *reinterpret_cast<uint2*>(hr + i) = *reinterpret_cast<uint2*>(h);
        *reinterpret_cast<uint2*>(lr + i) = *reinterpret_cast<uint2*>(l);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4 * NV; ++k) sh[g * 128 * NV + k * 32 + lane] = cm[k];
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * NV; i += 512) {
    uint32_t a = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) a = max(a, sh[k * 128 * NV + i]);
    // slot i: lane i % 32, its element i / 32 (group i / 128, component i / 32 % 4)
    const int c = 4 * (i / 128 * 32 + (i & 31)) + (i >> 5 & 3);
    if (c < C && a) atomicMax(bits + c, a);
  }
  if (which == 0 && jobs.count && lane == 0 && rows_kept) atomicAdd(jobs.count, rows_kept);
}

// bits[c] = largest finite magnitude of column c (as bits; zeroed before): 32 x W
// columns per block, 8 warps on every 8th row, a slice of rows per blockIdx.y
template <int W>
__global__ void __launch_bounds__(256) k_col_max(const float* __restrict__ src, int64_t R, int64_t C,
                                                 uint32_t* __restrict__ bits, const void* keep, int kdt, int64_t limit) {
  __shared__ uint32_t sh[8][32 * W];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + lane) * W;
  uint32_t m[W] = {};
  if (c < C) {
    const int64_t step = (int64_t)gridDim.y * 8;
    for (int64_t r = (int64_t)blockIdx.y * 8 + g; r < R; r += 8 * step) {
      float v[8][W];
      bool k[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // all in flight; past the end: the first one again
        const int64_t q = r + i * step < R ? r + i * step : r;
        const float* p = src + q * C + c;
        if constexpr (W == 4) {
          const float4 f = *reinterpret_cast<const float4*>(p);
          v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w;
        } else {
          v[i][0] = *p;
        }
        k[i] = kept(keep, kdt, limit, q);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) m[j] = max(m[j], k[i] ? f16_finite_bits(v[i][j]) : 0u);
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) sh[g][j * 32 + lane] = m[j];
  __syncthreads();
  if (threadIdx.x < 32 * W) {
    uint32_t a = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) a = max(a, sh[k][threadIdx.x]);
    const int64_t col = ((int64_t)blockIdx.x * 32 + lane) * W + g;
    if (col < C) atomicMax(bits + col, a);   // a maximum: the order does not matter
  }
}

// 64 x 64 tiles through shared memory: rows of the source in (16-byte groups when
// VEC), columns out, 4 rows (8 bytes of a plane) per lane.
template <bool VEC>
__global__ void __launch_bounds__(256) k_split_cols(const SplitJobs jobs, int64_t C) {
  __shared__ float tile[64][65];
  __shared__ float ups[64];
  __shared__ uint32_t rows_kept[2];
  // blocks[i] tiles of 64 rows each, 64-column tiles side by side
  const int ct = (int)((C + 63) / 64);
  const int64_t c0 = (int64_t)(blockIdx.x % ct) * 64;
  int rt = (int)(blockIdx.x / ct);
  const int which = rt >= jobs.blocks[0];
  if (which) rt -= jobs.blocks[0];
  const F16Split& job = jobs.j[which];
  const float* __restrict__ src = job.src;
  const uint32_t* __restrict__ bits = jobs.bits[which];
  const int64_t R = job.R, Rp = pad64(R), r0 = (int64_t)rt * 64;
  const int nr = (int)min((int64_t)64, R - r0), nc = (int)min((int64_t)64, C - c0), t = threadIdx.x;
  const float* p = src + r0 * C + c0;
  constexpr int kStep = VEC ? 16 : 4;                     // rows between a thread's
  const int tx = VEC ? (t & 15) * 4 : t & 63, ty = VEC ? t >> 4 : t >> 6;
  float v[16];
  if (VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 q = ty + 16 * i < nr && tx < nc ? *reinterpret_cast<const float4*>(p + (int64_t)(ty + 16 * i) * C + tx)
                                                   : make_float4(0.f, 0.f, 0.f, 0.f);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  } else {
    const float* q = p + (int64_t)ty * C + tx;
#pragma unroll
    for (int i = 0; i < 16; ++i, q += 4 * C) v[i] = ty + 4 * i < nr && tx < nc ? *q : 0.0f;
  }
  if (t < 64) {
    const bool k = t < nr && kept(job.keep, job.keep_dtype, job.limit, r0 + t, jobs.count && c0 == 0 ? jobs.err : nullptr);
    const uint32_t b = __ballot_sync(0xffffffffu, k);
    if ((t & 31) == 0) {
      rows_kept[t >> 5] = b;
      if (which == 0 && jobs.count && c0 == 0 && b) atomicAdd(jobs.count, __popc(b));
    }
    float up = 1.0f, iv = 1.0f;
    if (t < nc) f16_scale(bits[c0 + t], &up, &iv);
    ups[t] = up;
    if (rt == 0 && t < nc) job.cinv[c0 + t] = iv;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) tile[ty + kStep * (VEC ? i >> 2 : i)][tx + (VEC ? i & 3 : 0)] = v[i];
  __syncthreads();
  const int r = (t & 15) * 4;
  const uint32_t k4 = rows_kept[r >> 5] >> (r & 31);
  __half* h0 = job.chi + c0 * Rp + r0 + r;
  __half* l0 = job.clo + c0 * Rp + r0 + r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (t >> 4) + 16 * i;
    if (c >= nc) break;
    const float up = ups[c];
    __align__(8) __half h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) f16_split(k4 >> k & 1 ? tile[r + k][c] * up : 0.0f, &h[k], &l[k]);
    *reinterpret_cast<uint2*>(h0 + c * Rp) = *reinterpret_cast<uint2*>(h);
    *reinterpret_cast<uint2*>(l0 + c * Rp) = *reinterpret_cast<uint2*>(l);
  }
}

// ------------------------------------------------------------------ launch
CUtensorMap map_of(const F16Operand& o, const __half* plane) {
  const uint64_t pb = (uint64_t)o.pitch * 2;
  if (o.mn_major) {
    const uint64_t dims[3] = {64, (uint64_t)o.rows, (uint64_t)(o.cols + 63) / 64};
    const uint64_t st[2] = {pb, (uint64_t)(o.grouped ? 256 : 128)};
    const uint32_t box[3] = {64, BK, 2};
    return encode_f16_map(3, plane, dims, st, box);
  }
  if (o.grouped) {
    const uint64_t dims[3] = {64, (uint64_t)(o.cols + 63) / 64, (uint64_t)o.rows}, st[2] = {256, pb};
    const uint32_t box[3] = {64, 1, 128};
    return encode_f16_map(3, plane, dims, st, box);
  }
  const uint64_t dims[3] = {(uint64_t)o.cols, (uint64_t)o.rows, 1}, st[2] = {pb, pb * (uint64_t)o.rows};
  const uint32_t box[3] = {BK, 128, 1};
  return encode_f16_map(3, plane, dims, st, box);
}

template <int MODE>
cudaLaunchConfig_t config(int grid, cudaLaunchAttribute* at) {
  static const bool ready = [] {   // once, whichever thread comes first
    MALUS_CUDA(cudaFuncSetAttribute(k_gemm_f16<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    // the register split draws on what the launch reserves: fewer would wait forever
    cudaFuncAttributes fa;
    MALUS_CUDA(cudaFuncGetAttributes(&fa, k_gemm_f16<MODE>));
    if (fa.numRegs < kRegsLaunch) panic("gemm_f16: %d registers per thread at launch, %d needed", fa.numRegs, kRegsLaunch);
    return true;
  }();
  (void)ready;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream();
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cfg;
}

// Pairs resident at once: one per TPC, fewer where the device places fewer.
int max_pairs() {
  static int n = [] {
    cudaLaunchAttribute at[1];
    cudaLaunchConfig_t cfg = config<kStore>(kNumSMs, at);
    int c = 0;
    MALUS_CUDA(cudaOccupancyMaxActiveClusters(&c, k_gemm_f16<kStore>, &cfg));
    if (c < 1) panic("gemm_f16: no CTA pair can be resident");
    return std::min(c, kNumSMs / 2);
  }();
  return n;
}

// out: [splits][M][N], rows ldo floats apart (a multiple of 4, 16-byte aligned
// base), slices sstride; null in kLse mode.
template <int MODE>
void launch(const F16Gemm& g, Params& p, float* out, int64_t ldo, int64_t sstride) {
  p.M = g.M; p.N = g.N; p.K = g.K;
  p.tiles_m = (g.M + 2 * BM - 1) / (2 * BM);
  p.tiles_n = (g.N + BN - 1) / BN;
  p.inner_m = p.tiles_m <= p.tiles_n;
  p.a_mn = g.a.mn_major; p.b_mn = g.b.mn_major;
  p.a_grouped = g.a.grouped;
  p.a_k0 = g.a.k0; p.b_k0 = g.b.k0;
  p.a_inv = g.a.inv; p.b_inv = g.b.inv;
  p.inv_all = (g.a.inv ? 1.0f : g.a.inv_all) * (g.b.inv ? 1.0f : g.b.inv_all);
  p.err = device_error_word();
  const int units = p.tiles_m * p.tiles_n * p.splits;
  // half the chain where it costs little (16384 x 384 x 65, three products: 59 us, 57
  // with 4; 2048 x 768 x 50304: 360 us with 4, 418 with 2)
  p.chunk = units <= max_pairs() && (p.nst + p.splits - 1) / p.splits <= kShortUnit ? kShortChunk : kChunk;
  // a chunk lies within one block of scales
  p.align = MODE == kByM || MODE == kByN ? p.chunk : 1;
  cudaLaunchAttribute at[1];
  cudaLaunchConfig_t cfg = config<MODE>(2 * std::min(units, max_pairs()), at);
  CUtensorMap mo = {};
  if (MODE != kLse) {
    const uint64_t dims[3] = {(uint64_t)g.N, (uint64_t)g.M, (uint64_t)p.splits};
    const uint64_t st[2] = {(uint64_t)ldo * 4, (uint64_t)sstride * 4};
    const uint32_t box[3] = {32, 32, 1};
    mo = encode_f32_map(3, out, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const int pid = prof_begin(0, 2.0 * g.M * (double)g.N * g.K,
                             4.0 * ((double)g.M * g.K + (double)g.N * g.K) + 4.0 * (double)g.M * g.N);
  MALUS_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_f16<MODE>, map_of(g.a, g.a.hi), map_of(g.a, g.a.lo), map_of(g.b, g.b.hi),
                                map_of(g.b, g.b.lo), mo, p));
  count_launch();
  after_launch("k_gemm_f16");
  prof_end(pid);
}

// K slices: the count with the least time in stages of the longest-working pair
// (a slice costs about 4 stages of its own: the pipeline's fill, its store and
// its part of the join).
int splits_for(int tiles, int nst, int pairs) {
  int best = 1;
  double best_t = 1e30;
  for (int s = 1; s <= 64 && s * 4 <= std::max(4, nst); ++s) {
    const double waves = (double)(((int64_t)tiles * s + pairs - 1) / pairs);
    const double t = waves * ((double)((nst + s - 1) / s) + 4.0) + (s > 1 ? 4.0 + 0.25 * s : 0.0);
    if (t < best_t) { best_t = t; best = s; }
  }
  return best;
}

}  // namespace

static void launch_store(const F16Gemm& g, Params& p, float* out, int64_t ldo, int64_t sstride) {
  static_assert(kF16Block % (kChunk * BK) == 0 && kChunk % kShortChunk == 0, "a chunk crosses no block of scales");
  const F16Operand& s = g.a.block_inv ? g.a : g.b;
  p.block_inv = s.block_inv;
  p.block_pitch = s.block_pitch;
  if (g.a.block_inv) launch<kByM>(g, p, out, ldo, sstride);
  else if (g.b.block_inv) launch<kByN>(g, p, out, ldo, sstride);
  else launch<kStore>(g, p, out, ldo, sstride);
}

void gemm_f16(const F16Gemm& g) {
  if (g.M <= 0 || g.N <= 0) return;
  if (g.K <= 0) panic("gemm_f16 with K = %d", g.K);
  Params p{};
  p.nst = (g.K + BK - 1) / BK;
  const int tiles = ((g.M + 2 * BM - 1) / (2 * BM)) * ((g.N + BN - 1) / BN);
  p.splits = splits_for(tiles, p.nst, max_pairs());
  p.count = g.count;
  if (p.splits == 1 && g.ldo % 4 == 0 && ((uintptr_t)g.out & 15) == 0) {
    p.accumulate = g.accumulate;
    launch_store(g, p, g.out, g.ldo, (int64_t)g.M * g.ldo);
    return;
  }
  // K slices, or rows that a TMA store cannot address: through a workspace
  const int64_t ldw = ((int64_t)g.N + 3) / 4 * 4, sstride = (int64_t)g.M * ldw;
  float* ws = static_cast<float*>(scratch_alloc((size_t)sstride * p.splits * 4));
  launch_store(g, p, ws, ldw, sstride);
  const unsigned gx = (unsigned)((g.N + 1023) / 1024);
  for (int m0 = 0; m0 < g.M; m0 += 65535) {
    const dim3 grid(gx, (unsigned)std::min(65535, g.M - m0));
    float* o = g.out + (int64_t)m0 * g.ldo;
    const float* w = ws + (int64_t)m0 * ldw;
    if (g.ldo % 4 == 0 && ((uintptr_t)g.out & 15) == 0)
      k_f16_join<true><<<grid, 256, 0, stream()>>>(w, p.splits, sstride, g.N, ldw, o, g.ldo, g.accumulate);
    else k_f16_join<false><<<grid, 256, 0, stream()>>>(w, p.splits, sstride, g.N, ldw, o, g.ldo, g.accumulate);
    count_launch();
  }
  after_launch("k_f16_join");
  scratch_free(ws);
}

int f16_lse_parts(int N) { return BN / kCols * ((N + BN - 1) / BN); }

void gemm_f16_lse(const F16Gemm& g, float2* part, float* at, const void* target, int tgt_dtype) {
  if (g.M <= 0) return;
  Params p{};
  p.nst = (g.K + BK - 1) / BK;
  p.splits = 1;
  p.part = part;
  p.at = at;
  p.target = target;
  p.tdt = tgt_dtype;
  if (g.out) launch<kBoth>(g, p, g.out, g.ldo, (int64_t)g.M * g.ldo);
  else launch<kLse>(g, p, nullptr, 0, 0);
}

void f16_split_rows(const float* src, int64_t R, int64_t C, __half* hi, __half* lo, float* inv) {
  if (R == 0) return;
  const bool vec = C % 4 == 0 && ((uintptr_t)src & 15) == 0;
  const int64_t Cp = pad64(C);
  const int pid = prof_begin(1, 0.0, 8.0 * (double)R * (double)C);
  // a warp per row up to 4096 columns, which its second pass finds in L1
  if (C <= 4096) {
    const unsigned grid = (unsigned)std::min<int64_t>((R + 7) / 8, kNumSMs * 8);
    if (vec) k_split_rows<32, true><<<grid, 256, 0, stream()>>>(src, R, C, Cp, hi, lo, inv);
    else k_split_rows<32, false><<<grid, 256, 0, stream()>>>(src, R, C, Cp, hi, lo, inv);
  } else {
    const unsigned grid = (unsigned)std::min<int64_t>(R, kNumSMs * 4);
    if (vec) k_split_rows<512, true><<<grid, 512, 0, stream()>>>(src, R, C, Cp, hi, lo, inv);
    else k_split_rows<512, false><<<grid, 512, 0, stream()>>>(src, R, C, Cp, hi, lo, inv);
  }
  count_launch();
  after_launch("k_split_rows");
  prof_end(pid);
}

namespace {

void col_max(const float* src, int64_t R, int64_t C, uint32_t* bits, const void* keep, int keep_dtype, int64_t limit) {
  const bool vec = C % 4 == 0 && ((uintptr_t)src & 15) == 0;
  const int64_t cb = vec ? (C + 127) / 128 : (C + 31) / 32;
  const unsigned ry = (unsigned)std::max<int64_t>(1, std::min<int64_t>((R + 63) / 64, kNumSMs * 4 / cb));   // one wave
  if (vec) k_col_max<4><<<dim3((unsigned)cb, ry), 256, 0, stream()>>>(src, R, C, bits, keep, keep_dtype, limit);
  else k_col_max<1><<<dim3((unsigned)cb, ry), 256, 0, stream()>>>(src, R, C, bits, keep, keep_dtype, limit);
  count_launch();
  after_launch("k_col_max");
}

void split_cols(SplitJobs jobs, int n, int64_t C, bool vec) {
  int64_t tiles = 0;
  for (int i = 0; i < 2; ++i) {
    jobs.blocks[i] = i < n ? (int)(pad64(jobs.j[i].R) / 64) : 0;
    tiles += jobs.blocks[i];
  }
  const int64_t blocks = tiles * ((C + 63) / 64);
  if (blocks > INT32_MAX) panic("f16_split: %lld tiles", (long long)blocks);
  if (vec) k_split_cols<true><<<(unsigned)blocks, 256, 0, stream()>>>(jobs, C);
  else k_split_cols<false><<<(unsigned)blocks, 256, 0, stream()>>>(jobs, C);
  count_launch();
  after_launch("k_split_cols");
}

}  // namespace

void f16_split_cols(const F16Split& job, int64_t C, int* count) {
  if (C == 0 || job.R == 0) return;
  const int pid = prof_begin(1, 0.0, 8.0 * (double)job.R * (double)C);
  SplitJobs jobs{};
  jobs.j[0] = job;
  jobs.count = count;
  jobs.err = device_error_word();
  jobs.bits[0] = static_cast<uint32_t*>(scratch_alloc((size_t)C * 4));
  MALUS_CUDA(cudaMemsetAsync(jobs.bits[0], 0, (size_t)C * 4, stream()));
  col_max(job.src, job.R, C, jobs.bits[0], job.keep, job.keep_dtype, job.limit);
  split_cols(jobs, 1, C, C % 4 == 0 && ((uintptr_t)job.src & 15) == 0);
  scratch_free(jobs.bits[0]);
  prof_end(pid);
}

void f16_split_both(const F16Split* job, int n, int64_t C, uint32_t* bits, int* count) {
  // one read for the rows' planes and the columns' maxima where a warp's registers
  // hold a row: 50304 x 768 measured 47 us (the copy rate) against 52 and 33 apart
  bool fit = C <= 1024 && C % 4 == 0;
  double bytes = 0.0;
  for (int i = 0; i < n; ++i) {
    fit = fit && ((uintptr_t)job[i].src & 15) == 0;
    bytes += 16.0 * (double)job[i].R * (double)C;
  }
  if (!fit) {
    for (int i = 0; i < n; ++i) {
      f16_split_rows(job[i].src, job[i].R, C, job[i].rhi, job[i].rlo, job[i].rinv);
      f16_split_cols(job[i], C, i == 0 ? count : nullptr);
    }
    return;
  }
  const int pid = prof_begin(1, 0.0, bytes);
  SplitJobs jobs{};
  jobs.count = count;
  jobs.err = device_error_word();
  // one block per SM over both, by their rows: the maxima meet in one word per column
  double rows = 0.0;
  for (int i = 0; i < n; ++i) rows += (double)job[i].R;
  unsigned grid = 0;
  for (int i = 0; i < n; ++i) {
    jobs.j[i] = job[i];
    jobs.bits[i] = bits + i * C;
    const int64_t most = std::max<int64_t>(1, (int64_t)(kNumSMs * ((double)job[i].R / rows)));
    jobs.blocks[i] = (int)std::min<int64_t>((job[i].R + 15) / 16, most);
    grid += (unsigned)jobs.blocks[i];
  }
  const int Cp = (int)pad64(C), nv = (Cp + 127) / 128;
  auto go = [&](auto kernel, int NV) {
    const int smem = 16 * 128 * NV * 4;
    MALUS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kernel<<<grid, 512, smem, stream()>>>(jobs, (int)C, Cp);
  };
  switch (nv) {
    case 1: go(k_split_rows_max<1>, 1); break;
    case 2: go(k_split_rows_max<2>, 2); break;
    case 3: go(k_split_rows_max<3>, 3); break;
    case 4: go(k_split_rows_max<4>, 4); break;
    case 5: go(k_split_rows_max<5>, 5); break;
    case 6: go(k_split_rows_max<6>, 6); break;
    case 7: go(k_split_rows_max<7>, 7); break;
    default: go(k_split_rows_max<8>, 8); break;
  }
  count_launch();
  after_launch("k_split_rows_max");
  jobs.count = nullptr;   // they are counted
  split_cols(jobs, n, C, true);
  prof_end(pid);
}

}  // namespace malus
