// The head's cross entropy for small problems, where the time of a call is its
// launches: f32 multiply-adds straight from x and weight (no planes), three
// launches in all.
//   1. logits = x W^T into a scratch (and the row counter is cleared)
//   2. rows: nll, and dl = softmax - onehot in place (loss_rows.cu; counts the rows)
//   3. dx and dweight, and the loss, in one grid
// A product's tile belongs to a block; where a product has few tiles and a long K,
// to a cluster of 8 blocks that each take a slice of K and add their tiles up, in
// slice order, through distributed shared memory.
#include "linear_xent.cuh"
#include "loss_rows.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace malus {
namespace {

constexpr int kCluster = 8, kThreads = 256, BK = 32;
// one stage of both operands, [BK][rows + 4] each, for either tile shape
constexpr int kStage = BK * (16 + 4 + 128 + 4);
static_assert(kStage >= BK * (64 + 4 + 64 + 4) && 2 * kStage >= 64 * 64 && 8 * kStage <= 48 * 1024, "shared memory");

// out[m * ldo + n] = sum_k a(m, k) b(n, k), element (i, k) at i * s + k * sk; divided
// by max(1, count[0]) where count is set.
struct Mul {
  const float *a, *b;
  int64_t sam, sak, sbn, sbk;
  int M, N, K;
  float* out;
  int64_t ldo;
  int tiles_n, tiles;
  int narrow;      // 16 x 128 tiles, else 64 x 64
  int split;       // a cluster per tile
  // That operand is x along the tokens, against dl: what is not finite reads as 0.
  // A token that is not counted has dl = 0, whatever its x holds; in one that is,
  // an x that is not finite has made its whole row of dl NaN already.
  int finite_a, finite_b;
};
struct Small {
  Mul m[2];
  int blocks[2];   // of each product, multiples of kCluster
  int* count;
  int clear, use_count;
  float *nll, *loss;   // with loss: one more cluster, whose first block takes the mean
  int64_t n;
};

// This thread's elements of an operand's [ROWS][BK] blocks along K.  Where K is
// contiguous a warp takes 8 of K (32 bytes) of 4 rows, which falls into 32 different
// banks, and the thread's elements are 8 rows apart; else a warp takes 32 rows (16
// of them twice), and the thread's elements lie along K.
template <int ROWS>
struct Walk {
  static constexpr int kPer = ROWS * BK / kThreads, kPitch = ROWS + 4;
  const float* p;
  int64_t step, advance;   // to the thread's next element; to the next block
  int i, k, di, dk, n;
  int at, at_step;         // in shared memory
  bool finite;

  __device__ __forceinline__ Walk(const float* base, int64_t si, int64_t sk, int i0, int rows, int k0, bool finite_only) {
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    const bool kc = sk == 1;
    i = kc ? w / 4 * 4 + lane / 8 : t % ROWS;
    k = kc ? w % 4 * 8 + lane % 8 : t / ROWS;
    di = kc ? 8 : 0;
    dk = kc ? 0 : kThreads / ROWS;
    at = k * kPitch + i;
    at_step = kc ? 8 : dk * kPitch;
    i += i0;
    k += k0;
    n = rows;
    p = base + i * si + k * sk;
    step = kc ? 8 * si : dk * sk;
    advance = BK * sk;
    finite = finite_only;
  }
  __device__ __forceinline__ void fetch(int k1, float (&v)[kPer]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      v[j] = i + j * di < n && k + j * dk < k1 ? p[j * step] : 0.0f;
      if (finite && !isfinite(v[j])) v[j] = 0.0f;
    }
    p += advance;
    k += BK;
  }
  __device__ __forceinline__ void put(float* sh, const float (&v)[kPer]) const {
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh[at + j * at_step] = v[j];
  }
};

// Tile `tile` of product m over K slice [k0, k1): TM x 4 sums per thread, left in
// sh as [BM][BN].  Two stages: while one is multiplied the next one's loads run.
template <int BM, int BN, int TM>
__device__ __forceinline__ void tile_sums(const Mul& m, int tile, int k0, int k1, float* sh) {
  static_assert(BM * BN == kThreads * TM * 4 && BK * (BM + 4 + BN + 4) <= kStage, "tile");
  const int m0 = tile / m.tiles_n * BM, n0 = tile % m.tiles_n * BN;
  const int tx = threadIdx.x % (BN / 4), ty = threadIdx.x / (BN / 4);
  float acc[TM][4] = {};
  Walk<BM> wa(m.a, m.sam, m.sak, m0, m.M, k0, m.finite_a);
  Walk<BN> wb(m.b, m.sbn, m.sbk, n0, m.N, k0, m.finite_b);
  float va[Walk<BM>::kPer], vb[Walk<BN>::kPer];
  wa.fetch(k1, va);
  wb.fetch(k1, vb);
  int stage = 0;
  for (int k = k0; k < k1; k += BK, stage ^= 1) {
    float* as = sh + stage * kStage;
    float* bs = as + BK * (BM + 4);
    wa.put(as, va);
    wb.put(bs, vb);
    __syncthreads();   // also: everyone is done with this stage's last block but one
    if (k + BK < k1) {
      wa.fetch(k1, va);
      wb.fetch(k1, vb);
    }
#pragma unroll
    for (int q = 0; q < BK; ++q) {
      float a[TM];
      if constexpr (TM == 4) *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(as + q * (BM + 4) + ty * 4);
      else *reinterpret_cast<float2*>(a) = *reinterpret_cast<const float2*>(as + q * (BM + 4) + ty * 2);
      const float4 b = *reinterpret_cast<const float4*>(bs + q * (BN + 4) + tx * 4);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        acc[i][0] = fmaf(a[i], b.x, acc[i][0]);
        acc[i][1] = fmaf(a[i], b.y, acc[i][1]);
        acc[i][2] = fmaf(a[i], b.z, acc[i][2]);
        acc[i][3] = fmaf(a[i], b.w, acc[i][3]);
      }
    }
  }
  __syncthreads();   // the operands make room for the sums
#pragma unroll
  for (int i = 0; i < TM; ++i)
    *reinterpret_cast<float4*>(sh + (ty * TM + i) * BN + tx * 4) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
}

// Elements [first, last) of the tile: the sum of the `parts` blocks' tiles, out.
template <int BM, int BN>
__device__ __forceinline__ void tile_out(const Mul& m, int tile, cg::cluster_group& cl, float* sum, int parts, int first,
                                         int last, float f) {
  const int m0 = tile / m.tiles_n * BM, n0 = tile % m.tiles_n * BN;
  for (int e = first + threadIdx.x; e < last; e += kThreads) {
    float v = 0.0f;
    if (parts == 1) {
      v = sum[e];
    } else {
#pragma unroll
      for (int p = 0; p < kCluster; ++p) v += cl.map_shared_rank(sum, p)[e];
    }
    const int r = m0 + e / BN, c = n0 + e % BN;
    if (r < m.M && c < m.N) m.out[r * m.ldo + c] = v * f;
  }
}

__global__ void __launch_bounds__(kThreads) k_head_small(const Small s) {
  __shared__ __align__(16) float sh[2 * kStage];
  __shared__ double red[kThreads / 32];
  cg::cluster_group cl = cg::this_cluster();
  int b = (int)blockIdx.x;
  if (s.clear && b == 0 && threadIdx.x == 0) *s.count = 0;
  if (b >= s.blocks[0] + s.blocks[1]) {   // the loss
    if (b > s.blocks[0] + s.blocks[1]) return;
    double a = 0.0;
    for (int64_t i = threadIdx.x; i < s.n; i += kThreads) a += (double)s.nll[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
      a = 0.0;
      for (int i = 0; i < kThreads / 32; ++i) a += red[i];
      s.loss[0] = (float)(a / (double)max(1, *s.count));
    }
    return;
  }
  const int which = b >= s.blocks[0];
  if (which) b -= s.blocks[0];
  const Mul& m = s.m[which];
  const int rank = b % kCluster, tile = m.split ? b / kCluster : b;
  if (tile >= m.tiles) return;   // with split: the whole cluster
  const int k0 = m.split ? (int)((int64_t)m.K * rank / kCluster) : 0;
  const int k1 = m.split ? (int)((int64_t)m.K * (rank + 1) / kCluster) : m.K;
  const float f = s.use_count ? 1.0f / (float)max(1, *s.count) : 1.0f;
  if (m.narrow) tile_sums<16, 128, 2>(m, tile, k0, k1, sh);
  else tile_sums<64, 64, 4>(m, tile, k0, k1, sh);
  const int size = m.narrow ? 16 * 128 : 64 * 64;
  if (!m.split) {
    __syncthreads();
    if (m.narrow) tile_out<16, 128>(m, tile, cl, sh, 1, 0, size, f);
    else tile_out<64, 64>(m, tile, cl, sh, 1, 0, size, f);
    return;
  }
  cl.sync();
  const int first = size / kCluster * rank, last = first + size / kCluster;
  if (m.narrow) tile_out<16, 128>(m, tile, cl, sh, kCluster, first, last, f);
  else tile_out<64, 64>(m, tile, cl, sh, kCluster, first, last, f);
  cl.sync();   // the others may still read this block's tile
}

// Tile shape and split of a product: narrow tiles for up to 16 rows; a cluster per
// tile where the tiles leave most SMs idle and every slice of K is worth its
// exchange.  Returns its blocks.
int plan(Mul& m) {
  m.narrow = m.M <= 16;
  const int bm = m.narrow ? 16 : 64, bn = m.narrow ? 128 : 64;
  m.tiles_n = (m.N + bn - 1) / bn;
  m.tiles = (m.M + bm - 1) / bm * m.tiles_n;
  m.split = m.tiles < kNumSMs && m.K >= kCluster * BK;
  return m.split ? m.tiles * kCluster : (m.tiles + kCluster - 1) / kCluster * kCluster;
}

void launch(const Small& s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(s.blocks[0] + s.blocks[1] + (s.loss ? kCluster : 0)));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kCluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MALUS_CUDA(cudaLaunchKernelEx(&cfg, k_head_small, s));
  count_launch();
  after_launch("k_head_small");
}

}  // namespace

// Measured against half planes, the whole call: training 128 x 181 x 1586 43 us
// against 93, 256 x 384 x 1000 (9.8e7) 59 against 76, 256 x 768 x 1000 (2.0e8) 83
// against 82; and 100 x 100 x 10000 (1.3e8) 118 against 77, 16384 x 64 x 64 (6.7e7)
// 146 against 78, where a gradient sums over more than its slices can hide.  The
// loss alone sums over D only: 64 x 384 x 2000 (4.9e7) 23 against 33, 256 x 384 x
// 1000 (9.8e7) 30 against 33, 1000 x 384 x 500 (2.0e8) 45 against 33.
bool head_small(int64_t n, int64_t D, int64_t V, bool grad) {
  const double rows = n <= 16 ? 16.0 : (double)((n + 63) / 64 * 64);   // of x, padded to the tile
  const double work = rows * (double)D * (double)V;
  if (n > 16384) return false;
  return grad ? work <= 1.0e8 && std::max(n, V) <= 2560 : work <= 6.0e7;
}

void head_small_run(const float* x, const float* w, const void* tgt, int tdt, bool tied, int64_t n, int64_t D, int64_t V,
                    float* nll, float* loss, float* dx, float* dw) {
  const int64_t ld = (V + 63) / 64 * 64;
  float* logits = static_cast<float*>(scratch_alloc((size_t)(n * ld) * 4 + 16));
  int* count = reinterpret_cast<int*>(logits + n * ld);
  Small s{};
  s.count = count;
  s.n = n;
  s.clear = 1;
  const int N = (int)n, Di = (int)D, Vi = (int)V;
  s.m[0] = Mul{x, w, D, 1, tied ? D : 1, tied ? 1 : V, N, Vi, Di, logits, ld};
  s.blocks[0] = plan(s.m[0]);
  const int pid = prof_begin(2, 2.0 * (double)n * D * V * (1 + (dx ? 1 : 0) + (dw ? 1 : 0)), 0.0);
  launch(s);
  xent_rows_f32(logits, ld, n, V, tgt, tdt, nll, count, dx || dw);
  if (!dx && !dw) {
    loss_mean(nll, n, count, loss);
  } else {
    Small g = s;
    g.clear = 0;
    g.use_count = 1;
    g.nll = nll;
    g.loss = loss;
    g.blocks[0] = g.blocks[1] = 0;
    int i = 0;
    if (dx) {
      g.m[i] = Mul{logits, w, ld, 1, tied ? 1 : V, tied ? D : 1, N, Di, Vi, dx, D};
      g.blocks[i] = plan(g.m[i]);
      ++i;
    }
    if (dw) {
      if (tied) {
        g.m[i] = Mul{logits, x, 1, ld, 1, D, Vi, Di, N, dw, D};
        g.m[i].finite_b = 1;
      } else {
        g.m[i] = Mul{x, logits, 1, D, 1, ld, Di, Vi, N, dw, V};
        g.m[i].finite_a = 1;
      }
      g.blocks[i] = plan(g.m[i]);
    }
    launch(g);
  }
  prof_end(pid);
  scratch_free(logits);
}

}  // namespace malus
