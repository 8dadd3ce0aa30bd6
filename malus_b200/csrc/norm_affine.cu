// Affine layer norm over the last axis, forward and backward:
//
//   mean = sum(x) / D,  rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)
//   xhat = (x - mean) * rstd,  y = xhat * w + b
//   g = dy * w,  dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Bound by HBM: the forward reads x and writes y (8 B per element), the
// backward reads x and dy and writes dx (12 B).  A row stays in registers
// between the passes over it (the variance is the two-pass one, of the
// centred values) up to 8192 elements, held by 8 to 256 threads of a block, so
// each element is read once.  The backward keeps the
// same columns in the same thread for all the rows it walks: dw and db grow in
// registers and leave as one partial row per block, summed in block order
// by a second kernel (no atomics: the same bits every run).
#include "common.cuh"

#include <vector>

namespace malus {
namespace {

// Sum of v over the TPR threads of a row: part of a warp, a warp, or several warps
// of the block, which then meet at a barrier of their own (group grp's).  `sh`
// holds one float per warp and alternates between two banks, so one barrier per
// call is enough.
constexpr int sh_floats(int tpr) { return tpr > 32 ? 256 / 32 : 1; }
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*sh)[sh_floats(TPR)], int& bank) {
  constexpr int W = TPR < 32 ? TPR : 32;
  const int lane = threadIdx.x & 31;
  const unsigned mask = W == 32 ? 0xffffffffu : ((1u << (W & 31)) - 1u) << (lane & ~(W - 1));
#pragma unroll
  for (int o = W / 2; o; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  if constexpr (TPR > 32) {
    const int grp = threadIdx.x / TPR;
    float* s = sh[bank] + grp * (TPR / 32);
    bank ^= 1;
    if (lane == 0) s[(threadIdx.x % TPR) >> 5] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(TPR) : "memory");
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += s[i];
  }
  return v;
}

// Element index of slot (k, j) of thread t of a row: 16-byte groups of 4 when
// VEC, else single elements, consecutive threads side by side in both.
template <int TPR, bool VEC>
__device__ __forceinline__ int col_of(int t, int k, int j) {
  return VEC ? (k * TPR + t) * 4 + j : (k * 4 + j) * TPR + t;
}

template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void load_row(const float* __restrict__ p, int t, int D, float (&v)[NV * 4]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if constexpr (VEC) {
      const int c = col_of<TPR, true>(t, k, 0);
      float4 q = c < D ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[4 * k] = q.x; v[4 * k + 1] = q.y; v[4 * k + 2] = q.z; v[4 * k + 3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = col_of<TPR, false>(t, k, j);
        v[4 * k + j] = c < D ? p[c] : 0.0f;
      }
    }
  }
}

template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void store_row(float* __restrict__ p, int t, int D, const float (&v)[NV * 4]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if constexpr (VEC) {
      const int c = col_of<TPR, true>(t, k, 0);
      if (c < D) *reinterpret_cast<float4*>(p + c) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = col_of<TPR, false>(t, k, j);
        if (c < D) p[c] = v[4 * k + j];
      }
    }
  }
}

constexpr int kBlock = 256;

template <int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(kBlock)
k_norm_fwd(const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
           float* __restrict__ y, float* __restrict__ stats, int64_t rows, int D, float eps) {
  constexpr int BLOCK = kBlock, RPB = BLOCK / TPR;
  __shared__ float sh[2][sh_floats(TPR)];
  int bank = 0;
  const int t = threadIdx.x % TPR;
  const int64_t step = (int64_t)gridDim.x * RPB;
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < rows; r += step) {
    float v[NV * 4];
    load_row<TPR, NV, VEC>(x + r * D, t, D, v);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) s += v[i];
    const float mean = row_sum<TPR>(s, sh, bank) / (float)D;
    float q = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = v[4 * k + j] - mean;
        v[4 * k + j] = d;
        if (col_of<TPR, VEC>(t, k, j) < D) q += d * d;
      }
    const float var = row_sum<TPR>(q, sh, bank) / (float)D;
    const float rstd = 1.0f / sqrtf(var + eps);
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) v[i] *= rstd;
    if (w) {
      float a[NV * 4];
      load_row<TPR, NV, VEC>(w, t, D, a);
#pragma unroll
      for (int i = 0; i < NV * 4; ++i) v[i] *= a[i];
    }
    if (b) {
      float a[NV * 4];
      load_row<TPR, NV, VEC>(b, t, D, a);
#pragma unroll
      for (int i = 0; i < NV * 4; ++i) v[i] += a[i];
    }
    store_row<TPR, NV, VEC>(y + r * D, t, D, v);
    if (stats && t == 0) {
      stats[2 * r] = mean;
      stats[2 * r + 1] = rstd;
    }
  }
}

// part: [gridDim.x][2][D] partial dw and db (null: neither is wanted); dx may be null.
template <int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(kBlock)
k_norm_bwd(const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ stats,
           const float* __restrict__ dy, float* __restrict__ dx, float* __restrict__ part, int64_t rows, int D) {
  constexpr int BLOCK = kBlock, RPB = BLOCK / TPR;
  __shared__ float sh[2][sh_floats(TPR)];
  extern __shared__ float fold[];   // RPB > 1: [RPB][D], the row groups' partial sums
  int bank = 0;
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  float wv[NV * 4], dw[NV * 4], db[NV * 4];
  if (w) {
    load_row<TPR, NV, VEC>(w, t, D, wv);
  } else {
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) wv[i] = 1.0f;
  }
#pragma unroll
  for (int i = 0; i < NV * 4; ++i) dw[i] = db[i] = 0.0f;
  const int64_t step = (int64_t)gridDim.x * RPB;
  for (int64_t r = (int64_t)blockIdx.x * RPB + grp; r < rows; r += step) {
    float v[NV * 4], g[NV * 4];
    load_row<TPR, NV, VEC>(x + r * D, t, D, v);
    load_row<TPR, NV, VEC>(dy + r * D, t, D, g);
    const float mean = stats[2 * r], rstd = stats[2 * r + 1];
    float s = 0.0f, sx = 0.0f;
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) {   // slots past the row have dy = 0: they add nothing
      v[i] = (v[i] - mean) * rstd;
      dw[i] += g[i] * v[i];
      db[i] += g[i];
      g[i] *= wv[i];
      s += g[i];
      sx += g[i] * v[i];
    }
    if (!dx) continue;   // uniform over the grid
    const float ms = row_sum<TPR>(s, sh, bank) / (float)D;
    const float msx = row_sum<TPR>(sx, sh, bank) / (float)D;
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) g[i] = ((g[i] - ms) - v[i] * msx) * rstd;
    store_row<TPR, NV, VEC>(dx + r * D, t, D, g);
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * D;
  if constexpr (RPB == 1) {
    store_row<TPR, NV, VEC>(pw, t, D, dw);
    store_row<TPR, NV, VEC>(pw + D, t, D, db);
  } else {
    for (int q = 0; q < 2; ++q) {
      __syncthreads();
      store_row<TPR, NV, VEC>(fold + (int64_t)grp * D, t, D, q ? db : dw);
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += BLOCK) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < RPB; ++i) s += fold[i * D + c];
        pw[q * D + c] = s;
      }
    }
  }
}

// out[c] = sum over the nb partial rows, in order within each of the 32 groups of
// rows and then over the groups.
__global__ void __launch_bounds__(1024) k_norm_fold(const float* __restrict__ part, int nb, int D,
                                                    float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, W = 2 * (int64_t)D;   // column of the partial row
  float s = 0.0f;
  if (c < W) {
    const int per = (nb + 31) / 32, lo = g * per, hi = min(nb, lo + per);
    for (int i = lo; i < hi; i += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + k < hi ? part[(int64_t)(i + k) * W + c] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  }
  sh[g][lane] = s;
  __syncthreads();
  s = sh[lane][g];   // group `lane` of column g
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t col = (int64_t)blockIdx.x * 32 + g;
  if (lane == 0 && col < W) {
    float* out = col < D ? dw : db;
    if (out) out[col < D ? col : col - D] = s;
  }
}

// Rows longer than a block's registers hold: each pass reads the row again.
__global__ void __launch_bounds__(kBlock) k_norm_fwd_long(const float* __restrict__ x, const float* __restrict__ w,
                                                       const float* __restrict__ b, float* __restrict__ y,
                                                       float* __restrict__ stats, int64_t rows, int64_t D, float eps) {
  __shared__ float sh[2][sh_floats(kBlock)];
  int bank = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* xr = x + r * D;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < D; c += kBlock) s += xr[c];
    const float mean = row_sum<kBlock>(s, sh, bank) / (float)D;
    float q = 0.0f;
    for (int64_t c = threadIdx.x; c < D; c += kBlock) {
      const float d = xr[c] - mean;
      q += d * d;
    }
    const float rstd = 1.0f / sqrtf(row_sum<kBlock>(q, sh, bank) / (float)D + eps);
    for (int64_t c = threadIdx.x; c < D; c += kBlock) {
      float v = (xr[c] - mean) * rstd;
      if (w) v *= w[c];
      if (b) v += b[c];
      y[r * D + c] = v;
    }
    if (stats && threadIdx.x == 0) {
      stats[2 * r] = mean;
      stats[2 * r + 1] = rstd;
    }
  }
}

__global__ void __launch_bounds__(kBlock) k_norm_dx_long(const float* __restrict__ x, const float* __restrict__ w,
                                                      const float* __restrict__ stats, const float* __restrict__ dy,
                                                      float* __restrict__ dx, int64_t rows, int64_t D) {
  __shared__ float sh[2][sh_floats(kBlock)];
  int bank = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float *xr = x + r * D, *gr = dy + r * D;
    const float mean = stats[2 * r], rstd = stats[2 * r + 1];
    float s = 0.0f, sx = 0.0f;
    for (int64_t c = threadIdx.x; c < D; c += kBlock) {
      const float g = gr[c] * (w ? w[c] : 1.0f);
      s += g;
      sx += g * ((xr[c] - mean) * rstd);
    }
    const float ms = row_sum<kBlock>(s, sh, bank) / (float)D;
    const float msx = row_sum<kBlock>(sx, sh, bank) / (float)D;
    for (int64_t c = threadIdx.x; c < D; c += kBlock) {
      const float g = gr[c] * (w ? w[c] : 1.0f);
      dx[r * D + c] = ((g - ms) - (xr[c] - mean) * rstd * msx) * rstd;
    }
  }
}

// Partial dw / db of a slice of rows per blockIdx.y, one column per thread.
__global__ void __launch_bounds__(256) k_norm_dw_long(const float* __restrict__ x, const float* __restrict__ stats,
                                                      const float* __restrict__ dy, float* __restrict__ part,
                                                      int64_t rows, int64_t D) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = dy[r * D + c];
    dw += g * ((x[r * D + c] - stats[2 * r]) * stats[2 * r + 1]);
    db += g;
  }
  part[(int64_t)blockIdx.y * 2 * D + c] = dw;
  part[(int64_t)blockIdx.y * 2 * D + D + c] = db;
}

bool aligned16(std::initializer_list<const void*> ps) {
  uintptr_t a = 0;
  for (const void* p : ps) a |= (uintptr_t)p;
  return (a & 15) == 0;
}

constexpr int kFwdNv = 8, kBwdNv = 4;
constexpr int64_t kMaxRow = 8192;   // longest row held in registers

// Threads per row, and the float4 groups `nv` that each holds.  Few threads for short
// rows (200000 x 96 forward: 29 us with 8 threads a row, 51 with 32), up to `most`
// groups each; a warp up to 1024 elements; beyond, up to 6 groups each (16384 x 1281
// forward: 38 us with 64 threads, 56 with 256; but 8192 x 2048: 32 with 64 threads
// and 8 groups, 27 with 256 and 2) until 256 threads hold 8.
struct RowCfg { int tpr, nv; };
RowCfg row_cfg(int64_t D, int most) {
  int tpr = 8;
  while (tpr < 32 && D > 4 * most * tpr) tpr *= 2;
  if (D > 1024)
    for (tpr = 64; tpr < 256 && D > 4 * 6 * tpr;) tpr *= 2;
  return {tpr, (int)((D + 4 * tpr - 1) / (4 * tpr))};
}

// Whether row_cfg(D, MOST) ever gives NV groups with TPR threads: only those exist.
template <int MOST>
constexpr bool reached(int tpr, int nv) {
  if (tpr == 8) return nv <= MOST;
  if (tpr == 16) return nv > MOST / 2 && nv <= MOST;
  if (tpr == 32) return nv > MOST / 2 && nv <= 8;   // to 1024 elements
  if (tpr == 64) return nv == 5 || nv == 6;         // from 1025 on
  return nv >= 4 && nv <= (tpr == 128 ? 6 : 8);
}
template <int MOST, int TPR, bool VEC, int NV = 1, class F>
void with_nv(int nv, F&& f) {
  if constexpr (NV <= 8) {
    if (nv != NV) return with_nv<MOST, TPR, VEC, NV + 1>(nv, f);
    if constexpr (reached<MOST>(TPR, NV)) return f.template operator()<TPR, NV, VEC>();
  }
  panic("layernorm_affine: no kernel of %d threads per row and %d groups", TPR, nv);
}
template <int MOST, bool VEC, class F>
void with_tpr(RowCfg c, F&& f) {
  switch (c.tpr) {
    case 8: with_nv<MOST, 8, VEC>(c.nv, f); break;
    case 16: with_nv<MOST, 16, VEC>(c.nv, f); break;
    case 32: with_nv<MOST, 32, VEC>(c.nv, f); break;
    case 64: with_nv<MOST, 64, VEC>(c.nv, f); break;
    case 128: with_nv<MOST, 128, VEC>(c.nv, f); break;
    default: with_nv<MOST, 256, VEC>(c.nv, f); break;
  }
}
template <int MOST, class F>
void with_cfg(int64_t D, bool vec, F&& f) {
  if (vec) with_tpr<MOST, true>(row_cfg(D, MOST), f);
  else with_tpr<MOST, false>(row_cfg(D, MOST), f);
}

struct FwdLaunch {
  const float *x, *w, *b;
  float *y, *stats;
  int64_t rows;
  int D;
  float eps;
  template <int TPR, int NV, bool VEC>
  void operator()() const {
    constexpr int BLOCK = kBlock, RPB = BLOCK / TPR;
    const int64_t need = (rows + RPB - 1) / RPB;
    const unsigned grid = (unsigned)std::min<int64_t>(need, (int64_t)kNumSMs * (2048 / BLOCK));
    k_norm_fwd<TPR, NV, VEC><<<grid, BLOCK, 0, stream()>>>(x, w, b, y, stats, rows, D, eps);
  }
};

struct BwdLaunch {
  const float *x, *w, *stats, *dy;
  float *dx, *dw, *db;
  int64_t rows;
  int D;
  template <int TPR, int NV, bool VEC>
  void operator()() const {
    constexpr int BLOCK = kBlock, RPB = BLOCK / TPR;
    const int64_t need = (rows + RPB - 1) / RPB;
    // one resident wave: every block leaves one partial row
    static int per_sm = [] {
      int n = 0;
      MALUS_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k_norm_bwd<TPR, NV, VEC>, BLOCK,
                                                               RPB > 1 ? (size_t)RPB * NV * 4 * TPR * 4 : 0));
      return std::max(1, n);
    }();
    const int grid = (int)std::min<int64_t>(need, (int64_t)kNumSMs * per_sm);
    const size_t smem = RPB > 1 ? (size_t)RPB * D * 4 : 0;
    const bool cols = dw || db;
    float* part = cols ? static_cast<float*>(scratch_alloc((size_t)grid * 2 * D * 4)) : nullptr;
    k_norm_bwd<TPR, NV, VEC><<<grid, BLOCK, smem, stream()>>>(x, w, stats, dy, dx, part, rows, D);
    if (cols) {
      k_norm_fold<<<(2 * D + 31) / 32, 1024, 0, stream()>>>(part, grid, D, dw, db);
      count_launch();
      scratch_free(part);
    }
  }
};

}  // namespace

void norm_affine_fwd(const float* x, const float* w, const float* b, float* y, float* stats, int64_t rows,
                     int64_t D, float eps) {
  if (rows == 0) return;
  const int pid = prof_begin_named("k_norm_fwd", 4.0 * (2.0 * rows * D + 2.0 * D));
  if (D > kMaxRow) {
    k_norm_fwd_long<<<(unsigned)std::min<int64_t>(rows, kNumSMs * 8), kBlock, 0, stream()>>>(x, w, b, y, stats, rows, D,
                                                                                         eps);
  } else {
    const bool vec = D % 4 == 0 && aligned16({x, w, b, y});
    const FwdLaunch f{x, w, b, y, stats, rows, (int)D, eps};
    with_cfg<kFwdNv>(D, vec, f);
  }
  count_launch();
  after_launch("k_norm_fwd");
  prof_end(pid);
}

void norm_affine_bwd(const float* x, const float* w, const float* stats, const float* dy, float* dx, float* dw,
                     float* db, int64_t rows, int64_t D) {
  if (rows == 0) {
    if (dw) MALUS_CUDA(cudaMemsetAsync(dw, 0, D * 4, stream()));
    if (db) MALUS_CUDA(cudaMemsetAsync(db, 0, D * 4, stream()));
    return;
  }
  const int pid = prof_begin_named("k_norm_bwd", 4.0 * ((dx ? 3.0 : 2.0) * rows * D + 3.0 * D));
  if (D > kMaxRow) {
    if (dx) {
      k_norm_dx_long<<<(unsigned)std::min<int64_t>(rows, kNumSMs * 8), kBlock, 0, stream()>>>(x, w, stats, dy, dx, rows, D);
      count_launch();
    }
    if (dw || db) {
      const int nb = (int)std::min<int64_t>(rows, 32);
      float* part = static_cast<float*>(scratch_alloc((size_t)nb * 2 * D * 4));
      k_norm_dw_long<<<dim3((unsigned)((D + 255) / 256), nb), 256, 0, stream()>>>(x, stats, dy, part, rows, D);
      k_norm_fold<<<(unsigned)((2 * D + 31) / 32), 1024, 0, stream()>>>(part, nb, (int)D, dw, db);
      count_launch(2);
      scratch_free(part);
    }
  } else {
    const bool vec = D % 4 == 0 && aligned16({x, w, dy, dx});
    with_cfg<kBwdNv>(D, vec, BwdLaunch{x, w, stats, dy, dx, dw, db, rows, (int)D});
    count_launch();
  }
  after_launch("k_norm_bwd");
  prof_end(pid);
}

}  // namespace malus

using namespace malus;

namespace {

void check_vector(int64_t h, size_t D, const char* what) {
  if (!h) return;
  const auto* t = tb(h);
  if (t->dtype != MALUS_F32) panic("layernorm_affine %s must be f32, got dtype %d", what, t->dtype);
  if (t->ndim != 1 || t->shape[0] != D)
    panic("layernorm_affine %s must have shape [%zu] (x's last axis), got rank %d with %zu elements", what, D, t->ndim,
          t->len);
}

// Rows and width of x seen as [rows, D].
void rows_of(int64_t x, size_t* rows, size_t* D) {
  const auto* t = tb(x);
  if (t->dtype != MALUS_F32) panic("layernorm_affine expects an f32 tensor, got dtype %d", t->dtype);
  if (t->ndim < 1) panic("layernorm_affine needs a tensor of rank 1 or more");
  *D = t->shape[t->ndim - 1];
  if (*D == 0) panic("layernorm_affine over an empty last axis");
  if (*D > (size_t)1 << 30) panic("layernorm_affine last axis of %zu elements (limit 2^30)", *D);
  *rows = t->len / *D;
}

}  // namespace

extern "C" {

int64_t malus_layernorm_affine_fwd(int64_t x, int64_t weight, int64_t bias, float eps, int64_t* stats) {
  size_t rows, D;
  rows_of(x, &rows, &D);
  check_vector(weight, D, "weight");
  check_vector(bias, D, "bias");
  if (!(eps >= 0.0f)) panic("layernorm_affine eps must not be negative, got %g", (double)eps);
  const int64_t y = alloc_shape(shape_of(x));
  const int64_t st = stats ? alloc_f32({rows, 2}) : 0;
  norm_affine_fwd(fptr(x), weight ? fptr(weight) : nullptr, bias ? fptr(bias) : nullptr, fptr(y),
                  st ? fptr(st) : nullptr, (int64_t)rows, (int64_t)D, eps);
  if (stats) *stats = st;
  return y;
}

void malus_layernorm_affine_bwd(int64_t x, int64_t weight, int64_t stats, int64_t dout, int64_t* dx,
                                int64_t* dweight, int64_t* dbias) {
  size_t rows, D;
  rows_of(x, &rows, &D);
  check_vector(weight, D, "weight");
  if (tb(stats)->dtype != MALUS_F32 || tb(stats)->len != 2 * rows)
    panic("layernorm_affine stats must be the [%zu, 2] tensor of the forward pass", rows);
  if (tb(dout)->dtype != MALUS_F32 || !same_shape(x, dout))
    panic("layernorm_affine gradient must be f32 with x's shape");
  const int64_t hx = dx ? alloc_shape(shape_of(x)) : 0;
  const int64_t hw = dweight ? alloc_f32({D}) : 0;
  const int64_t hb = dbias ? alloc_f32({D}) : 0;
  norm_affine_bwd(fptr(x), weight ? fptr(weight) : nullptr, fptr(stats), fptr(dout), hx ? fptr(hx) : nullptr,
                  hw ? fptr(hw) : nullptr, hb ? fptr(hb) : nullptr, (int64_t)rows, (int64_t)D);
  if (dx) *dx = hx;
  if (dweight) *dweight = hw;
  if (dbias) *dbias = hb;
}

}  // extern "C"
