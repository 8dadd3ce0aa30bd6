// LM head and softmax cross entropy in one operator, the logits never kept
// whole:
//
//   logits = x W^T,  nll = logsumexp(logits) - logits[target]
//   dl = (softmax(logits) - onehot(target)) / rows,  dx = dl W,  dW = dl^T x
//
// Training takes the tokens in pieces: a piece's logits become half planes of dl
// (loss_rows.cu), feed both gradient products and make room for the next piece.
// That is the three products (6 N D V flops) and nothing computed twice.  dx and
// dweight each have planes of their own: dx sums over the vocabulary, where one scale
// serves; dweight sums over the tokens, and there each entry's gradients are scaled
// by their own largest, so that the row of a token that is hardly ever predicted is
// as accurate as any other.  A piece holds at most kPieceBytes of logits (or 64 rows
// of them, which is more from V = 2^21 on) and, with both gradients, as much again
// for the second set of planes.  Per logit that is 4 B written and read, then 4 B
// written and read for each product.  In every form the product's epilogue reduces
// each row of a tile to its maximum, sum of exponentials and target logit; the loss
// alone stores no logits.
//
// The loss of a few rows (a token being scored) reads the weight once as it is, with
// f32 multiply-adds: nothing is split, and that one read is what bounds it.
//
// All other products run as three half-precision ones (gemm_f16.cuh).  x and weight
// are split twice, by rows and by columns, so that every product's operands are
// scaled along the axis it does not sum over.
#include "gemm_f16.cuh"
#include "linear_xent.cuh"
#include "loss_rows.cuh"

#include <utility>

namespace malus {
namespace {

constexpr size_t kPieceBytes = (size_t)512 << 20;

// Half planes of an operand, in one scratch block with their scales.
struct Planes {
  __half *hi, *lo;
  float* inv;
  int64_t rows, pitch;
  Planes(int64_t r, int64_t cols) : rows(r), pitch(pad64(cols)) {
    const size_t plane = (size_t)rows * pitch;
    hi = static_cast<__half*>(scratch_alloc(plane * 4 + (size_t)f16_scales(rows) * 4));
    lo = hi + plane;
    inv = reinterpret_cast<float*>(lo + plane);
  }
  ~Planes() { scratch_free(hi); }
  Planes(const Planes&) = delete;
  // rows [r0, r0 + n), read along K from column k0
  F16Operand kmajor(int64_t r0, int64_t n, int64_t k0 = 0) const {
    return {hi + r0 * pitch, lo + r0 * pitch, n, pitch, pitch, false, k0, inv + r0, 1.0f};
  }
};

void train(const float* x, const float* w, const void* tgt, int tdt, bool tied, int64_t n, int64_t D, int64_t V,
           int64_t ld, float* nll, float* loss, float* dx, float* dw) {
  // a token, and a vocabulary entry, per row; then an embedding axis per row, with
  // the tokens that are not counted as zeros: whatever they hold, dl is 0 there
  Planes xr(n, D), wv(V, D), xc(dw ? D : 0, n), wd(dx ? D : 0, V);
  // the row count, and the column maxima of x and of weight
  const size_t words = 4 + (size_t)(D + std::max(D, V));
  int* count = static_cast<int*>(scratch_alloc(words * 4));
  uint32_t* bits = reinterpret_cast<uint32_t*>(count + 4);
  MALUS_CUDA(cudaMemsetAsync(count, 0, words * 4, stream()));
  const F16Split sx{x, n, xr.hi, xr.lo, xr.inv, xc.hi, xc.lo, xc.inv, tgt, tdt, V};
  const F16Split sw = tied ? F16Split{w, V, wv.hi, wv.lo, wv.inv, wd.hi, wd.lo, wd.inv, nullptr, 0, 0}
                           : F16Split{w, D, wd.hi, wd.lo, wd.inv, wv.hi, wv.lo, wv.inv, nullptr, 0, 0};
  if (dw && dx && tied) {
    const F16Split both[2] = {sx, sw};
    f16_split_both(both, 2, D, bits, count);
  } else {
    if (dw) f16_split_both(&sx, 1, D, bits, count);
    else f16_split_rows(x, n, D, xr.hi, xr.lo, xr.inv);
    if (dx) f16_split_both(&sw, 1, tied ? D : V, bits + D, nullptr);
    else if (tied) f16_split_rows(w, V, D, wv.hi, wv.lo, wv.inv);
    else f16_split_cols(sw, V);
  }
  if (!dw) xent_count(tgt, tdt, n, V, count);
  // Pieces of whole 256-row tiles, of even size; of 64 rows (the products' step in K)
  // where 256 do not fit the bound.
  const int64_t fit = (int64_t)(kPieceBytes / ((size_t)ld * 4));
  const int64_t unit = fit >= 256 ? 256 : 64, most = std::max(unit, fit / unit * unit);
  const int64_t pieces = (n + most - 1) / most;
  const int64_t piece = ((n + pieces - 1) / pieces + unit - 1) / unit * unit;
  const size_t rows = (size_t)std::min(piece, n), row_bytes = (size_t)ld * 4;
  float* logits = static_cast<float*>(scratch_alloc(rows * row_bytes));
  __half* over = reinterpret_cast<__half*>(logits);   // planes in place of the logits
  __half* entry = dw ? over : nullptr;
  __half* even = dx && dw ? static_cast<__half*>(scratch_alloc(rows * row_bytes)) : dx ? over : nullptr;
  // the scales of `entry`, and the rows' statistics
  const int parts = f16_lse_parts((int)V);
  const int64_t inv_pitch = f16_scales(ld), inv_rows = ((int64_t)rows + kF16Block - 1) / kF16Block;
  float* inv = static_cast<float*>(scratch_alloc((size_t)(inv_rows * inv_pitch) * 4 + rows * ((size_t)parts * 8 + 4)));
  float2* part = reinterpret_cast<float2*>(inv + inv_rows * inv_pitch);
  float* at = reinterpret_cast<float*>(part + rows * parts);
  for (int64_t r0 = 0; r0 < n; r0 += piece) {
    const int64_t m = std::min(piece, n - r0);
    const void* t = static_cast<const char*>(tgt) + r0 * (int64_t)dtype_size(tdt);
    F16Gemm g{(int)m, (int)V, (int)D, xr.kmajor(r0, m), wv.kmajor(0, V), logits, ld, false, nullptr};
    gemm_f16_lse(g, part, at, t, tdt);
    xent_planes(logits, ld, m, V, {part, parts, at, t, tdt}, nll + r0, even, entry, inv, inv_pitch);
    if (dx) {
      const F16Operand dl{even, even + 64, m, ld, 2 * ld, false, 0, nullptr, 1.0f / (1 << kDlExp), true};
      gemm_f16({(int)m, (int)D, (int)V, dl, wd.kmajor(0, D), dx + r0 * D, D, false, count});
    }
    if (dw) {
      const F16Operand dl{entry, entry + 64, m, ld, 2 * ld, true, 0, nullptr, 1.0f, true, inv, inv_pitch};
      const F16Operand xt = xc.kmajor(0, D, r0);
      if (tied) gemm_f16({(int)V, (int)D, (int)m, dl, xt, dw, D, r0 > 0, count});
      else gemm_f16({(int)D, (int)V, (int)m, xt, dl, dw, V, r0 > 0, count});
    }
  }
  scratch_free(inv);
  if (even != over) scratch_free(even);
  scratch_free(logits);
  loss_mean(nll, n, count, loss);
  scratch_free(count);
}

void loss_only(const float* x, const float* w, const void* tgt, int tdt, bool tied, int64_t n, int64_t D, int64_t V,
               float* nll, float* loss) {
  Planes xr(n, D), wv(V, D);
  f16_split_rows(x, n, D, xr.hi, xr.lo, xr.inv);
  if (tied) f16_split_rows(w, V, D, wv.hi, wv.lo, wv.inv);
  else f16_split_cols(F16Split{w, D, nullptr, nullptr, nullptr, wv.hi, wv.lo, wv.inv, nullptr, 0, 0}, V);
  const int parts = f16_lse_parts((int)V);
  // a piece's statistics (8 B per 128 logits) within the same bound
  const int64_t piece = std::min<int64_t>(n, std::max<int64_t>(256, (int64_t)(kPieceBytes / ((size_t)parts * 8 + 4))));
  float2* part = static_cast<float2*>(scratch_alloc((size_t)piece * (parts * 8 + 4)));
  float* at = reinterpret_cast<float*>(part + piece * parts);
  for (int64_t r0 = 0; r0 < n; r0 += piece) {
    const int64_t m = std::min(piece, n - r0);
    const void* t = static_cast<const char*>(tgt) + r0 * (int64_t)dtype_size(tdt);
    F16Gemm g{(int)m, (int)V, (int)D, xr.kmajor(r0, m), wv.kmajor(0, V), nullptr, 0, false, nullptr};
    gemm_f16_lse(g, part, at, t, tdt);
    xent_join({part, parts, at, t, tdt}, V, m, nll + r0, nullptr);
  }
  scratch_free(part);
  loss_mean_counted(nll, n, tgt, tdt, V, loss);
}

// ------------------------------------------------------------- few rows
constexpr int kFewRows = 8;
constexpr int kFewSmem = 96 * 1024;   // x rows held in shared memory
constexpr int kFewWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;

// Running maximum and sum of exponentials.
struct Run {
  float m = -INFINITY, s = 0.0f;
  __device__ __forceinline__ void add(float z) {
    const float mn = fmaxf(m, z), m0 = mn == -INFINITY ? 0.0f : mn;
    s = s * exp2f((m - m0) * kLog2e) + exp2f((z - m0) * kLog2e);
    m = mn;
  }
  __device__ __forceinline__ void join(float om, float os) {
    const float mn = fmaxf(m, om), m0 = mn == -INFINITY ? 0.0f : mn;
    s = s * exp2f((m - m0) * kLog2e) + os * exp2f((om - m0) * kLog2e);
    m = mn;
  }
};

__device__ __forceinline__ int64_t target_at(const void* t, int dt, int64_t i) {
  return dt == MALUS_I64 ? ((const int64_t*)t)[i] : (int64_t)((const int32_t*)t)[i];
}

// weight [V, D]: a warp takes four vocabulary entries at a time against all N rows
// of x, its lanes along D.  The 4 N sums are reduced by halving: each exchange
// leaves half as many to a lane, until every lane has one logit (or a share of
// it), whose running softmax it keeps.  part: [N][gridDim.x].
template <int N, bool VEC>
__global__ void __launch_bounds__(32 * kFewWarps, N <= 2 ? 4 : 2)
k_head_few_rows(const float* __restrict__ x, const float* __restrict__ w, int n, int D, int V, const void* tgt, int tdt,
                float2* __restrict__ part, float* __restrict__ at) {
  extern __shared__ __align__(16) float xs[];   // [N][Dp], zeros past n and D
  __shared__ float2 sh[kFewWarps][4 * N];
  const int Dp = (D + 127) / 128 * 128, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < N * Dp; i += blockDim.x) {
    const int r = i / Dp, c = i % Dp;
    xs[i] = r < n && c < D ? x[(int64_t)r * D + c] : 0.0f;
  }
  __syncthreads();
  // which of the 4 N logits (entry j, row i at j * N + i) ends in this lane
  int idx = 0, left = 4 * N;
#pragma unroll
  for (int o = 16; o; o >>= 1)
    if (left > 1) {
      left /= 2;
      if (lane & o) idx += left;
    }
  const int my_row = idx % N, my_entry = idx / N;
  const int64_t t = my_row < n ? target_at(tgt, tdt, my_row) : -1;
  Run run;
  const int step = (int)gridDim.x * kFewWarps * 4;
  for (int v0 = ((int)blockIdx.x * kFewWarps + warp) * 4; v0 < V; v0 += step) {
    float a[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) a[i] = 0.0f;
#pragma unroll 2
    for (int c = 0; c < Dp; c += 128) {
      float4 q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* p = w + (int64_t)min(v0 + j, V - 1) * D;
        if (VEC) {
          const int e = c + 4 * lane;
          q[j] = e < D ? *reinterpret_cast<const float4*>(p + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          const int e = c + lane;
          q[j] = make_float4(e < D ? p[e] : 0.f, e + 32 < D ? p[e + 32] : 0.f, e + 64 < D ? p[e + 64] : 0.f,
                             e + 96 < D ? p[e + 96] : 0.f);
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float* p = xs + i * Dp + c;
        const float4 u = VEC ? *reinterpret_cast<const float4*>(p + 4 * lane)
                             : make_float4(p[lane], p[lane + 32], p[lane + 64], p[lane + 96]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j * N + i] = fmaf(q[j].x, u.x, fmaf(q[j].y, u.y, fmaf(q[j].z, u.z, fmaf(q[j].w, u.w, a[j * N + i]))));
      }
    }
    int cnt = 4 * N;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      if (cnt > 1) {
        cnt /= 2;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i)
          if (i < cnt) {
            const float give = lane & o ? a[i] : a[i + cnt], keep = lane & o ? a[i + cnt] : a[i];
            a[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
      } else {
        a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
      }
    }
    const int v = v0 + my_entry;
    if (v < V) {
      run.add(a[0]);
      if (v == t) at[my_row] = a[0];   // the lanes of a logit write the same value
    }
  }
  sh[warp][idx] = make_float2(run.m, run.s);
  __syncthreads();
  if (threadIdx.x < n) {
    Run r;
    for (int k = 0; k < kFewWarps; ++k)
      for (int j = 0; j < 4; ++j) r.join(sh[k][j * N + threadIdx.x].x, sh[k][j * N + threadIdx.x].y);
    part[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = make_float2(r.m, r.s);
  }
}

// weight [D, V]: a block takes 32 W columns, its warps a slice of D each, and joins
// their sums through shared memory.  part: [N][gridDim.x].
template <int N, int W>
__global__ void __launch_bounds__(32 * kFewWarps, 3)
k_head_few_cols(const float* __restrict__ x, const float* __restrict__ w, int n, int D, int V, const void* tgt, int tdt,
                float2* __restrict__ part, float* __restrict__ at) {
  extern __shared__ __align__(16) float xs[];   // [D][N], then [warps][N][32 W]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* sums = xs + (int64_t)D * N;
  for (int i = threadIdx.x; i < N * D; i += blockDim.x) xs[i] = i % N < n ? x[(int64_t)(i % N) * D + i / N] : 0.0f;
  __syncthreads();
  const int c = ((int)blockIdx.x * 32 + lane) * W;
  const int d0 = (int)((int64_t)D * warp / kFewWarps), d1 = (int)((int64_t)D * (warp + 1) / kFewWarps);
  float a[N][W];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) a[i][j] = 0.0f;
  if (c < V) {
    for (int d = d0; d < d1; d += 8) {
      float q[8][W];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float* p = w + (int64_t)min(d + k, d1 - 1) * V + c;
        if constexpr (W == 4) *reinterpret_cast<float4*>(q[k]) = *reinterpret_cast<const float4*>(p);
        else q[k][0] = *p;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (d + k < d1)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float u = xs[(d + k) * N + i];
#pragma unroll
            for (int j = 0; j < W; ++j) a[i][j] = fmaf(q[k][j], u, a[i][j]);
          }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) sums[(warp * N + i) * 32 * W + lane * W + j] = a[i][j];
  __syncthreads();
  // a warp per row: logits of the block's columns, their running softmax
  for (int i = warp; i < n; i += kFewWarps) {
    const int64_t t = target_at(tgt, tdt, i);
    Run r;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int col = j * 32 + lane, v = (int)blockIdx.x * 32 * W + col;
      float z = 0.0f;
      for (int k = 0; k < kFewWarps; ++k) z += sums[(k * N + i) * 32 * W + col];
      if (v < V) {
        r.add(z);
        if (v == t) at[i] = z;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
      r.join(__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o));
    if (lane == 0) part[(int64_t)i * gridDim.x + blockIdx.x] = make_float2(r.m, r.s);
  }
}

// The rows' nll from their parts and the loss, in one block: a warp per row.
__global__ void __launch_bounds__(32 * kFewRows)
k_head_few_end(const float2* __restrict__ part, int parts, const float* __restrict__ at, const void* tgt, int tdt, int n,
               int V, float* __restrict__ nll, float* __restrict__ loss, int32_t* __restrict__ err) {
  __shared__ float sh[kFewRows];
  const int lane = threadIdx.x & 31, i = threadIdx.x >> 5;
  float v = 0.0f;
  bool counted = false;
  if (i < n) {
    const int64_t t = target_at(tgt, tdt, i);
    counted = t >= 0 && t < V;
    if (t >= V && lane == 0) atomicExch(err, 4);
    const float2* p = part + (int64_t)i * parts;
    float m = -INFINITY, sum = 0.0f;
#pragma unroll 8
    for (int k = lane; k < parts; k += 32) m = fmaxf(m, p[k].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float m0 = m == -INFINITY ? 0.0f : m;
#pragma unroll 8
    for (int k = lane; k < parts; k += 32) sum += p[k].y * exp2f((p[k].x - m0) * kLog2e);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (counted) v = logf(sum) - (at[i] - m);
    if (lane == 0) nll[i] = v;
  }
  if (lane == 0) sh[i] = v;
  const int count = __syncthreads_count(counted && lane == 0);
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int k = 0; k < kFewRows; ++k) s += (double)sh[k];
    loss[0] = (float)(s / (double)max(1, count));
  }
}

template <int N>
void few(const float* x, const float* w, const void* tgt, int tdt, bool tied, int n, int D, int V, float* nll,
         float* loss) {
  // tied: two blocks' worth of warps per SM and more, as the registers allow; else a block per 32 or 128 columns
  const bool vec = (tied ? D : V) % 4 == 0 && ((uintptr_t)w & 15) == 0;
  const int grid = tied ? std::min((V + 4 * kFewWarps - 1) / (4 * kFewWarps), kNumSMs * 4)
                        : (V + (vec ? 127 : 31)) / (vec ? 128 : 32);
  float2* part = static_cast<float2*>(scratch_alloc((size_t)n * (grid * 8 + 4)));
  float* at = reinterpret_cast<float*>(part + (int64_t)n * grid);
  const int pid = prof_begin_named("k_head_few", 4.0 * (double)V * D);
  auto go = [&](auto kernel, size_t smem) {
    // the limit is the function's, for every thread's calls: always the same one
    MALUS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem));
    kernel<<<grid, 32 * kFewWarps, smem, stream()>>>(x, w, n, D, V, tgt, tdt, part, at);
  };
  const size_t rows = (size_t)N * ((D + 127) / 128 * 128) * 4;
  const size_t cols = (size_t)N * (D + kFewWarps * (vec ? 128 : 32)) * 4;
  if (tied) vec ? go(k_head_few_rows<N, true>, rows) : go(k_head_few_rows<N, false>, rows);
  else vec ? go(k_head_few_cols<N, 4>, cols) : go(k_head_few_cols<N, 1>, cols);
  prof_end(pid);
  k_head_few_end<<<1, 32 * kFewRows, 0, stream()>>>(part, grid, at, tgt, tdt, n, V, nll, loss, device_error_word());
  count_launch(2);
  after_launch("k_head_few");
  scratch_free(part);
}

thread_local int t_mode = -1;   // one thread's choice leaves the others' results alone

// Rows that take this path: x in shared memory beside the block's sums.
bool few_rows(int64_t n, int64_t D) {
  if (n < 1 || n > kFewRows || t_mode != -1) return false;
  const int64_t N = n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8;
  return N * (D + 127 + kFewWarps * 128) * 4 <= kFewSmem;
}

}  // namespace
}  // namespace malus

using namespace malus;

extern "C" {

int32_t malus_linear_xent_mode(int32_t mode) {
  if (mode < -1 || mode > 1) panic("malus_linear_xent_mode(%d): -1, 0 or 1", mode);
  return std::exchange(t_mode, (int)mode);
}

int64_t malus_linear_xent(int64_t x, int64_t weight, int64_t targets, int32_t tied, int64_t* nll, int64_t* dx,
                          int64_t* dweight) {
  const Shape sx = shape_of(x), sw = shape_of(weight);
  if (tb(x)->dtype != MALUS_F32 || tb(weight)->dtype != MALUS_F32) panic("linear_xent expects f32 x and weight");
  const int tdt = tb(targets)->dtype;
  if (tdt != MALUS_I32 && tdt != MALUS_I64) panic("linear_xent targets must be Tensor<i32> or Tensor<i64>");
  if (sx.ndim < 1) panic("linear_xent x must have rank 1 or more");
  if (sw.ndim != 2) panic("linear_xent weight must be rank-2, got rank %d", sw.ndim);
  const size_t D = sx.d[sx.ndim - 1], V = tied ? sw.d[0] : sw.d[1];
  if (D == 0 || V == 0) panic("linear_xent over an empty axis (D = %zu, V = %zu)", D, V);
  if ((tied ? sw.d[1] : sw.d[0]) != D)
    panic("linear_xent weight [%zu, %zu] does not match x's last axis %zu (tied = %d: weight is %s)", sw.d[0], sw.d[1],
          D, (int)tied, tied ? "[V, D]" : "[D, V]");
  const size_t n = tb(x)->len / D;
  if (tb(targets)->len != n) panic("linear_xent x has %zu rows but targets has %zu elements", n, tb(targets)->len);
  const int64_t ld = ((int64_t)V + 63) / 64 * 64;
  if (ld > kMaxRowLogits) panic("linear_xent vocabulary is limited to %lld entries, got %zu", (long long)kMaxRowLogits, V);
  if (n > (size_t)1 << 27 || D > (size_t)1 << 24) panic("linear_xent x of %zu rows of %zu is past its limits", n, D);

  const float *xp = fptr(x), *wp = fptr(weight);
  const void* tp = vptr(targets);
  const int64_t loss = alloc_f32({1}), hn = alloc_f32({n});
  const int64_t hx = dx ? alloc_shape(sx) : 0, hw = dweight ? alloc_shape(sw) : 0;
  if (!hx && !hw && few_rows((int64_t)n, (int64_t)D)) {
    auto go = n <= 1 ? few<1> : n <= 2 ? few<2> : n <= 4 ? few<4> : few<8>;
    go(xp, wp, tp, tdt, tied != 0, (int)n, (int)D, (int)V, fptr(hn), fptr(loss));
    if (nll) *nll = hn;
    else tensor_release(hn);
    if (dx) *dx = 0;
    if (dweight) *dweight = 0;
    return loss;
  }
  if (n && (t_mode < 0 ? head_small((int64_t)n, (int64_t)D, (int64_t)V, hx || hw) : t_mode == 1 && n <= 16384)) {
    head_small_run(xp, wp, tp, tdt, tied != 0, (int64_t)n, (int64_t)D, (int64_t)V, fptr(hn), fptr(loss),
                   hx ? fptr(hx) : nullptr, hw ? fptr(hw) : nullptr);
    if (nll) *nll = hn;
    else tensor_release(hn);
    if (dx) *dx = hx;
    if (dweight) *dweight = hw;
    return loss;
  }
  if (n == 0) {
    MALUS_CUDA(cudaMemsetAsync(fptr(loss), 0, 4, stream()));
    if (hw) MALUS_CUDA(cudaMemsetAsync(fptr(hw), 0, V * D * 4, stream()));
  } else if (hx || hw) {
    train(xp, wp, tp, tdt, tied != 0, (int64_t)n, (int64_t)D, (int64_t)V, ld, fptr(hn), fptr(loss),
          hx ? fptr(hx) : nullptr, hw ? fptr(hw) : nullptr);
  } else {
    loss_only(xp, wp, tp, tdt, tied != 0, (int64_t)n, (int64_t)D, (int64_t)V, fptr(hn), fptr(loss));
  }
  if (nll) *nll = hn;
  else tensor_release(hn);
  if (dx) *dx = hx;
  if (dweight) *dweight = hw;
  return loss;
}

}  // extern "C"
