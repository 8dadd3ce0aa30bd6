// Softmax losses by rows: the cross entropy of a logits row against its target
// (for the head, linear_xent.cu), and distillation from a teacher's top logits:
//
//   p = softmax over the row's entries of teacher / T,  q = softmax(logits / T)
//   kl = T^2 sum_k p_k (log p_k - log q[id_k]),  dlogits = T (q - p) / rows
//
// Bound by HBM: a row is read once and held in registers, by one block or by a
// cluster of up to 8 that exchange their maximum and sum through distributed
// shared memory, so the gradient row is written without reading the logits
// again (4 B read and 4 B written per logit).
#include "gemm_f16.cuh"
#include "loss_rows.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace malus {
namespace {

constexpr int kNV = 8;            // float4 groups a thread holds
constexpr int kThreads = 512;     // usual most per block; twice that for the longest rows
constexpr int kMaxThreads = 1024;
constexpr int kMaxCluster = 8;
constexpr int kMaxEntries = 1024; // teacher entries of a row
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kErrId = 4;         // the error word's code for an id out of range

__device__ __forceinline__ int64_t id_at(const void* p, int dtype, int64_t i) {
  return dtype == MALUS_I64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}
__device__ __forceinline__ float wmax(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float wsum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row of V floats at `row` as 16-byte groups from the aligned address at or
// below it: group i covers elements 4 i - shift .. 4 i - shift + 3, and the
// groups that reach past either end of the row are read and written by element.
struct RowSlice {
  int shift;        // elements between the aligned address and the row
  int64_t g0, g1;   // this block's groups
};
__device__ __forceinline__ RowSlice slice_of(const float* row, int64_t V, int rank, int cs) {
  RowSlice s;
  s.shift = (int)(((uintptr_t)row >> 2) & 3);
  const int64_t groups = (V + s.shift + 3) / 4, per = (groups + cs - 1) / cs;
  s.g0 = rank * per;
  s.g1 = s.g0 + per < groups ? s.g0 + per : groups;
  return s;
}
__device__ __forceinline__ float4 load_group(const float* __restrict__ row, int64_t V, int64_t e) {
  if (e >= 0 && e + 4 <= V) return *reinterpret_cast<const float4*>(row + e);
  float4 q;
  const float ninf = -INFINITY;
  q.x = e >= 0 && e < V ? row[e] : ninf;
  q.y = e + 1 >= 0 && e + 1 < V ? row[e + 1] : ninf;
  q.z = e + 2 >= 0 && e + 2 < V ? row[e + 2] : ninf;
  q.w = e + 3 >= 0 && e + 3 < V ? row[e + 3] : ninf;
  return q;
}
__device__ __forceinline__ void store_group(float* __restrict__ row, int64_t V, int64_t e, float4 q, bool vec) {
  if (vec && e >= 0 && e + 4 <= V) {
    *reinterpret_cast<float4*>(row + e) = q;
    return;
  }
  if (e >= 0 && e < V) row[e] = q.x;
  if (e + 1 >= 0 && e + 1 < V) row[e + 1] = q.y;
  if (e + 2 >= 0 && e + 2 < V) row[e + 2] = q.z;
  if (e + 3 >= 0 && e + 3 < V) row[e + 3] = q.w;
}

// Maximum and sum of exponentials of the row whose groups the cluster's threads
// hold in v: v becomes exp((v - max) * c), and the sum is over the whole row.
// Elements of -inf give 0; a row of -inf only, or with a +inf or NaN, gives NaN
// probabilities as the formula does.  Every block has read its slice when this
// returns.
struct RowStat { float max, sum; };
__device__ __forceinline__ RowStat row_stat(float4 (&v)[kNV], int n, float c, cg::cluster_group& cl, float* red,
                                            float2* mine) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kNV; ++k)
    if (k < n) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
  m = wmax(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = -INFINITY;
  for (int i = 0; i < warps; ++i) m = fmaxf(m, red[i]);
  // exponentials against the block's own maximum; the blocks are joined below
  const float m0 = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < kNV; ++k)
    if (k < n) {
      v[k].x = exp2f((v[k].x - m0) * c);
      v[k].y = exp2f((v[k].y - m0) * c);
      v[k].z = exp2f((v[k].z - m0) * c);
      v[k].w = exp2f((v[k].w - m0) * c);
      s += (v[k].x + v[k].y) + (v[k].z + v[k].w);
    }
  s = wsum(s);
  if (lane == 0) red[32 + warp] = s;
  __syncthreads();
  s = 0.0f;
  for (int i = 0; i < warps; ++i) s += red[32 + i];
  const int cs = (int)cl.num_blocks();
  if (cs == 1) return {m, s};
  if (threadIdx.x == 0) *mine = make_float2(m, s);
  cl.sync();
  float M = -INFINITY;
  for (int r = 0; r < cs; ++r) M = fmaxf(M, cl.map_shared_rank(mine, r)->x);
  // a block of -inf only has the sum 0 (or NaN) whatever its factor
  auto factor = [&](float bm) { return bm == -INFINITY ? 1.0f : exp2f((bm - M) * c); };
  float S = 0.0f;
  for (int r = 0; r < cs; ++r) {
    const float2 o = *cl.map_shared_rank(mine, r);
    S += o.y * factor(o.x);
  }
  const float f = factor(m);
#pragma unroll
  for (int k = 0; k < kNV; ++k)
    if (k < n) v[k] = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
  cl.sync();   // no block leaves while another still reads its pair
  return {M, S};
}

// Four elements of the row's gradient, magnitudes at most 1, as the half planes
// that the head's products read: hi in the first half of the row's memory, lo in
// the second.
__device__ __forceinline__ void store_planes(float* row, int64_t ld, int64_t e, float4 q) {
  constexpr float up = (float)(1 << kF16Exp);
  const float x[4] = {q.x * up, q.y * up, q.z * up, q.w * up};
  __align__(8) __half h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = __float2half_rn(x[j]);
    l[j] = __float2half_rn(x[j] - __half2float(h[j]));
  }
  __half* p = reinterpret_cast<__half*>(row);
  *reinterpret_cast<uint2*>(p + e) = *reinterpret_cast<uint2*>(h);
  *reinterpret_cast<uint2*>(p + ld + e) = *reinterpret_cast<uint2*>(l);
}

__global__ void __launch_bounds__(kMaxThreads)
k_xent_rows(float* __restrict__ logits, int64_t ld, int64_t V, const void* __restrict__ tgt, int tdt, int64_t row0,
            float* __restrict__ nll) {
  __shared__ float red[64];
  __shared__ float2 mine;
  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t r = blockIdx.x / cs;
  float* row = logits + r * ld;
  const RowSlice sl = slice_of(row, ld, rank, cs);   // the pitch is whole groups
  const int64_t t = id_at(tgt, tdt, row0 + r);
  const bool counted = t >= 0 && t < V;
  float zt = 0.0f;
  if (counted) {
    if (rank == 0 && threadIdx.x == 0) zt = row[t];
    float4 v[kNV];
    int n = 0;
#pragma unroll
    for (int k = 0; k < kNV; ++k) {
      const int64_t g = sl.g0 + (int64_t)k * blockDim.x + threadIdx.x;
      if (g < sl.g1) {
        v[k] = load_group(row, V, 4 * g);
        n = k + 1;
      }
    }
    const RowStat st = row_stat(v, n, kLog2e, cl, red, &mine);
    if (rank == 0 && threadIdx.x == 0) nll[row0 + r] = logf(st.sum) - (zt - st.max);
    const float inv = 1.0f / st.sum;
#pragma unroll
    for (int k = 0; k < kNV; ++k)
      if (k < n) {
        const int64_t e = 4 * (sl.g0 + (int64_t)k * blockDim.x + threadIdx.x);
        float4 q = make_float4(v[k].x * inv, v[k].y * inv, v[k].z * inv, v[k].w * inv);
        if (t >= e && t < e + 4) {
          if (t == e) q.x -= 1.0f;
          if (t == e + 1) q.y -= 1.0f;
          if (t == e + 2) q.z -= 1.0f;
          if (t == e + 3) q.w -= 1.0f;
        }
        store_planes(row, ld, e, q);   // columns from V on hold exp(-inf) = 0
      }
  } else {
    if (rank == 0 && threadIdx.x == 0) nll[row0 + r] = 0.0f;
    for (int64_t g = sl.g0 + threadIdx.x; g < sl.g1; g += blockDim.x)
      store_planes(row, ld, 4 * g, make_float4(0.f, 0.f, 0.f, 0.f));
  }
}

__global__ void __launch_bounds__(1024) k_xent_count(const void* __restrict__ tgt, int tdt, int64_t n, int64_t V,
                                                     int* __restrict__ count, int32_t* __restrict__ err) {
  __shared__ int sh[32];
  int c = 0;
  bool bad = false;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int64_t t = id_at(tgt, tdt, i);
    c += t >= 0 && t < V;
    bad |= t >= V;
  }
  if (bad) atomicExch(err, kErrId);
#pragma unroll
  for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    int s = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) s += sh[i];
    count[0] = s;
  }
}

__global__ void __launch_bounds__(1024) k_loss_mean(const float* __restrict__ v, int64_t n,
                                                    const int* __restrict__ count, float* __restrict__ loss) {
  __shared__ double sh[32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += (double)v[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) s += sh[i];
    loss[0] = (float)(s / (double)max(1, count[0]));
  }
}

// nll of a row from its parts' (maximum, sum of exponentials) and its target's
// logit; a warp per row
__global__ void __launch_bounds__(256) k_xent_join(const float2* __restrict__ part, int parts,
                                                   const float* __restrict__ at, const void* __restrict__ tgt, int tdt,
                                                   int64_t V, int64_t n, float* __restrict__ nll) {
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < n; r += (int64_t)gridDim.x * 8) {
    const int64_t t = id_at(tgt, tdt, r);
    if (t < 0 || t >= V) {
      if (lane == 0) nll[r] = 0.0f;
      continue;
    }
    float M = -INFINITY;
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, part[r * parts + i].x);
    M = wmax(M);
    float s = 0.0f;
    for (int i = lane; i < parts; i += 32) {
      const float2 o = part[r * parts + i];
      s += o.y * (o.x == -INFINITY ? 1.0f : exp2f((o.x - M) * kLog2e));   // -inf only: the sum is 0 or NaN
    }
    s = wsum(s);
    if (lane == 0) nll[r] = logf(s) - (at[r] - M);
  }
}

// ---- distillation ----
// An entry is there when its id lies in [0, V) and its logit is not -inf.
__device__ __forceinline__ bool entry_there(int64_t id, float te, int64_t V) {
  return id >= 0 && id < V && te != -INFINITY;
}

// count[0] += rows with an entry (whole numbers: the order does not matter)
__global__ void __launch_bounds__(256) k_distill_count(const void* __restrict__ ids, int idt,
                                                       const float* __restrict__ teacher, int64_t n, int K, int64_t V,
                                                       int* __restrict__ count, int32_t* __restrict__ err) {
  __shared__ int sh[8];
  const int lane = threadIdx.x & 31;
  int c = 0;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < n; r += (int64_t)gridDim.x * 8) {
    bool any = false, bad = false;
    for (int k = lane; k < K; k += 32) {
      const int64_t id = id_at(ids, idt, r * K + k);
      any |= entry_there(id, teacher[r * K + k], V);
      bad |= id >= V;
    }
    if (bad) atomicExch(err, kErrId);
    c += __any_sync(0xffffffffu, any) ? 1 : 0;
  }
  if (lane == 0) sh[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    c = 0;
    for (int i = 0; i < 8; ++i) c += sh[i];
    if (c) atomicAdd(count, c);
  }
}

// The teacher's side of one row, by the block's first warp: p[k] (0 where there
// is no entry) and whether there is any entry.  lp[k] = log p[k].
__device__ __forceinline__ bool teacher_row(const void* ids, int idt, const float* teacher, int64_t r, int K, int64_t V,
                                            float c, int64_t* id, float* p, float* lp) {
  const int lane = threadIdx.x & 31;
  float m = -INFINITY;
  bool any = false;
  for (int k = lane; k < K; k += 32) {
    int64_t i = id_at(ids, idt, r * K + k);
    const float te = teacher[r * K + k];
    if (!entry_there(i, te, V)) i = -1;
    id[k] = i;
    p[k] = te;
    if (i >= 0) {
      m = fmaxf(m, te);
      any = true;
    }
  }
  m = wmax(m);
  any = __any_sync(0xffffffffu, any);
  float s = 0.0f;
  for (int k = lane; k < K; k += 32) {
    const float z = (p[k] - m) * c;   // base-2 units
    const float e = id[k] >= 0 ? exp2f(z) : 0.0f;
    lp[k] = z * kLn2;
    p[k] = e;
    s += e;
  }
  s = wsum(s);
  const float ls = logf(s);
  for (int k = lane; k < K; k += 32) {
    lp[k] -= ls;
    p[k] = id[k] >= 0 ? p[k] / s : 0.0f;
  }
  return any;
}

__global__ void __launch_bounds__(kMaxThreads)
k_distill_rows(const float* __restrict__ logits, int64_t V, const void* __restrict__ ids, int idt,
               const float* __restrict__ teacher, int K, float T, const int* __restrict__ count,
               float* __restrict__ kl, float* __restrict__ dl) {
  __shared__ float red[64];
  __shared__ float2 mine;
  __shared__ int any_sh;
  extern __shared__ int64_t dyn[];
  int64_t* id = dyn;
  float* p = reinterpret_cast<float*>(dyn + K);
  float* lp = p + K;
  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t r = blockIdx.x / cs;
  const float* row = logits + r * V;
  const RowSlice sl = slice_of(row, V, rank, cs);
  const float c = kLog2e / T;
  float4 v[kNV];
  int n = 0;
#pragma unroll
  for (int k = 0; k < kNV; ++k) {
    const int64_t g = sl.g0 + (int64_t)k * blockDim.x + threadIdx.x;
    if (g < sl.g1) {
      v[k] = load_group(row, V, 4 * g - sl.shift);
      n = k + 1;
    }
  }
  if (threadIdx.x < 32) {
    const bool any = teacher_row(ids, idt, teacher, r, K, V, c, id, p, lp);
    if (threadIdx.x == 0) any_sh = any;
  }
  const RowStat st = row_stat(v, n, c, cl, red, &mine);   // its barriers also publish the teacher's side
  const bool counted = any_sh != 0;
  if (rank == 0 && threadIdx.x < 32) {
    float s = 0.0f;
    if (counted) {
      const float lz = logf(st.sum);
      for (int k = threadIdx.x; k < K; k += 32)
        if (p[k] != 0.0f) s += p[k] * (lp[k] - ((row[id[k]] - st.max) * (c * kLn2) - lz));
      s = wsum(s);
    }
    if (threadIdx.x == 0) kl[r] = s * (T * T);
  }
  if (!dl) return;
  float* out = dl + r * V;
  const bool vec = (((uintptr_t)out >> 2) & 3) == (unsigned)sl.shift;
  const float scale = T / (float)max(1, *count), inv = scale / st.sum;
#pragma unroll
  for (int k = 0; k < kNV; ++k)
    if (k < n) {
      const int64_t e = 4 * (sl.g0 + (int64_t)k * blockDim.x + threadIdx.x) - sl.shift;
      const float4 q = counted ? make_float4(v[k].x * inv, v[k].y * inv, v[k].z * inv, v[k].w * inv)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
      store_group(out, V, e, q, vec);
    }
  if (!counted) return;   // uniform over the cluster
  // The teacher's entries, after the whole row is written.  An id listed more
  // than once is handled by its first entry, which takes the others' p in order.
  if (cs > 1) cl.sync();
  else __syncthreads();
  if (rank != 0) return;
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    if (id[k] < 0) continue;
    bool first = true;
    for (int j = 0; j < k && first; ++j) first = id[j] != id[k];
    if (!first) continue;
    float s = 0.0f;
    for (int j = k; j < K; ++j)
      if (id[j] == id[k]) s += p[j];
    const float q = exp2f((row[id[k]] - st.max) * c) / st.sum;
    out[id[k]] = scale * (q - s);
  }
}

// Blocks per row and threads per block for rows of `groups` 16-byte groups;
// false when a cluster's registers do not hold the row.
bool row_launch(int64_t groups, int* cs, int* threads) {
  for (*cs = 1; *cs <= kMaxCluster; *cs *= 2) {
    const int64_t per = (groups + *cs - 1) / *cs;
    const int most = *cs < kMaxCluster ? kThreads : kMaxThreads;
    if (per <= (int64_t)most * kNV) {
      *threads = (int)std::max<int64_t>(32, ((per + kNV - 1) / kNV + 31) / 32 * 32);
      return true;
    }
  }
  return false;
}

template <class K, class... A>
void launch_rows(K kernel, int64_t rows, int cs, int threads, size_t smem, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cs));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cs;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MALUS_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
}

}  // namespace

void xent_count(const void* targets, int tgt_dtype, int64_t n, int64_t V, int* count) {
  k_xent_count<<<1, 1024, 0, stream()>>>(targets, tgt_dtype, n, V, count, device_error_word());
  count_launch();
  after_launch("k_xent_count");
}

void xent_rows(float* logits, int64_t ld, int64_t n, int64_t V, const void* targets, int tgt_dtype, int64_t row0,
               float* nll) {
  if (n == 0) return;
  int cs, threads;
  if (!row_launch(ld / 4, &cs, &threads)) panic("xent_rows: rows of %lld logits", (long long)V);
  const int pid = prof_begin_named("k_xent_rows", 8.0 * (double)n * (double)ld);
  launch_rows(k_xent_rows, n, cs, threads, 0, logits, ld, V, targets, tgt_dtype, row0, nll);
  count_launch();
  after_launch("k_xent_rows");
  prof_end(pid);
}

void xent_join(const float2* part, int parts, const float* at, const void* targets, int tgt_dtype, int64_t V, int64_t n,
               float* nll) {
  if (n == 0) return;
  k_xent_join<<<grid_for((size_t)n * 32, 256), 256, 0, stream()>>>(part, parts, at, targets, tgt_dtype, V, n, nll);
  count_launch();
  after_launch("k_xent_join");
}

void loss_mean(const float* v, int64_t n, const int* count, float* loss) {
  k_loss_mean<<<1, 1024, 0, stream()>>>(v, n, count, loss);
  count_launch();
  after_launch("k_loss_mean");
}

}  // namespace malus

using namespace malus;

extern "C" {

int64_t malus_distill(int64_t logits, int64_t ids, int64_t teacher, float temperature, int64_t* kl,
                      int64_t* dlogits) {
  const Shape s = shape_of(logits), si = shape_of(ids);
  if (tb(logits)->dtype != MALUS_F32 || tb(teacher)->dtype != MALUS_F32)
    panic("distill logits and teacher logits must be f32");
  const int idt = tb(ids)->dtype;
  if (idt != MALUS_I32 && idt != MALUS_I64) panic("distill ids must be Tensor<i32> or Tensor<i64>");
  if (s.ndim != 2) panic("distill logits must be rank-2 [N, V], got rank %d", s.ndim);
  if (si.ndim != 2 || si.d[0] != s.d[0])
    panic("distill ids must be rank-2 [%zu, K], got rank %d with %zu elements", s.d[0], si.ndim, tb(ids)->len);
  if (!same_shape(ids, teacher)) panic("distill ids and teacher logits must have the same shape");
  if (!(temperature > 0.0f) || !std::isfinite(temperature))
    panic("distill temperature must be positive and finite, got %g", (double)temperature);
  const int64_t n = (int64_t)s.d[0], V = (int64_t)s.d[1], K = (int64_t)si.d[1];
  if (V == 0) panic("distill over an empty vocabulary");
  if (K < 1 || K > kMaxEntries) panic("distill takes 1 to %d teacher entries per row, got %lld", kMaxEntries, (long long)K);
  int cs, threads;
  // a row may start up to 3 elements past an aligned address
  if (V > kMaxRowLogits - 4 || !row_launch((V + 3 + 3) / 4, &cs, &threads))
    panic("distill rows are limited to %lld logits, got %lld", (long long)kMaxRowLogits - 4, (long long)V);
  if (n > (int64_t)1 << 27) panic("distill is limited to 2^27 rows, got %lld", (long long)n);
  const float* x = fptr(logits);
  const void* idp = vptr(ids);
  const float* te = fptr(teacher);
  const int64_t loss = alloc_f32({1}), hk = alloc_f32({s.d[0]});
  const int64_t hd = dlogits ? alloc_shape(s) : 0;
  int* count = static_cast<int*>(scratch_alloc(4));
  MALUS_CUDA(cudaMemsetAsync(count, 0, 4, stream()));
  if (n) {
    k_distill_count<<<grid_for((size_t)n * 32, 256), 256, 0, stream()>>>(idp, idt, te, n, (int)K, V, count,
                                                                        device_error_word());
    const int pid = prof_begin_named("k_distill_rows", (hd ? 8.0 : 4.0) * (double)n * (double)V);
    launch_rows(k_distill_rows, n, cs, threads, (size_t)K * 16, x, V, idp, idt, te, (int)K, temperature,
                (const int*)count, fptr(hk), hd ? fptr(hd) : (float*)nullptr);
    count_launch(2);
    after_launch("k_distill_rows");
    prof_end(pid);
  }
  loss_mean(fptr(hk), n, count, fptr(loss));
  scratch_free(count);
  if (kl) *kl = hk;
  else tensor_release(hk);
  if (dlogits) *dlogits = hd;
  return loss;
}

}  // extern "C"
