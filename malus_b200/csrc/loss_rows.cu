// Softmax losses by rows: the cross entropy of a logits row against its target
// (for the head, linear_xent.cu), and distillation from a teacher's top logits:
//
//   p = softmax over the row's entries of teacher / T,  q = softmax(logits / T)
//   kl = T^2 sum_k p_k (log p_k - log q[id_k]),  dlogits = T (q - p) / rows
//
// Bound by HBM: a row is read once and held in registers, so its gradient is
// written without reading the logits again (4 B read and 4 B written per logit).
// Rows up to 1024 logits take a warp each.  Longer ones take a block, or a
// cluster of up to 8 blocks that exchange their maximum and sum through
// distributed shared memory.  The blocks stay and walk the rows: while a row is
// in registers (maximum, exponentials, exchange, gradient), the bulk copy of the
// next one is already landing in shared memory, which keeps reads in flight
// through the phases that wait.
#include "gemm_f16.cuh"
#include "loss_rows.cuh"
#include "tc_common.cuh"

#include <cooperative_groups.h>
#include <mutex>
#include <map>

namespace cg = cooperative_groups;

namespace malus {
namespace {

constexpr int kNV = 8;            // float4 groups a thread holds
constexpr int kThreads = 448;     // most per block: two blocks per SM with 72 registers each
constexpr int kMaxThreads = 1024; // for rows that eight such blocks do not hold
constexpr int kMaxCluster = 8;
constexpr int kMaxEntries = 1024; // teacher entries of a row
constexpr int kShort = 32 * kNV * 4 - 4;   // longest row of a warp (it may start 3 past a 16-byte group)
constexpr int kWarps = 8;         // rows per block of the short-row kernels
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

// A row of V floats as 16-byte groups from the aligned address at or below it:
// group i covers elements 4 i - shift .. 4 i - shift + 3.  Groups [w0, w1) lie
// wholly in the row; the one before or after them reaches past its end and is read
// and written by element.
struct RowSlice {
  const float4* base;   // group 0
  int shift;            // elements between the aligned address and the row
  int g0, g1;           // this block's groups
  int w0, w1;
};
// (the cluster has 2^lc blocks)
__device__ __forceinline__ RowSlice slice_of(const float* row, int V, int rank, int lc) {
  RowSlice s;
  s.shift = (int)(((uintptr_t)row >> 2) & 3);
  s.base = reinterpret_cast<const float4*>(row - s.shift);
  const int groups = (V + s.shift + 3) >> 2, per = (groups + (1 << lc) - 1) >> lc;
  s.g0 = min(rank * per, groups);
  s.g1 = min(s.g0 + per, groups);
  s.w0 = s.shift ? 1 : 0;
  s.w1 = (V + s.shift) >> 2;
  return s;
}
__device__ __forceinline__ float4 load_edge(const float* __restrict__ row, int V, int e) {
  const float ninf = -INFINITY;
  return make_float4(e >= 0 && e < V ? row[e] : ninf, e + 1 >= 0 && e + 1 < V ? row[e + 1] : ninf,
                     e + 2 >= 0 && e + 2 < V ? row[e + 2] : ninf, e + 3 >= 0 && e + 3 < V ? row[e + 3] : ninf);
}
__device__ __forceinline__ void store_edge(float* __restrict__ row, int V, int e, float4 q) {
  if (e >= 0 && e < V) row[e] = q.x;
  if (e + 1 >= 0 && e + 1 < V) row[e + 1] = q.y;
  if (e + 2 >= 0 && e + 2 < V) row[e + 2] = q.z;
  if (e + 3 >= 0 && e + 3 < V) row[e + 3] = q.w;
}

// Maximum and sum of exponentials of a row whose groups the threads hold in v,
// -inf where a thread has none: v becomes exp((v - max) * c) after the join below,
// and the sum is over the whole row.  Elements of -inf give 0; a row of -inf only,
// or with a +inf or NaN, gives NaN probabilities as the formula does.
struct RowStat { float max, sum; };

// The warp's maximum; v becomes exp against it and the sum is the warp's.  The
// exponential is the hardware's base-2 one (relative error 2^-22; results
// below 2^-126 are 0).
__device__ __forceinline__ RowStat warp_stat(float4 (&v)[kNV], float c) {
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kNV; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
  m = wmax(m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < kNV; ++k) {
    v[k].x = tc::exp2_hw((v[k].x - m0) * c);
    v[k].y = tc::exp2_hw((v[k].y - m0) * c);
    v[k].z = tc::exp2_hw((v[k].z - m0) * c);
    v[k].w = tc::exp2_hw((v[k].w - m0) * c);
    s += (v[k].x + v[k].y) + (v[k].z + v[k].w);
  }
  return {m, wsum(s)};
}
// a part of -inf only has the sum 0 (or NaN) whatever its factor
__device__ __forceinline__ float join_factor(float m, float M, float c) {
  return m == -INFINITY ? 1.0f : tc::exp2_hw((m - M) * c);
}

// A wait of at most the bound; false (and an error word of `code`) when it runs out.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, int32_t* err, int code) {
  if (tc::mbar_try(bar, parity)) return true;
  const uint64_t t0 = tc::gtimer();
  while (!tc::mbar_try(bar, parity))
    if (tc::gtimer() - t0 > tc::kWaitNs) {
      atomicExch(err, code);
      return false;
    }
  return true;
}

constexpr int kTable = kMaxCluster * kMaxThreads / 32;
// Joins the warps of a cluster of blocks (or of one block).  Every warp sends its
// pair into each block's table by an asynchronous store that counts on that
// block's barrier, and every warp waits for its own block's barrier and reduces
// the table.  (A cluster barrier in its place also waits until the gradient
// stores of the row before are acknowledged.)  Two tables alternate: a warp sends
// into one again only after it has every block's pairs of the row between, which
// they send when they are done with this one.
struct Join {
  float2* table;     // [2][kTable]
  uint32_t bar[2];
  uint32_t uses;
  bool dead;
  int32_t* err;

  __device__ __forceinline__ void init(float2* t, uint64_t* bars, int32_t* e, cg::cluster_group& cl) {
    table = t;
    uses = 0;
    dead = false;
    err = e;
    for (int i = 0; i < 2; ++i) {
      bar[i] = tc::smem_u32(bars + i);
      if (threadIdx.x == 0) tc::mbar_init(bar[i], 1);
    }
    if (threadIdx.x == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    cl.sync();   // every block's barriers exist before another counts on them
  }
  // `f` is what brings this warp's exponentials to the row's maximum.
  __device__ __forceinline__ RowStat operator()(RowStat w, float c, cg::cluster_group& cl, float* f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int cs = (int)cl.num_blocks(), total = cs * warps, turn = uses & 1;
    float2* t = table + turn * kTable;
    if (cs == 1) {
      if (lane == 0) t[warp] = make_float2(w.max, w.sum);
      __syncthreads();
    } else {
      if (threadIdx.x == 0) tc::mbar_expect_tx(bar[turn], (uint32_t)total * 8);
      if (lane < cs) {
        const uint64_t v = ((uint64_t)__float_as_uint(w.sum) << 32) | __float_as_uint(w.max);
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];"
                     ::"r"(tc::cluster_addr(tc::smem_u32(t + cl.block_rank() * warps + warp), lane)), "l"(v),
                       "r"(tc::cluster_addr(bar[turn], lane))
                     : "memory");
      }
      if (!dead) dead = !wait_for(bar[turn], (uses >> 1) & 1, err, 52);
    }
    ++uses;
    float M = -INFINITY;
    for (int i = lane; i < total; i += 32) M = fmaxf(M, t[i].x);
    M = wmax(M);
    float S = 0.0f;
    for (int i = lane; i < total; i += 32) S += t[i].y * join_factor(t[i].x, M, c);
    *f = join_factor(w.max, M, c);
    return {M, wsum(S)};
  }
};

// The landing buffer: the slice of the next row, brought by a bulk copy of its
// whole 16-byte groups.  A copy that does not arrive within the wait's
// bound is reported in the error word; no further copy is then issued or waited for.
struct Landing {
  float4* buf;
  uint32_t bar;
  uint32_t parity;
  bool dead;
  int32_t* err;

  __device__ __forceinline__ void init(float4* b, uint64_t* mbar, int32_t* e) {
    buf = b;
    bar = tc::smem_u32(mbar);
    parity = 0;
    dead = false;
    err = e;
    if (threadIdx.x == 0) {
      tc::mbar_init(bar, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ __forceinline__ void issue(const RowSlice& s) {
    if (threadIdx.x != 0 || dead) return;
    const int i0 = max(s.g0, s.w0), i1 = min(s.g1, s.w1);
    const uint32_t bytes = i1 > i0 ? (uint32_t)(i1 - i0) * 16 : 0;
    tc::mbar_expect_tx(bar, bytes);
    if (bytes)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   ::"r"(tc::smem_u32(buf + (i0 - s.g0))), "l"(s.base + i0), "r"(bytes), "r"(bar)
                   : "memory");
  }
  __device__ __forceinline__ void wait() {
    if (dead) return;
    dead = !wait_for(bar, parity, err, 51);
    parity ^= 1;
  }
  // this thread's groups t + k * blockDim.x of the landed slice into v, -inf past
  // its end; a group that reaches past the row (first, last) comes from memory
  __device__ __forceinline__ void take(float4 (&v)[kNV], const RowSlice& s, const float* row, int V) const {
    const int len = s.g1 - s.g0, nt = (int)blockDim.x, t = (int)threadIdx.x;
    const int last = s.w1 < s.g1 ? s.w1 - s.g0 : -1;
    const bool head = s.shift && s.g0 == 0;
#pragma unroll
    for (int k = 0; k < kNV; ++k) {
      const int i = t + k * nt;
      v[k] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (i < len) v[k] = buf[i];
      if (i == last || (head && i == 0)) v[k] = load_edge(row, V, 4 * (s.g0 + i) - s.shift);
    }
  }
};

// Four elements of the row's gradient, magnitudes at most 1, as the half planes
// that the head's products read: hi in the first half of the row's memory, lo in
// the second.
__device__ __forceinline__ void store_planes(float* row, int ld, int e, float4 q) {
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

// the gradient of a row's groups that this thread holds in v (exponentials):
// groups g + k * step below g1
__device__ __forceinline__ void xent_store(float* row, int ld, const float4 (&v)[kNV], int g, int g1, int step, float f,
                                           int t) {
#pragma unroll
  for (int k = 0; k < kNV; ++k)
    if (g + k * step < g1) {
      const int e = 4 * (g + k * step);
      float4 q = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
      const unsigned o = (unsigned)(t - e);
      if (o < 4) {
        if (o == 0) q.x -= 1.0f;
        if (o == 1) q.y -= 1.0f;
        if (o == 2) q.z -= 1.0f;
        if (o == 3) q.w -= 1.0f;
      }
      store_planes(row, ld, e, q);   // columns from V on hold exp(-inf) = 0
    }
}
// Group g (of a row whose memory goes on to its pitch) with -inf from column V on.
__device__ __forceinline__ float4 cut_group(float4 q, int e, int V) {
  const float ninf = -INFINITY;
  return make_float4(e < V ? q.x : ninf, e + 1 < V ? q.y : ninf, e + 2 < V ? q.z : ninf, e + 3 < V ? q.w : ninf);
}

__global__ void __launch_bounds__(32 * kWarps)
k_xent_rows_warp(float* __restrict__ logits, int ld, int64_t rows, int V, const void* __restrict__ tgt, int tdt,
                 int64_t row0, float* __restrict__ nll) {
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * kWarps) {
    float* row = logits + r * ld;
    const int64_t t = id_at(tgt, tdt, row0 + r);
    if (t < 0 || t >= V) {
      if (lane == 0) nll[row0 + r] = 0.0f;
      for (int g = lane; g < ld / 4; g += 32) store_planes(row, ld, 4 * g, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    const float zt = row[t];
    float4 v[kNV];
#pragma unroll
    for (int k = 0; k < kNV; ++k) {
      const int g = k * 32 + lane;
      v[k] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (4 * g < V) v[k] = cut_group(reinterpret_cast<const float4*>(row)[g], 4 * g, V);
    }
    const RowStat st = warp_stat(v, kLog2e);   // the whole row is in registers after it
    if (lane == 0) nll[row0 + r] = logf(st.sum) - (zt - st.max);
    xent_store(row, ld, v, lane, ld / 4, 32, 1.0f / st.sum, (int)t);
  }
}

template <int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > kThreads ? 1 : 2)
k_xent_rows(float* __restrict__ logits, int ld, int64_t rows, int V, const void* __restrict__ tgt, int tdt,
            int64_t row0, float* __restrict__ nll, int32_t* __restrict__ err) {
  extern __shared__ __align__(16) float4 land[];
  __shared__ float2 table[2 * kTable];
  __shared__ uint64_t bar, jbar[2];
  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), lc = 31 - __clz(cs), rank = (int)cl.block_rank();
  const int64_t step = gridDim.x >> lc;
  Landing L;
  L.init(land, &bar, err);
  Join join;
  join.init(table, jbar, err, cl);
  int64_t r = blockIdx.x >> lc;
  RowSlice sl = slice_of(logits + r * ld, ld, rank, lc);   // the pitch is whole groups: the same in every row
  if (r < rows) L.issue(sl);
  for (; r < rows; r += step) {
    float* row = logits + r * ld;
    const int64_t t = id_at(tgt, tdt, row0 + r);
    const bool counted = t >= 0 && t < V;
    float zt = 0.0f;
    if (counted && rank == 0 && threadIdx.x == 0) zt = row[t];
    L.wait();
    const int g = sl.g0 + (int)threadIdx.x;
    float4 v[kNV];
    L.take(v, sl, row, ld);
    if (4 * sl.g1 > V) {   // what lies behind the row is no logit
#pragma unroll
      for (int k = 0; k < kNV; ++k) {
        const int e = 4 * (g + k * (int)blockDim.x);
        if (e + 4 > V) v[k] = cut_group(v[k], e, V);
      }
    }
    __syncthreads();   // the buffer is free
    sl.base += step * (ld / 4);
    if (r + step < rows) L.issue(sl);
    if (counted) {
      float f;
      const RowStat st = join(warp_stat(v, kLog2e), kLog2e, cl, &f);
      if (rank == 0 && threadIdx.x == 0) nll[row0 + r] = logf(st.sum) - (zt - st.max);
      xent_store(row, ld, v, g, sl.g1, blockDim.x, f / st.sum, (int)t);
    } else {
      if (rank == 0 && threadIdx.x == 0) nll[row0 + r] = 0.0f;
#pragma unroll
      for (int k = 0; k < kNV; ++k)
        if (g + k * (int)blockDim.x < sl.g1)
          store_planes(row, ld, 4 * (g + k * (int)blockDim.x), make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
  if (cs > 1) cl.sync();   // no block leaves while another may still send to it
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

// loss = sum of v / max(1, count); with parts, v[r] is first the sum of the row's parts
__global__ void __launch_bounds__(1024) k_loss_mean(float* __restrict__ v, const float* __restrict__ part, int parts,
                                                    int64_t n, const int* __restrict__ count, float* __restrict__ loss) {
  __shared__ double sh[32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    if (parts) {
      float a = 0.0f;
      for (int j = 0; j < parts; ++j) a += part[i * parts + j];
      v[i] = a;
    }
    s += (double)v[i];
  }
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

// An entry of a row: its id (-1: none), p and log p, and for the first entry with
// this id the p of all of them, -1 for the others.
struct __align__(16) Entry {
  int id;
  float p, lp, own;
};

// The teacher's side, a warp per row.  flag[r]: the row has an entry; count[0] +=
// such rows (whole numbers: the order does not matter).
__global__ void __launch_bounds__(256)
k_teacher(const void* __restrict__ ids, int idt, const float* __restrict__ teacher, int64_t n, int K, int64_t V,
          float c, Entry* __restrict__ ent, int* __restrict__ flag, int* __restrict__ count,
          int32_t* __restrict__ err) {
  extern __shared__ int sid[];   // [8][K]: the rows' ids, -1 where there is no entry
  __shared__ int sh[8];
  const int lane = threadIdx.x & 31;
  int* mine = sid + (threadIdx.x >> 5) * K;
  int rows = 0;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < n; r += (int64_t)gridDim.x * 8) {
    const int64_t o = r * K;
    float m = -INFINITY;
    bool any = false, bad = false;
    for (int k = lane; k < K; k += 32) {
      const int64_t id = id_at(ids, idt, o + k);
      const float te = teacher[o + k];
      bad |= id >= V;
      const bool there = entry_there(id, te, V);
      mine[k] = there ? (int)id : -1;
      if (there) {
        m = fmaxf(m, te);
        any = true;
      }
    }
    if (bad) atomicExch(err, kErrId);
    m = wmax(m);
    any = __any_sync(0xffffffffu, any);
    float s = 0.0f;
    for (int k = lane; k < K; k += 32) {
      const float z = (teacher[o + k] - m) * c;   // base-2 units
      const float e = mine[k] >= 0 ? exp2f(z) : 0.0f;
      ent[o + k] = {mine[k], e, z * kLn2, -1.0f};
      s += e;
    }
    s = wsum(s);
    const float ls = logf(s);
    for (int k = lane; k < K; k += 32) {
      ent[o + k].lp -= ls;
      ent[o + k].p = ent[o + k].p == 0.0f ? 0.0f : ent[o + k].p / s;
    }
    __syncwarp();   // the other lanes' ids and p
    for (int k = lane; k < K; k += 32) {
      const int id = mine[k];
      if (id < 0) continue;
      float sum = ent[o + k].p;
      for (int j = 0; j < K; ++j)
        if (mine[j] == id && j != k) {
          if (j < k) {
            sum = -1.0f;
            break;
          }
          sum += ent[o + j].p;
        }
      ent[o + k].own = sum;
    }
    __syncwarp();   // the ids are rewritten by the next row
    if (lane == 0) flag[r] = any;
    rows += any;
  }
  if (lane == 0) sh[threadIdx.x >> 5] = rows;
  __syncthreads();
  if (threadIdx.x == 0) {
    rows = 0;
    for (int i = 0; i < 8; ++i) rows += sh[i];
    if (rows) atomicAdd(count, rows);
  }
}

struct Distill {
  const float* logits;
  const Entry* ent;
  const int *flag, *count;
  int64_t rows, V_;
  int K;
  float T;
  float *part, *dl;   // part: [rows][parts], the row's kl in pieces
  int parts;
  int land;           // float4s of the landing buffer
  int32_t* err;
  __device__ __forceinline__ const float* row(int64_t r) const { return logits + r * V_; }
  __device__ __forceinline__ int width() const { return (int)V_; }
  __device__ __forceinline__ int V() const { return (int)V_; }
};

// q of the groups g + k * step in v into the row's gradient (`vec`: its groups
// are aligned like the logits')
__device__ __forceinline__ void distill_store(float* out, int V, const RowSlice& sl, const float4 (&v)[kNV], int g,
                                              int step, float f, bool vec) {
  float4* base = reinterpret_cast<float4*>(out - sl.shift);
#pragma unroll
  for (int k = 0; k < kNV; ++k)
    if (g + k * step < sl.g1) {
      const int i = g + k * step;
      const float4 q = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
      if (vec && i >= sl.w0 && i < sl.w1) base[i] = q;
      else store_edge(out, V, 4 * i - sl.shift, q);
    }
}
// The part of an entry with logit z in its row's kl.
__device__ __forceinline__ float entry_kl(const Entry& e, float z, RowStat st, float log_sum, float inv_T) {
  return e.p != 0.0f ? e.p * (e.lp - ((z - st.max) * inv_T - log_sum)) : 0.0f;
}

__global__ void __launch_bounds__(32 * kWarps) k_distill_rows_warp(const Distill d) {
  const int lane = threadIdx.x & 31, V = (int)d.V_;
  const float scale = d.dl ? d.T / (float)max(1, *d.count) : 0.0f, c = kLog2e / d.T;
  for (int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); r < d.rows; r += (int64_t)gridDim.x * kWarps) {
    const float* row = d.logits + r * d.V_;
    const RowSlice sl = slice_of(row, V, 0, 0);
    const bool counted = d.flag[r];
    float* out = d.dl + r * d.V_;
    if (!counted) {
      if (lane == 0) d.part[r] = 0.0f;
      if (d.dl)
        for (int e = lane; e < V; e += 32) out[e] = 0.0f;
      continue;
    }
    float4 v[kNV];
#pragma unroll
    for (int k = 0; k < kNV; ++k) {
      const int g = k * 32 + lane;
      v[k] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (g >= sl.w0 && g < sl.w1) v[k] = sl.base[g];
      else if (g < sl.g1) v[k] = load_edge(row, V, 4 * g - sl.shift);
    }
    const RowStat st = warp_stat(v, c);
    const bool vec = (((uintptr_t)out >> 2) & 3) == (unsigned)sl.shift;
    if (d.dl) {
      distill_store(out, V, sl, v, lane, 32, scale / st.sum, vec);
      __syncwarp();   // the entries' columns are written again
    }
    const float ls = logf(st.sum), inv_T = 1.0f / d.T;
    float kl = 0.0f;
    for (int k = lane; k < d.K; k += 32) {
      const Entry e = d.ent[r * d.K + k];
      if (e.id < 0) continue;
      const float z = row[e.id];
      kl += entry_kl(e, z, st, ls, inv_T);
      if (d.dl && e.own != -1.0f) out[e.id] = scale * (tc::exp2_hw((z - st.max) * c) / st.sum - e.own);
    }
    kl = wsum(kl);
    if (lane == 0) d.part[r] = kl * (d.T * d.T);
  }
}

template <int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > kThreads ? 1 : 2) k_distill_rows(const Distill d) {
  extern __shared__ __align__(16) float4 land[];
  __shared__ float2 table[2 * kTable];
  __shared__ uint64_t bar, jbar[2];
  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), lc = 31 - __clz(cs), rank = (int)cl.block_rank(), V = (int)d.V_;
  const int64_t step = gridDim.x >> lc;
  Landing L;
  L.init(land, &bar, d.err);
  Join join;
  join.init(table, jbar, d.err, cl);
  const float scale = d.dl ? d.T / (float)max(1, *d.count) : 0.0f, c = kLog2e / d.T;
  int64_t r = blockIdx.x >> lc;
  RowSlice sl = slice_of(d.logits + r * d.V_, V, rank, lc);
  if (r < d.rows) L.issue(sl);
  // Entry k of a row is thread k's (and k + blockDim.x, ...), in the block whose
  // slice holds its column.  Its logit is read from the landing buffer and kept in
  // ze; the first entry of the next row is fetched a row ahead.
  float* ze = reinterpret_cast<float*>(land + d.land);
  const int tid = (int)threadIdx.x, nt = (int)blockDim.x;
  Entry first = {-1, 0.0f, 0.0f, -1.0f};
  if (r < d.rows && tid < d.K) first = d.ent[r * d.K + tid];
  const float inv_T = 1.0f / d.T;
  for (; r < d.rows; r += step) {
    const float* row = d.logits + r * d.V_;
    const RowSlice cur = sl;
    const bool counted = d.flag[r];
    L.wait();
    float4 v[kNV];
    L.take(v, cur, row, V);
    // columns of this block's slice, and the buffer as floats from its first one
    const int e0 = max(0, 4 * cur.g0 - cur.shift), e1 = min(V, 4 * cur.g1 - cur.shift);
    const Entry mine = first;
    if (counted)
      for (int k = tid; k < d.K; k += nt) {
        const int id = k == tid ? mine.id : d.ent[r * d.K + k].id;
        // a group that reaches past the row did not land
        if (id >= e0 && id < e1) {
          const int q = id + cur.shift;
          ze[k] = q >= 4 * cur.w0 && q < 4 * cur.w1 ? reinterpret_cast<const float*>(land)[q - 4 * cur.g0] : row[id];
        }
      }
    __syncthreads();   // the buffer is free
    if (r + step < d.rows) {
      sl = slice_of(row + step * d.V_, V, rank, lc);
      L.issue(sl);
      if (tid < d.K) first = d.ent[(r + step) * d.K + tid];
    }
    float* out = d.dl + r * d.V_;
    const int wp = (d.K + 31) / 32;   // warps of a block whose lanes have entries (at most all)
    float* part = d.part + r * d.parts + rank * (d.parts / cs);
    if (!counted) {
      if (tid < d.parts / cs) part[tid] = 0.0f;
      if (d.dl)
        for (int e = e0 + tid; e < e1; e += nt) out[e] = 0.0f;
      continue;   // uniform over the cluster
    }
    float f;
    const RowStat st = join(warp_stat(v, c), c, cl, &f);
    if (d.dl) {
      const bool vec = (((uintptr_t)out >> 2) & 3) == (unsigned)cur.shift;
      distill_store(out, V, cur, v, cur.g0 + tid, nt, f * scale / st.sum, vec);
      __syncthreads();   // the entries' columns are written again, by other threads of the block
    }
    if ((tid >> 5) < wp) {
      const float ls = logf(st.sum);
      float kl = 0.0f;
      for (int k = tid; k < d.K; k += nt) {
        const Entry e = k == tid ? mine : d.ent[r * d.K + k];
        if (e.id < e0 || e.id >= e1) continue;
        const float z = ze[k];
        kl += entry_kl(e, z, st, ls, inv_T);
        if (d.dl && e.own != -1.0f) out[e.id] = scale * (tc::exp2_hw((z - st.max) * c) / st.sum - e.own);
      }
      kl = wsum(kl);
      if ((tid & 31) == 0) part[tid >> 5] = kl * (d.T * d.T);
    }
  }
  if (cs > 1) cl.sync();   // no block leaves while another may still send to it
}

// ---- rows that fit a block's shared memory ----
// A row of up to kRingGroups 16-byte groups lies whole in shared memory, in chunks
// of two groups per thread.  One warp feeds it: as soon as every other warp is done
// with a chunk, the same chunk of the block's next row is on its way.  The other
// warps pass over the row twice: maximum and sum of exponentials as the chunks
// arrive, then the gradient.  Reads of the next row overlap the second pass and its
// stores, and nothing but one block barrier per row joins the warps.
constexpr int kRingWarps = 24, kRingChunks = 16;
constexpr int kRingGroups = 225 * 64;   // 225 KB

struct Ring {
  float4* row;                // [groups]
  uint32_t full, empty;       // kRingChunks barriers each
  int chunk, chunks, groups;  // groups: the row's, for any alignment
  uint32_t parity;            // of the row being read
  bool dead;
  int32_t* err;

  __device__ __forceinline__ uint32_t full_of(int j) const { return full + 8 * j; }
  __device__ __forceinline__ uint32_t empty_of(int j) const { return empty + 8 * j; }
  __device__ __forceinline__ void wait(uint32_t bar, uint32_t par, int code) {
    if (!dead) dead = !wait_for(bar, par, err, code);
  }
  __device__ __forceinline__ void release(int j) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(empty_of(j));
  }
};

// The feeding warp: rows first, first + step, ... below rows.
template <class Op>
__device__ __forceinline__ void ring_feed(Ring& R, const Op& op, int64_t first, int64_t step) {
  const int lane = threadIdx.x & 31;
  for (int64_t r = first, it = 0; r < op.rows && !R.dead; r += step, ++it) {
    const RowSlice s = slice_of(op.row(r), op.width(), 0, 0);
    for (int j = 0; j < R.chunks; ++j) {
      if (it) R.wait(R.empty_of(j), (uint32_t)(it - 1) & 1, 53);
      if (R.dead) break;
      const int lo = j * R.chunk, hi = min(lo + R.chunk, R.groups);
      // groups that are not four logits of the row: written by element, -inf past its end
      const int w0 = s.w0, w1 = (op.V() + s.shift) >> 2;
      if (lane == 0 && lo == 0 && w0) R.row[0] = load_edge(op.row(r), op.V(), -s.shift);
      for (int g = max(lo, w1) + lane; g < hi; g += 32) R.row[g] = load_edge(op.row(r), op.V(), 4 * g - s.shift);
      __syncwarp();
      if (lane == 0) {
        const int i0 = max(lo, w0), i1 = min(hi, w1);
        const uint32_t bytes = i1 > i0 ? (uint32_t)(i1 - i0) * 16 : 0;
        tc::mbar_expect_tx(R.full_of(j), bytes);
        if (bytes)
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(tc::smem_u32(R.row + i0)), "l"(s.base + i0), "r"(bytes), "r"(R.full_of(j))
                       : "memory");
      }
    }
  }
}

// First pass over the landed row: its maximum and sum, in every thread.  With
// `once` the chunks are given back as they are read.
__device__ __forceinline__ RowStat ring_stat(Ring& R, float c, float2* table, bool once) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2, lane = tid & 31, warps = nt >> 5;
  const float ninf = -INFINITY;
  float m = ninf, s = 0.0f;
  for (int j = 0; j < R.chunks; ++j) {
    R.wait(R.full_of(j), R.parity, 54);
    const int g = j * R.chunk + tid;
    float4 a = make_float4(ninf, ninf, ninf, ninf), b = a;
    if (g < R.groups) a = R.row[g];
    if (g + nt < R.groups) b = R.row[g + nt];
    if (once) R.release(j);
    const float mx = fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w)));
    const float mn = fmaxf(m, mx), m0 = mn == ninf ? 0.0f : mn;
    s *= tc::exp2_hw((m - m0) * c);
    m = mn;
    s += ((tc::exp2_hw((a.x - m0) * c) + tc::exp2_hw((a.y - m0) * c)) +
          (tc::exp2_hw((a.z - m0) * c) + tc::exp2_hw((a.w - m0) * c))) +
         ((tc::exp2_hw((b.x - m0) * c) + tc::exp2_hw((b.y - m0) * c)) +
          (tc::exp2_hw((b.z - m0) * c) + tc::exp2_hw((b.w - m0) * c)));
  }
  float2* t = table + R.parity * kRingWarps;   // two alternate: the barrier between keeps them apart
  float M = wmax(m);
  s = wsum(s * join_factor(m, M, c));
  if (lane == 0) t[tid >> 5] = make_float2(M, s);
  asm volatile("bar.sync 1, %0;" ::"r"(nt) : "memory");
  const float2 o = lane < warps ? t[lane] : make_float2(ninf, 0.0f);
  M = wmax(o.x);
  return {M, wsum(o.y * join_factor(o.x, M, c))};
}

// Second pass: f(group, its four exponentials exp((x - max) * c)), chunk by chunk.
template <class F>
__device__ __forceinline__ void ring_map(Ring& R, RowStat st, float c, F&& f) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2;
  const float m0 = st.max == -INFINITY ? 0.0f : st.max;
  for (int j = 0; j < R.chunks; ++j) {
    const int g = j * R.chunk + tid;
    float4 q[2];
    if (g < R.groups) q[0] = R.row[g];
    if (g + nt < R.groups) q[1] = R.row[g + nt];
    R.release(j);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g + i * nt < R.groups)
        f(g + i * nt, make_float4(tc::exp2_hw((q[i].x - m0) * c), tc::exp2_hw((q[i].y - m0) * c),
                                  tc::exp2_hw((q[i].z - m0) * c), tc::exp2_hw((q[i].w - m0) * c)));
  }
}

struct XentRows {
  float* logits;
  int ld, V_;
  int64_t rows;
  const void* tgt;
  int tdt;
  int64_t row0;
  float* nll;
  int32_t* err;
  __device__ __forceinline__ float* row(int64_t r) const { return logits + r * ld; }
  __device__ __forceinline__ int width() const { return ld; }   // groups cover the pitch
  __device__ __forceinline__ int V() const { return V_; }       // logits among them
};

__device__ __forceinline__ void ring_rows(Ring& R, const XentRows& d, float2* table, int64_t first, int64_t step) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2;
  int64_t next = first < d.rows ? id_at(d.tgt, d.tdt, d.row0 + first) : -1;
  for (int64_t r = first; r < d.rows; r += step, R.parity ^= 1) {
    float* row = d.row(r);
    const int64_t t = next;
    if (r + step < d.rows) next = id_at(d.tgt, d.tdt, d.row0 + r + step);
    if (t < 0 || t >= d.V_) {
      if (tid == 0) d.nll[d.row0 + r] = 0.0f;
      for (int j = 0; j < R.chunks; ++j) {   // the copies must have left the row before it is written
        R.wait(R.full_of(j), R.parity, 54);
        R.release(j);
      }
      asm volatile("bar.sync 1, %0;" ::"r"(nt) : "memory");
      for (int g = tid; g < R.groups; g += nt) store_planes(row, d.ld, 4 * g, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    const float zt = tid == 0 ? row[t] : 0.0f;
    const RowStat st = ring_stat(R, kLog2e, table, false);   // its barrier: the whole row has landed
    if (tid == 0) d.nll[d.row0 + r] = logf(st.sum) - (zt - st.max);
    const float f = 1.0f / st.sum;
    ring_map(R, st, kLog2e, [&](int g, float4 e) {
      float4 q = make_float4(e.x * f, e.y * f, e.z * f, e.w * f);
      const unsigned o = (unsigned)((int)t - 4 * g);
      if (o < 4) {
        if (o == 0) q.x -= 1.0f;
        if (o == 1) q.y -= 1.0f;
        if (o == 2) q.z -= 1.0f;
        if (o == 3) q.w -= 1.0f;
      }
      store_planes(row, d.ld, 4 * g, q);   // columns from V on hold exp(-inf) = 0
    });
  }
}

__device__ __forceinline__ void ring_rows(Ring& R, const Distill& d, float2* table, int64_t first, int64_t step) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2, V = (int)d.V_;
  const float scale = d.dl ? d.T / (float)max(1, *d.count) : 0.0f, c = kLog2e / d.T, inv_T = 1.0f / d.T;
  // Entry k of a row is thread k's (and k + nt, ...); the first of them is fetched a row ahead.
  Entry next = {-1, 0.0f, 0.0f, -1.0f};
  int next_flag = 0;
  if (first < d.rows) {
    next_flag = d.flag[first];
    if (tid < d.K) next = d.ent[first * d.K + tid];
  }
  for (int64_t r = first; r < d.rows; r += step, R.parity ^= 1) {
    const float* row = d.row(r);
    const RowSlice s = slice_of(row, V, 0, 0);
    float* out = d.dl + r * d.V_;
    float* part = d.part + r * d.parts;
    const Entry mine = next;
    const bool counted = next_flag;
    if (r + step < d.rows) {
      next_flag = d.flag[r + step];
      if (tid < d.K) next = d.ent[(r + step) * d.K + tid];
    }
    if (!counted) {
      if (tid < d.parts) part[tid] = 0.0f;
      for (int j = 0; j < R.chunks; ++j) {
        R.wait(R.full_of(j), R.parity, 54);
        R.release(j);
      }
      asm volatile("bar.sync 1, %0;" ::"r"(nt) : "memory");   // as every row: keeps the tables' turns
      if (d.dl)
        for (int e = tid; e < V; e += nt) out[e] = 0.0f;
      continue;
    }
    const float z0 = mine.id >= 0 ? row[mine.id] : 0.0f;
    const RowStat st = ring_stat(R, c, table, d.dl == nullptr);
    if (d.dl) {
      const bool vec = (((uintptr_t)out >> 2) & 3) == (unsigned)s.shift;
      float4* base = reinterpret_cast<float4*>(out - s.shift);
      const float f = scale / st.sum;
      ring_map(R, st, c, [&](int g, float4 e) {
        const float4 q = make_float4(e.x * f, e.y * f, e.z * f, e.w * f);
        if (vec && g >= s.w0 && g < s.w1) base[g] = q;
        else store_edge(out, V, 4 * g - s.shift, q);
      });
      asm volatile("bar.sync 1, %0;" ::"r"(nt) : "memory");   // the entries' columns are written again
    }
    if (tid < 32 * d.parts) {
      const float ls = logf(st.sum);
      float kl = 0.0f;
      for (int k = tid; k < d.K; k += nt) {
        const Entry e = k == tid ? mine : d.ent[r * d.K + k];
        if (e.id < 0) continue;
        const float z = k == tid ? z0 : row[e.id];
        kl += entry_kl(e, z, st, ls, inv_T);
        if (d.dl && e.own != -1.0f) out[e.id] = scale * (tc::exp2_hw((z - st.max) * c) / st.sum - e.own);
      }
      kl = wsum(kl);
      if ((tid & 31) == 0) part[tid >> 5] = kl * (d.T * d.T);
    }
  }
}

template <class Op>
__global__ void __launch_bounds__(32 * (kRingWarps + 1), 1) k_softmax_ring(const Op op, int groups) {
  extern __shared__ __align__(16) float4 land[];
  __shared__ uint64_t full[kRingChunks], empty[kRingChunks];
  __shared__ float2 table[2 * kRingWarps];
  const int warps = (int)(blockDim.x >> 5) - 1;
  Ring R;
  R.row = land;
  R.full = tc::smem_u32(full);
  R.empty = tc::smem_u32(empty);
  R.chunk = 64 * warps;
  R.chunks = (groups + R.chunk - 1) / R.chunk;
  R.groups = groups;
  R.parity = 0;
  R.dead = false;
  R.err = op.err;
  if (threadIdx.x == 0) {
    for (int j = 0; j < R.chunks; ++j) {
      tc::mbar_init(R.full_of(j), 1);
      tc::mbar_init(R.empty_of(j), (uint32_t)warps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if ((int)(threadIdx.x >> 5) == warps) ring_feed(R, op, blockIdx.x, gridDim.x);
  else ring_rows(R, op, table, blockIdx.x, gridDim.x);
}

template <class Op>
void launch_ring(const Op& op, int groups) {
  const int warps = std::min(kRingWarps, (groups + 511) / 512);   // 16 groups a thread, or a little more
  const size_t smem = (size_t)groups * 16;
  static std::mutex mu;
  static std::map<int, int> resident;   // blocks per SM, asked of the driver once per row length
  static size_t most = 0;
  std::lock_guard<std::mutex> lk(mu);
  if (smem > most) {
    MALUS_CUDA(cudaFuncSetAttribute(k_softmax_ring<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    most = smem;
  }
  int& res = resident[groups];
  if (!res) {
    MALUS_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&res, k_softmax_ring<Op>, 32 * (warps + 1), smem));
    if (res < 1) panic("softmax rows: no block of %d threads with %zu bytes can be resident", 32 * (warps + 1), smem);
  }
  const unsigned grid = (unsigned)std::min<int64_t>(op.rows, (int64_t)kNumSMs * res);
  k_softmax_ring<Op><<<grid, 32 * (warps + 1), smem, stream()>>>(op, groups);
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

// Blocks that stay: exactly as many clusters as the device holds at once (one
// more would start when the others have walked all their rows).
// `more`: dynamic shared memory behind the landing buffer.
template <class K, class... A>
void launch_rows(K kernel, int64_t rows, int64_t groups, int cs, int threads, size_t more, A... args) {
  const size_t smem = (size_t)((groups + cs - 1) / cs) * 16 + more;
  cudaLaunchConfig_t cfg = {};
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
  // asked of the driver once per kernel and row length
  static std::mutex mu;
  static std::map<std::pair<int64_t, size_t>, int> resident;
  static std::map<K, size_t> smem_set;
  std::lock_guard<std::mutex> lk(mu);
  if (size_t& most = smem_set[kernel]; smem > most) {
    MALUS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    most = smem;
  }
  int& res = resident[{groups, more}];
  if (!res) {
    cfg.gridDim = dim3((unsigned)(kNumSMs / cs * cs));
    MALUS_CUDA(cudaOccupancyMaxActiveClusters(&res, kernel, &cfg));
    if (res < 1) panic("softmax rows: no cluster of %d blocks can be resident", cs);
  }
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(rows, res) * cs));
  MALUS_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
}
unsigned warp_row_blocks(int64_t rows) {
  return (unsigned)std::min<int64_t>((rows + kWarps - 1) / kWarps, kNumSMs * 4);
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
  const int pid = prof_begin_named("k_xent_rows", 8.0 * (double)n * (double)ld);
  if (ld <= kShort)
    k_xent_rows_warp<<<warp_row_blocks(n), 32 * kWarps, 0, stream()>>>(logits, (int)ld, n, (int)V, targets, tgt_dtype, row0, nll);
  else if (ld / 4 <= kRingGroups)
    launch_ring(XentRows{logits, (int)ld, (int)V, n, targets, tgt_dtype, row0, nll, device_error_word()}, (int)(ld / 4));
  else if (!row_launch(ld / 4, &cs, &threads)) panic("softmax rows of %lld logits", (long long)V);
  else launch_rows(threads > kThreads ? k_xent_rows<kMaxThreads> : k_xent_rows<kThreads>, n, ld / 4, cs, threads, 0, logits, (int)ld, n, (int)V, targets, tgt_dtype, row0, nll, device_error_word());
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

void loss_mean(float* v, int64_t n, const int* count, float* loss) {
  k_loss_mean<<<1, 1024, 0, stream()>>>(v, nullptr, 0, n, count, loss);
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
  if (V > kMaxRowLogits - 4)
    panic("distill rows are limited to %lld logits, got %lld", (long long)kMaxRowLogits - 4, (long long)V);
  if (n > (int64_t)1 << 27) panic("distill is limited to 2^27 rows, got %lld", (long long)n);
  const float* x = fptr(logits);
  const void* idp = vptr(ids);
  const float* te = fptr(teacher);
  const int64_t loss = alloc_f32({1}), hk = alloc_f32({s.d[0]});
  const int64_t hd = dlogits ? alloc_shape(s) : 0;
  // a row may start 3 past an aligned address
  const int64_t groups = (V + 3 + 3) / 4;
  int cs = 1, threads = 0, parts = 1;
  const bool ring = V > kShort && groups <= kRingGroups;
  if (ring) {
    parts = std::min((int)(K + 31) / 32, std::min(kRingWarps, (int)(groups + 511) / 512));
  } else if (V > kShort) {
    if (!row_launch(groups, &cs, &threads)) panic("softmax rows of %lld logits", (long long)V);
    parts = cs * std::min((int)(K + 31) / 32, threads / 32);
  }
  char* ws = static_cast<char*>(scratch_alloc(16 + (size_t)(n * K) * sizeof(Entry) + (size_t)n * 4 * (1 + parts)));
  int* count = reinterpret_cast<int*>(ws);
  Entry* ent = reinterpret_cast<Entry*>(ws + 16);
  int* flag = reinterpret_cast<int*>(ent + n * K);
  float* part = reinterpret_cast<float*>(flag + n);
  MALUS_CUDA(cudaMemsetAsync(count, 0, 4, stream()));
  if (n) {
    const int land = (int)((groups + cs - 1) / cs);
    const Distill d{x, ent, flag, count, n, V, (int)K, temperature, part, hd ? fptr(hd) : nullptr, parts, land,
                    device_error_word()};
    k_teacher<<<grid_for((size_t)n * 32, 256), 256, (size_t)K * 32, stream()>>>(
        idp, idt, te, n, (int)K, V, kLog2e / temperature, ent, flag, count, device_error_word());
    const int pid = prof_begin_named("k_distill_rows", (hd ? 8.0 : 4.0) * (double)n * (double)V);
    if (V <= kShort) k_distill_rows_warp<<<warp_row_blocks(n), 32 * kWarps, 0, stream()>>>(d);
    else if (ring) launch_ring(d, (int)groups);
    else launch_rows(threads > kThreads ? k_distill_rows<kMaxThreads> : k_distill_rows<kThreads>, n, groups, cs, threads,
                     (size_t)K * 4, d);
    count_launch(2);
    after_launch("k_distill_rows");
    prof_end(pid);
  }
  k_loss_mean<<<1, 1024, 0, stream()>>>(fptr(hk), part, parts, n, count, fptr(loss));
  count_launch();
  after_launch("k_loss_mean");
  scratch_free(ws);
  if (kl) *kl = hk;
  else tensor_release(hk);
  if (dlogits) *dlogits = hd;
  return loss;
}

}  // extern "C"
