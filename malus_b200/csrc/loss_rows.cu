// Softmax losses by rows: for the head (linear_xent.cu) the cross entropy of a logits
// row against its target, and half planes of its gradient by tiles (k_xent_planes); and
// distillation from a teacher's top logits:
//
//   p = softmax over the row's entries of teacher / T,  q = softmax(logits / T)
//   kl = T^2 sum_k p_k (log p_k - log q[id_k]),  dlogits = T (q - p) / rows
//
// Rows, bound by HBM: 4 B read and 4 B written per logit.  Rows up to 1020 logits take
// a warp each, held in registers.  Longer ones take a block that stays and walks
// rows through a ring of shared-memory chunks: one warp feeds the ring by bulk
// copies, the others pass over a row twice, maximum and sum of exponentials first,
// then the gradient.  A row of up to 57 600 logits stays in the ring between the
// passes, and each of its chunks makes way for the next row's as the second pass
// is done with it, so reads, arithmetic and stores of neighbouring rows overlap and
// one block barrier per row is all that joins the warps.  Longer rows are fed
// twice, the second time mostly from L2.  (Rows held in registers over clusters of
// blocks, joined through distributed shared memory, measured 176 us against 137
// for 2048 x 50304 with its gradient: two such blocks per SM spend most of a row
// waiting for one another.)
#include "gemm_f16.cuh"
#include "loss_rows.cuh"
#include "tc_common.cuh"

#include <mutex>
#include <map>

namespace malus {
namespace {

constexpr int kNV = 8;            // float4 groups a lane holds of a short row, at most
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
struct RowView {
  const float4* base;   // group 0
  int shift;            // elements between the aligned address and the row
  int groups, w0, w1;
};
__device__ __forceinline__ RowView view_row(const float* row, int V) {
  RowView s;
  s.shift = (int)(((uintptr_t)row >> 2) & 3);
  s.base = reinterpret_cast<const float4*>(row - s.shift);
  s.groups = (V + s.shift + 3) >> 2;
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

// Maximum of a row and sum of exp((x - max) * c) over it.  Elements of -inf add 0;
// a row of -inf only, or with a +inf or NaN, gives NaN probabilities as the formula
// does.
struct RowStat { float max, sum; };

// Of a row held by one warp in v (-inf where a lane has no group); v becomes the
// exponentials.  The exponential is the hardware's base-2 one (relative error
// 2^-22; results below 2^-126 are 0).
template <int NV>
__device__ __forceinline__ RowStat warp_stat(float4 (&v)[NV], float c) {
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < NV; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
  m = wmax(m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
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

// Four probabilities (times `one`) from column e on, less 1 at the target.
__device__ __forceinline__ float4 less_hot(float4 q, int t, int e, float one = 1.0f) {
  const unsigned o = (unsigned)(t - e);
  if (o < 4) {
    if (o == 0) q.x -= one;
    if (o == 1) q.y -= one;
    if (o == 2) q.z -= one;
    if (o == 3) q.w -= one;
  }
  return q;
}

// The cross entropy's rows; the gradient in place.
struct XentRows {
  float* logits;
  bool grad;           // whether the gradient is wanted
  int ld, V_;
  int64_t rows;
  const void* tgt;
  int tdt;
  float* nll;
  int* count;          // counts the rows
  int32_t* err;
  __device__ __forceinline__ const float* row(int64_t r) const { return logits + r * ld; }
  __device__ __forceinline__ int width() const { return ld; }   // groups cover the pitch
  __device__ __forceinline__ int V() const { return V_; }       // logits among them
  // four elements of a row's gradient
  __device__ __forceinline__ void store(float* row_out, int e, float4 q) const {
    *reinterpret_cast<float4*>(row_out + e) = q;
  }
  // a row's value, by one thread
  __device__ __forceinline__ void tell(int64_t r, int64_t t, bool counted, float v) const {
    nll[r] = v;
    if (counted) atomicAdd(count, 1);   // whole numbers: the order does not matter
    else if (t >= V_) atomicExch(err, kErrId);
  }
};

template <int NV>
__global__ void __launch_bounds__(32 * kWarps) k_xent_rows_warp(const XentRows d) {
  const int lane = threadIdx.x & 31, ld = d.ld, V = d.V_;
  for (int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); r < d.rows; r += (int64_t)gridDim.x * kWarps) {
    float* row = d.logits + r * ld;
    const int64_t t = id_at(d.tgt, d.tdt, r);
    if (t < 0 || t >= V) {
      if (lane == 0) d.tell(r, t, false, 0.0f);
      if (!d.grad) continue;
      for (int g = lane; g < ld / 4; g += 32) d.store(row, 4 * g, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    const float zt = row[t];
    float4 v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int e = 4 * (k * 32 + lane);
      v[k] = e + 4 <= V ? *reinterpret_cast<const float4*>(row + e) : load_edge(row, V, e);
    }
    const RowStat st = warp_stat(v, kLog2e);   // the whole row is in registers after it
    __syncwarp();   // shuffles order no memory: every lane has read the row before one writes over it
    if (lane == 0) d.tell(r, t, true, logf(st.sum) - (zt - st.max));
    if (!d.grad) continue;
    const float f = 1.0f / st.sum;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int e = 4 * (k * 32 + lane);
      if (e < ld)   // columns from V on hold exp(-inf) = 0
        d.store(row, e, less_hot(make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f), (int)t, e));
    }
  }
}

__global__ void __launch_bounds__(1024) k_xent_count(const void* __restrict__ tgt, int tdt, int64_t n, int64_t V,
                                                     int* __restrict__ count, int32_t* __restrict__ err) {
  __shared__ int sh[32];
  int c = 0;
  bool bad = false;
  for (int64_t i = threadIdx.x; i < n; i += 8 * 1024) {
    int64_t t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = i + k * 1024 < n ? id_at(tgt, tdt, i + k * 1024) : -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      c += t[k] >= 0 && t[k] < V;
      bad |= t[k] >= V;
    }
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

// loss = sum of v / max(1, count); with parts, v[r] is first the sum of the row's
// parts; without count, the rows are counted here by their targets.
__global__ void __launch_bounds__(1024) k_loss_mean(float* __restrict__ v, const float* __restrict__ part, int parts,
                                                    int64_t n, const int* __restrict__ count, float* __restrict__ loss,
                                                    const void* __restrict__ tgt, int tdt, int64_t V,
                                                    int32_t* __restrict__ err) {
  __shared__ double sh[32];
  __shared__ int shc[32];
  double s = 0.0;
  int c = 0;
  if (parts) {
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
      float a = 0.0f;
#pragma unroll 8
      for (int j = 0; j < parts; ++j) a += part[i * parts + j];
      v[i] = a;
      s += (double)a;
    }
  } else {
    for (int64_t i = threadIdx.x; i < n; i += 8 * 1024) {
      float a[8];
      int64_t t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = i + k * 1024 < n;
        a[k] = in ? v[i + k * 1024] : 0.0f;
        t[k] = in && tgt ? id_at(tgt, tdt, i + k * 1024) : -1;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s += (double)a[k];
        c += t[k] >= 0 && t[k] < V;
        if (t[k] >= V) atomicExch(err, kErrId);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if ((threadIdx.x & 31) == 0) {
    sh[threadIdx.x >> 5] = s;
    shc[threadIdx.x >> 5] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    c = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) {
      s += sh[i];
      c += shc[i];
    }
    loss[0] = (float)(s / (double)max(1, count ? count[0] : c));
  }
}

// nll of row r from its parts' (maximum, sum of exponentials) and its target's logit,
// and what its gradient takes, by W threads (a warp, or one)
template <int W>
__device__ __forceinline__ XentStat join_row(const XentParts& p, int64_t V, int64_t r) {
  const int lane = W == 32 ? threadIdx.x & 31 : 0;
  const int64_t t = id_at(p.tgt, p.tdt, r);
  if (t < 0 || t >= V) return {0.0f, 0.0f, -1, 0.0f};
  const float2* part = p.part + r * p.parts;
  float M = -INFINITY, s = 0.0f;
  for (int i = lane; i < p.parts; i += W) M = fmaxf(M, part[i].x);
  if (W == 32) M = wmax(M);
  for (int i = lane; i < p.parts; i += W) {
    const float2 o = part[i];
    s += o.y * (o.x == -INFINITY ? 1.0f : exp2f((o.x - M) * kLog2e));   // -inf only: the sum is 0 or NaN
  }
  if (W == 32) s = wsum(s);
  return {M == -INFINITY ? 0.0f : M, 1.0f / s, (int)t, logf(s) - (p.at[r] - M)};
}
__global__ void __launch_bounds__(256) k_xent_join(const XentParts p, int64_t V, int64_t n, float* __restrict__ nll,
                                                   XentStat* __restrict__ stat) {
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < n; r += (int64_t)gridDim.x * 8) {
    const XentStat s = join_row<32>(p, V, r);
    if ((threadIdx.x & 31) == 0) {
      nll[r] = s.nll;
      if (stat) stat[r] = s;
    }
  }
}

// A tile of kF16Block rows and 64 columns of f32 logits to the half planes of dl =
// softmax - onehot, in the grouped layout of F16Operand, in one pass: 4 B read per
// logit and 4 B written per set of planes (2048 x 50304, both sets: 197 us, 6.3 TB/s; with
// 256 threads of 16 groups each 265 us).  EVEN: at one scale,
// 2^kDlExp, for a product that sums over the vocabulary, where the largest of a
// token's gradients sets the accuracy.  ENTRY: scaled per vocabulary entry by the
// largest of its column in the tile, for the product that sums over the tokens:
// there each entry's row of dweight has a size of its own, from 1 down to the
// smallest floats.  One of the sets may lie over the logits: a tile's planes cover
// just the bytes of its logits.  Columns from V on are zeros, and rows left out.
// Rows of few parts (stat null) are joined here, by every tile of theirs, and the
// first one writes their nll.
constexpr int kTileThreads = 512;
static_assert(kTileThreads >= kF16Block, "a thread per row");

// Two scaled values as halves, hi and what is left.
__device__ __forceinline__ void split_pair(float x, float y, uint32_t* h, uint32_t* l) {
  const __half2 hi = __floats2half2_rn(x, y);
  const float2 b = __half22float2(hi);
  const __half2 lo = __floats2half2_rn(x - b.x, y - b.y);
  *h = *reinterpret_cast<const uint32_t*>(&hi);
  *l = *reinterpret_cast<const uint32_t*>(&lo);
}
__device__ __forceinline__ void store_split(__half* p, float4 v) {
  uint2 h, l;
  split_pair(v.x, v.y, &h.x, &l.x);
  split_pair(v.z, v.w, &h.y, &l.y);
  *reinterpret_cast<uint2*>(p) = h;
  *reinterpret_cast<uint2*>(p + 64) = l;
}

template <bool EVEN, bool ENTRY>
__global__ void __launch_bounds__(kTileThreads, 1024 / kTileThreads)
k_xent_planes(const float* logits, int64_t ld, int64_t n, int64_t V, const XentStat* __restrict__ stat, const XentParts p,
              float* __restrict__ nll, __half* even, __half* entry, float* __restrict__ inv, int64_t inv_pitch) {
  constexpr int kStep = kTileThreads / 16, kRows = kF16Block / kStep, kTileWarps = kTileThreads / 32;
  constexpr float one = (float)(1 << kDlExp);
  __shared__ XentStat st[kF16Block];
  __shared__ __align__(16) float sh[kTileWarps][64], ups[64];
  const int groups = (int)(ld / 64), g = (int)(blockIdx.x % groups), tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t block = blockIdx.x / groups, r0 = block * kF16Block;
  const int c = g * 64 + 4 * tx, rows = (int)min((int64_t)kF16Block, n - r0);
  float4 q[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = ty + kStep * i;
    q[i] = r < rows ? *reinterpret_cast<const float4*>(logits + (r0 + r) * ld + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (threadIdx.x < kF16Block) {
    const int64_t r = r0 + threadIdx.x;
    XentStat s = {0.0f, 0.0f, -1, 0.0f};
    if (threadIdx.x < rows) {
      s = stat ? stat[r] : join_row<1>(p, V, r);
      if (!stat && g == 0) nll[r] = s.nll;
    }
    st[threadIdx.x] = s;
  }
  __syncthreads();
  float cm[4] = {};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const XentStat s = st[ty + kStep * i];
    if (s.target < 0) {
      q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      continue;
    }
    const float f = s.inv_sum * one;   // dl times 2^kDlExp
    q[i].x = tc::exp2_hw((q[i].x - s.max) * kLog2e) * f;
    q[i].y = tc::exp2_hw((q[i].y - s.max) * kLog2e) * f;
    q[i].z = tc::exp2_hw((q[i].z - s.max) * kLog2e) * f;
    q[i].w = tc::exp2_hw((q[i].w - s.max) * kLog2e) * f;
    if (c + 4 > V) {
      if (c >= V) q[i].x = 0.0f;
      if (c + 1 >= V) q[i].y = 0.0f;
      if (c + 2 >= V) q[i].z = 0.0f;
      q[i].w = 0.0f;
    }
    q[i] = less_hot(q[i], s.target, c, one);
    if (ENTRY) {   // a NaN passes by: its row makes all of dweight NaN
      cm[0] = fmaxf(cm[0], fabsf(q[i].x));
      cm[1] = fmaxf(cm[1], fabsf(q[i].y));
      cm[2] = fmaxf(cm[2], fabsf(q[i].z));
      cm[3] = fmaxf(cm[3], fabsf(q[i].w));
    }
  }
  float4 up = make_float4(one, one, one, one);
  if (ENTRY) {
#pragma unroll
    for (int j = 0; j < 4; ++j) cm[j] = fmaxf(cm[j], __shfl_xor_sync(0xffffffffu, cm[j], 16));
    if ((threadIdx.x & 16) == 0)
      *reinterpret_cast<float4*>(&sh[threadIdx.x >> 5][4 * tx]) = make_float4(cm[0], cm[1], cm[2], cm[3]);
    __syncthreads();
    if (threadIdx.x < 64) {   // a column's scale
      float m = 0.0f, u, iv;
      for (int k = 0; k < kTileWarps; ++k) m = fmaxf(m, sh[k][threadIdx.x]);
      f16_scale(__float_as_uint(m), &u, &iv);
      ups[threadIdx.x] = u;
      inv[block * inv_pitch + g * 64 + threadIdx.x] = iv * (1.0f / one);
    }
    __syncthreads();
    up = *reinterpret_cast<const float4*>(ups + 4 * tx);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = ty + kStep * i;
    if (r >= rows) break;
    const int64_t at = (r0 + r) * 2 * ld + g * 128 + 4 * tx;
    if (EVEN) store_split(even + at, q[i]);
    if (ENTRY) store_split(entry + at, make_float4(q[i].x * up.x, q[i].y * up.y, q[i].z * up.z, q[i].w * up.w));
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
  extern __shared__ int sid[];   // [8][2][K]: the rows' ids (-1: no entry) and p
  __shared__ int sh[8];
  const int lane = threadIdx.x & 31;
  int* mine = sid + (threadIdx.x >> 5) * 2 * K;
  float* ps = reinterpret_cast<float*>(mine + K);
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
      ps[k] = te;
      if (there) {
        m = fmaxf(m, te);
        any = true;
      }
    }
    if (bad) atomicExch(err, kErrId);
    m = wmax(m);
    any = __any_sync(0xffffffffu, any);
    float s = 0.0f;
    for (int k = lane; k < K; k += 32)
      if (mine[k] >= 0) s += exp2f((ps[k] - m) * c);
    s = wsum(s);
    const float ls = logf(s);
    __syncwarp();   // the other lanes' ids
    for (int k = lane; k < K; k += 32) {
      const int id = mine[k];
      const float z = (ps[k] - m) * c;   // base-2 units
      float sum = id >= 0 ? exp2f(z) / s : -1.0f;
      const float p = id >= 0 ? sum : 0.0f;
      if (id >= 0)
#pragma unroll 8
        for (int j = 0; j < K; ++j)
          if (mine[j] == id && j != k) {
            if (j < k) {
              sum = -1.0f;
              break;
            }
            sum += exp2f((ps[j] - m) * c) / s;
          }
      ent[o + k] = {id, p, z * kLn2 - ls, sum};
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
  int32_t* err;
  __device__ __forceinline__ const float* row(int64_t r) const { return logits + r * V_; }
  __device__ __forceinline__ int width() const { return (int)V_; }
  __device__ __forceinline__ int V() const { return (int)V_; }
};

// The part of an entry with logit z in its row's kl.
__device__ __forceinline__ float entry_kl(const Entry& e, float z, RowStat st, float log_sum, float inv_T) {
  return e.p != 0.0f ? e.p * (e.lp - ((z - st.max) * inv_T - log_sum)) : 0.0f;
}

template <int NV>
__global__ void __launch_bounds__(32 * kWarps) k_distill_rows_warp(const Distill d) {
  const int lane = threadIdx.x & 31, V = (int)d.V_;
  const float scale = d.dl ? d.T / (float)max(1, *d.count) : 0.0f, c = kLog2e / d.T;
  for (int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); r < d.rows; r += (int64_t)gridDim.x * kWarps) {
    const float* row = d.logits + r * d.V_;
    const RowView sl = view_row(row, V);
    const bool counted = d.flag[r];
    float* out = d.dl + r * d.V_;
    if (!counted) {
      if (lane == 0) d.part[r] = 0.0f;
      if (d.dl)
        for (int e = lane; e < V; e += 32) out[e] = 0.0f;
      continue;
    }
    float4 v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int g = k * 32 + lane;
      v[k] = g >= sl.w0 && g < sl.w1 ? sl.base[g] : load_edge(row, V, 4 * g - sl.shift);
    }
    const RowStat st = warp_stat(v, c);
    const bool vec = (((uintptr_t)out >> 2) & 3) == (unsigned)sl.shift;
    if (d.dl) {
      const float f = scale / st.sum;
      float4* base = reinterpret_cast<float4*>(out - sl.shift);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int g = k * 32 + lane;
        const float4 q = make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f);
        if (vec && g >= sl.w0 && g < sl.w1) base[g] = q;
        else if (g < sl.groups) store_edge(out, V, 4 * g - sl.shift, q);
      }
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

// ---- longer rows: the ring ----
constexpr int kRingWarps = 24, kRingSlots = 16;
constexpr int kRingGroups = 225 * 64;   // 225 KB of 16-byte groups

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

// Chunks of two groups per thread, fed one after another into `slots` slots: a
// row's chunks once where each has a slot of its own (STAY), else twice.
template <bool STAY_>
struct Ring {
  static constexpr bool STAY = STAY_;
  float4* buf;
  uint32_t full, empty;       // kRingSlots barriers each
  int chunk, chunks, slots;   // groups per chunk, chunks per row (of any alignment)
  int groups;
  bool dead;
  int slot;                   // of the next chunk (unless STAY: then chunk j has slot j)
  uint32_t round;             // how often the slots went round (STAY: rows done)
  int32_t* err;

  __device__ __forceinline__ uint32_t full_of(int i) const { return full + 8 * i; }
  __device__ __forceinline__ uint32_t empty_of(int i) const { return empty + 8 * i; }
  __device__ __forceinline__ int at(int j) const { return STAY ? j : slot; }
  __device__ __forceinline__ void step() {   // after each chunk
    if (!STAY && ++slot == slots) {
      slot = 0;
      ++round;
    }
  }
  __device__ __forceinline__ void row_done() {
    if (STAY) ++round;
  }
  __device__ __forceinline__ void wait_full(int i, uint32_t rnd) {
    if (!dead) dead = !wait_for(full_of(i), rnd & 1, err, 54);
  }
  // this warp is done with slot i
  __device__ __forceinline__ void release(int i) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(empty_of(i));
  }
};

// The feeding warp: rows first, first + step, ... below rows.  At most 32 groups
// follow a row's whole ones: its pitch is less than 64 elements longer, or its
// alignment adds one.
template <class R_, class Op>
__device__ __forceinline__ void ring_feed(R_& R, const Op& op, int64_t first, int64_t step) {
  const int lane = threadIdx.x & 31;
  // groups that are not four logits of the row are written by element, -inf past
  // its end: the first (lane 0) and those from w1 on (one per lane); they are
  // fetched a row ahead
  auto w1_of = [&](const RowView& v) { return (op.V() + v.shift) >> 2; };   // whole groups of logits end here
  RowView s, ns;
  float4 head, tail, nhead, ntail;
  auto fetch = [&](int64_t r) {
    ns = view_row(op.row(r), op.width());
    if (lane == 0 && ns.w0) nhead = load_edge(op.row(r), op.V(), -ns.shift);
    ntail = load_edge(op.row(r), op.V(), 4 * (w1_of(ns) + lane) - ns.shift);
  };
  if (first < op.rows) fetch(first);
  for (int64_t r = first; r < op.rows && !R.dead; r += step, R.row_done()) {
    s = ns;
    head = nhead;
    tail = ntail;
    if (r + step < op.rows) fetch(r + step);
    const int w1 = w1_of(s);
    for (int j = 0; j < (R_::STAY ? 1 : 2) * R.chunks; ++j, R.step()) {
      const int slot = R.at(j);
      if (R.round && !R.dead) R.dead = !wait_for(R.empty_of(slot), (R.round - 1) & 1, R.err, 53);
      if (R.dead) break;
      // what this slot held was written by element at its row's ends, and read, before
      // the copy may land on it
      tc::fence_async_smem();
      const int lo = (j < R.chunks ? j : j - R.chunks) * R.chunk, hi = min(lo + R.chunk, R.groups);
      float4* at = R.buf + slot * R.chunk - lo;
      if (lane == 0 && lo == 0 && s.w0) at[0] = head;
      if (w1 + lane >= lo && w1 + lane < hi) at[w1 + lane] = tail;
      __syncwarp();
      if (lane == 0) {
        const int i0 = max(lo, s.w0), i1 = min(hi, w1);
        const uint32_t bytes = i1 > i0 ? (uint32_t)(i1 - i0) * 16 : 0;
        tc::mbar_expect_tx(R.full_of(slot), bytes);
        if (bytes)
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(tc::smem_u32(at + i0)), "l"(s.base + i0), "r"(bytes), "r"(R.full_of(slot))
                       : "memory");
      }
    }
  }
}

template <class R_>
__device__ __forceinline__ void ring_barrier(const R_& R) {   // of the warps that do not feed
  asm volatile("bar.sync 1, %0;" ::"r"(R.chunk / 2) : "memory");
}

// First pass over a row: its maximum and sum, in every thread.  With `once` there
// is no second pass and the chunks are given back here (a row that does not stay
// is fed twice all the same: ring_skip).
template <class R_>
__device__ __forceinline__ RowStat ring_stat(R_& R, float c, float2* table, uint32_t turn, bool once) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2, lane = tid & 31, warps = nt >> 5;
  const float ninf = -INFINITY;
  const bool give = once || !R_::STAY;
  float m = ninf, s = 0.0f;
  for (int j = 0; j < R.chunks; ++j, R.step()) {
    const int slot = R.at(j);
    R.wait_full(slot, R.round);
    const int g = j * R.chunk + tid;
    const float4* at = R.buf + slot * R.chunk + tid;
    float4 a = make_float4(ninf, ninf, ninf, ninf), b = a;
    if (g < R.groups) a = at[0];
    if (g + nt < R.groups) b = at[nt];
    if (give) R.release(slot);
    const float mx = fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w)));
    const float mn = fmaxf(m, mx), m0 = mn == ninf ? 0.0f : mn;
    s *= tc::exp2_hw((m - m0) * c);
    m = mn;
    s += ((tc::exp2_hw((a.x - m0) * c) + tc::exp2_hw((a.y - m0) * c)) +
          (tc::exp2_hw((a.z - m0) * c) + tc::exp2_hw((a.w - m0) * c))) +
         ((tc::exp2_hw((b.x - m0) * c) + tc::exp2_hw((b.y - m0) * c)) +
          (tc::exp2_hw((b.z - m0) * c) + tc::exp2_hw((b.w - m0) * c)));
  }
  float2* t = table + (turn & 1) * kRingWarps;   // two alternate: the barrier between keeps them apart
  float M = wmax(m);
  s = wsum(s * join_factor(m, M, c));
  if (lane == 0) t[tid >> 5] = make_float2(M, s);
  ring_barrier(R);
  const float2 o = lane < warps ? t[lane] : make_float2(ninf, 0.0f);
  M = wmax(o.x);
  return {M, wsum(o.y * join_factor(o.x, M, c))};
}

// Gives a row's chunks back unread, `times` over; they have landed when it returns.
template <class R_>
__device__ __forceinline__ void ring_skip(R_& R, int times) {
  for (int j = 0; j < times * R.chunks; ++j, R.step()) {
    R.wait_full(R.at(j), R.round);
    R.release(R.at(j));
  }
}

// Second pass: f(group, its four exponentials exp((x - max) * c)), chunk by chunk.
template <class R_, class F>
__device__ __forceinline__ void ring_map(R_& R, RowStat st, float c, F&& f) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2;
  const float m0 = st.max == -INFINITY ? 0.0f : st.max;
  for (int j = 0; j < R.chunks; ++j, R.step()) {
    const int slot = R.at(j);
    if (!R_::STAY) R.wait_full(slot, R.round);
    const int g = j * R.chunk + tid;
    const float4* at = R.buf + slot * R.chunk + tid;
    float4 q[2];
    if (g < R.groups) q[0] = at[0];
    if (g + nt < R.groups) q[1] = at[nt];
    R.release(slot);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g + i * nt < R.groups)
        f(g + i * nt, make_float4(tc::exp2_hw((q[i].x - m0) * c), tc::exp2_hw((q[i].y - m0) * c),
                                  tc::exp2_hw((q[i].z - m0) * c), tc::exp2_hw((q[i].w - m0) * c)));
  }
}

template <class R_>
__device__ __forceinline__ void ring_rows(R_& R, const XentRows& d, float2* table, int64_t first, int64_t step) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2;
  int64_t next = first < d.rows ? id_at(d.tgt, d.tdt, first) : -1;
  uint32_t turn = 0;
  for (int64_t r = first; r < d.rows; r += step, ++turn, R.row_done()) {
    float* row = d.logits + r * d.ld;
    const int64_t t = next;
    if (r + step < d.rows) next = id_at(d.tgt, d.tdt, r + step);
    if (t < 0 || t >= d.V_) {
      if (tid == 0) d.tell(r, t, false, 0.0f);
      ring_skip(R, R_::STAY ? 1 : 2);   // the copies have left the row before it is written
      ring_barrier(R);
      if (d.grad)
        for (int g = tid; g < R.groups; g += nt) d.store(row, 4 * g, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    const float zt = tid == 0 ? row[t] : 0.0f;
    const RowStat st = ring_stat(R, kLog2e, table, turn, !d.grad);   // its barrier: a row that stays has landed
    if (tid == 0) d.tell(r, t, true, logf(st.sum) - (zt - st.max));
    if (!d.grad) {
      if (!R_::STAY) ring_skip(R, 1);
      continue;
    }
    const float f = 1.0f / st.sum;
    ring_map(R, st, kLog2e, [&](int g, float4 e) {   // columns from V on hold exp(-inf) = 0
      d.store(row, 4 * g, less_hot(make_float4(e.x * f, e.y * f, e.z * f, e.w * f), (int)t, 4 * g));
    });
  }
}

template <class R_>
__device__ __forceinline__ void ring_rows(R_& R, const Distill& d, float2* table, int64_t first, int64_t step) {
  const int tid = (int)threadIdx.x, nt = R.chunk / 2, V = (int)d.V_;
  const float scale = d.dl ? d.T / (float)max(1, *d.count) : 0.0f, c = kLog2e / d.T, inv_T = 1.0f / d.T;
  // Entry k of a row is thread k's (and k + nt, ...); the first of them is fetched a row ahead.
  Entry next = {-1, 0.0f, 0.0f, -1.0f};
  int next_flag = 0;
  if (first < d.rows) {
    next_flag = d.flag[first];
    if (tid < d.K) next = d.ent[first * d.K + tid];
  }
  uint32_t turn = 0;
  for (int64_t r = first; r < d.rows; r += step, ++turn, R.row_done()) {
    const float* row = d.row(r);
    const RowView s = view_row(row, V);
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
      ring_skip(R, R_::STAY ? 1 : 2);
      ring_barrier(R);   // as every row: keeps the tables' turns
      if (d.dl)
        for (int e = tid; e < V; e += nt) out[e] = 0.0f;
      continue;
    }
    const float z0 = mine.id >= 0 ? row[mine.id] : 0.0f;
    const RowStat st = ring_stat(R, c, table, turn, d.dl == nullptr);
    if (!d.dl && !R_::STAY) ring_skip(R, 1);
    if (d.dl) {
      const bool vec = (((uintptr_t)out >> 2) & 3) == (unsigned)s.shift;
      float4* base = reinterpret_cast<float4*>(out - s.shift);
      const float f = scale / st.sum;
      ring_map(R, st, c, [&](int g, float4 e) {
        const float4 q = make_float4(e.x * f, e.y * f, e.z * f, e.w * f);
        if (vec && g >= s.w0 && g < s.w1) base[g] = q;
        else store_edge(out, V, 4 * g - s.shift, q);
      });
      ring_barrier(R);   // the entries' columns are written again
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

template <bool STAY, class Op>
__global__ void __launch_bounds__(32 * (kRingWarps + 1), 1) k_softmax_ring(const Op op, int groups, int slots) {
  extern __shared__ __align__(16) float4 land[];
  __shared__ uint64_t full[kRingSlots], empty[kRingSlots];
  __shared__ float2 table[2 * kRingWarps];
  const int warps = (int)(blockDim.x >> 5) - 1;
  Ring<STAY> R;
  R.buf = land;
  R.full = tc::smem_u32(full);
  R.empty = tc::smem_u32(empty);
  R.chunk = 64 * warps;
  R.chunks = (groups + R.chunk - 1) / R.chunk;
  R.slots = slots;
  R.groups = groups;
  R.slot = 0;
  R.round = 0;
  R.dead = false;
  R.err = op.err;
  if (threadIdx.x == 0) {
    for (int j = 0; j < slots; ++j) {
      tc::mbar_init(R.full_of(j), 1);
      tc::mbar_init(R.empty_of(j), (uint32_t)warps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if ((int)(threadIdx.x >> 5) == warps) ring_feed(R, op, blockIdx.x, gridDim.x);
  else ring_rows(R, op, table, blockIdx.x, gridDim.x);
}

// Warps of the ring for rows of `groups` groups: 16 groups a thread, or a little
// more.  A row that stays has all its chunks in slots, the last one cut short.
int ring_warps(int64_t groups) { return (int)std::min<int64_t>(kRingWarps, (groups + 511) / 512); }

template <bool STAY, class Op>
void launch_ring(const Op& op, int groups) {
  const int warps = ring_warps(groups), chunk = 64 * warps;
  const int slots = STAY ? (groups + chunk - 1) / chunk : kRingGroups / chunk;
  const size_t smem = (size_t)(STAY ? groups : slots * chunk) * 16;
  auto* kernel = k_softmax_ring<STAY, Op>;
  static std::mutex mu;
  static std::map<int, int> resident;   // blocks per SM, asked of the driver once per row length
  static size_t most = 0;
  std::lock_guard<std::mutex> lk(mu);
  if (smem > most) {
    MALUS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    most = smem;
  }
  int& res = resident[groups];
  if (!res) {
    MALUS_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&res, kernel, 32 * (warps + 1), smem));
    if (res < 1) panic("softmax rows: no block of %d threads with %zu bytes can be resident", 32 * (warps + 1), smem);
  }
  const unsigned grid = (unsigned)std::min<int64_t>(op.rows, (int64_t)kNumSMs * res);
  kernel<<<grid, 32 * (warps + 1), smem, stream()>>>(op, groups, slots);
}
template <class Op>
void launch_ring(const Op& op, int groups) {
  if (groups <= kRingGroups) launch_ring<true>(op, groups);
  else launch_ring<false>(op, groups);
}

// Short rows: f(number of float4 groups a lane holds, as a constant; blocks).
template <class F>
void with_warp_rows(int64_t groups, int64_t rows, F&& f) {
  const int nv = (int)((groups + 31) / 32);
  const unsigned blocks = (unsigned)std::min<int64_t>((rows + kWarps - 1) / kWarps, kNumSMs * (nv > 2 ? 4 : 8));
  if (nv <= 1) f.template operator()<1>(blocks);
  else if (nv <= 2) f.template operator()<2>(blocks);
  else if (nv <= 4) f.template operator()<4>(blocks);
  else f.template operator()<kNV>(blocks);
}
struct XentShort {
  const XentRows& d;
  template <int NV>
  void operator()(unsigned blocks) const { k_xent_rows_warp<NV><<<blocks, 32 * kWarps, 0, stream()>>>(d); }
};
struct DistillShort {
  const Distill& d;
  template <int NV>
  void operator()(unsigned blocks) const { k_distill_rows_warp<NV><<<blocks, 32 * kWarps, 0, stream()>>>(d); }
};

}  // namespace

void xent_count(const void* targets, int tgt_dtype, int64_t n, int64_t V, int* count) {
  k_xent_count<<<1, 1024, 0, stream()>>>(targets, tgt_dtype, n, V, count, device_error_word());
  count_launch();
  after_launch("k_xent_count");
}

void xent_planes(const float* logits, int64_t ld, int64_t n, int64_t V, const XentParts& p, float* nll, __half* even,
                 __half* entry, float* inv, int64_t inv_pitch) {
  const int64_t blocks = (n + kF16Block - 1) / kF16Block * (ld / 64);
  if (blocks > INT32_MAX) panic("xent_planes: %lld tiles", (long long)blocks);
  // up to 1024 entries a tile's threads join their rows themselves (training 16384 x 384
  // x 65: 130 us, 136 with a launch for it)
  XentStat* stat = nullptr;
  if (p.parts > 8) {
    stat = static_cast<XentStat*>(scratch_alloc((size_t)n * sizeof(XentStat)));
    xent_join(p, V, n, nll, stat);
  }
  const int pid = prof_begin_named("k_xent_planes", (even && entry ? 12.0 : 8.0) * (double)n * (double)ld);
  auto go = [&](auto kernel) {
    kernel<<<(unsigned)blocks, kTileThreads, 0, stream()>>>(logits, ld, n, V, stat, p, nll, even, entry, inv, inv_pitch);
  };
  if (even && entry) go(k_xent_planes<true, true>);
  else if (even) go(k_xent_planes<true, false>);
  else go(k_xent_planes<false, true>);
  count_launch();
  after_launch("k_xent_planes");
  prof_end(pid);
  scratch_free(stat);
}

void xent_rows_f32(float* logits, int64_t ld, int64_t n, int64_t V, const void* targets, int tgt_dtype, float* nll,
                   int* count, bool grad) {
  if (n == 0) return;
  const XentRows d{logits, grad, (int)ld, (int)V, n, targets, tgt_dtype, nll, count, device_error_word()};
  const int pid = prof_begin_named("k_xent_rows", (grad ? 8.0 : 4.0) * (double)n * (double)ld);
  if (ld <= kShort) with_warp_rows(ld / 4, n, XentShort{d});
  else launch_ring(d, (int)(ld / 4));
  count_launch();
  after_launch("k_xent_rows");
  prof_end(pid);
}

void xent_join(const XentParts& p, int64_t V, int64_t n, float* nll, XentStat* stat) {
  if (n == 0) return;
  k_xent_join<<<grid_for((size_t)n * 32, 256), 256, 0, stream()>>>(p, V, n, nll, stat);
  count_launch();
  after_launch("k_xent_join");
}

void loss_mean(float* v, int64_t n, const int* count, float* loss) {
  k_loss_mean<<<1, 1024, 0, stream()>>>(v, nullptr, 0, n, count, loss, nullptr, 0, 0, nullptr);
  count_launch();
  after_launch("k_loss_mean");
}

void loss_mean_counted(float* v, int64_t n, const void* targets, int tgt_dtype, int64_t V, float* loss) {
  k_loss_mean<<<1, 1024, 0, stream()>>>(v, nullptr, 0, n, nullptr, loss, targets, tgt_dtype, V, device_error_word());
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
  if (temperature < 0x1p-60f || temperature > 0x1p60f)   // its square and its inverse stay floats
    panic("distill temperature must lie between 2^-60 and 2^60, got %g", (double)temperature);
  const int64_t n = (int64_t)s.d[0], V = (int64_t)s.d[1], K = (int64_t)si.d[1];
  if (V == 0) panic("distill over an empty vocabulary");
  if (K < 1 || K > kMaxEntries) panic("distill takes 1 to %d teacher entries per row, got %lld", kMaxEntries, (long long)K);
  if (V > kMaxRowLogits) panic("distill rows are limited to %lld logits, got %lld", (long long)kMaxRowLogits, (long long)V);
  if (n > (int64_t)1 << 27) panic("distill is limited to 2^27 rows, got %lld", (long long)n);
  const float* x = fptr(logits);
  const void* idp = vptr(ids);
  const float* te = fptr(teacher);
  const int64_t loss = alloc_f32({1}), hk = alloc_f32({s.d[0]});
  const int64_t hd = dlogits ? alloc_shape(s) : 0;
  // a row may start 3 past an aligned address
  const int64_t groups = (V + 3 + 3) / 4;
  const int parts = V > kShort ? std::min((int)(K + 31) / 32, ring_warps(groups)) : 1;
  char* ws = static_cast<char*>(scratch_alloc(16 + (size_t)(n * K) * sizeof(Entry) + (size_t)n * 4 * (1 + parts)));
  int* count = reinterpret_cast<int*>(ws);
  Entry* ent = reinterpret_cast<Entry*>(ws + 16);
  int* flag = reinterpret_cast<int*>(ent + n * K);
  float* part = reinterpret_cast<float*>(flag + n);
  MALUS_CUDA(cudaMemsetAsync(count, 0, 4, stream()));
  if (n) {
    const Distill d{x, ent, flag, count, n, V, (int)K, temperature, part, hd ? fptr(hd) : nullptr, parts,
                    device_error_word()};
    if (K > 512)   // past the default limit from 768 on; the same limit for every thread's calls
      MALUS_CUDA(cudaFuncSetAttribute(k_teacher, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxEntries * 64));
    k_teacher<<<grid_for((size_t)n * 32, 256), 256, (size_t)K * 64, stream()>>>(
        idp, idt, te, n, (int)K, V, kLog2e / temperature, ent, flag, count, device_error_word());
    const int pid = prof_begin_named("k_distill_rows", (hd ? 8.0 : 4.0) * (double)n * (double)V);
    if (V <= kShort) with_warp_rows(groups, n, DistillShort{d});
    else launch_ring(d, (int)groups);
    count_launch(2);
    after_launch("k_distill_rows");
    prof_end(pid);
  }
  k_loss_mean<<<1, 1024, 0, stream()>>>(fptr(hk), part, parts, n, count, fptr(loss), nullptr, 0, 0, nullptr);
  count_launch();
  after_launch("k_loss_mean");
  scratch_free(ws);
  if (kl) *kl = hk;
  else tensor_release(hk);
  if (dlogits) *dlogits = hd;
  return loss;
}

}  // extern "C"
