// f32 GEMM through three half-precision products (gemm_f16.cu).
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

namespace malus {

// A matrix of f32 values held as two half planes: value = (hi + lo) * inv, with
// inv a power of two per row of the product's M or N (or one for all).  Both
// planes have `pitch` halves per stored row, a multiple of 64, zero past the
// matrix.  K-major: stored rows are M (or N), columns K.  MN-major: stored rows
// are K, columns M (or N).
struct F16Operand {
  const __half *hi, *lo;
  int64_t rows, cols, pitch;
  bool mn_major;
  int64_t k0;          // first K column read (K-major only; a multiple of 64)
  const float* inv;    // per M (or N) index; null: inv_all
  float inv_all;
  // Each 64 columns of a stored row hold their hi halves, then their lo halves
  // (`lo` is hi + 64, pitch covers both).
  bool grouped = false;
  // MN-major only, in place of inv: a scale per kF16Block rows of K and M (or N)
  // index, rows of block_pitch floats, padded as f16_scales says.
  const float* block_inv = nullptr;
  int64_t block_pitch = 0;
};
constexpr int kF16Block = 256;   // rows of K under one block_inv: an accumulator's

// out[m * ldo + n] = A B^T / max(1, count[0]) (count null: as it is), added to
// what is there with accumulate.  A B operand with per-row scales has them
// padded to whole tiles of 256 (f16_scales).
struct F16Gemm {
  int M, N, K;
  F16Operand a, b;
  float* out;
  int64_t ldo;
  bool accumulate;
  const int* count;
};
void gemm_f16(const F16Gemm& g);

// Row statistics of A B^T: part[m * parts + i] = (maximum, sum of exp(value -
// maximum)) over the i-th 128 columns, parts = f16_lse_parts(N), and at[m] = the
// value in column target[m] (rows whose target lies outside [0, N) get none).  The
// product itself is stored too where out is not null (16-byte rows).
int f16_lse_parts(int N);
void gemm_f16_lse(const F16Gemm& g, float2* part, float* at, const void* target, int tgt_dtype);

// Planes of a row-major R x C matrix: its rows (rhi/rlo [R][pad64(C)], rinv[R]), and
// its columns (chi/clo [C][pad64(R)], cinv[C]).  Each plane row is scaled by the
// power of two that brings its largest finite magnitude into [2^13, 2^14).
// keep (columns only, may be null): rows whose keep id lies outside [0, limit)
// are taken as zeros.
struct F16Split {
  const float* src;
  int64_t R;
  __half *rhi, *rlo;
  float* rinv;
  __half *chi, *clo;
  float* cinv;
  const void* keep;
  int keep_dtype;
  int64_t limit;
};
void f16_split_rows(const float* src, int64_t R, int64_t C, __half* hi, __half* lo, float* inv);
// With count (zero before), here and below: count[0] has the first matrix's kept rows
// after it, and ids at or past its limit are reported in the error word.
void f16_split_cols(const F16Split& job, int64_t C, int* count = nullptr);
// Both of one or two matrices (R > 0) of C columns.  bits: n * C words, zero.
void f16_split_both(const F16Split* jobs, int n, int64_t C, uint32_t* bits, int* count);
__host__ __device__ inline int64_t pad64(int64_t v) { return (v + 63) / 64 * 64; }

// floats behind the scales of `rows` plane rows: a GEMM reads whole tiles of them
inline int64_t f16_scales(int64_t rows) { return (rows + 255) / 256 * 256; }

constexpr int kF16Exp = 13;   // scaled magnitudes stay below 2^(kF16Exp + 1)

// The power of two that brings a magnitude (its bits) into [2^13, 2^14), and its
// inverse; 1 for zero.  Both stay normal numbers.
__device__ __forceinline__ void f16_scale(uint32_t bits, float* up, float* inv) {
  int e = (int)(bits >> 23) - 127;              // floor(log2), -127 for subnormals
  int s = bits ? kF16Exp - e : 0;
  s = s > 126 ? 126 : s < -113 ? -113 : s;
  *up = __uint_as_float((uint32_t)(s + 127) << 23);
  *inv = __uint_as_float((uint32_t)(127 - s) << 23);
}
__device__ __forceinline__ uint32_t f16_finite_bits(float x) {   // bits of |x|; 0 for inf and NaN
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b >= 0x7f800000u ? 0u : b;
}
__device__ __forceinline__ void f16_split(float x, __half* h, __half* l) {
  *h = __float2half_rn(x);
  *l = __float2half_rn(x - __half2float(*h));
}

}  // namespace malus
