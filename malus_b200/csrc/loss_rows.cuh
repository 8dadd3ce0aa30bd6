// Row kernels of the softmax losses (loss_rows.cu): one pass over a row of
// logits gives its maximum, the sum of exponentials, the row's loss and, where
// wanted, the gradient row.
#pragma once
#include "common.cuh"

namespace malus {

// count[0] = rows whose target lies in [0, V); a target at or past V is reported
// in the runtime's error word (and its row left out, as a negative one's).
void xent_count(const void* targets, int tgt_dtype, int64_t n, int64_t V, int* count);

// Rows [0, n) of f32 logits (row pitch ld >= V, a multiple of 64) against
// targets[row0 ..]: nll[row0 + r] = logsumexp - logits[target] (0 for rows left
// out), and the half planes of 2^kF16Exp (softmax - onehot): hi in the first ld
// halves of row r of `planes` (pitch ld floats), lo in the next ld; zeros for rows
// left out and for the columns from V to ld.  planes may be logits itself where
// xent_rows_in_place(ld).
bool xent_rows_in_place(int64_t ld);
void xent_rows(const float* logits, float* planes, int64_t ld, int64_t n, int64_t V, const void* targets, int tgt_dtype,
               int64_t row0, float* nll);

// The same with the gradient as f32 in place (none without grad), counting the rows
// into count[0] (cleared before) and reporting targets at or past V.  A row takes
// any length: f32 in place only ever overwrites what has been read.
void xent_rows_f32(float* logits, int64_t ld, int64_t n, int64_t V, const void* targets, int tgt_dtype, float* nll,
                   int* count, bool grad);

// nll[r] of n rows from the statistics of gemm_f16_lse
void xent_join(const float2* part, int parts, const float* at, const void* targets, int tgt_dtype, int64_t V, int64_t n,
               float* nll);

// loss[0] = sum of v[0 .. n) / max(1, count[0])
void loss_mean(float* v, int64_t n, const int* count, float* loss);

// The same, counting the rows whose target lies in [0, V) (and reporting those at or
// past V).
void loss_mean_counted(float* v, int64_t n, const void* targets, int tgt_dtype, int64_t V, float* loss);

constexpr int64_t kMaxRowLogits = (int64_t)1 << 24;   // longest row

}  // namespace malus
