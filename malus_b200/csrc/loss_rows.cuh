// Row kernels of the softmax losses (loss_rows.cu): one pass over a row of
// logits gives its maximum, the sum of exponentials, the row's loss and, where
// wanted, the gradient row.
#pragma once
#include "common.cuh"

namespace malus {

// count[0] = rows whose target lies in [0, V); a target at or past V is reported
// in the runtime's error word (and its row left out, as a negative one's).
void xent_count(const void* targets, int tgt_dtype, int64_t n, int64_t V, int* count);

// Rows [0, n) of f32 logits (row pitch ld >= V, a multiple of 4) against targets[row0 ..]:
//   nll[row0 + r] = logsumexp - logits[target]   (0 for rows left out)
// and, with grad, the row in place becomes (softmax - onehot) (0 for rows left
// out and for the columns from V to ld).
void xent_rows(float* logits, int64_t ld, int64_t n, int64_t V, const void* targets, int tgt_dtype, int64_t row0,
               float* nll, bool grad);

// v[0 .. n) *= 1 / max(1, count[0])
void scale_by_count(float* v, int64_t n, const int* count);

// loss[0] = sum of v[0 .. n) / max(1, count[0])
void loss_mean(const float* v, int64_t n, const int* count, float* loss);

constexpr int64_t kMaxRowLogits = 262144;   // longest row (pitch) xent_rows takes

}  // namespace malus
