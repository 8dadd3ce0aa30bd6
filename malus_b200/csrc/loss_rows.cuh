// Row kernels of the softmax losses (loss_rows.cu): one pass over a row of
// logits gives its maximum, the sum of exponentials, the row's loss and, where
// wanted, the gradient row.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

namespace malus {

// count[0] = rows whose target lies in [0, V); a target at or past V is reported
// in the runtime's error word (and its row left out, as a negative one's).
void xent_count(const void* targets, int tgt_dtype, int64_t n, int64_t V, int* count);

// The statistics that gemm_f16_lse leaves of n rows, and their targets.
struct XentParts {
  const float2* part;
  int parts;
  const float* at;
  const void* tgt;
  int tdt;
};
// What a row's gradient takes: its maximum, 1 / (sum of exponentials), and its target
// (-1: the row is left out); and its value.
struct __align__(16) XentStat {
  float max, inv_sum;
  int target;
  float nll;
};
// nll[r], and stat[r] where not null
void xent_join(const XentParts& p, int64_t V, int64_t n, float* nll, XentStat* stat);

constexpr int kDlExp = 15;   // magnitudes of softmax - onehot are at most 1: 2^15 is half's last power of two

// nll[r], and half planes of softmax - onehot, from n > 0 rows of f32 logits (row pitch
// ld >= V, a multiple of 64; what lies from V on is not looked at), in the grouped
// layout with a pitch of 2 ld halves: `even` all at 2^kDlExp; `entry` scaled per
// kF16Block rows and vocabulary entry, with the inverse scales in inv (rows of
// inv_pitch >= ld floats).  Either may be null, not both, and one of them may lie over
// the logits.
void xent_planes(const float* logits, int64_t ld, int64_t n, int64_t V, const XentParts& p, float* nll, __half* even,
                 __half* entry, float* inv, int64_t inv_pitch);

// Rows [0, n) of f32 logits (row pitch ld >= V, a multiple of 64) against their
// targets: nll[r] = logsumexp - logits[target] (0 for rows left out) and, with grad,
// softmax - onehot in place; zeros for rows left out and for the columns from V to ld.
// Counts the rows into count[0] (cleared before) and reports targets at or past V.
void xent_rows_f32(float* logits, int64_t ld, int64_t n, int64_t V, const void* targets, int tgt_dtype, float* nll,
                   int* count, bool grad);

// loss[0] = sum of v[0 .. n) / max(1, count[0])
void loss_mean(float* v, int64_t n, const int* count, float* loss);

// The same, counting the rows whose target lies in [0, V) (and reporting those at or
// past V).
void loss_mean_counted(float* v, int64_t n, const void* targets, int tgt_dtype, int64_t V, float* loss);

constexpr int64_t kMaxRowLogits = (int64_t)1 << 24;   // longest row

}  // namespace malus
