// LM head and softmax cross entropy in one operator, the logits never kept
// whole:
//
//   logits = x W^T,  nll = logsumexp(logits) - logits[target]
//   dl = (softmax(logits) - onehot(target)) / rows,  dx = dl W,  dW = dl^T x
//
// Tokens are taken in pieces: a piece's logits live in a scratch of at most
// kPieceBytes, become dl in place, feed both gradient products and make room
// for the next piece.  Training costs the three products (6 N D V flops) and
// nothing is computed twice.
#include "loss_rows.cuh"

namespace malus {
namespace {

constexpr size_t kPieceBytes = (size_t)512 << 20;

}  // namespace
}  // namespace malus

using namespace malus;

extern "C" {

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
  const bool grad = hx || hw;
  int* count = static_cast<int*>(scratch_alloc(4));
  xent_count(tp, tdt, (int64_t)n, (int64_t)V, count);
  const size_t piece = std::max<size_t>(64, std::min<size_t>((n + 63) / 64 * 64, kPieceBytes / (ld * 4) / 64 * 64));
  float* logits = static_cast<float*>(scratch_alloc(piece * ld * 4));
  for (size_t r0 = 0; r0 < n; r0 += piece) {
    const int m = (int)std::min(piece, n - r0);
    const GemmOperand X = plain_operand(xp + r0 * D, 1, m, D, D, 0);
    const GemmOperand W = plain_operand(wp, 1, sw.d[0], sw.d[1], sw.d[1], 0);
    const GemmOperand L = plain_operand(logits, 1, m, V, ld, 0);
    GemmArgs g{};
    g.M = m; g.N = (int)V; g.K = (int)D; g.batch = 1;
    g.A = X; g.B = W; g.b_trans = tied != 0;
    g.C = logits; g.ldc = ld;
    gemm(g);
    xent_rows(logits, ld, m, (int64_t)V, tp, tdt, (int64_t)r0, fptr(hn), grad);
    if (hx) {
      GemmArgs q{};
      q.M = m; q.N = (int)D; q.K = (int)V; q.batch = 1;
      q.A = L; q.B = W; q.b_trans = tied == 0;
      q.C = fptr(hx) + r0 * D; q.ldc = D;
      gemm(q);
    }
    if (hw) {
      GemmArgs q{};
      q.K = m; q.batch = 1;
      q.a_trans = true;
      if (tied) { q.M = (int)V; q.N = (int)D; q.A = L; q.B = X; }
      else { q.M = (int)D; q.N = (int)V; q.A = X; q.B = L; }
      q.C = fptr(hw); q.ldc = q.N;
      q.beta = r0 ? 1.0f : 0.0f;
      gemm(q);
    }
  }
  scratch_free(logits);
  if (hx && n) scale_by_count(fptr(hx), n * D, count);
  if (hw) {
    if (n) scale_by_count(fptr(hw), V * D, count);
    else MALUS_CUDA(cudaMemsetAsync(fptr(hw), 0, V * D * 4, stream()));
  }
  loss_mean(fptr(hn), (int64_t)n, count, fptr(loss));
  scratch_free(count);
  if (nll) *nll = hn;
  else tensor_release(hn);
  if (dx) *dx = hx;
  if (dweight) *dweight = hw;
  return loss;
}

}  // extern "C"
