// LM head and softmax cross entropy in one operator, the logits never kept
// whole:
//
//   logits = x W^T,  nll = logsumexp(logits) - logits[target]
//   dl = (softmax(logits) - onehot(target)) / rows,  dx = dl W,  dW = dl^T x
//
// Training takes the tokens in pieces: a piece's logits live in a scratch of at
// most kPieceBytes, become the half planes of dl in place (loss_rows.cu), feed
// both gradient products and make room for the next piece.  That is the three
// products (6 N D V flops) and nothing computed twice; the scratch costs 4 B
// written and read per logit, then 4 B written and read by each product.  The
// loss alone stores no logits: the product's epilogue reduces each row of a tile
// to its maximum, sum of exponentials and target logit.
//
// All products run as three half-precision ones (gemm_f16.cuh).  x and weight
// are split twice, by rows and by columns, so that every product's operands are
// scaled along the axis it does not sum over.
#include "gemm_f16.cuh"
#include "loss_rows.cuh"

namespace malus {
namespace {

constexpr size_t kPieceBytes = (size_t)512 << 20;
// rows per statistics buffer of the loss alone (8 B per 128 logits)
constexpr size_t kLossRows = (size_t)1 << 18;

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
           int64_t ld, const Planes& wv, const Planes& xr, const int* count, float* nll, float* dx, float* dw) {
  // x by columns, tokens that are not counted as zeros: whatever they hold, dl
  // is 0 there; weight by columns (tied) or rows: an embedding axis per row
  Planes xc(dw ? D : 0, n), wd(dx ? D : 0, V);
  if (dw) f16_split_cols(x, n, D, xc.hi, xc.lo, xc.inv, tgt, tdt, V);
  if (dx && tied) f16_split_cols(w, V, D, wd.hi, wd.lo, wd.inv, nullptr, 0, 0);
  if (dx && !tied) f16_split_rows(w, D, V, wd.hi, wd.lo, wd.inv);
  // pieces of whole 256-row tiles, of even size
  const bool in_place = xent_rows_in_place(ld);
  const int64_t most = std::max<int64_t>(256, (int64_t)(kPieceBytes / ((size_t)ld * (in_place ? 4 : 8))) / 256 * 256);
  const int64_t pieces = (n + most - 1) / most;
  const int64_t piece = ((n + pieces - 1) / pieces + 255) / 256 * 256;
  float* logits = static_cast<float*>(scratch_alloc((size_t)std::min(piece, n) * ld * 4));
  float* planes = in_place ? logits : static_cast<float*>(scratch_alloc((size_t)std::min(piece, n) * ld * 4));
  const __half* hi = reinterpret_cast<const __half*>(planes);
  constexpr float inv = 1.0f / (1 << kF16Exp);
  for (int64_t r0 = 0; r0 < n; r0 += piece) {
    const int64_t m = std::min(piece, n - r0);
    F16Gemm g{(int)m, (int)V, (int)D, xr.kmajor(r0, m), wv.kmajor(0, V), logits, ld, false, nullptr};
    gemm_f16(g);
    xent_rows(logits, planes, ld, m, V, tgt, tdt, r0, nll);
    if (dx) {
      const F16Operand dl{hi, hi + ld, m, ld, 2 * ld, false, 0, nullptr, inv};
      gemm_f16({(int)m, (int)D, (int)V, dl, wd.kmajor(0, D), dx + r0 * D, D, false, count});
    }
    if (dw) {
      const F16Operand dl{hi, hi + ld, m, ld, 2 * ld, true, 0, nullptr, inv};
      const F16Operand xt = xc.kmajor(0, D, r0);
      if (tied) gemm_f16({(int)V, (int)D, (int)m, dl, xt, dw, D, r0 > 0, count});
      else gemm_f16({(int)D, (int)V, (int)m, xt, dl, dw, V, r0 > 0, count});
    }
  }
  if (!in_place) scratch_free(planes);
  scratch_free(logits);
}

void loss_only(const void* tgt, int tdt, int64_t n, int64_t D, int64_t V, const Planes& wv, const Planes& xr,
               float* nll) {
  const int parts = f16_lse_parts((int)V);
  const int64_t piece = std::min<int64_t>(n, kLossRows);
  float2* part = static_cast<float2*>(scratch_alloc((size_t)piece * (parts * 8 + 4)));
  float* at = reinterpret_cast<float*>(part + piece * parts);
  for (int64_t r0 = 0; r0 < n; r0 += piece) {
    const int64_t m = std::min(piece, n - r0);
    const void* t = static_cast<const char*>(tgt) + r0 * (int64_t)dtype_size(tdt);
    F16Gemm g{(int)m, (int)V, (int)D, xr.kmajor(r0, m), wv.kmajor(0, V), nullptr, 0, false, nullptr};
    gemm_f16_lse(g, part, at, t, tdt);
    xent_join(part, parts, at, t, tdt, V, m, nll + r0);
  }
  scratch_free(part);
}

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
  int* count = static_cast<int*>(scratch_alloc(4));
  xent_count(tp, tdt, (int64_t)n, (int64_t)V, count);
  if (n == 0) {
    if (hw) MALUS_CUDA(cudaMemsetAsync(fptr(hw), 0, V * D * 4, stream()));
  } else {
    const int64_t N = (int64_t)n;
    Planes wv(V, D);   // a vocabulary entry per row
    if (tied) f16_split_rows(wp, V, D, wv.hi, wv.lo, wv.inv);
    else f16_split_cols(wp, D, V, wv.hi, wv.lo, wv.inv, nullptr, 0, 0);
    Planes xr(N, D);   // a token per row
    f16_split_rows(xp, N, D, xr.hi, xr.lo, xr.inv);
    if (hx || hw) train(xp, wp, tp, tdt, tied != 0, N, (int64_t)D, (int64_t)V, ld, wv, xr, count, fptr(hn),
                        hx ? fptr(hx) : nullptr, hw ? fptr(hw) : nullptr);
    else loss_only(tp, tdt, N, (int64_t)D, (int64_t)V, wv, xr, fptr(hn));
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
