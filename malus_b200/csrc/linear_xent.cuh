// The head's cross entropy by the size of the problem (linear_xent.cu).
#pragma once
#include "common.cuh"

namespace malus {

// Whether a problem takes f32 multiply-adds (head_small.cu).
bool head_small(int64_t n, int64_t D, int64_t V, bool grad);
// loss, nll, and dx and dw where not null.
void head_small_run(const float* x, const float* w, const void* tgt, int tdt, bool tied, int64_t n, int64_t D, int64_t V,
                    float* nll, float* loss, float* dx, float* dw);

}  // namespace malus
