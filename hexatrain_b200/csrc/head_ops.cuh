// head_ops.cuh -- the operators on rows of logits, for callers within the library:
// top_logits.cu, distill.cu, sample_logits.cu.  Each checks its arguments, fails
// by hx::Error and enqueues on the runtime's stream.
#pragma once

#include "hx_internal.cuh"

namespace hx {
namespace head {

struct TopArgs {
    const void* logits;
    size_t stride;
    float* values;
    int32_t* indices;
    float* lse;  // may be NULL
    int* err;
    uint32_t vocab, k;
    float tau;
};
void top_logits(hx_runtime* rt, int dtype, uint32_t rows, TopArgs a);

struct DistillArgs {
    const void* logits;
    void* d_logits;  // NULL: forward only
    size_t stride, grad_stride;
    const float* teacher_values;
    const int32_t* teacher_indices;
    const float* teacher_lse;  // NULL: renormalised record
    const int32_t* labels;     // NULL: no hard targets
    const float* grad_loss;    // NULL: 1 for every row
    float* loss;               // NULL in the backward
    float* stats;              // [rows, 3] logsumexp(l/tau), logsumexp(l), q_T/p_T; may be NULL in the fused form
    int* err;
    uint32_t vocab, k;
    float tau, kd, ce, grad_scale;
    int exact_inverse = 0;  // set by distill(): 1 / tau is exact (tau a power of two)
};
// backward: the gradient from a.stats; otherwise the loss, with the gradient where
// a.d_logits is given.
void distill(hx_runtime* rt, int dtype, uint32_t rows, DistillArgs a, bool backward);

struct SampleArgs {
    const void* logits;
    size_t stride;
    const float* uniform;
    const float* temperature;  // NULL: 1
    const int32_t* top_k;      // NULL or <= 0: the whole vocabulary
    const float* top_p;        // NULL or >= 1: off
    const float* min_p;        // NULL or <= 0: off
    int32_t* tokens;
    float* log_probs;  // may be NULL
    uint32_t vocab;
};
void sample_logits(hx_runtime* rt, int dtype, uint32_t rows, const SampleArgs& a);

}  // namespace head
}  // namespace hx
