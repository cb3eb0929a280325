// distill.cu -- distillation from a teacher's top logits, forward and backward.
//
// Row by row, with z = l / tau, p = softmax(z) and teacher entries (t_j, i_j):
//   q_j = exp(t_j/tau - logsumexp_j(t_j/tau))             (renormalised record), or
//   q_j = exp(t_j/tau - lse_teacher), q_T = 1 - sum_j q_j (record with a tail bucket),
//   KL  = sum_j q_j (log q_j - log p_{i_j}) [+ q_T (log q_T - log p_T)],
//   p_T = the student's mass outside the record, summed directly: 1 - sum p
//         would cancel where the student is sure,
//   loss = kd tau^2 KL + ce (logsumexp(l) - l_label),
//   dloss/dl_i = kd tau (p_i c_i - q_i) + ce (softmax(l)_i - [i = label]),
//   c_i = 1 (renormalised, or i named by the record), 1 - q_T/p_T (elsewhere).
// No counterpart in the reference, whose loss is the hard-label cross-entropy
// (tiny_language_model_cpu.cpp:77); that is kd = 0, ce = 1 here.
#include <cmath>

#include "head_rows.cuh"

namespace hx {
namespace head {

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
};

constexpr int kDistillThreads = 256;

// One block per row; the row is read once for the maximum, once for the sums
// and once for the gradient.
template <class T, bool kBackward>
__global__ void __launch_bounds__(kDistillThreads)
distill_row_kernel(const DistillArgs a)
{
    HX_PDL_PROLOGUE();
    constexpr int NT = kDistillThreads;
    extern __shared__ uint32_t named[];  // bit i: the record names token i (tail only)
    __shared__ float red[NT / 32];
    const size_t row = blockIdx.x;
    const int V = int(a.vocab), k = int(a.k), tid = threadIdx.x;
    const T* l = static_cast<const T*>(a.logits) + row * a.stride;
    const bool tail = a.teacher_lse != nullptr;

    // the teacher's record: thread j holds entry j
    int idx = -1;
    float logq = -INFINITY, q = 0.f, lj = 0.f;
    if (tail) {
        for (int w = tid; w < (V + 31) / 32; w += NT) named[w] = 0u;
        __syncthreads();
    }
    if (tid < k) {
        idx = a.teacher_indices[row * k + tid];
        if (idx >= V) {
            atomicCAS(a.err, 0, kBadIndexCode);
            idx = -1;
        }
        if (idx >= 0) {
            logq = __fdiv_rn(a.teacher_values[row * k + tid], a.tau);
            lj = to_float(l[idx]);
            if (tail) atomicOr(&named[idx >> 5], 1u << (idx & 31));
        }
    }
    const bool has = __syncthreads_or(idx >= 0 && (tail || logq != -INFINITY)) != 0;
    if (tail) {
        logq -= a.teacher_lse[row];
    } else {
        const float mt = block_reduce<NT>(logq, red, MaxOp());
        const float st = block_reduce<NT>(has && idx >= 0 ? expf(logq - mt) : 0.f, red, SumOp());
        logq -= mt + logf(st);
    }
    if (idx >= 0 && has) q = expf(logq);
    int label = a.labels ? a.labels[row] : -1;
    if (label >= V) {
        if (tid == 0) atomicCAS(a.err, 0, kBadIndexCode);
        label = -1;
    }
    const float l_label = label >= 0 ? to_float(l[label]) : 0.f;

    const float c_tau = __fdiv_rn(kLog2e, a.tau);
    float lse_tau, lse_1, ratio = 0.f;
    if (!kBackward) {
        float m = -INFINITY;
        for (int i = tid; i < V; i += NT) m = fmaxf(m, to_float(l[i]));
        m = block_reduce<NT>(m, red, MaxOp());
        const float off = m == -INFINITY ? 0.f : m;
        float s = 0.f, s1 = 0.f, sT = 0.f;
        for (int i = tid; i < V; i += NT) {
            const float d = to_float(l[i]) - off;
            const float e = tc::exp2_approx(d * c_tau);
            s += e;
            s1 += tc::exp2_approx(d * kLog2e);
            if (tail && !((named[i >> 5] >> (i & 31)) & 1u)) sT += e;
        }
        s = block_reduce<NT>(s, red, SumOp());
        s1 = block_reduce<NT>(s1, red, SumOp());
        lse_tau = __fdiv_rn(off, a.tau) + logf(s);
        lse_1 = off + logf(s1);
        float kl = q > 0.f ? q * (logq - (__fdiv_rn(lj, a.tau) - lse_tau)) : 0.f;
        kl = block_reduce<NT>(kl, red, SumOp());
        if (tail) {
            sT = block_reduce<NT>(sT, red, SumOp());
            const float sq = block_reduce<NT>(q, red, SumOp());
            const float pT = sT / s;
            const float qT = has && pT > 0.f ? fmaxf(1.f - sq, 0.f) : 0.f;
            if (qT > 0.f) {
                kl += qT * (logf(qT) - logf(pT));
                ratio = qT / pT;
            }
        }
        if (tid == 0) {
            float loss = a.kd != 0.f ? a.kd * a.tau * a.tau * kl : 0.f;
            if (label >= 0) loss += a.ce * (lse_1 - l_label);
            if (a.loss) a.loss[row] = loss;
            if (a.stats) {
                a.stats[row * 3] = lse_tau;
                a.stats[row * 3 + 1] = lse_1;
                a.stats[row * 3 + 2] = ratio;
            }
        }
    } else {
        lse_tau = a.stats[row * 3];
        lse_1 = a.stats[row * 3 + 1];
        ratio = a.stats[row * 3 + 2];
    }
    if (!a.d_logits) return;

    T* d = static_cast<T*>(a.d_logits) + row * a.grad_stride;
    const float gs = a.grad_scale * (a.grad_loss ? a.grad_loss[row] : 1.f);
    const float A = has ? gs * a.kd * a.tau : 0.f, B = label >= 0 ? gs * a.ce : 0.f;
    const float o_tau = lse_tau * kLog2e, o_1 = lse_1 * kLog2e;
    auto p_tau = [&](float x) { return tc::exp2_approx(fmaf(x, c_tau, -o_tau)); };
    auto p_1 = [&](float x) { return tc::exp2_approx(fmaf(x, kLog2e, -o_1)); };
    const float rest = A * (1.f - ratio);
    __syncthreads();  // every entry's logit is read before d may overwrite it
    for (int i = tid; i < V; i += NT) {
        const float x = to_float(l[i]);
        float g = 0.f;
        if (A != 0.f) g = rest * p_tau(x);
        if (B != 0.f) g += B * p_1(x);
        d[i] = from_float<T>(g);
    }
    // the record's tokens and the label, whose gradients have terms of their own
    const bool label_named = __syncthreads_or(label >= 0 && idx == label) != 0;
    if (idx >= 0) {
        float g = 0.f;
        if (A != 0.f) g = A * (p_tau(lj) - q);
        if (B != 0.f) g += B * (p_1(lj) - (idx == label ? 1.f : 0.f));
        d[idx] = from_float<T>(g);
    }
    if (tid == 0 && label >= 0 && !label_named) {
        float g = 0.f;
        if (A != 0.f) g = rest * p_tau(l_label);
        if (B != 0.f) g += B * (p_1(l_label) - 1.f);
        d[label] = from_float<T>(g);
    }
}

template <class T>
void launch_distill(hx_runtime* rt, const DistillArgs& a, uint32_t rows, bool backward)
{
    const size_t smem = a.teacher_lse ? size_t((a.vocab + 31) / 32) * 4 : 0;
    auto k = backward ? distill_row_kernel<T, true> : distill_row_kernel<T, false>;
    pdl_launch(k, rows, kDistillThreads, smem, rt->stream, a);
    HX_LAUNCHED(rt);
}

void distill(hx_runtime* rt, int dtype, uint32_t rows, DistillArgs a, bool backward)
{
    check_logits("distillation", dtype, rows, a.vocab, a.logits, a.stride);
    require(a.k >= 1 && a.k <= kMaxTop && a.k <= a.vocab, HX_ERR_ARGUMENT,
            "distillation: record length must be in [1, min(256, vocabulary)]");
    require(std::isfinite(a.tau) && a.tau > 0.f && std::isfinite(1.f / a.tau), HX_ERR_ARGUMENT,
            "distillation: temperature must be positive and finite");
    require(std::isfinite(a.kd) && std::isfinite(a.ce) && std::isfinite(a.grad_scale), HX_ERR_ARGUMENT,
            "distillation: weights and gradient scale must be finite");
    if (rows == 0) return;
    require(a.teacher_values && a.teacher_indices, HX_ERR_ARGUMENT, "distillation: null teacher record");
    if (a.d_logits) {
        require(a.grad_stride >= a.vocab, HX_ERR_ARGUMENT, "distillation: gradient row stride below the vocabulary size");
        require(reinterpret_cast<uintptr_t>(a.d_logits) % element_bytes(dtype) == 0, HX_ERR_ARGUMENT,
                "distillation: gradient not aligned to its type");
        require(a.d_logits != a.logits || a.grad_stride == a.stride, HX_ERR_ARGUMENT,
                "distillation: a gradient in place needs the logits' row stride");
    }
    a.err = rt->device_error();
    ProfScope prof(rt, kTagSoftmaxCe, 6.0 * rows * a.vocab,
                   double(element_bytes(dtype)) * rows * a.vocab * (a.d_logits ? 2.0 : 1.0));
    if (dtype == HX_DTYPE_F32) launch_distill<float>(rt, a, rows, backward);
    else if (dtype == HX_DTYPE_BF16) launch_distill<__nv_bfloat16>(rt, a, rows, backward);
    else launch_distill<__half>(rt, a, rows, backward);
}

}  // namespace head
}  // namespace hx

extern "C" {

int hx_distill_forward_device(hx_runtime* rt, int dtype, uint32_t rows, uint32_t vocab, const void* logits,
                              size_t stride, uint32_t k, const float* teacher_values, const int32_t* teacher_indices,
                              const float* teacher_lse, const int32_t* labels, float temperature, float kd_weight,
                              float ce_weight, float* loss, float* stats) {
    return hx_guard(rt, [&] {
        hx::require(rows == 0 || (loss && stats), HX_ERR_ARGUMENT, "distillation: null output");
        hx::head::distill(rt, dtype, rows,
                          {logits, nullptr, stride, 0, teacher_values, teacher_indices, teacher_lse, labels, nullptr,
                           loss, stats, nullptr, vocab, k, temperature, kd_weight, ce_weight, 1.f}, false);
    });
}

int hx_distill_backward_device(hx_runtime* rt, int dtype, uint32_t rows, uint32_t vocab, const void* logits,
                               size_t stride, uint32_t k, const float* teacher_values, const int32_t* teacher_indices,
                               const float* teacher_lse, const int32_t* labels, float temperature, float kd_weight,
                               float ce_weight, const float* stats, const float* grad_loss, float grad_scale,
                               void* d_logits, size_t grad_stride) {
    return hx_guard(rt, [&] {
        hx::require(rows == 0 || (stats && d_logits), HX_ERR_ARGUMENT, "distillation: null statistics or output");
        hx::head::distill(rt, dtype, rows,
                          {logits, d_logits, stride, grad_stride, teacher_values, teacher_indices, teacher_lse, labels,
                           grad_loss, nullptr, const_cast<float*>(stats), nullptr, vocab, k, temperature, kd_weight,
                           ce_weight, grad_scale}, true);
    });
}

int hx_distill_forward_backward_device(hx_runtime* rt, int dtype, uint32_t rows, uint32_t vocab, const void* logits,
                                       size_t stride, uint32_t k, const float* teacher_values,
                                       const int32_t* teacher_indices, const float* teacher_lse, const int32_t* labels,
                                       float temperature, float kd_weight, float ce_weight, const float* grad_loss,
                                       float grad_scale, float* loss, void* d_logits, size_t grad_stride) {
    return hx_guard(rt, [&] {
        hx::require(rows == 0 || (loss && d_logits), HX_ERR_ARGUMENT, "distillation: null output");
        hx::head::distill(rt, dtype, rows,
                          {logits, d_logits, stride, grad_stride, teacher_values, teacher_indices, teacher_lse, labels,
                           grad_loss, loss, nullptr, nullptr, vocab, k, temperature, kd_weight, ce_weight, grad_scale},
                          false);
    });
}

}  // extern "C"
