// top_logits.cu -- the k largest logits of every row and its log-sum-exp.
//
// Order: value descending, index ascending among equals; NaN after -inf.  With
// keys whose ascending order is that of descending values, the k-th key is the
// smallest t with count(key <= t) >= k; the record is every key below t and
// the first keys equal to t in index order.  lse = m/tau + log sum exp((l-m)/tau).
// No counterpart in the reference, whose sampler sorts the whole row on the
// host (nicopedia_generation.h:286-395).
#include <cmath>

#include "head_rows.cuh"

namespace hx {
namespace head {

struct TopArgs {
    const void* logits;
    size_t stride;
    float* values;
    int32_t* indices;
    float* lse;  // may be NULL
    uint32_t vocab, k;
    float tau;
};

constexpr int kTopThreads = 256;

// One block per row: the k-th key by bisection over 32 bits, every step a
// counting pass over the row.
template <class T>
__global__ void __launch_bounds__(kTopThreads)
top_row_kernel(const TopArgs a)
{
    HX_PDL_PROLOGUE();
    constexpr int NT = kTopThreads;
    __shared__ float redf[NT / 32];
    __shared__ int redi[NT / 32];
    __shared__ uint64_t list[kMaxTop];
    __shared__ int s_count;
    const size_t row = blockIdx.x;
    const int V = int(a.vocab), k = int(a.k), tid = threadIdx.x;
    const T* l = static_cast<const T*>(a.logits) + row * a.stride;

    if (a.lse) {
        float m = -INFINITY;
        for (int i = tid; i < V; i += NT) m = fmaxf(m, to_float(l[i]));
        m = block_reduce<NT>(m, redf, MaxOp());
        const float off = m == -INFINITY ? 0.f : m, c = __fdiv_rn(kLog2e, a.tau);
        float s = 0.f;
        for (int i = tid; i < V; i += NT) s += tc::exp2_approx((to_float(l[i]) - off) * c);
        s = block_reduce<NT>(s, redf, SumOp());
        if (tid == 0) a.lse[row] = m == INFINITY ? m : __fdiv_rn(off, a.tau) + logf(s);
    }

    // smallest t with count(key <= t) >= k
    uint32_t lo = 0, hi = 0xffffffffu;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int c = 0;
        for (int i = tid; i < V; i += NT) c += descending_key(to_float(l[i])) <= mid;
        c = block_reduce<NT>(c, redi, SumOp());
        if (c >= k) hi = mid; else lo = mid + 1;
    }
    const uint32_t t = lo;
    if (tid == 0) s_count = 0;
    __syncthreads();
    for (int i = tid; i < V; i += NT) {
        const uint32_t key = descending_key(to_float(l[i]));
        if (key < t) list[atomicAdd(&s_count, 1)] = (uint64_t(key) << 32) | uint32_t(i);
    }
    __syncthreads();
    int have = s_count;  // below k
    for (int base = 0; base < V && have < k; base += NT) {
        const int i = base + tid;
        const bool eq = i < V && descending_key(to_float(l[i])) == t;
        const unsigned votes = __ballot_sync(0xffffffffu, eq);
        if ((tid & 31) == 0) redi[tid >> 5] = __popc(votes);
        __syncthreads();
        int before = have, total = have;
        for (int w = 0; w < NT / 32; ++w) {
            if (w < (tid >> 5)) before += redi[w];
            total += redi[w];
        }
        before += __popc(votes & ((1u << (tid & 31)) - 1));
        if (eq && before < k) list[before] = (uint64_t(t) << 32) | uint32_t(i);
        have = total;
        __syncthreads();
    }
    if (tid < k) {
        const uint64_t mine = list[tid];
        int rank = 0;
        for (int j = 0; j < k; ++j) rank += list[j] < mine;
        a.values[row * k + rank] = from_descending_key(uint32_t(mine >> 32));
        a.indices[row * k + rank] = int32_t(uint32_t(mine));
    }
}

template <class T>
void launch_top(hx_runtime* rt, const TopArgs& a, uint32_t rows)
{
    pdl_launch(top_row_kernel<T>, rows, kTopThreads, 0, rt->stream, a);
    HX_LAUNCHED(rt);
}

void top_logits(hx_runtime* rt, int dtype, uint32_t rows, const TopArgs& a)
{
    check_logits("top logits", dtype, rows, a.vocab, a.logits, a.stride);
    require(a.k >= 1 && a.k <= kMaxTop && a.k <= a.vocab, HX_ERR_ARGUMENT,
            "top logits: k must be in [1, min(256, vocabulary)]");
    require(std::isfinite(a.tau) && a.tau > 0.f && std::isfinite(1.f / a.tau), HX_ERR_ARGUMENT,
            "top logits: temperature must be positive and finite");
    if (rows == 0) return;
    require(a.values && a.indices, HX_ERR_ARGUMENT, "top logits: null output");
    ProfScope prof(rt, kTagSoftmaxCe, 4.0 * rows * a.vocab, double(element_bytes(dtype)) * rows * a.vocab);
    if (dtype == HX_DTYPE_F32) launch_top<float>(rt, a, rows);
    else if (dtype == HX_DTYPE_BF16) launch_top<__nv_bfloat16>(rt, a, rows);
    else launch_top<__half>(rt, a, rows);
}

}  // namespace head
}  // namespace hx

extern "C" int hx_top_logits_device(hx_runtime* rt, int dtype, uint32_t rows, uint32_t vocab, const void* logits,
                                    size_t stride, uint32_t k, float temperature, float* values, int32_t* indices,
                                    float* lse) {
    return hx_guard(rt, [&] {
        hx::head::top_logits(rt, dtype, rows, {logits, stride, values, indices, lse, vocab, k, temperature});
    });
}
