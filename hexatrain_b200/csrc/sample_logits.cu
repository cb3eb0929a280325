// sample_logits.cu -- next-token sampling on the device from given random
// numbers: temperature, top-k, top-p and min-p, each row with its own.
//
// The token order is that of the host sampler (sampling.cu; the reference's
// sampleTopKChecked, nicopedia_generation.h:286-395): scaled logit descending,
// index ascending among equals.  Masses are whole numbers,
//   y_i = (max - l_i) * (1/T),  w_i = floor(2^31 exp(-y_i)),
// so that every sum is exact in 64 bits, whatever its order, and one u gives
// one token on every launch; a token below 2^-31 of the most likely one has no
// mass, less than the spacing of a 24-bit random number can reach.  Every
// filter keeps the head of the order, so each is one prefix mass:
//   top-k: the mass M of the first k;
//   top-p: the shortest prefix with mass >= max(1, floor(M floor(2^32 p) / 2^32));
//   min-p: the tokens with y <= max(0, -log(min_p));
//   W = the smallest of them.
// The token is the first whose prefix mass exceeds floor(W floor(2^32 u) / 2^32);
// its log-probability is -y - log(W / 2^31).  T <= 0, not finite or without a finite 1/T: the first
// largest logit, log-probability 0.  A row whose logits are all -inf gets token
// -1 and -inf; one with a NaN or +inf gets -1 and NaN.
#include <cmath>

#include "head_rows.cuh"

namespace hx {
namespace head {

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

// floor(mass * f / 2^32) for f <= 2^32
__device__ __forceinline__ uint64_t scaled_mass(uint64_t mass, uint64_t f) {
    return (__umul64hi(mass, f) << 32) | ((mass * f) >> 32);
}
__device__ __forceinline__ uint64_t fraction32(float x) {  // floor(2^32 x) for x clamped to [0, 1]
    return uint64_t(double(fminf(fmaxf(x, 0.f), 1.f)) * 4294967296.0);
}
__device__ __forceinline__ uint64_t mass_of(float y) { return uint64_t(expf(-y) * 2147483648.0f); }

constexpr int kSampleThreads = 256;

// One block per row; every search is a bisection over the 32 bits of y, each
// step a pass over the row.
template <class T>
__global__ void __launch_bounds__(kSampleThreads)
sample_row_kernel(const SampleArgs a)
{
    HX_PDL_PROLOGUE();
    constexpr int NT = kSampleThreads;
    __shared__ float redf[NT / 32];
    __shared__ uint64_t redu[NT / 32];
    __shared__ int redi[NT / 32];
    __shared__ int s_token;
    const size_t row = blockIdx.x;
    const int V = int(a.vocab), tid = threadIdx.x;
    const T* l = static_cast<const T*>(a.logits) + row * a.stride;

    float m = -INFINITY;
    bool nan = false;
    for (int i = tid; i < V; i += NT) {
        const float x = to_float(l[i]);
        nan |= x != x;
        m = fmaxf(m, x);
    }
    m = block_reduce<NT>(m, redf, MaxOp());
    nan = __syncthreads_or(nan || m == INFINITY) != 0;
    if (nan || m == -INFINITY) {
        if (tid == 0) {
            a.tokens[row] = -1;
            if (a.log_probs) a.log_probs[row] = nan ? __uint_as_float(0x7fc00000u) : -INFINITY;
        }
        return;
    }
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    float inv_t = __fdiv_rn(1.f, temp);
    const bool greedy = !(temp > 0.f) || temp == INFINITY || inv_t == INFINITY;
    if (greedy) inv_t = 1.f;
    auto y_of = [&](int i) { return __fmul_rn(__fsub_rn(m, to_float(l[i])), inv_t); };
    auto mass_to = [&](uint32_t t) {  // mass of the keys <= t
        uint64_t w = 0;
        for (int i = tid; i < V; i += NT) {
            const float y = y_of(i);
            if (__float_as_uint(y) <= t) w += mass_of(y);
        }
        return block_reduce<NT>(w, redu, SumOp());
    };
    auto count_to = [&](uint32_t t) {
        int c = 0;
        for (int i = tid; i < V; i += NT) c += __float_as_uint(y_of(i)) <= t;
        return block_reduce<NT>(c, redi, SumOp());
    };
    // the key whose prefix mass first exceeds `amount`, and the mass before it
    auto cross = [&](uint64_t amount, uint64_t& before) {
        uint32_t lo = 0, hi = 0x7f800000u;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (mass_to(mid) > amount) hi = mid; else lo = mid + 1;
        }
        before = lo ? mass_to(lo - 1) : 0;
        return lo;
    };

    uint64_t W;
    int top_k = greedy ? 1 : a.top_k ? a.top_k[row] : 0;
    if (top_k <= 0 || top_k >= V) {
        W = mass_to(0x7f800000u);
    } else {
        uint32_t lo = 0, hi = 0x7f800000u;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (count_to(mid) >= top_k) hi = mid; else lo = mid + 1;
        }
        const int above = lo ? count_to(lo - 1) : 0;
        W = (lo ? mass_to(lo - 1) : 0) + uint64_t(top_k - above) * mass_of(__uint_as_float(lo));
    }
    const float p = a.top_p && !greedy ? a.top_p[row] : 1.f;
    if (p < 1.f) {
        uint64_t need = scaled_mass(W, fraction32(p));
        if (need < 1) need = 1;
        uint64_t before;
        const uint32_t t = cross(need - 1, before);
        const uint64_t w = mass_of(__uint_as_float(t));
        W = before + ((need - 1 - before) / w + 1) * w;
    }
    const float mp = a.min_p && !greedy ? a.min_p[row] : 0.f;
    if (mp > 0.f) {
        const float limit = fmaxf(-logf(mp), 0.f);
        uint64_t w = 0;
        for (int i = tid; i < V; i += NT) {
            const float y = y_of(i);
            if (y <= limit) w += mass_of(y);
        }
        w = block_reduce<NT>(w, redu, SumOp());
        if (w < W) W = w;
    }
    uint64_t u = fraction32(a.uniform[row]);
    if (u > 0xffffffffull) u = 0xffffffffull;
    const uint64_t target = scaled_mass(W, u);
    uint64_t before;
    const uint32_t t = cross(target, before);
    const uint64_t nth = (target - before) / mass_of(__uint_as_float(t));
    // the nth key equal to t, in index order
    if (tid == 0) s_token = -1;
    uint64_t have = 0;
    for (int base = 0; base < V && have <= nth; base += NT) {
        const int i = base + tid;
        const bool eq = i < V && __float_as_uint(y_of(i)) == t;
        const unsigned votes = __ballot_sync(0xffffffffu, eq);
        if ((tid & 31) == 0) redi[tid >> 5] = __popc(votes);
        __syncthreads();
        uint64_t mine = have, total = have;
        for (int w = 0; w < NT / 32; ++w) {
            if (w < (tid >> 5)) mine += redi[w];
            total += redi[w];
        }
        mine += __popc(votes & ((1u << (tid & 31)) - 1));
        if (eq && mine == nth) s_token = i;
        have = total;
        __syncthreads();
    }
    if (tid == 0) {
        a.tokens[row] = s_token;
        if (a.log_probs)
            a.log_probs[row] = greedy ? 0.f : -__uint_as_float(t) - logf(float(W) * (1.f / 2147483648.f));
    }
}

template <class T>
void launch_sample(hx_runtime* rt, const SampleArgs& a, uint32_t rows)
{
    pdl_launch(sample_row_kernel<T>, rows, kSampleThreads, 0, rt->stream, a);
    HX_LAUNCHED(rt);
}

void sample_logits(hx_runtime* rt, int dtype, uint32_t rows, const SampleArgs& a)
{
    check_logits("sampling", dtype, rows, a.vocab, a.logits, a.stride);
    if (rows == 0) return;
    require(a.uniform && a.tokens, HX_ERR_ARGUMENT, "sampling: null random numbers or output");
    ProfScope prof(rt, kTagSoftmaxCe, 4.0 * rows * a.vocab, double(element_bytes(dtype)) * rows * a.vocab);
    if (dtype == HX_DTYPE_F32) launch_sample<float>(rt, a, rows);
    else if (dtype == HX_DTYPE_BF16) launch_sample<__nv_bfloat16>(rt, a, rows);
    else launch_sample<__half>(rt, a, rows);
}

}  // namespace head
}  // namespace hx

extern "C" int hx_sample_logits_device(hx_runtime* rt, int dtype, uint32_t rows, uint32_t vocab, const void* logits,
                                       size_t stride, const float* uniform, const float* temperature,
                                       const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
                                       float* log_probs) {
    return hx_guard(rt, [&] {
        hx::head::sample_logits(rt, dtype, rows, {logits, stride, uniform, temperature, top_k, top_p, min_p, tokens,
                                                  log_probs, vocab});
    });
}
