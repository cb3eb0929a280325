// head_rows.cuh -- shared parts of the kernels over rows of logits (top logits,
// distillation, device sampling): element types, block reductions, sort keys.
//
// All of them take [rows, vocab] logits in float32, bfloat16 or float16 with
// any row stride and work in float32; every offset is formed in 64 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "hx_internal.cuh"
#include "tc_ptx.cuh"

namespace hx {
namespace head {

constexpr uint32_t kMaxVocab = 262144;  // 16 slices of 16384 logits
constexpr uint32_t kMaxTop = 256;       // entries of a top-logits record

// Error-word code of a teacher index or label outside the vocabulary.
constexpr int kBadIndexCode = kHeadIndexCode;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Unsigned key whose ascending order is the descending order of x: +inf first,
// -inf last before NaN; the two zeros are equal.
__device__ __forceinline__ uint32_t descending_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float from_descending_key(uint32_t k) {
    if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((k & 0x80000000u) ? k : ~k & 0x7fffffffu);
}

constexpr float kLog2e = 1.44269504088896340736f;

struct SumOp {
    template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct MaxOp {
    template <class T> __device__ __forceinline__ T operator()(T a, T b) const { return a > b ? a : b; }
};

template <class T, class Op>
__device__ __forceinline__ T warp_reduce(T v, Op op) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Reduction over the block's NT threads; every thread gets the result.
// `scratch` holds NT / 32 values and may be reused after the call returns.
template <int NT, class T, class Op>
__device__ __forceinline__ T block_reduce(T v, T* scratch, Op op) {
    v = warp_reduce(v, op);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    T r = scratch[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) r = op(r, scratch[w]);
    __syncthreads();
    return r;
}

inline size_t element_bytes(int dtype)
{
    require(dtype == HX_DTYPE_F32 || dtype == HX_DTYPE_BF16 || dtype == HX_DTYPE_F16, HX_ERR_ARGUMENT,
            "unknown logit type (HX_DTYPE_F32, HX_DTYPE_BF16 or HX_DTYPE_F16)");
    return dtype == HX_DTYPE_F32 ? 4 : 2;
}

inline void check_logits(const char* op, int dtype, uint32_t rows, uint32_t vocab, const void* logits, size_t stride)
{
    const size_t bytes = element_bytes(dtype);
    const std::string name(op);
    require(vocab >= 1, HX_ERR_ARGUMENT, name + ": empty vocabulary");
    require(vocab <= kMaxVocab, HX_ERR_UNSUPPORTED,
            name + ": vocabulary over " + std::to_string(kMaxVocab) + " is not supported");
    require(rows <= 0x7fffffffu, HX_ERR_UNSUPPORTED, name + ": over 2^31 - 1 rows");
    require(stride >= vocab, HX_ERR_ARGUMENT, name + ": row stride below the vocabulary size");
    require(rows == 0 || logits, HX_ERR_ARGUMENT, name + ": null logits");
    require(reinterpret_cast<uintptr_t>(logits) % bytes == 0, HX_ERR_ARGUMENT, name + ": logits not aligned to their type");
}

}  // namespace head
}  // namespace hx
