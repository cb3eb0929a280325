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
constexpr float kLn2 = 0.69314718055994530942f;

// Whether a row's sum of exponentials against a reference serves.  Against one of the
// row's logits it is 1 or more, and too large only where another lies far above.
// Where the logits looked at are masked the reference is 0 and may lie far above
// all of the row: below 2^-126 ex2.approx gives 0, so that part of a small sum is missing.
__device__ __forceinline__ bool sum_serves(float sum) { return sum > 0x1p-60f && sum < 0x1p60f; }

// Exponentials of a row against one of its logits are 2^(l c - o), c = log2(e) / tau,
// o = ref c rounded; a row's sum and its uses share o, and its rounding cancels.
// From kFarOffset on (a row at its type's lowest value) the rounding alone is an
// exponent of 64 and more.  There two logits are equal or, times c, over 2^7 apart, an
// exponential is 1 or 0, and a power of two for c gives the same with o exact.
constexpr float kFarOffset = 0x1p31f;
__device__ __forceinline__ float scale_against(float ref, float c) {
    if (fabsf(ref * c) < kFarOffset) return c;
    const int exponent = int(__float_as_uint(ref) >> 23 & 255u);  // |ref| times the scale in [2^125, 2^126)
    return __uint_as_float(uint32_t(min(379 - exponent, 254)) << 23);
}
// For sums that take c as it is: beyond the bound their exponentials are 0, and no
// sum serves.
__device__ __forceinline__ float offset_against(float ref, float c) {
    const float o = ref * c;
    return fabsf(o) < kFarOffset ? o : INFINITY;
}

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

// The largest of the warp's values (not NaN).
__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
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

// ---- chunks -------------------------------------------------------------------
// A row is seen as 16-byte chunks that are aligned in memory; the first begins
// `lead` elements before the row, and chunk c holds elements [c EPV - lead, + EPV).
// Chunks at the ends are read and written by element.
constexpr int kPerThread = 32;  // logits of a lane where a warp holds a row in registers

template <class T>
struct Chunk {
    static constexpr int EPV = 16 / int(sizeof(T));   // elements of a 16-byte chunk
    static constexpr int N = kPerThread / EPV;        // chunks of kPerThread elements
    static __device__ __forceinline__ void unpack(const uint4& raw, float (&x)[EPV]);
    static __device__ __forceinline__ uint4 pack(const float (&x)[EPV]);
};
template <>
__device__ __forceinline__ void Chunk<float>::unpack(const uint4& raw, float (&x)[4]) {
    x[0] = __uint_as_float(raw.x);
    x[1] = __uint_as_float(raw.y);
    x[2] = __uint_as_float(raw.z);
    x[3] = __uint_as_float(raw.w);
}
template <>
__device__ __forceinline__ uint4 Chunk<float>::pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
template <>
__device__ __forceinline__ void Chunk<__nv_bfloat16>::unpack(const uint4& raw, float (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bfloat16 is the upper half of a float32
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <>
__device__ __forceinline__ uint4 Chunk<__nv_bfloat16>::pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void Chunk<__half>::unpack(const uint4& raw, float (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ uint4 Chunk<__half>::pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 b = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Launch of `rows` teams of `slices` CTAs each, a cluster per row when there
// are several (over 8 only for a kernel that is opted in to them).
template <class... KArgs, class... Args>
inline void launch_rows(void (*kernel)(KArgs...), unsigned grid, int threads, int slices, bool cluster, size_t smem,
                        cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster && slices > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = slices;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    cfg.attrs = attr;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    if (e != cudaSuccess) (void)cudaGetLastError();  // reported here, not by the next launch
    check_cuda(e, "kernel launch");
}

// Teams of `slices` CTAs (a cluster where there are several) that the GPU holds at
// once: persistent kernels launch no more, since one that had to wait would
// take a second round of its own.  Asked once for each shape.
template <class... KArgs>
inline int resident_teams(hx_runtime* rt, void (*kernel)(KArgs...), int threads, size_t smem, int slices) {
    struct Known {
        const void* kernel;
        size_t smem;
        int device, slices, teams;
    };
    static thread_local std::vector<Known> known;
    const void* id = reinterpret_cast<const void*>(kernel);
    for (const Known& x : known)
        if (x.kernel == id && x.smem == smem && x.device == rt->device && x.slices == slices) return x.teams;
    int teams = 0;
    if (slices == 1) {
        HX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&teams, kernel, threads, smem));
        teams *= rt->sm_count;
    } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(slices));
        cfg.blockDim = dim3(unsigned(threads));
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(slices);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        HX_CUDA(cudaOccupancyMaxActiveClusters(&teams, kernel, &cfg));
    }
    require(teams >= 1, HX_ERR_UNSUPPORTED, "the device does not hold " + std::to_string(slices) + " blocks of a row");
    if (known.size() >= 256) known.clear();
    known.push_back({id, smem, rt->device, slices, teams});
    return teams;
}

// The chunks a row can take: the largest lead that any of the rows has.
inline long row_chunks(const void* logits, size_t stride, uint32_t rows, uint32_t vocab, int elem_bytes) {
    const int epv = 16 / elem_bytes;
    const uintptr_t base = reinterpret_cast<uintptr_t>(logits);
    const bool same = rows <= 1 || stride * elem_bytes % 16 == 0;
    const long lead = same ? long(base % 16) / elem_bytes : epv - 1;
    return (long(vocab) + lead + epv - 1) / epv;
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
