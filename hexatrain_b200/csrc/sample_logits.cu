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
// its log-probability is -y - log(W / 2^31).  T <= 0, not finite or without a finite
// 1/T: the first largest logit, log-probability 0.  A row whose logits are all
// -inf gets token -1 and -inf; one with a NaN or +inf gets -1 and NaN.
//
// No row is sorted: a histogram of masses (and counts, for top-k) over y finds the
// bucket in which a prefix crosses an amount, and the bucket's few tokens are
// collected and sorted; a bucket with too many gets a histogram of its own, over
// the bits of y, which order it.
#include <cmath>

#include "head_ops.cuh"
#include "head_rows.cuh"

namespace hx {
namespace head {

// floor(mass * f / 2^32) for f <= 2^32
__device__ __forceinline__ uint64_t scaled_mass(uint64_t mass, uint64_t f) {
    return (__umul64hi(mass, f) << 32) | ((mass * f) >> 32);
}
__device__ __forceinline__ uint64_t fraction32(float x) {  // floor(2^32 x) for x clamped to [0, 1]
    return uint64_t(double(fminf(fmaxf(x, 0.f), 1.f)) * 4294967296.0);
}
// floor(2^31 exp(-y)), at most 2^31.  expf in full: the masses are the definition.
__device__ __forceinline__ uint32_t mass_of(float y) { return __float2uint_rz(expf(-y) * 2147483648.0f); }
__device__ __forceinline__ uint32_t mass_of_key(uint32_t key) { return mass_of(__uint_as_float(key)); }

// Shared memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t remote_u32(uint32_t addr) {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
    return x;
}
__device__ __forceinline__ void remote_store(uint32_t addr, uint64_t x) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(x) : "memory");
}
__device__ __forceinline__ void remote_store_u32(uint32_t addr, uint32_t x) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}
__device__ __forceinline__ uint32_t remote_add(uint32_t addr, uint32_t x) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(x) : "memory");
    return old;
}

// Adds to a shared word where `if_not` is not 0, without a branch.
__device__ __forceinline__ void add_shared(uint32_t addr, uint32_t x, uint32_t if_not) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p red.shared::cta.add.u32 [%0], %1;\n\t}" ::"r"(addr),
                 "r"(x), "r"(if_not)
                 : "memory");
}

constexpr float kNoMass = 24.f;               // tokens beyond have no mass: exp(-24) < 2^-31
constexpr uint32_t kNoMassKey = 0x41c00000u;  // the bits of 24.0
constexpr int kFine = 512;                    // buckets of a bucket's own histogram
constexpr int kList = 256;                    // tokens that are collected and sorted at once
// A top_k that is taken from one list: with it the tokens of the bucket in which it
// ends have to fit.  Counting alone against masses for all, top_k 1, 50 and 200 for all
// rows: 256x32768 float32 49, 55 and 74 us (62, 64, 66), 4096x4096 float16 58, 72 and 107
// (82, 90, 92): better but for the widest.
constexpr int kFew = 224;
// Buckets of the row's histogram, equal steps of y: few tokens in each, and few
// threads of a warp in the same.
__host__ __device__ constexpr int coarse_buckets(int nt) { return nt == 128 ? 512 : 2048; }

// A pass over the row, asked for by the first warp of the first CTA.
enum SampleStep { kDone = 0, kCoarse, kFineStep, kCollect, kNth };
struct SampleCommand {
    int step;
    int b0, b1;       // of the tokens in the row's buckets [b0, b1]
    int c0, c1;       // kCollect: and in [c0, c1]
    uint32_t lo, hi;  // those with keys in [lo, hi)
    int shift;        // kFineStep: bucket = (key - lo) >> shift
    uint32_t nth;     // kNth: which of the tokens with key lo
    int masses;       // kCoarse: masses too, not counts alone
};

// What the thinking warp keeps between passes.
enum Goal { kTopK, kTopP, kToken };
struct Thought {
    int goal, pending, head_count, shift, bucket;  // pending: the step whose result is awaited
    bool by_count, head, planned, masses;
    uint64_t W, amount, mass, least, plan_mass;
    uint32_t count, lo, hi;  // mass and tokens before [lo, hi)
    int plan_b1;
};

// A histogram: in a slice mass = high 2^16 + low, in the first CTA then the row's
// masses, high 2^32 + low, and counts.
template <int N>
struct Histogram {
    uint32_t low[N], high[N], count[N];
    uint64_t lane_mass[33];  // before a lane's buckets, and in all
    uint32_t lane_count[33];
    __device__ __forceinline__ uint64_t mass(int b) const { return (uint64_t(high[b]) << 32) | low[b]; }
};
template <int NB>
struct SampleShared {
    Histogram<NB> coarse;
    Histogram<kFine> fine;
    uint64_t list[kList];  // key 2^32 + index
    uint64_t scan[32];
    float maxima[16];
    uint64_t min_mass[16];  // within min-p's limit
    uint32_t nth_counts[16];
    uint32_t listed, key_min, key_max;  // of what a collection found
    SampleCommand command;
    Thought thought;
};

// The largest element of a chunk, NaN if one is NaN.
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float chunk_max(const uint4& raw, float) {
    return max_or_nan(max_or_nan(__uint_as_float(raw.x), __uint_as_float(raw.y)),
                      max_or_nan(__uint_as_float(raw.z), __uint_as_float(raw.w)));
}
__device__ __forceinline__ float chunk_max(const uint4& raw, __nv_bfloat16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
    const __nv_bfloat162 x = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_or_nan(__low2float(x), __high2float(x));
}
__device__ __forceinline__ float chunk_max(const uint4& raw, __half) {
    const __half2* h = reinterpret_cast<const __half2*>(&raw);
    const __half2 x = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_or_nan(__low2float(x), __high2float(x));
}

// A warp's prefix sums of 64-bit numbers.
__device__ __forceinline__ uint64_t warp_scan(uint64_t x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// The thinking warp's functions are called, not inlined, and their loops not
// unrolled: a row passes through all of this code once, so its length is what
// the instruction cache has to bring in for every row.

// One warp sorts the first c <= kList entries of the list.
__device__ __noinline__ void sort_list(uint64_t* list, int c) {
    const int lane = threadIdx.x & 31;
    int size = 32;
    while (size < c) size *= 2;
    for (int i = c + lane; i < size; i += 32) list[i] = ~0ull;
    __syncwarp();
#pragma unroll 1
    for (int k = 2; k <= size; k *= 2)
#pragma unroll 1
        for (int j = k / 2; j > 0; j /= 2) {
#pragma unroll
            for (int q = 0; q < kList / 64; ++q) {
                const int t = lane + 32 * q, i = 2 * t - (t & (j - 1));
                if (t >= size / 2) break;
                const uint64_t a = list[i], b = list[i + j];
                if ((a > b) == ((i & k) == 0)) {
                    list[i] = b;
                    list[i + j] = a;
                }
            }
            __syncwarp();
        }
}
// Prefixes before each lane's N / 32 buckets.
template <int N>
__device__ __noinline__ void lane_prefixes(Histogram<N>& h) {
    const int lane = threadIdx.x & 31;
    constexpr int per = N / 32;
    uint64_t w = 0;
    uint32_t k = 0;
#pragma unroll 4
    for (int i = 0; i < per; ++i) {  // (each lane from a place of its own: no bank conflicts)
        const int b = lane * per + ((i + lane) & (per - 1));
        w += h.mass(b);
        k += h.count[b];
    }
    const uint64_t ws = warp_scan(w);
    const uint32_t ks = uint32_t(warp_scan(k));
    h.lane_mass[lane] = ws - w;
    h.lane_count[lane] = ks - k;
    if (lane == 31) {
        h.lane_mass[32] = ws;
        h.lane_count[32] = ks;
    }
    __syncwarp();
}
struct Bucket {
    int at;
    uint64_t mass;  // before it
    uint32_t count;
};
// The bucket in which the prefix exceeds `want` (which lies in one).
template <int N>
__device__ __noinline__ Bucket find_bucket(const Histogram<N>& h, bool counted, uint64_t want) {
    const int lane = threadIdx.x & 31;
    constexpr int per = N / 32;
    const bool here = counted ? h.lane_count[lane] <= want && want < h.lane_count[lane + 1]
                              : h.lane_mass[lane] <= want && want < h.lane_mass[lane + 1];
    const int src = (__ffs(__ballot_sync(0xffffffffu, here)) - 1) & 31;
    uint64_t before = h.lane_mass[src];
    uint32_t tokens = h.lane_count[src];
    Bucket r{src * per, before, tokens};
#pragma unroll 1
    for (int i0 = 0; i0 < per; i0 += 32) {
        const int b = src * per + i0 + lane;
        const bool in = i0 + lane < per;
        const uint64_t w = in ? h.mass(b) : 0, we = before + warp_scan(w);
        const uint32_t k = in ? h.count[b] : 0, ke = tokens + uint32_t(warp_scan(k));
        const unsigned hit = __ballot_sync(0xffffffffu, in && want < (counted ? uint64_t(ke) : we));
        if (hit) {
            const int at = __ffs(hit) - 1;
            r = {src * per + i0 + at, __shfl_sync(0xffffffffu, we - w, at), __shfl_sync(0xffffffffu, ke - k, at)};
            break;
        }
        before = __shfl_sync(0xffffffffu, we, 31);
        tokens = __shfl_sync(0xffffffffu, ke, 31);
    }
    return r;
}
struct Found {
    uint64_t entry, prefix;  // the prefix mass with the entry
};
// Where the prefix of the sorted list's entries [from, to) exceeds `want`, given
// the mass and the count before them.
__device__ __noinline__ Found find_in_list(const uint64_t* list, int from, int to, uint64_t w0, uint64_t k0, bool counted,
                                           uint64_t want) {
    const int lane = threadIdx.x & 31;
    uint64_t e = 0, prefix = 0;
    unsigned hit = 0;
#pragma unroll 1
    for (int j0 = from; j0 < to && !hit; j0 += 32) {
        const int j = j0 + lane;
        e = j < to ? list[j] : 0;
        const uint32_t w = j < to ? mass_of_key(uint32_t(e >> 32)) : 0u;
        prefix = w0 + warp_scan(w);
        hit = __ballot_sync(0xffffffffu, j < to && (counted ? k0 + (j - from) == want : want < prefix && want >= prefix - w));
        w0 = __shfl_sync(0xffffffffu, prefix, 31);
    }
    const int src = (__ffs(hit) - 1) & 31;
    return {__shfl_sync(0xffffffffu, e, src), __shfl_sync(0xffffffffu, prefix, src)};
}
// The mass of the sorted list's entries with y <= limit.
__device__ __noinline__ uint64_t list_mass(const uint64_t* list, int c, float limit) {
    uint64_t w = 0;
#pragma unroll 1
    for (int j = threadIdx.x & 31; j < c; j += 32) {
        const float y = __uint_as_float(uint32_t(list[j] >> 32));
        if (y <= limit) w += mass_of(y);
    }
    return warp_reduce(w, SumOp());
}
// One block per row, or a cluster of them with a slice each, held in shared memory.
// The first warp of the first CTA thinks, all others make the passes that it asks
// for: the row's histogram, the collection of a bucket's tokens, rarely a bucket's
// own histogram or the nth of equal tokens.  Bound by the instructions of the passes (2 to 4
// a token; the first forms expf of every one) and by the latency
// between them: 256x32768 float32 57 us, 4096x4096 float16 74 us, one row of 1024
// 7 to 12 us.  Few-token filters (top_k <= kFew) need no masses but those of
// the tokens they keep: their histogram only counts.
template <class T, int NT>
__global__ void __launch_bounds__(NT, NT == 512 ? 2 : 8)
sample_kernel(const SampleArgs a, int slices, int log_slices)
{
    HX_PDL_PROLOGUE();
    constexpr int NB = coarse_buckets(NT), EPV = Chunk<T>::EPV;
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared<NB>& s = *reinterpret_cast<SampleShared<NB>*>(smem);
    uint4* held = reinterpret_cast<uint4*>(smem + ((sizeof(SampleShared<NB>) + 15) & ~size_t(15)));
    const int tid = threadIdx.x, lane = tid & 31, V = int(a.vocab);
    const int rank = int(blockIdx.x) & (slices - 1);
    const size_t row = blockIdx.x >> log_slices;
    const T* l = static_cast<const T*>(a.logits) + row * a.stride;
    const bool many = slices > 1, thinker = rank == 0 && tid < 32;
    auto sync = [&] {
        if (many) tc::cluster_sync(); else __syncthreads();
    };
    const int lead = int((reinterpret_cast<uintptr_t>(l) & 15) / sizeof(T));
    const int chunks = (V + lead + EPV - 1) / EPV, each = (chunks + slices - 1) >> log_slices;
    const int first = min(chunks, rank * each), n = min(chunks, first + each) - first;  // this CTA's chunks
    const int base = first * EPV - lead;                                                // element 0 of chunk 0

    // ---- the slice and its maximum ----
    float m = -INFINITY;
    auto keep = [&](int c, const uint4& raw) {
        held[c] = raw;
        m = max_or_nan(m, chunk_max(raw, T()));
    };
    const float uniform = thinker ? a.uniform[row] : 0.f;
    const float temp = a.temperature ? a.temperature[row] : 1.f;
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f, mp = a.min_p ? a.min_p[row] : 0.f;
    const int whole0 = lead > 0 && first == 0 ? 1 : 0, whole1 = max(whole0, min(n, (V + lead) / EPV - first));
    const uint4* from = reinterpret_cast<const uint4*>(l - lead) + first;
    for (int c0 = whole0 + tid; c0 < whole1; c0 += 4 * NT) {
        uint4 raw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c0 + q * NT < whole1) raw[q] = from[c0 + q * NT];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c0 + q * NT < whole1) keep(c0 + q * NT, raw[q]);
    }
    // the chunks that begin before the row or end after it
    if (tid < 2) {
        const int c = tid == 0 ? 0 : n - 1;
        if (n > 0 && (tid == 0 ? whole0 == 1 : whole1 < n && (c > 0 || whole0 == 0))) {
            float x[EPV];
#pragma unroll
            for (int r = 0; r < EPV; ++r) {
                const int i = base + c * EPV + r;
                x[r] = i >= 0 && i < V ? to_float(l[i]) : -INFINITY;
            }
            keep(c, Chunk<T>::pack(x));
        }
    }
    for (int b = tid; b < NB; b += NT) {
        s.coarse.low[b] = s.coarse.high[b] = s.coarse.count[b] = 0u;
    }
    bool nan = __syncthreads_or(!(m < INFINITY)) != 0;
    m = block_reduce<NT>(m, reinterpret_cast<float*>(s.scan), MaxOp());
    if (many) {
        tc::cluster_sync();  // every CTA has started
        // a NaN marks the whole row: no maximum is above +inf
        if (tid < slices)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(tc::cluster_addr(&s.maxima[rank], tid)),
                         "f"(nan ? INFINITY : m) : "memory");
        tc::cluster_sync();
        for (int r = 0; r < slices; ++r) m = fmaxf(m, s.maxima[r]);
        nan = m == INFINITY;
    }
    m += 0.f;  // a maximum of -0 would give +0 a y of -0, whose bits are no key
    if (nan || m == -INFINITY) {
        if (tid == 0 && rank == 0) {
            a.tokens[row] = -1;
            if (a.log_probs) a.log_probs[row] = nan ? __uint_as_float(0x7fc00000u) : -INFINITY;
        }
        return;  // the whole cluster
    }

    const float inv_t = __fdiv_rn(1.f, temp);
    if (!(temp > 0.f) || temp == INFINITY || inv_t == INFINITY) {  // the first largest logit
        int at = 0x7fffffff;
        for (int c = tid; c < n; c += NT) {
            float x[EPV];
            Chunk<T>::unpack(held[c], x);
#pragma unroll
            for (int r = 0; r < EPV; ++r)
                if (x[r] == m) at = min(at, base + c * EPV + r);
        }
        at = -block_reduce<NT>(-at, reinterpret_cast<int*>(s.scan), MaxOp());
        if (many) {
            if (tid == 0)
                remote_store_u32(tc::cluster_addr(&s.nth_counts[rank], 0), at);
            tc::cluster_sync();
            if (rank == 0)
                for (int r = 0; r < slices; ++r) at = min(at, int(s.nth_counts[r]));
        }
        if (tid == 0 && rank == 0) {
            a.tokens[row] = at;
            if (a.log_probs) a.log_probs[row] = 0.f;
        }
        return;  // the whole cluster
    }
    const float limit = mp > 0.f ? fmaxf(-logf(mp), 0.f) : -1.f;
    // the row's bucket of y < kNoMass
    constexpr float kScale = float(NB) / kNoMass;
    auto bucket_of = [](float y) {  // y kScale rounded: the low bits of its sum with 2^23
        return min(int(__float_as_uint(fmaf(y, kScale, 8388608.f)) - 0x4b000000u), NB - 1);
    };
    auto key_below = [](int b) { return b <= 1 ? 0u : __float_as_uint(float(b - 1) / kScale); };  // at most those of bucket b
    auto key_above = [](int b) { return min(kNoMassKey, __float_as_uint(float(b + 2) / kScale)); };  // above them

    // Goes on until a pass over the row is needed.
    auto think = [&](bool begin) {
        Thought t;
        if (begin) {
            t = Thought{};
            t.masses = top_k <= 0 || top_k > kFew;
        } else {
            t = s.thought;
        }
        auto ask = [&](const SampleCommand& c) {
            t.pending = c.step;
            __syncwarp();
            if (lane == 0) {
                s.command = c;
                s.listed = 0;
                s.key_min = 0xffffffffu;
                s.key_max = 0;
                s.thought = t;
            }
        };
        auto collect = [&](int b0, int b1, int c0, int c1, uint32_t lo, uint32_t hi) {
            ask({kCollect, b0, b1, c0, c1, lo, hi, 0, 0, 0});
        };
        const uint64_t u = min(fraction32(uniform), uint64_t(0xffffffffu)), p32 = fraction32(p);
        Found found{};
        bool have = false;  // `found` answers the goal
        auto one_key = [&] {  // the tokens of the only key lo have one mass
            const uint64_t w = mass_of_key(t.lo), nth = t.by_count ? t.amount - t.count : (t.amount - t.mass) / w;
            found = {uint64_t(t.lo) << 32, t.mass + (nth + 1) * w};
            if (t.goal == kToken) {
                t.amount = nth;
                t.pending = kNth;
            }
        };
        if (t.pending == kCoarse || begin) {  // the row's histogram is there
            lane_prefixes(s.coarse);
            const uint32_t tokens = s.coarse.lane_count[32];
            t.least = ~0ull;
            if (!t.masses) {
                // the first k, or all that have mass, in one list, if it holds them
                t.amount = min(uint32_t(top_k), tokens) - 1;
                const Bucket b = find_bucket(s.coarse, true, t.amount);
                if (b.count + s.coarse.count[b.at] <= uint32_t(kList)) {
                    t.head = true;
                    t.by_count = true;
                    t.goal = kTopK;
                    collect(0, b.at, 1, 0, 0, key_above(b.at));
                    return;
                }
                t.masses = true;
                ask({kCoarse, 0, NB - 1, 1, 0, 0, kNoMassKey, 0, 0, 1});
                return;
            }
            t.W = s.coarse.lane_mass[32];
            if (mp > 0.f) {
                t.least = 0;
                for (int r = 0; r < slices; ++r) t.least += s.min_mass[r];
            }
            t.goal = top_k > 0 && uint32_t(top_k) < tokens ? kTopK : p < 1.f ? kTopP : kToken;
            t.pending = kDone;
        } else if (t.pending == kCollect) {
            const int c = int(s.listed);
            if (c > kList) {
                if (t.planned) {  // together too many: one after the other
                    t.planned = false;
                    collect(t.bucket, t.bucket, 1, 0, t.lo, t.hi);
                    return;
                }
                // a histogram of this bucket's keys, or one key (16-bit logits tie)
                t.lo = max(t.lo, s.key_min);
                t.hi = min(t.hi, s.key_max + 1);
                if (t.hi - t.lo > 1) {
                    t.shift = 0;
                    while (((t.hi - 1 - t.lo) >> t.shift) >= uint32_t(kFine)) ++t.shift;
                    ask({kFineStep, t.bucket, t.bucket, 1, 0, t.lo, t.hi, t.shift, 0, 0});
                    return;
                }
                one_key();
            } else {
                sort_list(s.list, c);
                if (t.head) {
                    t.head_count = c;
                    if (mp > 0.f) t.least = list_mass(s.list, c, limit);
                    found = find_in_list(s.list, 0, c, 0, 0, true, t.amount);
                } else if (t.planned && t.plan_b1 < t.bucket) {
                    // the token's tokens come first in the list
                    int f = 0;
#pragma unroll 1
                    for (int j0 = 0; j0 < c; j0 += 32) {
                        const int j = j0 + lane;
                        f += __popc(__ballot_sync(
                            0xffffffffu, j < c && bucket_of(__uint_as_float(uint32_t(s.list[j] >> 32))) < t.bucket));
                    }
                    found = find_in_list(s.list, f, c, t.mass, t.count, t.by_count, t.amount);
                    t.W = min(found.prefix, t.least);
                    t.goal = kToken;
                    found = find_in_list(s.list, 0, f, t.plan_mass, 0, false, scaled_mass(t.W, u));
                } else {
                    found = find_in_list(s.list, 0, c, t.mass, t.count, t.by_count, t.amount);
                    if (t.planned) {  // both in one bucket
                        t.W = min(found.prefix, t.least);
                        t.goal = kToken;
                        found = find_in_list(s.list, 0, c, t.mass, 0, false, scaled_mass(t.W, u));
                    }
                }
            }
            have = true;
        } else {  // a bucket's histogram
            lane_prefixes(s.fine);
            const Bucket b = find_bucket(s.fine, t.by_count, t.by_count ? t.amount - t.count : t.amount - t.mass);
            t.mass += b.mass;
            t.count += b.count;
            t.hi = min(t.hi, t.lo + (uint32_t(b.at + 1) << t.shift));
            t.lo += uint32_t(b.at) << t.shift;
            if (t.hi - t.lo > 1) {
                collect(t.bucket, t.bucket, 1, 0, t.lo, t.hi);
                return;
            }
            one_key();
            have = true;
        }
#pragma unroll 1
        for (;;) {
            if (have) {  // the goal's answer
                if (t.goal == kToken) {
                    if (lane == 0) {
                        if (t.pending != kNth) a.tokens[row] = int32_t(uint32_t(found.entry));
                        if (a.log_probs)
                            a.log_probs[row] = -__uint_as_float(uint32_t(found.entry >> 32)) -
                                               logf(float(t.W) * (1.f / 2147483648.f));
                    }
                    const uint32_t key = uint32_t(found.entry >> 32);
                    ask({t.pending == kNth ? kNth : kDone, 0, NB - 1, 1, 0, key, key + 1, 0, uint32_t(t.amount), 0});
                    return;
                }
                t.W = found.prefix;
                t.goal = t.goal == kTopK && p < 1.f ? kTopP : kToken;
                have = false;
            }
            // the next goal
            t.by_count = t.goal == kTopK;
            if (t.goal == kTopK) {
                t.amount = uint64_t(top_k) - 1;
            } else if (t.goal == kTopP) {
                const uint64_t need = scaled_mass(t.W, p32);
                t.amount = need < 1 ? 0 : need - 1;
            } else {
                t.W = min(t.W, t.least);
                t.amount = scaled_mass(t.W, u);
            }
            if (t.head) {
                found = find_in_list(s.list, 0, t.head_count, 0, 0, t.by_count, t.amount);
                have = true;
                continue;
            }
            const Bucket b = find_bucket(s.coarse, t.by_count, t.amount);
            t.bucket = b.at;
            t.mass = b.mass;
            t.count = b.count;
            t.lo = key_below(b.at);
            t.hi = key_above(b.at);
            t.planned = t.goal == kTopP || (t.goal == kTopK && !(p < 1.f));
            if (!t.planned) {
                collect(b.at, b.at, 1, 0, t.lo, t.hi);
                return;
            }
            // W will lie in this bucket: but for that the token's bucket is known, and
            // its tokens are collected in the same pass
            const Bucket f1 = find_bucket(s.coarse, false, scaled_mass(min(b.mass, t.least), u));
            const Bucket f2 = find_bucket(s.coarse, false, scaled_mass(min(b.mass + s.coarse.mass(b.at), t.least), u));
            t.plan_mass = f1.mass;
            t.plan_b1 = f2.at;
            if (f2.at < b.at) {
                collect(b.at, b.at, f1.at, f2.at, key_below(f1.at), t.hi);
            } else if (f1.at == b.at) {
                collect(b.at, b.at, 1, 0, t.lo, t.hi);
            } else {  // the two adjoin: first the one, then the other
                t.planned = false;
                collect(b.at, b.at, 1, 0, t.lo, t.hi);
            }
            return;
        }
    };

    // ---- passes, the first the row's histogram ----
    SampleCommand cmd{kCoarse, 0, NB - 1, 1, 0, 0, kNoMassKey, 0, 0, top_k <= 0 || top_k > kFew};
    const T* element = reinterpret_cast<const T*>(held);
    auto y_of = [&](int i) { return __fmul_rn(__fsub_rn(m, to_float(element[i])), inv_t); };
#pragma unroll 1
    for (bool begin = true;; begin = false) {
        // a logit below which no key is below hi: y >= hi once (m - l)/T is above it
        // by more than the roundings
        const float least = m - __uint_as_float(cmd.hi) * temp * 1.00001f - fabsf(m) * 1e-5f;
        if (cmd.step == kCoarse || cmd.step == kFineStep) {
            const bool coarse = cmd.step == kCoarse;
            uint32_t* low = coarse ? s.coarse.low : s.fine.low;
            uint32_t* high = coarse ? s.coarse.high : s.fine.high;
            uint32_t* count = coarse ? s.coarse.count : s.fine.count;
            const int buckets = coarse ? NB : kFine;
            const uint32_t low_at = tc::smem_u32(low), high_at = tc::smem_u32(high), count_at = tc::smem_u32(count);
            if (!begin) {
                for (int b = tid; b < buckets; b += NT) {
                    low[b] = high[b] = count[b] = 0u;
                }
                sync();  // (a CTA's buckets may be read until here)
            }
            const bool counts = top_k > 0, masses = !coarse || cmd.masses, limited = coarse && mp > 0.f;
            uint64_t below = 0;
#pragma unroll 1
            for (int c = tid; c < n; c += NT) {
                const uint4 raw = held[c];
                if (!(chunk_max(raw, T()) >= least)) continue;
                float x[EPV];
                Chunk<T>::unpack(raw, x);
#pragma unroll
                for (int r = 0; r < EPV; ++r) {
                    const float y = __fmul_rn(__fsub_rn(m, x[r]), inv_t);
                    int b = bucket_of(y);
                    bool in = y < kNoMass;
                    if (!coarse) {
                        const uint32_t key = __float_as_uint(y);
                        in = b == cmd.b0 && key - cmd.lo < cmd.hi - cmd.lo;
                        b = in ? int((key - cmd.lo) >> cmd.shift) : 0;
                    }
                    if (masses) {
                        const uint32_t w = in ? mass_of(y) : 0u;
                        add_shared(low_at + b * 4, w & 0xffffu, w & 0xffffu);
                        add_shared(high_at + b * 4, w >> 16, w >> 16);
                        if (limited) below += y <= limit ? w : 0u;
                    }
                    if (counts) add_shared(count_at + b * 4, 1u, in);
                }
            }
            if (limited) {  // the slice's mass within the limit, to the first CTA
                below = block_reduce<NT>(below, s.scan, SumOp());
                if (tid == 0) {
                    if (many) remote_store(tc::cluster_addr(&s.min_mass[rank], 0), below); else s.min_mass[0] = below;
                }
            }
            sync();
            // the buckets of all slices, each CTA a share of them, to the first CTA, in place
            const int share = buckets >> log_slices;
#pragma unroll 1
            for (int b = rank * share + tid; b < (rank + 1) * share; b += NT) {
                uint64_t w = 0;
                uint32_t k = 0;
                if (many) {
                    for (int r = 0; r < slices; ++r) {
                        w += (uint64_t(remote_u32(tc::cluster_addr(high + b, r))) << 16) +
                             remote_u32(tc::cluster_addr(low + b, r));
                        if (counts) k += remote_u32(tc::cluster_addr(count + b, r));
                    }
                    remote_store_u32(tc::cluster_addr(low + b, 0), uint32_t(w));
                    remote_store_u32(tc::cluster_addr(high + b, 0), uint32_t(w >> 32));
                    remote_store_u32(tc::cluster_addr(count + b, 0), k);
                } else {
                    w = (uint64_t(high[b]) << 16) + low[b];
                    low[b] = uint32_t(w);
                    high[b] = uint32_t(w >> 32);
                }
            }
        } else if (cmd.step == kCollect) {
            const uint32_t counter = many ? tc::cluster_addr(&s.listed, 0) : 0, list = many ? tc::cluster_addr(s.list, 0) : 0;
            uint32_t key_min = 0xffffffffu, key_max = 0;
            // all of a warp's finds at once: the place of the first is asked for once
#pragma unroll 1
            for (int c0 = 0; c0 < n; c0 += NT) {
                const int c = c0 + tid;
                uint32_t mask = 0;
                float x[EPV];
                if (c < n && chunk_max(held[c], T()) >= least) {
                    Chunk<T>::unpack(held[c], x);
#pragma unroll
                    for (int r = 0; r < EPV; ++r) {
                        const uint32_t key = __float_as_uint(__fmul_rn(__fsub_rn(m, x[r]), inv_t));
                        mask |= uint32_t(key - cmd.lo < cmd.hi - cmd.lo) << r;
                    }
                    // of those few, the ones in the buckets
#pragma unroll 1
                    for (uint32_t rest = mask; rest; rest &= rest - 1) {
                        const int r = __ffs(rest) - 1;
                        const float y = y_of(c * EPV + r);
                        const int b = bucket_of(y);
                        if ((b >= cmd.b0 && b <= cmd.b1) || (b >= cmd.c0 && b <= cmd.c1)) {
                            key_min = min(key_min, __float_as_uint(y));
                            key_max = max(key_max, __float_as_uint(y));
                        } else {
                            mask &= ~(1u << r);
                        }
                    }
                }
                if (!__any_sync(0xffffffffu, mask != 0)) continue;
                int at = __popc(mask);
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, at, o);
                    if (lane >= o) at += y;
                }
                const int all = __shfl_sync(0xffffffffu, at, 31);
                uint32_t start = 0;
                if (lane == 0) start = many ? remote_add(counter, uint32_t(all)) : atomicAdd(&s.listed, uint32_t(all));
                at += int(__shfl_sync(0xffffffffu, start, 0)) - __popc(mask);
                for (; mask; mask &= mask - 1, ++at) {
                    const int i = c * EPV + __ffs(mask) - 1;
                    const uint64_t entry = (uint64_t(__float_as_uint(y_of(i))) << 32) | uint32_t(base + i);
                    if (at >= kList) break;
                    if (many) remote_store(list + at * 8, entry); else s.list[at] = entry;
                }
            }
            key_min = __reduce_min_sync(0xffffffffu, key_min);
            key_max = __reduce_max_sync(0xffffffffu, key_max);
            if (lane == 0 && key_min <= key_max) {
                if (many) {
                    asm volatile("red.shared::cluster.min.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.key_min, 0)), "r"(key_min)
                                 : "memory");
                    asm volatile("red.shared::cluster.max.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.key_max, 0)), "r"(key_max)
                                 : "memory");
                } else {
                    atomicMin(&s.key_min, key_min);
                    atomicMax(&s.key_max, key_max);
                }
            }
        } else {
            break;
        }
        sync();
        if (thinker) think(begin);
        sync();
        if (rank == 0) {
            cmd = s.command;
        } else {
            const uint32_t at = tc::cluster_addr(&s.command, 0);
            cmd = {int(remote_u32(at)), int(remote_u32(at + 4)), int(remote_u32(at + 8)), int(remote_u32(at + 12)),
                   int(remote_u32(at + 16)), remote_u32(at + 20), remote_u32(at + 24), int(remote_u32(at + 28)),
                   remote_u32(at + 32), int(remote_u32(at + 36))};
        }
    }
    if (cmd.step == kNth) {  // the nth token with key lo, in index order
        uint32_t mine = 0, before = 0;
        for (int i = tid; i < n * EPV; i += NT) mine += __float_as_uint(y_of(i)) == cmd.lo;
        mine = block_reduce<NT>(mine, reinterpret_cast<uint32_t*>(s.scan), SumOp());
        if (many) {
            if (tid < slices)
                remote_store_u32(tc::cluster_addr(&s.nth_counts[rank], tid), mine);
            tc::cluster_sync();
            for (int r = 0; r < rank; ++r) before += s.nth_counts[r];
        }
        if (cmd.nth >= before && cmd.nth < before + mine) {
            uint32_t have = before;
            uint32_t* votes_of = reinterpret_cast<uint32_t*>(s.scan);
#pragma unroll 1
            for (int i0 = 0; i0 < n * EPV && have <= cmd.nth; i0 += NT) {
                const int i = i0 + tid;
                const bool eq = i < n * EPV && __float_as_uint(y_of(i)) == cmd.lo;
                const unsigned votes = __ballot_sync(0xffffffffu, eq);
                if (lane == 0) votes_of[tid >> 5] = __popc(votes);
                __syncthreads();
                uint32_t at = have;
                for (int w = 0; w < NT / 32; ++w) {
                    if (w < (tid >> 5)) at += votes_of[w];
                    have += votes_of[w];
                }
                at += __popc(votes & ((1u << lane) - 1));
                if (eq && at == cmd.nth) a.tokens[row] = base + i;
                __syncthreads();
            }
        }
    }
    if (many) tc::cluster_sync();  // no CTA leaves while another may read it
}

template <class T, int NT>
void launch_sample(hx_runtime* rt, const SampleArgs& a, uint32_t rows, long chunks, int slices)
{
    const size_t smem = ((sizeof(SampleShared<coarse_buckets(NT)>) + 15) & ~size_t(15)) +
                        size_t((chunks + slices - 1) / slices) * 16;
    require(uint64_t(rows) * slices <= 0x7fffffffu, HX_ERR_UNSUPPORTED, "sampling: too many rows for one call");
    auto kernel = sample_kernel<T, NT>;
    static thread_local int opted[64] = {};
    if (!opted[rt->device & 63]) {
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 131072));
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        opted[rt->device & 63] = 1;
    }
    launch_rows(kernel, rows * unsigned(slices), NT, slices, true, smem, rt->stream, a, slices, __builtin_ctz(unsigned(slices)));
    HX_LAUNCHED(rt);
}

template <class T>
void launch_sample(hx_runtime* rt, const SampleArgs& a, uint32_t rows)
{
    constexpr int EPV = Chunk<T>::EPV;
    const long chunks = row_chunks(a.logits, a.stride, rows, a.vocab, sizeof(T));
    if (chunks <= 4096 / EPV + 1) {
        launch_sample<T, 128>(rt, a, rows, chunks, 1);
    } else {
        // slices of 64 KB, so that two blocks share an SM; more of them, down to
        // 4096 tokens, while the rows alone would leave SMs idle
        int s = 1;
        while (chunks > 4160L * s) s *= 2;
        while (s < 8 && long(rows) * s * 2 <= rt->sm_count && chunks * EPV / (2 * s) >= 4096) s *= 2;
        launch_sample<T, 512>(rt, a, rows, chunks, s);
    }
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
