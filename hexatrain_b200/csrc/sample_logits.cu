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
// No row is sorted.  y >= 0, so its bits order it: a histogram of counts and
// masses over the bits (64 buckets to an octave) finds the bucket in which a
// prefix crosses an amount; the bucket's few tokens are collected and sorted.
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
// floor(2^31 exp(-y)), at most 2^31.  expf in full: the masses are the definition.
__device__ __forceinline__ uint32_t mass_of(float y) { return __float2uint_rz(expf(-y) * 2147483648.0f); }
__device__ __forceinline__ uint32_t mass_of_key(uint32_t key) { return mass_of(__uint_as_float(key)); }

// Shared memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t remote_u32(uint32_t addr) {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
    return x;
}
__device__ __forceinline__ uint64_t remote_u64(uint32_t addr) {
    uint64_t x;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(addr) : "memory");
    return x;
}
__device__ __forceinline__ void remote_store(uint32_t addr, uint64_t x) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(x) : "memory");
}
__device__ __forceinline__ uint32_t remote_add(uint32_t addr, uint32_t x) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(x) : "memory");
    return old;
}

constexpr int kBuckets = 512;
constexpr uint32_t kHeadKey = 0x41000000u;    // bits of 8.0: the first histogram's end
constexpr uint32_t kTopKey = 0x42000000u;     // bits of 32.0: above it no token has mass
constexpr int kFirstShift = 17;               // 64 buckets to an octave, from 1/32
constexpr uint32_t kFirstKey = kHeadKey - (uint32_t(kBuckets) << kFirstShift);
constexpr int kList = 128;                    // tokens that are collected and sorted at once
constexpr int kPerLane = kBuckets / 32;

// A pass over the row, asked for by the first warp of the first CTA.
enum SampleStep { kDone = 0, kHistogram, kCollect, kNth };
struct SampleCommand {
    int step;
    uint32_t lo, hi;    // keys [lo, hi)
    uint32_t lo2, hi2;  // kCollect: and [lo2, hi2)
    int shift;          // kHistogram: bucket = (key - lo2) >> shift, 0 below lo2
    uint32_t nth;       // kNth: which of the tokens with key lo
    int level, sums;    // kHistogram: where to; with the sums beyond hi
};

// What the thinking warp keeps between passes.
enum Goal { kTopK, kTopP, kToken };
struct Thought {
    int goal, pending, head_count, refine_shift;  // pending: the step whose result is awaited, -1 at first
    bool by_count, head, planned;
    uint64_t W, amount, mass, least, total, plan_mass;
    uint32_t count, lo, hi, tokens;
    uint32_t plan_hi;           // the end of the second interval, for the token that follows
};

struct SampleShared {
    uint32_t low[kBuckets], high[kBuckets], count[kBuckets];  // this slice's: mass = high 2^16 + low
    uint64_t mass[2][kBuckets];                               // the row's, of the first histogram and the last
    uint32_t tokens[2][kBuckets];
    uint64_t lane_mass[2][33];                                // before a lane's buckets, and in all
    uint32_t lane_tokens[2][33];
    uint64_t list[kList];                                     // key 2^32 + index
    uint64_t scan[32];
    float maxima[16];
    uint64_t rest_mass[16], min_mass[16];                     // beyond the first histogram; within min-p's limit
    uint32_t rest_tokens[16], nth_counts[16];
    uint32_t listed;
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
__device__ __noinline__ void sort_list(SampleShared& s, int c) {
    const int lane = threadIdx.x & 31;
    int size = 32;
    while (size < c) size *= 2;
    for (int i = c + lane; i < size; i += 32) s.list[i] = ~0ull;
    __syncwarp();
#pragma unroll 1
    for (int k = 2; k <= size; k *= 2)
#pragma unroll 1
        for (int j = k / 2; j > 0; j /= 2) {
#pragma unroll 1
            for (int t = lane; t < size / 2; t += 32) {
                const int i = 2 * t - (t & (j - 1));
                const uint64_t a = s.list[i], b = s.list[i + j];
                if ((a > b) == ((i & k) == 0)) {
                    s.list[i] = b;
                    s.list[i + j] = a;
                }
            }
            __syncwarp();
        }
}
// Prefixes before each lane's 16 buckets.
__device__ __noinline__ void lane_prefixes(SampleShared& s, int level) {
    const int lane = threadIdx.x & 31;
    uint64_t w = 0;
    uint32_t k = 0;
    const ulonglong2* ms = reinterpret_cast<const ulonglong2*>(&s.mass[level][lane * kPerLane]);
    const uint4* ts = reinterpret_cast<const uint4*>(&s.tokens[level][lane * kPerLane]);
#pragma unroll
    for (int i = 0; i < kPerLane / 2; ++i) w += ms[i].x + ms[i].y;
#pragma unroll
    for (int i = 0; i < kPerLane / 4; ++i) k += ts[i].x + ts[i].y + ts[i].z + ts[i].w;
    const uint64_t ws = warp_scan(w);
    const uint32_t ks = uint32_t(warp_scan(k));
    s.lane_mass[level][lane] = ws - w;
    s.lane_tokens[level][lane] = ks - k;
    if (lane == 31) {
        s.lane_mass[level][32] = ws;
        s.lane_tokens[level][32] = ks;
    }
    __syncwarp();
}
struct Bucket {
    int at;
    uint64_t mass;  // before it
    uint32_t count;
};
// The bucket in which the prefix exceeds `want` (which lies in one).
__device__ __noinline__ Bucket find_bucket(const SampleShared& s, int level, bool counted, uint64_t want) {
    const int lane = threadIdx.x & 31;
    const bool here = counted ? s.lane_tokens[level][lane] <= want && want < s.lane_tokens[level][lane + 1]
                              : s.lane_mass[level][lane] <= want && want < s.lane_mass[level][lane + 1];
    const int src = (__ffs(__ballot_sync(0xffffffffu, here)) - 1) & 31;
    const int b = src * kPerLane + (lane & (kPerLane - 1));
    const uint64_t w = lane < kPerLane ? s.mass[level][b] : 0;
    const uint32_t k = lane < kPerLane ? s.tokens[level][b] : 0;
    const uint64_t we = s.lane_mass[level][src] + warp_scan(w);
    const uint32_t ke = s.lane_tokens[level][src] + uint32_t(warp_scan(k));
    const int at = (__ffs(__ballot_sync(0xffffffffu, lane < kPerLane && want < (counted ? uint64_t(ke) : we))) - 1) & 31;
    return {src * kPerLane + at, __shfl_sync(0xffffffffu, we - w, at), __shfl_sync(0xffffffffu, ke - k, at)};
}
struct Found {
    uint64_t entry, prefix;  // the prefix mass with the entry
};
// Where the prefix of the sorted list's entries [from, to) exceeds `want`, given
// the mass and the count before them.
__device__ __noinline__ Found find_in_list(const SampleShared& s, int from, int to, uint64_t w0, uint64_t k0, bool counted,
                                           uint64_t want) {
    const int lane = threadIdx.x & 31;
    uint64_t e = 0, prefix = 0;
    unsigned hit = 0;
#pragma unroll 1
    for (int j0 = from; j0 < to && !hit; j0 += 32) {
        const int j = j0 + lane;
        e = j < to ? s.list[j] : 0;
        const uint32_t w = j < to ? mass_of_key(uint32_t(e >> 32)) : 0u;
        prefix = w0 + warp_scan(w);
        hit = __ballot_sync(0xffffffffu, j < to && (counted ? k0 + (j - from) == want : want < prefix && want >= prefix - w));
        w0 = __shfl_sync(0xffffffffu, prefix, 31);
    }
    const int src = (__ffs(hit) - 1) & 31;
    return {__shfl_sync(0xffffffffu, e, src), __shfl_sync(0xffffffffu, prefix, src)};
}
// The first entry of the sorted list with a key >= `key`.
__device__ __forceinline__ int list_from(const SampleShared& s, int c, uint32_t key) {
    int at = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < c; j0 += 32) {
        const int j = j0 + (threadIdx.x & 31);
        at += __popc(__ballot_sync(0xffffffffu, j < c && uint32_t(s.list[j] >> 32) < key));
    }
    return at;
}

// One block per row, or a cluster of them with a slice each, held in shared memory.
// The first warp of the first CTA thinks, all others make the passes that it asks
// for: a histogram, the collection of a bucket's tokens, rarely the nth of equal
// tokens.  Most tokens lie far below the largest (beyond y = 8): the first pass
// gives them no buckets, only their sum.
template <class T, int NT>
__global__ void __launch_bounds__(NT, NT == 512 ? 2 : 8)
sample_kernel(const SampleArgs a, int slices, int log_slices)
{
    HX_PDL_PROLOGUE();
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem);
    uint4* held = reinterpret_cast<uint4*>(smem + ((sizeof(SampleShared) + 15) & ~size_t(15)));
    constexpr int EPV = Chunk<T>::EPV;
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
    if (nan || m == -INFINITY) {
        if (tid == 0 && rank == 0) {
            a.tokens[row] = -1;
            if (a.log_probs) a.log_probs[row] = nan ? __uint_as_float(0x7fc00000u) : -INFINITY;
        }
        return;  // the whole cluster
    }

    const float temp = a.temperature ? a.temperature[row] : 1.f;
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
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.nth_counts[rank], 0)), "r"(at)
                             : "memory");
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
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f, mp = a.min_p ? a.min_p[row] : 0.f;
    const float limit = mp > 0.f ? fmaxf(-logf(mp), 0.f) : INFINITY;
    const bool whole = top_k <= 0 || (mp > 0.f && limit > 8.f);

    // Goes on until a pass over the row is needed.
    auto think = [&](bool begin) {
        Thought t;
        if (begin) {
            t = Thought{};
            t.pending = -1;
            t.least = ~0ull;
        } else {
            t = s.thought;
        }
        auto ask = [&](int step, uint32_t lo, uint32_t hi, uint32_t lo2, uint32_t hi2, int shift, uint32_t nth, int sums) {
            t.pending = sums ? -2 : step;
            __syncwarp();
            if (lane == 0) {
                s.command = {step, lo, hi, lo2, hi2, shift, nth, sums ? 0 : 1, sums};
                s.listed = 0;
                s.thought = t;
            }
        };
        auto collect = [&](uint32_t lo, uint32_t hi, uint32_t lo2, uint32_t hi2) { ask(kCollect, lo, hi, lo2, hi2, 0, 0, 0); };
        auto finer = [&] {
            t.refine_shift = 0;
            while (((t.hi - 1 - t.lo) >> t.refine_shift) >= uint32_t(kBuckets)) ++t.refine_shift;
            ask(kHistogram, t.lo, t.hi, t.lo, 0, t.refine_shift, 0, 0);
        };
        auto bucket_lo = [](int b) { return b == 0 ? 0u : kFirstKey + (uint32_t(b) << kFirstShift); };
        auto bucket_hi = [](int b) { return kFirstKey + (uint32_t(b + 1) << kFirstShift); };
        const uint64_t u = min(fraction32(uniform), uint64_t(0xffffffffu)), p32 = fraction32(p);
        Found found{};
        bool have = false;  // `found` answers the goal
        if (begin) lane_prefixes(s, 0);
        const uint64_t head_mass = s.lane_mass[0][32];
        const uint32_t head_tokens = s.lane_tokens[0][32];
        if (t.pending < 0) {
            if (begin && !whole && uint32_t(top_k) > head_tokens) {  // the first k reach beyond the first histogram
                ask(kHistogram, 0, kHeadKey, kFirstKey, 0, kFirstShift, 0, 1);
                return;
            }
            t.total = head_mass;
            t.tokens = head_tokens;
            if (whole || t.pending == -2)
                for (int r = 0; r < slices; ++r) {
                    t.total += s.rest_mass[r];
                    t.tokens += s.rest_tokens[r];
                }
            if (mp > 0.f) {
                t.least = 0;
                for (int r = 0; r < slices; ++r) t.least += s.min_mass[r];
            }
            t.W = t.total;
            const bool counted = top_k > 0 && uint32_t(top_k) <= t.tokens;
            t.goal = counted ? kTopK : p < 1.f ? kTopP : kToken;
            // all that will be asked lies below this: where few tokens do, they
            // are collected once
            const uint64_t most = counted ? uint64_t(top_k) - 1
                                  : p < 1.f ? scaled_mass(t.total, p32) : scaled_mass(min(t.least, t.total), u);
            if (counted ? most < head_tokens : most < head_mass) {
                const Bucket b = find_bucket(s, 0, counted, most);
                if (b.count + s.tokens[0][b.at] <= uint32_t(kList)) {
                    t.head = true;
                    collect(0, bucket_hi(b.at), 0, 0);
                    return;
                }
            }
        } else if (t.head && t.head_count == 0) {
            t.head_count = int(s.listed);
            sort_list(s, t.head_count);
        } else if (t.pending == kCollect) {
            const int c = int(s.listed);
            if (c > kList) {
                if (t.planned) {  // together too many: one after the other
                    t.planned = false;
                    collect(t.lo, t.hi, 0, 0);
                } else {
                    finer();
                }
                return;
            }
            sort_list(s, c);
            const bool apart = t.planned && t.plan_hi <= t.lo;
            const int from = apart ? list_from(s, c, t.lo) : 0;
            found = find_in_list(s, from, c, t.mass, t.count, t.by_count, t.amount);
            have = true;
            if (t.planned) {  // the token that follows lies in the list too
                t.W = min(found.prefix, t.least);
                t.goal = kToken;
                found = find_in_list(s, 0, apart ? from : c, t.plan_mass, 0, false, scaled_mass(t.W, u));
            }
        }
#pragma unroll 1
        for (;;) {
            if (!have) {
                if (t.pending == kHistogram) {  // continue within [lo, hi)
                    lane_prefixes(s, 1);
                    const Bucket b = find_bucket(s, 1, t.by_count, t.by_count ? t.amount - t.count : t.amount - t.mass);
                    t.mass += b.mass;
                    t.count += b.count;
                    t.hi = min(t.hi, t.lo + (uint32_t(b.at + 1) << t.refine_shift));
                    t.lo += uint32_t(b.at) << t.refine_shift;
                } else {  // a new goal
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
                        found = find_in_list(s, 0, t.head_count, 0, 0, t.by_count, t.amount);
                        have = true;
                    } else if (t.by_count ? t.amount < head_tokens : t.amount < head_mass) {
                        const Bucket b = find_bucket(s, 0, t.by_count, t.amount);
                        t.lo = bucket_lo(b.at);
                        t.hi = bucket_hi(b.at);
                        t.mass = b.mass;
                        t.count = b.count;
                        t.planned = false;
                        if (t.goal == kTopP || (t.goal == kTopK && !(p < 1.f))) {
                            // W will lie in this bucket: but for that the token's bucket is
                            // known, and its tokens are collected in the same pass
                            const Bucket b1 = find_bucket(s, 0, false, scaled_mass(min(b.mass, t.least), u));
                            const Bucket b2 = find_bucket(s, 0, false, scaled_mass(min(b.mass + s.mass[0][b.at], t.least), u));
                            if (b2.count + s.tokens[0][b2.at] - b1.count + s.tokens[0][b.at] <= uint32_t(kList)) {
                                t.planned = true;
                                t.plan_mass = b1.mass;
                                t.plan_hi = bucket_hi(b2.at);
                                if (b2.at < b.at) {
                                    collect(t.lo, t.hi, bucket_lo(b1.at), t.plan_hi);
                                    return;
                                }
                                // one interval: the list begins at the token's first bucket
                                t.lo = bucket_lo(b1.at);
                                t.mass = b1.mass;
                                t.count = b1.count;
                            }
                        }
                    } else {  // beyond the first histogram
                        t.mass = head_mass;
                        t.count = head_tokens;
                        t.lo = kHeadKey;
                        t.hi = kTopKey;
                        finer();
                        return;
                    }
                }
                if (!have) {
                    if (t.hi - t.lo > 1) {
                        collect(t.lo, t.hi, 0, 0);
                        return;
                    }
                    // one key: its tokens have one mass
                    const uint64_t w = mass_of_key(t.lo);
                    const uint64_t nth = t.by_count ? t.amount - t.count : (t.amount - t.mass) / w;
                    found.prefix = t.mass + (nth + 1) * w;
                    if (t.goal == kToken) {
                        found.entry = uint64_t(t.lo) << 32;
                        t.amount = nth;
                    }
                }
            }
            if (t.goal == kToken) {
                if (lane == 0) {
                    if (have) a.tokens[row] = int32_t(uint32_t(found.entry));
                    if (a.log_probs)
                        a.log_probs[row] = -__uint_as_float(uint32_t(found.entry >> 32)) -
                                           logf(float(t.W) * (1.f / 2147483648.f));
                }
                ask(have ? kDone : kNth, t.lo, t.lo + 1, 0, 0, 0, uint32_t(t.amount), 0);
                return;
            }
            have = false;
            t.pending = kDone;
            t.W = found.prefix;
            t.goal = t.goal == kTopK && p < 1.f ? kTopP : kToken;
        }
    };

    // ---- passes, the first a histogram up to y = 8 with, where the filters need
    // it, the sum of the rest ----
    SampleCommand cmd{kHistogram, 0, kHeadKey, kFirstKey, 0, kFirstShift, 0, 0, whole};
    const T* element = reinterpret_cast<const T*>(held);
    auto y_of = [&](int i) { return __fmul_rn(__fsub_rn(m, to_float(element[i])), inv_t); };
#pragma unroll 1
    for (bool begin = true;; begin = false) {
        // a logit below which no key is below hi: y >= hi once (m - l)/T is above it
        // by more than the roundings
        const float least = m - __uint_as_float(cmd.hi) * temp * 1.00001f - fabsf(m) * 1e-5f;
        if (cmd.step == kHistogram) {
            for (int b = tid; b < kBuckets; b += NT) s.low[b] = s.high[b] = s.count[b] = 0u;
            __syncthreads();
            uint64_t rest = 0, below = 0;
            uint32_t tokens = 0;
#pragma unroll 1
            for (int c = tid; c < n; c += NT) {
                const uint4 raw = held[c];
                if (!cmd.sums && !(chunk_max(raw, T()) >= least)) continue;
                float x[EPV];
                Chunk<T>::unpack(raw, x);
#pragma unroll
                for (int r = 0; r < EPV; ++r) {
                    const float y = __fmul_rn(__fsub_rn(m, x[r]), inv_t);
                    const uint32_t key = __float_as_uint(y), w = mass_of(y);
                    if (key - cmd.lo < cmd.hi - cmd.lo) {
                        if (w) {
                            const uint32_t b = key < cmd.lo2 ? 0u : (key - cmd.lo2) >> cmd.shift;
                            atomicAdd(&s.low[b], w & 0xffffu);
                            atomicAdd(&s.high[b], w >> 16);
                            atomicAdd(&s.count[b], 1u);
                        }
                    } else if (key >= kHeadKey) {
                        rest += w;
                        tokens += w != 0;
                    }
                    if (y <= limit) below += w;
                }
            }
            if (cmd.level == 0) {  // the slice's sums to the first CTA
                rest = block_reduce<NT>(rest, s.scan, SumOp());
                below = block_reduce<NT>(below, s.scan, SumOp());
                tokens = block_reduce<NT>(tokens, reinterpret_cast<uint32_t*>(s.scan), SumOp());
                if (tid == 0) {
                    if (many) {
                        remote_store(tc::cluster_addr(&s.rest_mass[rank], 0), rest);
                        remote_store(tc::cluster_addr(&s.min_mass[rank], 0), below);
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.rest_tokens[rank], 0)),
                                     "r"(tokens) : "memory");
                    } else {
                        s.rest_mass[0] = rest;
                        s.min_mass[0] = below;
                        s.rest_tokens[0] = tokens;
                    }
                }
            }
            sync();
            // the buckets of all slices, each CTA a share of them, to the first CTA
            const int share = kBuckets >> log_slices;
#pragma unroll 1
            for (int b = rank * share + tid; b < (rank + 1) * share; b += NT) {
                if (many) {
                    uint64_t w = 0;
                    uint32_t k = 0;
                    for (int r = 0; r < slices; ++r) {
                        w += (uint64_t(remote_u32(tc::cluster_addr(&s.high[b], r))) << 16) +
                             remote_u32(tc::cluster_addr(&s.low[b], r));
                        k += remote_u32(tc::cluster_addr(&s.count[b], r));
                    }
                    remote_store(tc::cluster_addr(&s.mass[cmd.level][b], 0), w);
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.tokens[cmd.level][b], 0)),
                                 "r"(k) : "memory");
                } else {
                    s.mass[cmd.level][b] = (uint64_t(s.high[b]) << 16) + s.low[b];
                    s.tokens[cmd.level][b] = s.count[b];
                }
            }
        } else if (cmd.step == kCollect) {
            const uint32_t counter = many ? tc::cluster_addr(&s.listed, 0) : 0, list = many ? tc::cluster_addr(s.list, 0) : 0;
#pragma unroll 1
            for (int c = tid; c < n; c += NT) {
                if (!(chunk_max(held[c], T()) >= least)) continue;
#pragma unroll 1
                for (int i = c * EPV; i < (c + 1) * EPV; ++i) {
                    const uint32_t key = __float_as_uint(y_of(i));
                    if (key - cmd.lo >= cmd.hi - cmd.lo && key - cmd.lo2 >= cmd.hi2 - cmd.lo2) continue;
                    const uint64_t entry = (uint64_t(key) << 32) | uint32_t(base + i);
                    const uint32_t at = many ? remote_add(counter, 1u) : atomicAdd(&s.listed, 1u);
                    if (at >= kList) continue;
                    if (many) remote_store(list + at * 8, entry); else s.list[at] = entry;
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
            cmd = {int(remote_u32(at)), remote_u32(at + 4), remote_u32(at + 8), remote_u32(at + 12), remote_u32(at + 16),
                   int(remote_u32(at + 20)), remote_u32(at + 24), int(remote_u32(at + 28)), int(remote_u32(at + 32))};
        }
    }
    if (cmd.step == kNth) {  // the nth token with key lo, in index order
        uint32_t mine = 0, before = 0;
        for (int i = tid; i < n * EPV; i += NT) mine += __float_as_uint(y_of(i)) == cmd.lo;
        mine = block_reduce<NT>(mine, reinterpret_cast<uint32_t*>(s.scan), SumOp());
        if (many) {
            if (tid < slices)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.nth_counts[rank], tid)), "r"(mine)
                             : "memory");
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
    const size_t smem = ((sizeof(SampleShared) + 15) & ~size_t(15)) + size_t((chunks + slices - 1) / slices) * 16;
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
