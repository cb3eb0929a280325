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
// masses over the bits (32 buckets to an octave) finds the bucket in which a
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
constexpr uint32_t kTopKey = 0x42000000u;     // bits of 32.0: above it no token has mass
constexpr int kFirstShift = 18;               // 32 buckets to an octave
constexpr int kList = 512;                    // tokens that are collected and sorted at once

// What the cluster's first CTA has the others do.
enum SampleStep { kDone = 0, kHistogram, kCollect, kNth };
struct SampleCommand {
    int step;
    uint32_t lo, hi;  // keys [lo, hi)
    int shift;
    uint32_t nth;     // kNth: which of the tokens with key lo
};

struct SampleShared {
    uint32_t low[kBuckets], high[kBuckets], count[kBuckets];  // this slice's: mass = high 2^16 + low
    uint64_t mass[2][kBuckets];                               // the row's prefix masses before each bucket
    uint32_t tokens[2][kBuckets];                             // and counts; [0] of the first histogram
    uint64_t total[2];
    uint64_t list[kList];                                     // key 2^32 + index
    uint64_t scan[32];
    float maxima[16];
    uint64_t min_mass[16];
    uint32_t nth_counts[16];
    uint32_t listed, found_bucket;
    uint64_t found_mass;
    uint32_t found_count;
    SampleCommand command;
    int nan;
};

// Inclusive prefix sums over the block's threads; `total` is the last.
template <int NT>
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* scratch, uint64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += scratch[w];
        total += scratch[w];
    }
    __syncthreads();
    return x + before;
}

// Sorts n <= kList numbers; entries up to the next power of two are written.
template <int NT>
__device__ __forceinline__ void block_sort(uint64_t* list, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += NT) list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            for (int t = threadIdx.x; t < size / 2; t += NT) {
                const int i = 2 * t - (t & (j - 1));
                const uint64_t a = list[i], b = list[i + j];
                if ((a > b) == ((i & k) == 0)) {
                    list[i] = b;
                    list[i + j] = a;
                }
            }
            // strides up to 32 stay within a warp's 64 entries
            if (j > 32 || j == 1) __syncthreads(); else __syncwarp();
        }
}

// One block per row, or a cluster of them with a slice each; the slice is held in
// shared memory as y.  The first CTA decides, the others follow its commands.
// Every pass over a slice costs less than its load did; what a row takes beside
// them is the latency of the block's (and the cluster's) barriers, so few rows to
// an SM overlap.
template <class T, int NT>
__global__ void __launch_bounds__(NT)
sample_kernel(const SampleArgs a, int slices, int held)
{
    HX_PDL_PROLOGUE();
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(smem);
    float* y = reinterpret_cast<float*>(smem + ((sizeof(SampleShared) + 15) & ~size_t(15)));  // [held]
    constexpr int EPV = Chunk<T>::EPV;
    const int tid = threadIdx.x, lane = tid & 31, V = int(a.vocab);
    const int rank = int(blockIdx.x) & (slices - 1);
    const size_t row = blockIdx.x / unsigned(slices);
    const T* l = static_cast<const T*>(a.logits) + row * a.stride;
    const bool many = slices > 1;
    auto sync = [&] {
        if (many) tc::cluster_sync(); else __syncthreads();
    };
    // this CTA's chunks; y[p] is element p + base
    const int lead = int((reinterpret_cast<uintptr_t>(l) & 15) / sizeof(T));
    const int chunks = (V + lead + EPV - 1) / EPV, each = (chunks + slices - 1) / slices;
    const int first = min(chunks, rank * each), last = min(chunks, first + each);
    const int base = first * EPV - lead, n = (last - first) * EPV;

    // ---- the slice, its maximum ----
    if (tid == 0) s.nan = 0;
    float m = -INFINITY;
    bool nan = false;
    for (int c0 = first + tid; c0 < last; c0 += 4 * NT) {
        uint4 raw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = (c0 + q * NT) * EPV - lead;
            if (c0 + q * NT < last && i >= 0 && i + EPV <= V) raw[q] = *reinterpret_cast<const uint4*>(l + i);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = c0 + q * NT, i = c * EPV - lead;
            if (c >= last) break;
            float x[EPV];
            if (i >= 0 && i + EPV <= V) {
                Chunk<T>::unpack(raw[q], x);
            } else {
#pragma unroll
                for (int r = 0; r < EPV; ++r) x[r] = i + r >= 0 && i + r < V ? to_float(l[i + r]) : -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < EPV; ++r) {
                nan |= x[r] != x[r];
                m = fmaxf(m, x[r]);
            }
            float4* to = reinterpret_cast<float4*>(y + (c - first) * EPV);
#pragma unroll
            for (int r = 0; r < EPV; r += 4) to[r / 4] = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
        }
    }
    float* scratch = reinterpret_cast<float*>(s.scan);
    m = block_reduce<NT>(m, scratch, MaxOp());
    nan = __syncthreads_or(nan || m == INFINITY) != 0;
    if (many) {
        tc::cluster_sync();  // every CTA has started
        // a NaN marks the whole row: no maximum is above it
        if (tid < slices) {
            const uint32_t to = tc::cluster_addr(&s.maxima[rank], tid);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(nan ? INFINITY : m) : "memory");
        }
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
    float inv_t = __fdiv_rn(1.f, temp);
    const bool greedy = !(temp > 0.f) || temp == INFINITY || inv_t == INFINITY;
    if (greedy) inv_t = 1.f;
    int top_k = greedy ? 1 : a.top_k ? a.top_k[row] : 0;
    if (top_k <= 0 || top_k >= V) top_k = 0;
    const float p = a.top_p && !greedy ? a.top_p[row] : 1.f, mp = a.min_p && !greedy ? a.min_p[row] : 0.f;
    const float limit = mp > 0.f ? fmaxf(-logf(mp), 0.f) : INFINITY;

    for (int i = tid * 4; i < n; i += NT * 4) {
        float4 x = *reinterpret_cast<float4*>(y + i);
        x.x = __fmul_rn(__fsub_rn(m, x.x), inv_t);
        x.y = __fmul_rn(__fsub_rn(m, x.y), inv_t);
        x.z = __fmul_rn(__fsub_rn(m, x.z), inv_t);
        x.w = __fmul_rn(__fsub_rn(m, x.w), inv_t);
        *reinterpret_cast<float4*>(y + i) = x;
    }

    // ---- the commands ----
    // bucket of a key under (lo, shift): the first takes all below its range
    const uint32_t first_lo = kTopKey - (uint32_t(kBuckets) << kFirstShift);
    auto bucket_of = [](uint32_t key, uint32_t lo, int shift) { return key < lo ? 0u : (key - lo) >> shift; };
    auto histogram = [&](const SampleCommand& c, bool with_limit) {
        for (int b = tid; b < kBuckets; b += NT) s.low[b] = s.high[b] = s.count[b] = 0u;
        __syncthreads();
        uint64_t below = 0;
        const uint32_t from = with_limit ? first_lo : c.lo;
        for (int i = tid; i < n; i += NT) {
            const float v = y[i];
            const uint32_t key = __float_as_uint(v);
            if (key >= c.hi || (!with_limit && key < c.lo)) continue;
            const uint32_t w = mass_of(v);
            if (w == 0) continue;
            const uint32_t b = bucket_of(key, from, c.shift);
            atomicAdd(&s.low[b], w & 0xffffu);
            atomicAdd(&s.high[b], w >> 16);
            atomicAdd(&s.count[b], 1u);
            if (v <= limit) below += w;
        }
        if (with_limit && mp > 0.f) {
            below = block_reduce<NT>(below, s.scan, SumOp());
            if (tid == 0) {
                if (many) remote_store(tc::cluster_addr(&s.min_mass[rank], 0), below); else s.min_mass[0] = below;
            }
        }
        sync();
        // the buckets of all slices, each CTA a share of them, to the first CTA
        const int level = with_limit ? 0 : 1, share = kBuckets / slices;
        for (int b = rank * share + tid; b < (rank + 1) * share; b += NT) {
            uint64_t w = 0;
            uint32_t k = 0;
            for (int r = 0; r < slices; ++r) {
                if (many) {
                    w += (uint64_t(remote_u32(tc::cluster_addr(&s.high[b], r))) << 16) +
                         remote_u32(tc::cluster_addr(&s.low[b], r));
                    k += remote_u32(tc::cluster_addr(&s.count[b], r));
                } else {
                    w += (uint64_t(s.high[b]) << 16) + s.low[b];
                    k += s.count[b];
                }
            }
            if (many) {
                remote_store(tc::cluster_addr(&s.mass[level][b], 0), w);
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.tokens[level][b], 0)), "r"(k)
                             : "memory");
            } else {
                s.mass[level][b] = w;
                s.tokens[level][b] = k;
            }
        }
        sync();
    };
    auto collect = [&](const SampleCommand& c) {
        const uint32_t counter = many ? tc::cluster_addr(&s.listed, 0) : 0, list = many ? tc::cluster_addr(s.list, 0) : 0;
        for (int i = tid; i < n; i += NT) {
            const uint32_t key = __float_as_uint(y[i]);
            if (key < c.lo || key >= c.hi) continue;
            const uint64_t entry = (uint64_t(key) << 32) | uint32_t(i + base);
            if (many) {
                const uint32_t at = remote_add(counter, 1u);
                if (at < kList) remote_store(list + at * 8, entry);
            } else {
                const uint32_t at = atomicAdd(&s.listed, 1u);
                if (at < kList) s.list[at] = entry;
            }
        }
        sync();
    };
    // the token that is the nth with key lo, in index order
    auto nth_token = [&](const SampleCommand& c) {
        uint32_t mine = 0;
        for (int i = tid; i < n; i += NT) mine += __float_as_uint(y[i]) == c.lo;
        mine = block_reduce<NT>(mine, reinterpret_cast<uint32_t*>(s.scan), SumOp());
        uint32_t before = 0;
        if (many) {
            if (tid < slices)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(&s.nth_counts[rank], tid)), "r"(mine)
                             : "memory");
            tc::cluster_sync();
            for (int r = 0; r < rank; ++r) before += s.nth_counts[r];
        }
        if (c.nth < before || c.nth >= before + mine) return;
        uint32_t have = before;
        uint32_t* votes_of = reinterpret_cast<uint32_t*>(s.scan);
        for (int i0 = 0; i0 < n && have <= c.nth; i0 += NT) {
            const int i = i0 + tid;
            const bool eq = i < n && __float_as_uint(y[i]) == c.lo;
            const unsigned votes = __ballot_sync(0xffffffffu, eq);
            if (lane == 0) votes_of[tid >> 5] = __popc(votes);
            __syncthreads();
            uint32_t at = have;
            for (int w = 0; w < NT / 32; ++w) {
                if (w < (tid >> 5)) at += votes_of[w];
                have += votes_of[w];
            }
            at += __popc(votes & ((1u << lane) - 1));
            if (eq && at == c.nth) a.tokens[row] = i + base;
            __syncthreads();
        }
    };

    // The first histogram needs no command.
    SampleCommand cmd{kHistogram, first_lo, kTopKey, kFirstShift, 0};
    histogram(cmd, true);
    if (rank != 0) {
        for (;;) {
            tc::cluster_sync();
            const uint32_t at = tc::cluster_addr(&s.command, 0);
            cmd.step = int(remote_u32(at));
            cmd.lo = remote_u32(at + 4);
            cmd.hi = remote_u32(at + 8);
            cmd.shift = int(remote_u32(at + 12));
            cmd.nth = remote_u32(at + 16);
            if (cmd.step == kHistogram) histogram(cmd, false);
            else if (cmd.step == kCollect) collect(cmd);
            else {
                if (cmd.step == kNth) nth_token(cmd);
                break;
            }
        }
        tc::cluster_sync();
        return;
    }

    // ---- the first CTA ----
    auto issue = [&](const SampleCommand& c) {
        if (tid == 0) {
            s.command = c;
            s.listed = 0;
        }
        sync();
    };
    // turns bucket masses and counts into prefixes before each bucket
    auto prefixes = [&](int level) {
        constexpr int per = kBuckets / NT;
        uint64_t w[per], sum = 0;
        uint32_t k[per], count = 0;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            w[i] = s.mass[level][tid * per + i];
            k[i] = s.tokens[level][tid * per + i];
            sum += w[i];
            count += k[i];
        }
        uint64_t total, all;
        uint64_t at = block_scan<NT>(sum, s.scan, total) - sum;
        uint32_t c = uint32_t(block_scan<NT>(count, s.scan, all)) - count;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            s.mass[level][tid * per + i] = at;
            s.tokens[level][tid * per + i] = c;
            at += w[i];
            c += k[i];
        }
        if (tid == 0) s.total[level] = total;
        __syncthreads();
        return uint32_t(all);
    };
    const uint32_t positive = prefixes(0);  // tokens with mass
    const uint64_t total = s.total[0];
    auto mass_after = [&](int level, int b) { return b + 1 < kBuckets ? s.mass[level][b + 1] : s.total[level]; };

    struct Place {       // where a prefix crosses an amount
        uint32_t key;    // of the token
        int index;       // of the token; -1 when only its number among its equals is known
        uint32_t nth;
        uint64_t prefix; // mass up to and with the token
    };
    // the bucket that holds the token: by mass, or by number of tokens
    auto find_bucket = [&](int level, bool by_count, uint64_t amount) {
        for (int b = tid; b < kBuckets; b += NT) {
            const uint64_t at = by_count ? s.tokens[level][b] : s.mass[level][b];
            const uint64_t to = b + 1 < kBuckets ? (by_count ? s.tokens[level][b + 1] : s.mass[level][b + 1])
                                                 : (by_count ? ~0ull : s.total[level]);
            if (at <= amount && amount < to && (!by_count || b + 1 < kBuckets || s.mass[level][b] < s.total[level])) {
                s.found_bucket = b;
                s.found_mass = s.mass[level][b];
                s.found_count = s.tokens[level][b];
            }
        }
        __syncthreads();
        const int b = int(s.found_bucket);
        return b;
    };
    // within the sorted list of c tokens, mass and count before it given
    auto find_in_list = [&](int c, uint64_t mass, uint64_t count, bool by_count, uint64_t amount) {
        constexpr int per = kList / NT;
        uint64_t e[per], w[per], sum = 0;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int at = tid * per + i;
            e[i] = at < c ? s.list[at] : 0ull;
            w[i] = at < c ? mass_of_key(uint32_t(e[i] >> 32)) : 0u;
            sum += w[i];
        }
        uint64_t all;
        uint64_t at = mass + block_scan<NT>(sum, s.scan, all) - sum;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int j = tid * per + i;
            const bool here = by_count ? count + j == amount : at <= amount && amount < at + w[i];
            if (j < c && here) {
                s.found_mass = at + w[i];
                s.found_bucket = uint32_t(e[i] >> 32);
                s.found_count = uint32_t(e[i]);
            }
            at += w[i];
        }
        __syncthreads();
        Place r{s.found_bucket, int(s.found_count), 0, s.found_mass};
        __syncthreads();
        return r;
    };
    bool head = false;  // the list holds the head of the order, sorted
    int head_count = 0;
    auto cross = [&](bool by_count, uint64_t amount) {
        if (head) return find_in_list(head_count, 0, 0, by_count, amount);
        int level = 0, b = find_bucket(0, by_count, amount), shift = kFirstShift;
        uint64_t mass = s.found_mass;
        uint64_t count = s.found_count;
        uint32_t lo = b == 0 ? 0u : first_lo + (uint32_t(b) << shift), hi = first_lo + (uint32_t(b + 1) << shift);
        __syncthreads();
        for (;;) {
            if (hi - lo == 1) {  // one key: its tokens have one mass
                const uint64_t w = mass_of_key(lo);
                const uint64_t nth = by_count ? amount - count : (amount - mass) / w;
                return Place{lo, -1, uint32_t(nth), mass + (nth + 1) * w};
            }
            issue({kCollect, lo, hi, 0, 0});
            collect({kCollect, lo, hi, 0, 0});
            const int c = int(s.listed);
            if (c <= kList) {
                block_sort<NT>(s.list, c);
                return find_in_list(c, mass, count, by_count, amount);
            }
            // too many: a finer histogram of this bucket
            shift = 0;
            while (((hi - 1 - lo) >> shift) >= uint32_t(kBuckets)) ++shift;
            const SampleCommand finer{kHistogram, lo, hi, shift, 0};
            issue(finer);
            histogram(finer, false);
            prefixes(1);
            level = 1;
            // prefixes of this level count from the bucket's beginning
            b = find_bucket(1, by_count, by_count ? amount - count : amount - mass);
            mass += s.found_mass;
            count += s.found_count;
            const uint32_t start = lo + (uint32_t(b) << shift);
            hi = min(hi, lo + (uint32_t(b + 1) << shift));
            lo = start;
            __syncthreads();
        }
    };

    uint64_t W = total;
    uint64_t u = fraction32(a.uniform[row]);
    if (u > 0xffffffffull) u = 0xffffffffull;
    uint64_t least = ~0ull;
    if (mp > 0.f) {
        least = 0;
        for (int r = 0; r < slices; ++r) least += s.min_mass[r];
    }
    // The head of the order in one list, where all that is asked lies in it.
    {
        const bool counted = top_k > 0 && uint32_t(top_k) < positive;
        const uint64_t need = counted ? uint64_t(top_k) - 1
                              : p < 1.f ? scaled_mass(total, fraction32(p))
                                        : scaled_mass(least < total ? least : total, u);
        const int b = find_bucket(0, counted, need);
        const uint32_t tokens = b + 1 < kBuckets ? s.tokens[0][b + 1] : positive;
        __syncthreads();
        if (tokens <= uint32_t(kList)) {
            const SampleCommand c{kCollect, 0, first_lo + (uint32_t(b + 1) << kFirstShift), 0, 0};
            issue(c);
            collect(c);
            // tokens without mass may share the last bucket
            head_count = int(s.listed);
            head = head_count <= kList;
            if (head) block_sort<NT>(s.list, head_count);
        }
    }
    if (top_k > 0 && uint32_t(top_k) < positive) W = cross(true, uint64_t(top_k) - 1).prefix;
    if (p < 1.f) {
        uint64_t need = scaled_mass(W, fraction32(p));
        if (need < 1) need = 1;
        W = cross(false, need - 1).prefix;
    }
    if (least < W) W = least;
    const Place at = cross(false, scaled_mass(W, u));
    const SampleCommand end{at.index < 0 ? kNth : kDone, at.key, at.key + 1, 0, at.nth};
    issue(end);
    if (at.index < 0) nth_token(end);
    if (tid == 0) {
        if (at.index >= 0) a.tokens[row] = at.index;
        if (a.log_probs)
            a.log_probs[row] = greedy ? 0.f : -__uint_as_float(at.key) - logf(float(W) * (1.f / 2147483648.f));
    }
    if (many) tc::cluster_sync();
}

template <class T, int NT>
void launch_sample(hx_runtime* rt, const SampleArgs& a, uint32_t rows, long chunks, int slices)
{
    constexpr int EPV = Chunk<T>::EPV;
    const int held = int((chunks + slices - 1) / slices) * EPV;
    const size_t smem = ((sizeof(SampleShared) + 15) & ~size_t(15)) + size_t(held) * 4;
    require(uint64_t(rows) * slices <= 0x7fffffffu, HX_ERR_UNSUPPORTED, "sampling: too many rows for one call");
    auto kernel = sample_kernel<T, NT>;
    static thread_local int opted[64] = {};
    if (!opted[rt->device & 63]) {
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 131072));
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        opted[rt->device & 63] = 1;
    }
    launch_rows(kernel, rows * unsigned(slices), NT, slices, true, smem, rt->stream, a, slices, held);
    HX_LAUNCHED(rt);
}

template <class T>
void launch_sample(hx_runtime* rt, const SampleArgs& a, uint32_t rows)
{
    constexpr int EPV = Chunk<T>::EPV;
    const long chunks = row_chunks(a.logits, a.stride, rows, a.vocab, sizeof(T));
    if (chunks * EPV <= 4096 + 2 * EPV) {
        launch_sample<T, 128>(rt, a, rows, chunks, 1);
    } else {
        int s = 1;
        while (chunks * EPV > 16640L * s) s *= 2;
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
