// top_logits.cu -- the k largest logits of every row and its log-sum-exp.
//
// Order: value descending, index ascending among equals; NaN after -inf.  With
// keys whose ascending order is that of descending values, an entry is the
// number key 2^32 + index and the record is the k smallest entries in order.
// lse = ref/tau + log sum exp((l - ref)/tau); a NaN makes it NaN, else a +inf +inf.
// No row is sorted.  The k-th largest of the maxima of more than k groups of a row's
// logits is a lower bound of its k-th largest logit, and a close one: the few
// logits that reach it are collected and sorted.
// No counterpart in the reference, whose sampler sorts the whole row on the
// host (nicopedia_generation.h:286-395).
#include <cmath>

#include "head_ops.cuh"
#include "head_plan.cuh"
#include "head_stream.cuh"

namespace hx {
namespace head {

__device__ __forceinline__ uint64_t entry_of(uint32_t key, int index) { return (uint64_t(key) << 32) | uint32_t(index); }

// A warp's smallest t with count(key <= t) >= k over the keys of all lanes; any
// t with a count up to k + slack will do.  At least k keys exist.
template <int N>
__device__ __forceinline__ uint32_t warp_kth(const uint32_t (&key)[N], int k, int slack) {
    uint32_t lo = 0xffffffffu, hi = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        lo = min(lo, key[i]);
        hi = max(hi, key[i]);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
#pragma unroll 1
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += key[i] <= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= k) {
            hi = mid;
            if (c <= k + slack) break;
        } else {
            lo = mid + 1;
        }
    }
    return hi;
}

// One warp sorts the first n entries of a list that has room up to the next
// power of two.
__device__ __noinline__ void warp_sort_list(uint64_t* list, int n) {
    const int lane = threadIdx.x & 31;
    int size = 32;
    while (size < n) size *= 2;
    for (int i = n + lane; i < size; i += 32) list[i] = ~0ull;
    __syncwarp();
#pragma unroll 1
    for (int k = 2; k <= size; k *= 2)
#pragma unroll 1
        for (int j = k / 2; j > 0; j /= 2) {
#pragma unroll 2
            for (int t = lane; t < size / 2; t += 32) {
                const int i = 2 * t - (t & (j - 1));
                const uint64_t a = list[i], b = list[i + j];
                if ((a > b) == ((i & k) == 0)) {
                    list[i] = b;
                    list[i + j] = a;
                }
            }
            __syncwarp();
        }
}

__device__ __forceinline__ void write_entry(const TopArgs& a, size_t row, int rank, uint64_t entry) {
    a.values[row * a.k + rank] = from_descending_key(uint32_t(entry >> 32));
    a.indices[row * a.k + rank] = int32_t(uint32_t(entry));
}

// One warp's exact list of the `want` first entries of elements [e0, e1) of a row,
// unsorted, where the collection above `bound` did not serve: too many equal
// logits, or NaN.  The list has room for them.
template <class T>
__device__ __noinline__ int exact_list(const T* row, int e0, int e1, float bound, int want, uint64_t* list) {
    const int lane = threadIdx.x & 31;
    auto key_at = [&](int i) { return descending_key(to_float(row[i])); };
    auto count_to = [&](uint32_t t) {
        int c = 0;
        for (int i = e0 + lane; i < e1; i += 32) c += key_at(i) <= t;
        return __reduce_add_sync(0xffffffffu, c);
    };
    // the bound is often the k-th itself
    uint32_t t = descending_key(bound);
    if (!(t > 0 && count_to(t - 1) < want && count_to(t) >= want)) {
        uint32_t lo = 0, hi = 0xffffffffu;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (count_to(mid) >= want) hi = mid; else lo = mid + 1;
        }
        t = lo;
    }
    int have = 0;
    auto append = [&](bool equal) {
        for (int i0 = e0; i0 < e1 && have < want; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t key = i < e1 ? key_at(i) : 0u;
            const bool in = i < e1 && (equal ? key == t : key < t);
            const unsigned votes = __ballot_sync(0xffffffffu, in);
            const int at = have + __popc(votes & ((1u << lane) - 1));
            if (in && at < want) list[at] = entry_of(key, i);
            have += __popc(votes);
        }
    };
    append(false);
    append(true);
    __syncwarp();
    return want;
}

// ---- short rows: a warp per row ---------------------------------------------------
// Rows of up to 1024 logits (with the lead): 32 to a lane, in registers, read from
// the second of two buffers while the next row's copy is in flight.  Bound by the
// instructions of the selection (about 1400 a row at k = 32): 131072x1024 float32 218 us, 2.6 TB/s.
constexpr int kTopTeams = 4;
// Entries that a warp's list holds.
__host__ __device__ constexpr int top_list(int k) { return k <= 32 ? 128 : k <= 96 ? 256 : 512; }

template <class T>
__global__ void __launch_bounds__(32 * kTopTeams, 6)
top_warp_kernel(const TopArgs a, uint32_t rows)
{
    HX_PDL_PROLOGUE();
    constexpr int EPV = Chunk<T>::EPV, N = Chunk<T>::N, kChunks = 32 * N;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_full[kTopTeams * 2];
    __shared__ int s_aborted;
    const int k = int(a.k), V = int(a.vocab), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T* rows_at = reinterpret_cast<T*>(smem + warp * (2 * kChunks * 16));
    uint64_t* list = reinterpret_cast<uint64_t*>(smem + kTopTeams * 2 * kChunks * 16) + warp * top_list(k);
    uint64_t* full = s_full + warp * 2;
    const WaitState ws{a.err, &s_aborted};
    if (threadIdx.x == 0) s_aborted = 0;
    if (lane == 0) {
        tc::mbar_init(full, 1);
        tc::mbar_init(full + 1, 1);
        tc::fence_mbar_init();
    }
    __syncthreads();

    const uint32_t team = blockIdx.x * kTopTeams + warp, teams = gridDim.x * kTopTeams;
    auto span_of = [&](size_t row) { return Span<T>(static_cast<const T*>(a.logits) + row * a.stride, V, 0, 0); };
    auto issue = [&](size_t row, int b) {
        const Span<T> span = span_of(row);
        if (lane == 0) {
            const uint32_t bytes = uint32_t(span.w1 - span.w0) * 16;
            tc::mbar_arrive_expect_tx(full + b, bytes);
            if (bytes)
                bulk_load(rows_at + (b * kChunks + span.w0) * EPV, span.row - span.lead + span.w0 * EPV, bytes, full + b);
        }
    };
    auto partial = [&](const Span<T>& span) {
        const int r = lane & 7, pc = lane < 8 ? 0 : span.last - 1;
        return lane < 16 && r < EPV && !span.whole(pc) ? pc * EPV + r : -1;
    };
    auto partial_value = [&](const Span<T>& span) {
        const int p = partial(span), i = p - span.lead;
        return p >= 0 && i >= 0 && i < V ? span.row[i] : from_float<T>(-INFINITY);
    };
    for (int i = 0; i < 2; ++i)
        if (team + i * teams < rows) issue(team + i * teams, i);
    T px = from_float<T>(0.f);
    if (team < rows) px = partial_value(span_of(team));
    const float c = kLog2e / a.tau, inv_tau = 1.f / a.tau;
    unsigned n = 0;
    for (size_t row = team; row < rows; row += teams, ++n) {
        const int b = n & 1;
        const Span<T> span = span_of(row);
        T* l = rows_at + b * kChunks * EPV;
        stream_wait(full + b, (n >> 1) & 1, ws);
        if (partial(span) >= 0) l[partial(span)] = px;
        __syncwarp();
        if (row + teams < rows) px = partial_value(span_of(row + teams));
        // lane's chunks are lane, lane + 32, ...: position (32 j + lane) EPV + r
        float v[kPerThread];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int p = 32 * j + lane;
            float x[EPV];
            Chunk<T>::unpack(reinterpret_cast<const uint4*>(l)[p], x);
#pragma unroll
            for (int r = 0; r < EPV; ++r) v[j * EPV + r] = x[r];
        }
        if (span.last < kChunks) {
#pragma unroll
            for (int i = 0; i < kPerThread; ++i)
                if (32 * (i / EPV) + lane >= span.last) v[i] = -INFINITY;
        }
        float group[kPerThread / 4], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPerThread / 4; ++i) {
            group[i] = fmaxf(fmaxf(v[4 * i], v[4 * i + 1]), fmaxf(v[4 * i + 2], v[4 * i + 3]));
            top = fmaxf(top, group[i]);
        }
        top = warp_max(top);
        if (a.lse) {
            const float ref = fabsf(top) < INFINITY ? top : 0.f, scale = scale_against(ref, c), o = ref * scale;
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) s[i & 3] += tc::exp2_approx(fmaf(v[i], scale, -o));
            const float sum = warp_reduce((s[0] + s[1]) + (s[2] + s[3]), SumOp());
            if (lane == 0)
                a.lse[row] = top == INFINITY && sum == sum ? top : ref * inv_tau + (logf(sum) - kLn2 * fmaf(ref, scale, -o));
        }
        float bound;  // at least k logits reach it, and not many more
        // (groups: twice as many as k that have a logit)
        if (k <= 32 && 16 * k <= V) {  // the k-th of the 128 maxima of eight logits each
            uint32_t key[kPerThread / 8];
#pragma unroll
            for (int i = 0; i < kPerThread / 8; ++i) key[i] = descending_key(fmaxf(group[2 * i], group[2 * i + 1]));
            bound = from_descending_key(warp_kth(key, k, 4));
        } else if (k <= 96 && 8 * k <= V) {  // of the 256 maxima of four
            uint32_t key[kPerThread / 4];
#pragma unroll
            for (int i = 0; i < kPerThread / 4; ++i) key[i] = descending_key(group[i]);
            bound = from_descending_key(warp_kth(key, k, 4));
        } else {
            uint32_t key[kPerThread];
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) key[i] = descending_key(v[i]);
            bound = from_descending_key(warp_kth(key, k, 64));
        }
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) mask |= uint32_t(v[i] >= bound) << i;
        int mine = __popc(mask), count = __reduce_add_sync(0xffffffffu, mine);
        bool listed = false;
        if (!(bound > -INFINITY) || count > min(top_list(k), 384)) {
            // NaN, or many equal logits
            count = exact_list(l + span.lead, 0, V, bound, k, list);
            listed = true;
        }
        // first the places, lane 32 + bit, then each lane the entries of its share
        uint32_t* places = reinterpret_cast<uint32_t*>(list);
        if (!listed) {
            int at = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, at, o);
                if (lane >= o) at += y;
            }
            at -= mine;
            for (; mask; mask &= mask - 1) places[at++] = uint32_t(lane * 32 + __ffs(mask) - 1);
            __syncwarp();
            // from the end, so that an entry overwrites places already read
            for (int j0 = (count - 1) & ~31; j0 >= 0; j0 -= 32) {
                const int j = j0 + lane;
                uint64_t e = 0;
                if (j < count) {
                    const int bit = places[j] & 31, from = places[j] >> 5;
                    const int p = (32 * (bit / EPV) + from) * EPV + bit % EPV;
                    e = entry_of(descending_key(to_float(l[p])), p - span.lead);
                }
                __syncwarp();
                if (j < count) list[j] = e;
                __syncwarp();
            }
        }
        __syncwarp();
        if (row + 2 * size_t(teams) < rows) {  // the row is in registers and in the list
            tc::fence_proxy_async_smem();
            __syncwarp();
            issue(row + 2 * size_t(teams), b);
        }
        if (count <= 64) {
            // the rank of an entry is the number of smaller ones
            const uint64_t e0 = lane < count ? list[lane] : ~0ull, e1 = lane + 32 < count ? list[lane + 32] : ~0ull;
            int r0 = 0, r1 = 0;
#pragma unroll 4
            for (int j = 0; j < count; ++j) {
                const uint64_t x = list[j];
                r0 += x < e0;
                r1 += x < e1;
            }
            if (lane < count && r0 < k) write_entry(a, row, r0, e0);
            if (lane + 32 < count && r1 < k) write_entry(a, row, r1, e1);
        } else {
            warp_sort_list(list, count);
            for (int i = lane; i < k; i += 32) write_entry(a, row, i, list[i]);
        }
        __syncwarp();
    }
    if (s_aborted)  // leave with no copy in flight
        for (int i = 0; i < 2; ++i)
            for (int w = 0; n > unsigned(i) && w < 1000000 && !tc::mbar_try_wait(full + i, ((n - 1 - i) >> 1) & 1); ++w) {}
}

// ---- long rows: a block, or a cluster, per row --------------------------------------
// As the distillation's long rows (distill.cu): NT consumer threads stream, R row
// warps do what belongs to a row, R rows ahead and behind.  The consumers add
// the exponentials and keep the maxima of 512 groups of one row, then go back to the row
// before, still in the ring, for the logits that reach its bound.  The row's warp
// finds the bound (in a cluster one for all CTAs), sorts what was collected, and one
// CTA's warp, in turn, merges the CTAs' lists.  Bound
// by instructions, two looks at every chunk and the row warps' sorts: 2048x131072
// bfloat16, k 128, 276 us, 1.9 TB/s; 8192x16384 float32, k 64, 145 us, 3.7 TB/s.
struct TopPost {
    float o, bound;
};
// The running maxima of a thread's four groups (16-bit types two to a register),
// and the largest element of one chunk.
template <class T>
struct GroupMax;
template <>
struct GroupMax<float> {
    float g[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    __device__ __forceinline__ void add(const uint4& raw) {
        g[0] = fmaxf(g[0], __uint_as_float(raw.x));
        g[1] = fmaxf(g[1], __uint_as_float(raw.y));
        g[2] = fmaxf(g[2], __uint_as_float(raw.z));
        g[3] = fmaxf(g[3], __uint_as_float(raw.w));
    }
    __device__ __forceinline__ float of(int i) const { return g[i]; }
    static __device__ __forceinline__ float of_chunk(const uint4& raw) {
        return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)),
                     fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
    }
};
template <class H2>
struct GroupMax16 {
    H2 a, b;
    __device__ __forceinline__ void add(const uint4& raw) {
        const H2* h = reinterpret_cast<const H2*>(&raw);
        a = __hmax2(a, __hmax2(h[0], h[1]));
        b = __hmax2(b, __hmax2(h[2], h[3]));
    }
    __device__ __forceinline__ float of(int i) const {
        const H2 x = i < 2 ? a : b;
        return i & 1 ? __high2float(x) : __low2float(x);
    }
    static __device__ __forceinline__ float of_chunk(const uint4& raw) {
        const H2* h = reinterpret_cast<const H2*>(&raw);
        const H2 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(x), __high2float(x));
    }
};
template <>
struct GroupMax<__nv_bfloat16> : GroupMax16<__nv_bfloat162> {
    __device__ __forceinline__ GroupMax() { a = b = __float2bfloat162_rn(-INFINITY); }
};
template <>
struct GroupMax<__half> : GroupMax16<__half2> {
    __device__ __forceinline__ GroupMax() { a = b = __float2half2_rn(-INFINITY); }
};

template <class T, int NT>
__global__ void __launch_bounds__(NT + 32 + 32 * top_row_warps(NT), top_blocks(NT))
top_stream_kernel(const TopArgs a, uint32_t rows, const TopShape shape)
{
    HX_PDL_PROLOGUE();
    constexpr int EPV = Chunk<T>::EPV, NW = NT / 32, U = 16 / EPV, kSlot = U * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_aborted;
    const int k = int(a.k), V = int(a.vocab), ring = shape.ring, slices = shape.slices, R = shape.row_warps;
    const TopMemory mem(NT, kSlot, ring, R, k, slices);
    const int room = stream_list(k);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + mem.bars);
    uint64_t* empty = full + ring;
    uint64_t *formed = empty + ring, *summed = formed + R, *bounded = summed + R, *collected = bounded + R;
    uint64_t *joined = collected + R, *merged = joined + 2 * R;
    float* part = reinterpret_cast<float*>(smem + mem.part);
    float* groups = reinterpret_cast<float*>(smem + mem.groups);
    TopPost* posts = reinterpret_cast<TopPost*>(smem + mem.posts);
    int* counts = reinterpret_cast<int*>(smem + mem.counts);
    uint64_t* lists = reinterpret_cast<uint64_t*>(smem + mem.lists);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = int(blockIdx.x) & (slices - 1);
    const size_t team = blockIdx.x >> shape.log_slices, teams = gridDim.x >> shape.log_slices;
    const WaitState ws{a.err, &s_aborted};
    auto span_of = [&](size_t row) {
        return Span<T>(static_cast<const T*>(a.logits) + row * a.stride, V, rank, shape.log_slices);
    };

    if (tid == 0) {
        s_aborted = 0;
        for (int i = 0; i < ring; ++i) {
            tc::mbar_init(full + i, 1);
            tc::mbar_init(empty + i, NW);
        }
        for (int i = 0; i < R; ++i) {
            tc::mbar_init(formed + i, 1);
            tc::mbar_init(summed + i, NW);
            tc::mbar_init(bounded + i, 1);
            tc::mbar_init(collected + i, NW);
            tc::mbar_init(joined + 2 * i, 1);
            tc::mbar_init(joined + 2 * i + 1, 1);
            tc::mbar_init(merged + i, 1);
        }
        tc::fence_mbar_init();
    }
    if (slices > 1) tc::cluster_sync(); else __syncthreads();

    if (warp == NW) {
        stream_producer<T, kSlot>(smem, full, empty, ring, rows, team, teams, span_of, ws);
    } else if (warp > NW) {
        // ---- the rows' warps ----
        const int b = warp - NW - 1;
        float4* slots = reinterpret_cast<float4*>(smem + mem.slots) + b * 32;
        uint64_t* list = lists + b * room;
        const int half = (k + 1) & ~1;
        uint64_t* merge = reinterpret_cast<uint64_t*>(smem + mem.merge) + size_t(b) * slices * half;
        const float c = kLog2e / a.tau, inv_tau = 1.f / a.tau;
        uint32_t phase = 0, merges = 0;
        int merger = 0;  // the CTA that merges, in turn
        ClusterExchange joins{slots, joined + 2 * b, rank, slices};
        auto exchange = [&](float4 x) { return joins(x, make_float4(0.f, -INFINITY, -INFINITY, -INFINITY), ws); };
        // a logit to take the exponentials against: the largest of 32, loaded a row
        // ahead (a load waits long behind the rows' copies)
        auto sample_of = [&](size_t row) {
            return row < rows ? to_float(static_cast<const T*>(a.logits)[row * a.stride + size_t(lane) * V / 32]) : 0.f;
        };
        float sample = b < R ? sample_of(team + b * teams) : 0.f;
        if (b < R)
            for (size_t row = team + b * teams; row < rows; row += R * teams, phase ^= 1) {
                const Span<T> span = span_of(row);
                const int e0 = max(0, span.first * EPV - span.lead), e1 = min(V, span.last * EPV - span.lead);
                float ref = warp_max(sample);
                sample = sample_of(row + R * teams);
                if (!(fabsf(ref * c) < kFarOffset)) ref = 0.f;
                float scale = c, o = ref * c;
                if (lane == 0) {
                    posts[b].o = o;
                    counts[b] = 0;
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(formed + b);
                stream_wait(summed + b, phase, ws);
                // the bound: the k-th largest group maximum
                uint32_t key[kGroups / 32];
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kGroups / 32; ++i) {
                    const float g = groups[b * kGroups + i * 32 + lane];
                    top = fmaxf(top, g);
                    key[i] = descending_key(g);
                }
                top = warp_max(top);
                float bound = from_descending_key(warp_kth(key, k, k / 8));
                // in a cluster also: k / slices logits of every CTA reach the smallest
                // of these
                float shared_bound = -INFINITY;
                if (slices > 1) {
                    const int share = (k + slices - 1) >> shape.log_slices;
                    shared_bound = from_descending_key(warp_kth(key, share, share / 8));
                }
                float sum = warp_reduce(lane < NW ? part[b * NW + lane] : 0.f, SumOp());
                if (slices > 1) {
                    const float4 x = exchange(make_float4(sum, top, bound, -shared_bound));
                    sum = warp_reduce(x.x, SumOp());
                    top = warp_max(x.y);
                    bound = fmaxf(warp_max(x.z), -warp_max(x.w));
                }
                if (lane == 0) {
                    posts[b].bound = bound;
                    tc::mbar_arrive(bounded + b);
                }
                __syncwarp();
                if (a.lse) {
                    if (!sum_serves(sum) && top < INFINITY && top > -INFINITY) {
                        // the reference was far off: against the maximum
                        ref = top;
                        scale = scale_against(ref, c);
                        o = ref * scale;
                        sum = 0.f;
                        for (int i = e0 + lane; i < e1; i += 32)
                            sum += tc::exp2_approx(fmaf(to_float(span.row[i]), scale, -o));
                        sum = warp_reduce(sum, SumOp());
                        if (slices > 1) sum = warp_reduce(exchange(make_float4(sum, 0.f, 0.f, 0.f)).x, SumOp());
                    }
                    if (rank == 0 && lane == 0)
                        a.lse[row] = top == INFINITY && sum == sum ? top : ref * inv_tau + (logf(sum) - kLn2 * fmaf(ref, scale, -o));
                }
                stream_wait(collected + b, phase, ws);
                int n = counts[b];
                const int want = min(k, max(0, e1 - e0));
                // in a cluster the bound may pass a CTA's own k-th: fewer are enough there,
                // unless NaN leaves the row short
                if (n > room || (n < want && !(bound > -INFINITY))) {
                    n = exact_list(span.row, e0, e1, bound, want, list);
                } else {
                    for (int i = lane; i < n; i += 32) {
                        const int at = int(uint32_t(list[i]));
                        list[i] = entry_of(descending_key(to_float(span.row[at])), at);
                    }
                    __syncwarp();
                }
                if (slices == 1) {
                    warp_sort_list(list, n);
                    for (int i = lane; i < k; i += 32) write_entry(a, row, i, list[i]);
                    __syncwarp();
                } else {
                    warp_sort_list(list, n);
                    const int give = min(n, k);
                    if (rank == merger && lane == 0) tc::mbar_arrive_expect_tx(merged + b, uint32_t(slices) * half * 8);
                    __syncwarp();
                    for (int i = lane; i < half / 2; i += 32) {
                        const uint64_t x = 2 * i < give ? list[2 * i] : ~0ull, y = 2 * i + 1 < give ? list[2 * i + 1] : ~0ull;
                        store_async(tc::cluster_addr(merge + rank * half + 2 * i, merger),
                                    make_float4(__uint_as_float(uint32_t(x)), __uint_as_float(uint32_t(x >> 32)),
                                                __uint_as_float(uint32_t(y)), __uint_as_float(uint32_t(y >> 32))),
                                    tc::cluster_addr(merged + b, merger));
                    }
                    if (rank == merger) {
                        stream_wait(merged + b, merges & 1, ws);
                        ++merges;
                        // an entry's rank: its place in its own list and in every other
                        int top_step = 1;
                        while (top_step <= half) top_step *= 2;
                        for (int i = lane; i < slices * half; i += 32) {
                            const uint64_t x = merge[i];
                            if (x == ~0ull) continue;
                            int r = 0;
                            for (int q0 = 0; q0 < slices; q0 += 4) {  // four searches at a time
                                int at[4] = {0, 0, 0, 0};
                                for (int step = top_step / 2; step > 0; step /= 2)
#pragma unroll
                                    for (int q = 0; q < 4; ++q)
                                        if (q0 + q < slices && at[q] + step <= half &&
                                            merge[(q0 + q) * half + at[q] + step - 1] < x)
                                            at[q] += step;
                                r += at[0] + at[1] + at[2] + at[3];
                            }
                            if (r < k) write_entry(a, row, r, x);
                        }
                        __syncwarp();
                    }
                    merger = (merger + 1) & (slices - 1);
                }
            }
    } else {
        // ---- consumers ----
        const float c = kLog2e / a.tau;
        const bool sums = a.lse != nullptr;
        const uint4* mine = reinterpret_cast<const uint4*>(smem) + tid;
        RingCursor sums_at{0, 0}, back_at{0, 0};
        int sb = 0, gb = 0;
        uint32_t s_phase = 0, g_phase = 0;
        auto add_row = [&](size_t row) {
            const int chunks = span_of(row).chunks();
            stream_wait(formed + sb, s_phase, ws);
            const float o = posts[sb].o;
            float sum = 0.f;
            GroupMax<T> g;
            auto add = [&](const uint4& raw) {
                g.add(raw);
                if (sums) {
                    float e[EPV];
                    Chunk<T>::unpack(raw, e);
#pragma unroll
                    for (int r = 0; r < EPV; ++r) e[r] = tc::exp2_approx(fmaf(e[r], c, -o));
#pragma unroll
                    for (int w = EPV / 2; w > 0; w /= 2)
#pragma unroll
                        for (int r = 0; r < w; ++r) e[r] += e[r + w];
                    sum += e[0];
                }
            };
            for (int p0 = 0; p0 < chunks; p0 += kSlot) {
                stream_wait(full + sums_at.slot, sums_at.phase, ws);
                const uint4* from = mine + sums_at.slot * kSlot;
                if (p0 + kSlot <= chunks) {
                    uint4 raw[U];
#pragma unroll
                    for (int q = 0; q < U; ++q) raw[q] = from[q * NT];
#pragma unroll
                    for (int q = 0; q < U; ++q) add(raw[q]);
                } else {
#pragma unroll 1
                    for (int q = 0; q < U; ++q)
                        if (p0 + q * NT + tid < chunks) add(from[q * NT]);
                }
                sums_at.next(ring);
            }
            float* to = groups + sb * kGroups;
            if (NT == 512) {
                to[tid] = fmaxf(fmaxf(g.of(0), g.of(1)), fmaxf(g.of(2), g.of(3)));
            } else if (NT == 256) {
                to[tid] = fmaxf(g.of(0), g.of(1));
                to[tid + 256] = fmaxf(g.of(2), g.of(3));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) to[tid + 128 * i] = g.of(i);
            }
            if (sums) sum = warp_reduce(sum, SumOp());
            __syncwarp();
            if (lane == 0) {
                part[sb * NW + warp] = sum;
                tc::mbar_arrive(summed + sb);
            }
            if (++sb == R) { sb = 0; s_phase ^= 1; }
        };
        auto collect_row = [&](size_t row) {
            const Span<T> span = span_of(row);
            const int chunks = span.chunks();
            stream_wait(bounded + gb, g_phase, ws);
            const float bound = posts[gb].bound;
            uint64_t* list = lists + gb * room;
            // (not unrolled: few chunks hold one, and each thread few)
            auto take = [&](const uint4& raw, int p) {
                float x[EPV];
                Chunk<T>::unpack(raw, x);
                uint32_t mask = 0;
#pragma unroll
                for (int r = 0; r < EPV; ++r) mask |= uint32_t(x[r] >= bound) << r;
#pragma unroll 1
                for (; mask; mask &= mask - 1) {
                    const int i = (span.first + p) * EPV + __ffs(mask) - 1 - span.lead;
                    if (i < 0 || i >= V) continue;
                    const int at = atomicAdd(counts + gb, 1);
                    if (at >= room) break;
                    list[at] = uint32_t(i);  // the row's warp adds the key
                }
            };
            for (int p0 = 0; p0 < chunks; p0 += kSlot) {
                const uint4* from = mine + back_at.slot * kSlot;
                uint4 raw[U];
#pragma unroll
                for (int q = 0; q < U; ++q) raw[q] = from[q * NT];
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(empty + back_at.slot);
                uint32_t holds = 0;
#pragma unroll
                for (int q = 0; q < U; ++q)
                    holds |= uint32_t(p0 + q * NT + tid < chunks && GroupMax<T>::of_chunk(raw[q]) >= bound) << q;
#pragma unroll
                for (int q = 0; q < U; ++q)
                    if (holds >> q & 1u) take(raw[q], p0 + q * NT + tid);
                back_at.next(ring);
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(collected + gb);
            if (++gb == R) { gb = 0; g_phase ^= 1; }
        };
        const size_t ahead = top_adds_ahead(R) ? teams : 0;
        size_t next = team;
        for (size_t row = team; row < rows; row += teams) {
#pragma unroll 1
            for (; next <= row + ahead && next < rows; next += teams) add_row(next);
            collect_row(row);
        }
    }
    if (slices > 1) tc::cluster_sync();  // no CTA leaves while another may write to it
}

template <class T, int NT>
void launch_top_stream(hx_runtime* rt, const TopArgs& a, uint32_t rows, long chunks)
{
    constexpr int kSlot = 16 / Chunk<T>::EPV * NT;
    const int threads = NT + 32 + 32 * top_row_warps(NT);
    const size_t limit = stream_limit(top_blocks(NT));
    const TopShape shape = top_shape(NT, Chunk<T>::EPV, chunks, int(a.k), long(rows), rt->sm_count);
    const int s = shape.slices;
    require(shape.row_warps > 0, HX_ERR_UNSUPPORTED, "top logits: no room for the row");
    const size_t smem = TopMemory(NT, kSlot, shape.ring, shape.row_warps, int(a.k), s).bytes;
    auto kernel = top_stream_kernel<T, NT>;
    static thread_local int opted[64] = {};
    if (!opted[rt->device & 63]) {
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(limit)));
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        opted[rt->device & 63] = 1;
    }
    const int teams = resident_teams(rt, kernel, threads, smem, s);
    launch_rows(kernel, std::min<uint32_t>(rows, uint32_t(teams)) * unsigned(s), threads, s, true, smem, rt->stream, a, rows,
                shape);
    HX_LAUNCHED(rt);
}

// By the row's bytes: a warp while its registers hold the row, up to 16 KB 128 consumers,
// 32 KB 256, then 512.  134 MB of float32 logits, k 64, in us, the other variant in
// brackets: 14 KB 145 (154 by 256), 19 KB 98 (221 by 128), 30 KB 92 (82 by 512; bfloat16
// 86, 94), 36 KB 78 (127 by 256; bfloat16 88, 82).
template <class T>
void launch_top(hx_runtime* rt, const TopArgs& a, uint32_t rows)
{
    const long chunks = row_chunks(a.logits, a.stride, rows, a.vocab, sizeof(T));
    if (chunks <= 32 * Chunk<T>::N) {
        const size_t smem = kTopTeams * (2 * 32 * Chunk<T>::N * 16 + size_t(top_list(int(a.k))) * 8);
        auto kernel = top_warp_kernel<T>;
        static thread_local int opted[64] = {};
        if (!opted[rt->device & 63]) {
            HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536));
            opted[rt->device & 63] = 1;
        }
        const unsigned blocks =
            std::min((rows + kTopTeams - 1) / kTopTeams, unsigned(resident_teams(rt, kernel, 32 * kTopTeams, smem, 1)));
        launch_rows(kernel, blocks, 32 * kTopTeams, 1, false, smem, rt->stream, a, rows);
        HX_LAUNCHED(rt);
    } else if (chunks <= 1024) {
        launch_top_stream<T, 128>(rt, a, rows, chunks);
    } else if (chunks <= 2048) {
        launch_top_stream<T, 256>(rt, a, rows, chunks);
    } else {
        launch_top_stream<T, 512>(rt, a, rows, chunks);
    }
}

void top_logits(hx_runtime* rt, int dtype, uint32_t rows, TopArgs a)
{
    check_logits("top logits", dtype, rows, a.vocab, a.logits, a.stride);
    require(a.k >= 1 && a.k <= kMaxTop && a.k <= a.vocab, HX_ERR_ARGUMENT,
            "top logits: k must be in [1, min(256, vocabulary)]");
    require(std::isfinite(a.tau) && a.tau > 0.f && std::isfinite(1.f / a.tau), HX_ERR_ARGUMENT,
            "top logits: temperature must be positive and finite");
    if (rows == 0) return;
    require(a.values && a.indices, HX_ERR_ARGUMENT, "top logits: null output");
    a.err = rt->device_error();
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
        hx::head::top_logits(rt, dtype, rows, {logits, stride, values, indices, lse, nullptr, vocab, k, temperature});
    });
}
