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
//   c_i = S (renormalised, or i named by the record), S - q_T/p_T (elsewhere),
//   S the sum of all the q that the loss has: 1, but sum_j q_j where the bucket is
//   left out (q_T = 0 or p_T = 0), which may be anything.
// No counterpart in the reference, whose loss is the hard-label cross-entropy
// (tiny_language_model_cpu.cpp:77); that is kd = 0, ce = 1 here.
#include <cmath>

#include "head_ops.cuh"
#include "head_stream.cuh"

namespace hx {
namespace head {

// The record's entries, j = lane, lane + 32, ...: index, probability, the
// student's logit, and the position in the team's slice (-1 where it does not
// hold the token).  In shared memory, or in the registers of the one warp.
constexpr size_t kEntryBytes = 16;
struct EntriesShared {
    float* mem;
    int k;
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        int* whole = reinterpret_cast<int*>(mem + 2 * k);
        for (int j = threadIdx.x & 31; j < k; j += 32) f(j, mem[j], mem[k + j], whole[j], whole[k + j]);
    }
    __device__ __forceinline__ bool names(int p) const {
        const int* pos = reinterpret_cast<const int*>(mem + 3 * k);
        for (int j = 0; j < k; ++j)
            if (pos[j] == p) return true;
        return false;
    }
};
template <int N>
struct EntriesHeld {
    float q[N], l[N];
    int idx[N], pos[N], k;
    template <class F>
    __device__ __forceinline__ void each(F&& f) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (threadIdx.x & 31) + 32 * i;
            if (j < k) f(j, q[i], l[i], idx[i], pos[i]);
        }
    }
};

// The exponentials a call needs: of the soft targets' temperature, of the hard
// targets, or of both (two), where the temperature makes them differ.
struct Needs {
    bool soft, hard, two, tail, exact;  // exact: 1 / tau is (tau a power of two)
    float c, inv_tau;                   // c: log2(e) times the scale of the first exponential
    // `both`: the call writes the statistics of both
    __device__ __forceinline__ Needs(const DistillArgs& a, bool both)
        : soft(both || a.kd != 0.f), hard(both || (a.labels && a.ce != 0.f)), two(soft && hard && a.tau != 1.f),
          tail(a.teacher_lse != nullptr), exact(a.exact_inverse != 0), inv_tau(1.f / a.tau) {
        c = soft ? kLog2e / a.tau : kLog2e;
    }
};

// One number of a row to a lane: its label, the teacher's log-sum-exp, the
// gradient of its loss, the forward's statistics.
struct RowNumbers {
    const float* from;
    int step;
    float none;
    __device__ __forceinline__ RowNumbers(const DistillArgs& a, bool backward) : from(nullptr), step(1), none(1.f) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) {
            from = reinterpret_cast<const float*>(a.labels);
            none = __int_as_float(-1);
        }
        if (lane == 1) from = a.teacher_lse;
        if (lane == 2) from = a.grad_loss;
        if (lane >= 3 && lane < 6 && backward) {
            from = a.stats + (lane - 3);
            step = 3;
        }
    }
    __device__ __forceinline__ float of(size_t row) const { return from ? from[row * step] : none; }
};

// A row's record as one warp holds it: the same in every lane but the sums, of
// which each lane has a share.
struct Record {
    bool has, label_named;
    int label;
    float sq, kl;      // sum q; sum q (log q - (l - ref)/tau)
    float soft, hard;  // the named tokens' part of the row's sums (tail only)
    float ref;         // the logit the row's exponentials are taken against
    float l_label, A, B;  // A, B: the scales of the soft and the hard gradient
};

// One warp forms a row's record, in full precision: 1 - sum q and a KL near 0 keep
// few of the digits of what they are formed from.  The entries hold the teacher's
// indices and, as q, its values; `number` the row's numbers; logit(i) reads a logit
// of the row.
template <class Span, class Entries, class Logit>
__device__ __forceinline__ Record form_record(const DistillArgs& a, const Needs& n, const Span& span, float number,
                                              Entries& e, Logit logit) {
    const int V = int(a.vocab);
    Record rec{};
    int label = __float_as_int(__shfl_sync(0xffffffffu, number, 0));
    bool bad = label >= V, has = false, named = false;
    if (bad) label = -1;
    rec.label = label;
    rec.l_label = label >= 0 ? logit(label) : 0.f;
    // (a teacher that masks the whole row has a log-sum-exp of -inf, and no entries)
    const float lse_teacher = __shfl_sync(0xffffffffu, number, 1);
    float most = -INFINITY, ref = -INFINITY;
    e.each([&](int, float& t, float& l, int& idx, int& pos) {
        t = n.exact ? t * n.inv_tau : t / a.tau;
        l = 0.f;
        pos = -1;
        if (idx >= V) {
            bad = true;
            idx = -1;
        }
        if (idx >= 0) {
            l = logit(idx);
            most = fmaxf(most, t);
            ref = fmaxf(ref, l);
            has |= (n.tail ? lse_teacher : t) != -INFINITY;
            named |= idx == label;
            if (span.holds(idx)) pos = span.position(idx);
        }
    });
    if (bad) atomicCAS(a.err, 0, kBadIndexCode);
    rec.has = __any_sync(0xffffffffu, has);
    rec.label_named = __any_sync(0xffffffffu, named);
    ref = warp_max(ref);
    if (label >= 0) ref = fmaxf(ref, rec.l_label);
    if (ref == -INFINITY) ref = logit(0);
    rec.ref = fabsf(ref) < INFINITY ? ref : 0.f;
    float log_z;
    if (n.tail) {
        log_z = lse_teacher;
    } else {
        most = warp_max(most);
        float z = 0.f;
        e.each([&](int, float& t, float&, int& idx, int&) {
            if (rec.has && idx >= 0) z += expf(t - most);
        });
        log_z = most + logf(warp_reduce(z, SumOp()));
    }
    const float o = offset_against(rec.ref, n.c), o1 = offset_against(rec.ref, kLog2e);
    e.each([&](int, float& q, float& l, int& idx, int& pos) {
        const float logq = q - log_z;
        q = rec.has && idx >= 0 ? expf(logq) : 0.f;
        rec.sq += q;
        if (q > 0.f) rec.kl += q * (logq - (l - rec.ref) * n.inv_tau);
        if (n.tail && pos >= 0) {
            rec.soft += tc::exp2_approx(fmaf(l, n.c, -o));
            if (n.two) rec.hard += tc::exp2_approx(fmaf(l, kLog2e, -o1));
        }
    });
    const float gs = a.grad_scale * __shfl_sync(0xffffffffu, number, 2);
    rec.A = rec.has ? gs * a.kd * a.tau : 0.f;
    rec.B = label >= 0 ? gs * a.ce : 0.f;
    return rec;
}

// Sums over a thread's logits: of 2^(l c - o) and of 2^(l log2e - o1).  With a tail
// bucket the tokens that the record names have been set to -inf in shared memory
// before, so that the sum is that of the tail, without cancellation; their own
// part comes from the record.  The reference logit is one of the row's, so the
// exponents are at most those of the maximum over it: far from overflow unless
// the record misses the row's largest logits by 40 tau.
struct Sums {
    float soft, hard;
};
// (Scalar: the paired forms of these operations cost more in register moves than they save.)
template <int EPV>
__device__ __forceinline__ float tree_sum(float (&e)[EPV]) {
#pragma unroll
    for (int w = EPV / 2; w > 0; w /= 2)
#pragma unroll
        for (int r = 0; r < w; ++r) e[r] += e[r + w];
    return e[0];
}
template <int EPV>
__device__ __forceinline__ void add_chunk(Sums& s, const float (&x)[EPV], const Needs& n, float o, float o1) {
    float e[EPV];
#pragma unroll
    for (int r = 0; r < EPV; ++r) e[r] = tc::exp2_approx(fmaf(x[r], n.c, -o));
    s.soft += tree_sum(e);
    if (n.two) {
#pragma unroll
        for (int r = 0; r < EPV; ++r) e[r] = tc::exp2_approx(fmaf(x[r], kLog2e, -o1));
        s.hard += tree_sum(e);
    }
}

// A row's gradient: g = A 2^(l c - o) + B 2^(l c1 - o1), the second term only
// where both are needed.
struct Gradient {
    float A, B, c, o, c1, o1;
    template <int EPV>
    __device__ __forceinline__ void of(const float (&x)[EPV], float (&g)[EPV]) const {
#pragma unroll
        for (int r = 0; r < EPV; ++r) g[r] = A * tc::exp2_approx(fmaf(x[r], c, -o));
        if (B != 0.f) {
#pragma unroll
            for (int r = 0; r < EPV; ++r) g[r] = fmaf(B, tc::exp2_approx(fmaf(x[r], c1, -o1)), g[r]);
        } else if (A == 0.f) {  // a row without targets is zero, whatever its logits
#pragma unroll
            for (int r = 0; r < EPV; ++r) g[r] = 0.f;
        }
    }
};

// A row's result, from its sums (forward) or its statistics (backward).  A
// probability is inv 2^(l c - o): in the forward o = ref c, as in the sums, and
// inv = 1/s, so that the rounding of o cancels; the logarithm takes its
// residual, ref c - o, off again.  (c and c1 are the row's: scale_against.)
struct RowResult {
    float named, rest, c, o, inv, c1, o1, inv1, ratio;  // named, rest: the soft gradient's factors of p
    __device__ __forceinline__ void soft_factors(const Needs& n, const Record& rec, float sq) {
        const float mass = n.tail && ratio == 0.f ? sq : 1.f;
        named = rec.A * mass;
        rest = rec.A * (mass - ratio);
    }
    // A row masked as a whole by a low value: beyond 2^24 its log-sum-exp cannot hold the
    // logarithm of the number of its logits beside them, and its probabilities count as 0.
    static __device__ __forceinline__ float offset_of(float lse) {
        return fabsf(lse) > 0x1p24f && fabsf(lse) < INFINITY ? INFINITY : lse * kLog2e;
    }
    // statistics written by the forward
    __device__ __forceinline__ void from_statistics(const Needs& n, const Record& rec, float number, float sq) {
        c = n.c;
        c1 = kLog2e;
        o = offset_of(n.soft ? __shfl_sync(0xffffffffu, number, 3) : __shfl_sync(0xffffffffu, number, 4));
        o1 = offset_of(__shfl_sync(0xffffffffu, number, 4));
        ratio = __shfl_sync(0xffffffffu, number, 5);
        inv = inv1 = 1.f;
        soft_factors(n, rec, sq);
    }
    __device__ __forceinline__ void from_sums(const Needs& n, const Record& rec, float ref, float s_out, float s_named,
                                              float s_hard, float sq) {
        const float s = s_out + s_named;
        c = n.c;
        c1 = kLog2e;
        if (!(fabsf(ref) * fmaxf(n.c, kLog2e) < kFarOffset)) {
            c = scale_against(ref, n.c);
            c1 = scale_against(ref, kLog2e);
        }
        o = ref * c;
        o1 = ref * c1;
        // (a row without targets: its sums may be anything, and 0 / 0 is NaN)
        const bool none = rec.A == 0.f && rec.B == 0.f;
        inv = none ? 0.f : __fdividef(1.f, s);
        inv1 = n.two && !none ? __fdividef(1.f, s_hard) : inv;
        ratio = 0.f;
        if (n.tail && n.soft && rec.has && s_out > 0.f) {
            // (s / s_out overflows where s_out is near 2^-126: no mass either)
            const float r = fmaxf(1.f - sq, 0.f) * __fdividef(s, s_out);
            ratio = r < INFINITY ? r : 0.f;
        }
        soft_factors(n, rec, sq);
    }
    // one lane writes the row's loss and statistics
    __device__ __forceinline__ void write(const DistillArgs& a, const Needs& n, const Record& rec, size_t row, float ref,
                                          float s_out, float s_named, float s_hard, float sq, float kl) const {
        const float s = s_out + s_named, log_s = logf(s) - kLn2 * fmaf(ref, c, -o);
        const float log_1 = n.two ? logf(s_hard) - kLn2 * fmaf(ref, c1, -o1) : log_s;
        const float lse_tau = n.soft ? ref * n.inv_tau + log_s : 0.f, lse_1 = ref + log_1;
        float loss = 0.f;
        if (a.kd != 0.f && rec.has) {
            // sum q (log q - log p); the entries' share is against rec.ref
            kl += sq * ((ref - rec.ref) * n.inv_tau + log_s);
            if (ratio > 0.f) kl += fmaxf(1.f - sq, 0.f) * logf(ratio);
            loss = a.kd * a.tau * a.tau * kl;
        }
        if (rec.label >= 0 && a.ce != 0.f) loss += a.ce * ((ref - rec.l_label) + log_1);
        if (a.loss) a.loss[row] = loss;
        if (a.stats) {
            a.stats[row * 3] = lse_tau;
            a.stats[row * 3 + 1] = lse_1;
            a.stats[row * 3 + 2] = ratio;
        }
    }
    __device__ __forceinline__ Gradient dense(const Needs& n, const Record& rec) const {
        if (!n.two) return {((n.soft ? rest : 0.f) + (n.hard ? rec.B : 0.f)) * inv, 0.f, c, o, c1, 0.f};  // one softmax
        if (rest != 0.f) return {rest * inv, rec.B * inv1, c, o, c1, o1};
        return {rec.B * inv1, 0.f, c1, o1, c1, 0.f};
    }
    // the gradient of a token that the record names with probability q
    // (soft = named) or of an unnamed label (soft = rest, q = 0)
    __device__ __forceinline__ float token(const Needs& n, const Record& rec, float l, float soft, float q, bool is_label) const {
        const float e = tc::exp2_approx(fmaf(l, c, -o)) * inv;
        float g = rec.A != 0.f ? soft * e - rec.A * q : 0.f;
        if (rec.B != 0.f) g += rec.B * ((n.two ? tc::exp2_approx(fmaf(l, c1, -o1)) * inv1 : e) - (is_label ? 1.f : 0.f));
        return g;
    }
    // One warp writes the record's tokens, and the label, over the dense gradient.
    template <class T, class Entries>
    __device__ __forceinline__ void scatter(const Needs& n, const Record& rec, Entries& e, T* d, bool holds_label) const {
        e.each([&](int, float& q, float& l, int& idx, int& pos) {
            if (pos >= 0) d[idx] = from_float<T>(token(n, rec, l, named, q, idx == rec.label));
        });
        if ((threadIdx.x & 31) == 0 && holds_label && !rec.label_named)
            d[rec.label] = from_float<T>(token(n, rec, rec.l_label, rest, 0.f, true));
    }
};

// Writes one chunk's gradient; elements outside [e0, e1) are not the caller's.
template <class T, int EPV>
__device__ __forceinline__ void write_chunk(T* d, int base, int e0, int e1, const float (&g)[EPV]) {
    if (base >= e0 && base + EPV <= e1) {
        *reinterpret_cast<uint4*>(d + base) = Chunk<T>::pack(g);
    } else {
#pragma unroll
        for (int r = 0; r < EPV; ++r)
            if (base + r >= e0 && base + r < e1) d[base + r] = from_float<T>(g[r]);
    }
}

enum DistillPass { kForward = 1, kBackwardPass = 2, kFused = 3 };  // bit 0: the sums, bit 1: the gradient

// Joins the sums of the warps (and CTAs): each lane holds one part.
__device__ __forceinline__ void join_sums(float4 p, float& s_out, float& s_named, float& s_hard) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        p.x += __shfl_xor_sync(0xffffffffu, p.x, o);
        p.y += __shfl_xor_sync(0xffffffffu, p.y, o);
        p.z += __shfl_xor_sync(0xffffffffu, p.z, o);
    }
    s_out = p.x;
    s_named = p.y;
    s_hard = p.z;
}

// ---- long rows: a block, or a cluster, per row -----------------------------------
// Memory bound.  NT consumer threads do nothing but stream: the exponentials'
// sums of one row, then the gradient of the row before it.  All that belongs to a
// row as a whole is done by one of R further warps, up to R rows ahead and
// behind: its record, the join of the sums over the block and the cluster,
// the loss, and the record's tokens and the label written over the dense
// gradient.  While a row's sums are joined the consumers are on the next row, so the
// latency of the join (and of the cluster's exchange) is hidden; the ring
// (head_stream.cuh) holds two rows and the copies ahead, so the logits are read
// from memory once.  The exponentials are taken against the largest logit that
// the record or the label names, known before the row's sums begin: no maximum
// is looked for unless the sum overflows.
// Measured: 4096x65536 bf16 fused at one temperature 212 us, 5.1 TB/s of 6.55 (at two
// 293 us: four exponentials a logit fill the special-function unit for 236 us; the loss
// alone 144 us, two of them); 16384x8192 float32 fused 176 us, 6.1 TB/s, with a tail
// 189; 2048x32768 float16 backward 48 us.
struct StreamShape {
    int ring;        // slots
    int slices;      // CTAs of a row, a power of two
    int log_slices;
};
// Blocks of NT consumer threads on an SM: 512 consumers in all.
__host__ __device__ constexpr int stream_blocks(int nt) { return nt == 128 ? 4 : nt == 256 ? 2 : 1; }
__host__ __device__ constexpr int record_warps(int nt) { return nt == 128 ? 3 : 4; }
constexpr int stream_threads(int nt) { return nt + 32 + 32 * record_warps(nt); }

struct RowPost {  // from the row's warp to the consumers
    float o, o1;  // the sums' exponent offsets
    Gradient grad;
};

template <int NT, int kSlot>
struct StreamMemory {  // offsets into dynamic shared memory
    static constexpr int R = record_warps(NT);
    size_t bars, part, slots, posts, entries, bytes;
    __host__ __device__ StreamMemory(int ring, int k) {
        size_t at = size_t(ring) * kSlot * 16;
        bars = at; at += size_t(2 * ring + 6 * R) * 8;
        at = (at + 15) & ~size_t(15);
        part = at; at += R * (NT / 32) * 8;
        slots = at; at += R * 2 * 16 * 16;
        posts = at; at += R * 32;
        entries = at; at += R * kEntryBytes * size_t(k);
        bytes = at;
    }
};

template <class T, int NT, int kPass>
__global__ void __launch_bounds__(NT + 32 + 32 * record_warps(NT), stream_blocks(NT))
distill_stream_kernel(const DistillArgs a, uint32_t rows, const StreamShape shape)
{
    HX_PDL_PROLOGUE();
    constexpr int EPV = Chunk<T>::EPV, NW = NT / 32, R = record_warps(NT), U = 16 / EPV;
    constexpr int kSlot = U * NT;  // chunks of a slot
    constexpr bool kSums = kPass & 1, kGrad = kPass & 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_aborted;
    const int k = int(a.k), V = int(a.vocab), ring = shape.ring, slices = shape.slices;
    const StreamMemory<NT, kSlot> mem(ring, k);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + mem.bars);
    uint64_t* empty = full + ring;
    uint64_t *formed = empty + ring, *summed = formed + R, *result = summed + R, *written = result + R;
    uint64_t* joined = written + R;
    float2* part = reinterpret_cast<float2*>(smem + mem.part);
    RowPost* posts = reinterpret_cast<RowPost*>(smem + mem.posts);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = int(blockIdx.x) & (slices - 1);
    const size_t team = blockIdx.x >> shape.log_slices, teams = gridDim.x >> shape.log_slices;
    const bool marks = kSums && a.teacher_lse != nullptr;  // named logits are set to -inf
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
            tc::mbar_init(result + i, 1);
            tc::mbar_init(written + i, NW);
            tc::mbar_init(joined + 2 * i, 1);
            tc::mbar_init(joined + 2 * i + 1, 1);
        }
        tc::fence_mbar_init();
    }
    if (slices > 1) tc::cluster_sync(); else __syncthreads();

    if (warp == NW) {
        stream_producer<T, kSlot>(smem, full, empty, ring, rows, team, teams, span_of, ws);
    } else if (warp > NW) {
        // ---- the rows' warps ----
        const int b = warp - NW - 1;
        const EntriesShared e{reinterpret_cast<float*>(smem + mem.entries + b * kEntryBytes * k), k};
        float4* slots = reinterpret_cast<float4*>(smem + mem.slots) + b * 32;
        const Needs need(a, kPass == kForward);
        const RowNumbers numbers(a, !kSums);
        uint32_t phase = 0;
        RingCursor at{0, 0};  // of the row's first slot
        bool begun = false;
        auto skip = [&](size_t row) {
            if (row < rows)
                for (int c = span_of(row).chunks(); c > 0; c -= kSlot) at.next(ring);
        };
        if (marks)
            for (int i = 0; i < b; ++i) skip(team + i * teams);
        ClusterExchange joins{slots, joined + 2 * b, rank, slices};
        auto exchange = [&](float4 x) { return joins(x, make_float4(0.f, 0.f, 0.f, -INFINITY), ws); };
        for (size_t row = team + b * teams; row < rows; row += R * teams, phase ^= 1) {
            const Span<T> span = span_of(row);
            const float number = numbers.of(row);
            e.each([&](int j, float& t, float&, int& idx, int&) {
                idx = a.teacher_indices[row * k + j];
                t = a.teacher_values[row * k + j];
            });
            // The backward may write over the logits, and nothing tells a CTA how far the others
            // are: it reads its own slice alone, which is all that its gradient needs.
            const Record rec = form_record(a, need, span, number, e, [&](int i) {
                return kSums || span.holds(i) ? to_float(span.row[i]) : 0.f;
            });
            RowResult res;
            if (!kSums) {
                res.from_statistics(need, rec, number, warp_reduce(rec.sq, SumOp()));
                if (lane == 0) posts[b].grad = res.dense(need, rec);
            } else {
                if (lane == 0) {
                    posts[b].o = offset_against(rec.ref, need.c);
                    posts[b].o1 = offset_against(rec.ref, kLog2e);
                }
                if (marks) {
                    // Once the row has arrived its named logits leave the sums.  A slot's
                    // arrival can be told from the one before it only when that one
                    // is over: the row before, and with it every earlier one, has arrived.
                    if (b > 0 || begun) stream_wait(formed + (b > 0 ? b : R) - 1, b > 0 ? phase : phase ^ 1, ws);
                    begun = true;
                    const int first = at.slot;
                    for (int c = span.chunks(); c > 0; c -= kSlot, at.next(ring)) stream_wait(full + at.slot, at.phase, ws);
                    e.each([&](int, float&, float&, int&, int& pos) {
                        if (pos < 0) return;
                        int slot = first + pos / (kSlot * EPV);
                        if (slot >= ring) slot -= ring;
                        reinterpret_cast<T*>(smem)[slot * (kSlot * EPV) + pos % (kSlot * EPV)] = from_float<T>(-INFINITY);
                    });
                    tc::fence_proxy_async_smem();
                    for (int i = 1; i < R; ++i) skip(row + i * teams);
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(formed + b);
            if (kSums) {
                const float sq = warp_reduce(rec.sq, SumOp()), kl = warp_reduce(rec.kl, SumOp());
                float ref = rec.ref, s_out, s_named, s_hard;
                stream_wait(summed + b, phase, ws);
                const float2 p = lane < NW ? part[b * NW + lane] : make_float2(0.f, 0.f);
                join_sums(make_float4(p.x, rec.soft, p.y + rec.hard, 0.f), s_out, s_named, s_hard);
                if (slices > 1) join_sums(exchange(make_float4(s_out, s_named, s_hard, 0.f)), s_out, s_named, s_hard);
                if (!sum_serves(s_out + s_named) || (need.two && !sum_serves(s_hard))) {
                    // an overflow, or no reference of the row's: this warp finds the row's
                    // maximum and forms the sums against it
                    const int e0 = max(0, span.first * EPV - span.lead), e1 = min(V, span.last * EPV - span.lead);
                    float m = -INFINITY;
                    for (int i = e0 + lane; i < e1; i += 32) m = fmaxf(m, to_float(span.row[i]));
                    m = warp_max(m);
                    if (slices > 1) m = warp_max(exchange(make_float4(0.f, 0.f, 0.f, m)).w);
                    ref = m == -INFINITY ? 0.f : m;
                    const float c = scale_against(ref, need.c), c1 = scale_against(ref, kLog2e), o = ref * c, o1 = ref * c1;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int i = e0 + lane; i < e1; i += 32) {
                        const float l = to_float(span.row[i]), y = tc::exp2_approx(fmaf(l, c, -o));
                        if (marks && e.names(span.position(i))) x.y += y; else x.x += y;
                        if (need.two) x.z += tc::exp2_approx(fmaf(l, c1, -o1));
                    }
                    join_sums(x, s_out, s_named, s_hard);
                    if (slices > 1) join_sums(exchange(make_float4(s_out, s_named, s_hard, 0.f)), s_out, s_named, s_hard);
                }
                res.from_sums(need, rec, ref, s_out, s_named, s_hard, sq);
                if (kGrad) {
                    if (lane == 0) {
                        posts[b].grad = res.dense(need, rec);
                        tc::mbar_arrive(result + b);
                    }
                    __syncwarp();
                }
                if (lane == 0 && rank == 0) res.write(a, need, rec, row, ref, s_out, s_named, s_hard, sq, kl);
            }
            if (kGrad) {
                stream_wait(written + b, phase, ws);
                res.scatter(need, rec, e, static_cast<T*>(a.d_logits) + row * a.grad_stride,
                            rec.label >= 0 && span.holds(rec.label));
                __syncwarp();
            }
        }
    } else {
        // ---- consumers ----
        const Needs need(a, kPass == kForward);
        RingCursor sums_at{0, 0}, grad_at{0, 0};
        const uint4* mine = reinterpret_cast<const uint4*>(smem) + tid;
        int sb = 0, gb = 0;
        uint32_t s_phase = 0, g_phase = 0;
        auto add_row = [&](size_t row) {
            const Span<T> span = span_of(row);
            const int chunks = span.chunks();
            stream_wait(formed + sb, s_phase, ws);
            const float o = posts[sb].o, o1 = posts[sb].o1;
            Sums x{};
            auto add = [&](const uint4& raw) {
                float v[EPV];
                Chunk<T>::unpack(raw, v);
                add_chunk<EPV>(x, v, need, o, o1);
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
                if (!kGrad) {
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(empty + sums_at.slot);
                }
                sums_at.next(ring);
            }
            const float soft = warp_reduce(x.soft, SumOp()), hard = need.two ? warp_reduce(x.hard, SumOp()) : 0.f;
            if (lane == 0) {
                part[sb * NW + warp] = make_float2(soft, hard);
                tc::mbar_arrive(summed + sb);
            }
            if (++sb == R) { sb = 0; s_phase ^= 1; }
        };
        auto write_row = [&](size_t row) {
            const Span<T> span = span_of(row);
            T* d = static_cast<T*>(a.d_logits) + row * a.grad_stride;
            const int chunks = span.chunks();
            const int e0 = max(0, span.first * EPV - span.lead), e1 = min(V, span.last * EPV - span.lead);
            const int lead_d = int((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T));
            stream_wait((kSums ? result : formed) + gb, g_phase, ws);
            const Gradient grad = posts[gb].grad;
            if (lead_d == span.lead) {
                for (int p0 = 0; p0 < chunks; p0 += kSlot) {
                    if (!kSums) stream_wait(full + grad_at.slot, grad_at.phase, ws);
                    const uint4* from = mine + grad_at.slot * kSlot;
                    const int c0 = span.first + p0;
                    if (c0 >= span.w0 && c0 + kSlot <= span.w1) {
                        uint4* to = reinterpret_cast<uint4*>(d - span.lead) + c0 + tid;
                        uint4 raw[U];
#pragma unroll
                        for (int q = 0; q < U; ++q) raw[q] = from[q * NT];
#pragma unroll
                        for (int q = 0; q < U; ++q) {
                            float v[EPV], y[EPV];
                            Chunk<T>::unpack(raw[q], v);
                            grad.of(v, y);
                            to[q * NT] = Chunk<T>::pack(y);
                        }
                    } else {
#pragma unroll 1
                        for (int q = 0; q < U; ++q) {
                            const int p = p0 + q * NT + tid;
                            if (p >= chunks) break;
                            float v[EPV], y[EPV];
                            Chunk<T>::unpack(from[q * NT], v);
                            grad.of(v, y);
                            write_chunk<T, EPV>(d, (span.first + p) * EPV - span.lead, e0, e1, y);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(empty + grad_at.slot);
                    grad_at.next(ring);
                }
            } else {
                // the gradient's chunks lie across the logits': read the ring by element
                if (!kSums) {
                    RingCursor at = grad_at;
                    for (int p0 = 0; p0 < chunks; p0 += kSlot, at.next(ring)) stream_wait(full + at.slot, at.phase, ws);
                }
                const int d1 = e1 > e0 ? (e1 + lead_d + EPV - 1) / EPV : 0;
                for (int c = (e0 + lead_d) / EPV + tid; c < d1; c += NT) {
                    const int base = c * EPV - lead_d;
                    float v[EPV], y[EPV];
#pragma unroll
                    for (int r = 0; r < EPV; ++r) {
                        const int i = min(max(base + r, e0), e1 - 1), p = span.position(i);
                        int slot = grad_at.slot + p / (kSlot * EPV);
                        if (slot >= ring) slot -= ring;
                        v[r] = to_float(reinterpret_cast<const T*>(smem)[slot * (kSlot * EPV) + p % (kSlot * EPV)]);
                    }
                    grad.of(v, y);
                    write_chunk<T, EPV>(d, base, e0, e1, y);
                }
                __syncwarp();
                for (int p0 = 0; p0 < chunks; p0 += kSlot, grad_at.next(ring))
                    if (lane == 0) tc::mbar_arrive(empty + grad_at.slot);
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(written + gb);
            if (++gb == R) { gb = 0; g_phase ^= 1; }
        };
        if (kPass == kFused) {
            size_t row = team;
            if (row < rows) add_row(row);
            for (; row < rows; row += teams) {
                if (row + teams < rows) add_row(row + teams);
                write_row(row);
            }
        } else {
            for (size_t row = team; row < rows; row += teams) {
                if (kSums) add_row(row); else write_row(row);
            }
        }
    }
    if (slices > 1) tc::cluster_sync();  // no CTA leaves while another may write to it
}

// ---- short rows: a warp per row -------------------------------------------------
// Rows of up to kChunks chunks (4 or 8 KB).  Each warp streams rows of its own
// through two buffers in shared memory, the logits by cp.async.bulk and the record
// by cp.async, so that the next row is in flight while one is worked on and no
// barrier wider than the warp is met.  Measured: 131072x1024 float32 fused, k 32, 196 us,
// 5.7 TB/s; one row per 128 threads with the row in registers took 287 us.
constexpr int kWarpRows = 2, kWarpTeams = 4;

template <int kChunks>
struct WarpMemory {  // a warp's dynamic shared memory
    size_t record, bytes;
    __host__ __device__ explicit WarpMemory(int k) {
        size_t at = size_t(kWarpRows) * kChunks * 16;
        record = at; at += size_t(kWarpRows) * k * 8;
        bytes = (at + 15) & ~size_t(15);
    }
};

__device__ __forceinline__ void copy4_async(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(tc::smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void arrive_after_copies(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

template <class T, int kChunks, int kHeld, int kPass>
__global__ void __launch_bounds__(32 * kWarpTeams)
distill_warp_kernel(const DistillArgs a, uint32_t rows)
{
    HX_PDL_PROLOGUE();
    constexpr int EPV = Chunk<T>::EPV, U = 16 / EPV;
    constexpr bool kSums = kPass & 1, kGrad = kPass & 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t s_full[kWarpTeams * kWarpRows];
    __shared__ int s_aborted;
    const int k = int(a.k), V = int(a.vocab), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WarpMemory<kChunks> mem(k);
    uint8_t* mine = smem + warp * mem.bytes;
    uint64_t* full = s_full + warp * kWarpRows;
    EntriesHeld<kHeld> e;
    e.k = k;
    const bool marks = kSums && a.teacher_lse != nullptr;  // named logits are set to -inf
    const WaitState ws{a.err, &s_aborted};
    if (threadIdx.x == 0) s_aborted = 0;
    if (lane == 0) {
        for (int i = 0; i < kWarpRows; ++i) tc::mbar_init(full + i, 33);
        tc::fence_mbar_init();
    }
    __syncthreads();

    const uint32_t team = blockIdx.x * kWarpTeams + warp, teams = gridDim.x * kWarpTeams;
    auto span_of = [&](size_t row) { return Span<T>(static_cast<const T*>(a.logits) + row * a.stride, V, 0, 0); };
    auto buffer = [&](int b) { return reinterpret_cast<T*>(mine) + b * (kChunks * EPV); };
    auto issue = [&](size_t row, int b) {
        const Span<T> span = span_of(row);
        float* record = reinterpret_cast<float*>(mine + mem.record) + b * 2 * k;
        for (int j = lane; j < k; j += 32) {
            copy4_async(record + j, a.teacher_indices + row * k + j);
            copy4_async(record + k + j, a.teacher_values + row * k + j);
        }
        arrive_after_copies(full + b);
        if (lane == 0) {
            const uint32_t bytes = uint32_t(span.w1 - span.w0) * 16;
            tc::mbar_arrive_expect_tx(full + b, bytes);
            if (bytes) bulk_load(buffer(b) + span.w0 * EPV, span.row - span.lead + span.w0 * EPV, bytes, full + b);
        }
    };
    // an element of the row's partial chunks: the first (lanes 0-7), the last (8-15)
    auto partial = [&](const Span<T>& span) {
        const int r = lane & 7, pc = lane < 8 ? 0 : span.last - 1;
        return lane < 16 && r < EPV && !span.whole(pc) ? pc * EPV + r : -1;
    };
    auto partial_value = [&](const Span<T>& span) {
        const int p = partial(span), i = p - span.lead;
        return p >= 0 && i >= 0 && i < V ? span.row[i] : from_float<T>(-INFINITY);
    };

    for (int i = 0; i < kWarpRows; ++i)
        if (team + i * teams < rows) issue(team + i * teams, i);
    const RowNumbers numbers(a, !kSums);
    T px = from_float<T>(0.f);
    float number = 0.f;
    if (team < rows) {
        px = partial_value(span_of(team));
        number = numbers.of(team);
    }
    const Needs need(a, kPass == kForward);
    unsigned n = 0;
    int b = 0;
    for (size_t row = team; row < rows; row += teams, ++n) {
        const Span<T> span = span_of(row);
        T* l = buffer(b);
        const uint4* from = reinterpret_cast<const uint4*>(l) + lane;
        const int chunks = span.chunks();
        stream_wait(full + b, (n / kWarpRows) & 1, ws);
        if (partial(span) >= 0) l[partial(span)] = px;
        const float* record = reinterpret_cast<const float*>(mine + mem.record) + b * 2 * k;
        e.each([&](int j, float& t, float&, int& idx, int&) {
            idx = __float_as_int(record[j]);
            t = record[k + j];
        });
        __syncwarp();
        const Record rec = form_record(a, need, span, number, e, [&](int i) { return to_float(l[i + span.lead]); });
        RowResult res;
        if (!kSums) res.from_statistics(need, rec, number, warp_reduce(rec.sq, SumOp()));
        if (row + teams < rows) {  // the next row's numbers, while this one is worked on
            px = partial_value(span_of(row + teams));
            number = numbers.of(row + teams);
        }
        if (kSums) {
            float ref = rec.ref, s_out, s_named, s_hard;
            if (marks) {
                __syncwarp();
                e.each([&](int, float&, float&, int&, int& pos) {
                    if (pos >= 0) l[pos] = from_float<T>(-INFINITY);
                });
                __syncwarp();
            }
            {
                const float o = offset_against(ref, need.c), o1 = offset_against(ref, kLog2e);
                Sums x{};
                auto add = [&](const uint4& raw) {
                    float v[EPV];
                    Chunk<T>::unpack(raw, v);
                    add_chunk<EPV>(x, v, need, o, o1);
                };
                int p = 0;
                for (; p + 32 * U <= chunks; p += 32 * U) {
                    uint4 raw[U];
#pragma unroll
                    for (int q = 0; q < U; ++q) raw[q] = from[p + 32 * q];
#pragma unroll
                    for (int q = 0; q < U; ++q) add(raw[q]);
                }
#pragma unroll 1
                for (p += lane; p < chunks; p += 32) add(from[p - lane]);
                join_sums(make_float4(x.soft, rec.soft, x.hard + rec.hard, 0.f), s_out, s_named, s_hard);
            }
            if (!sum_serves(s_out + s_named) || (need.two && !sum_serves(s_hard))) {
                // an overflow, or no reference of the row's: against the row's maximum
                float m = -INFINITY;
#pragma unroll 1
                for (int i = lane; i < chunks * EPV; i += 32) m = fmaxf(m, to_float(l[i]));
                e.each([&](int, float&, float& x, int&, int& pos) {
                    if (pos >= 0) m = fmaxf(m, x);
                });
                m = warp_max(m);
                ref = m == -INFINITY ? 0.f : m;
                const float c = scale_against(ref, need.c), c1 = scale_against(ref, kLog2e), o = ref * c, o1 = ref * c1;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int i = lane; i < chunks * EPV; i += 32) {
                    x.x += tc::exp2_approx(fmaf(to_float(l[i]), c, -o));
                    if (need.two) x.z += tc::exp2_approx(fmaf(to_float(l[i]), c1, -o1));
                }
                if (marks)
                    e.each([&](int, float&, float& t, int&, int& pos) {
                        if (pos < 0) return;
                        x.y += tc::exp2_approx(fmaf(t, c, -o));
                        if (need.two) x.z += tc::exp2_approx(fmaf(t, c1, -o1));
                    });
                join_sums(x, s_out, s_named, s_hard);
            }
            const float sq = warp_reduce(rec.sq, SumOp()), kl = warp_reduce(rec.kl, SumOp());
            res.from_sums(need, rec, ref, s_out, s_named, s_hard, sq);
            if (lane == 0) res.write(a, need, rec, row, ref, s_out, s_named, s_hard, sq, kl);
        }
        if (kGrad) {
            T* d = static_cast<T*>(a.d_logits) + row * a.grad_stride;
            const Gradient grad = res.dense(need, rec);
            const int lead_d = int((reinterpret_cast<uintptr_t>(d) & 15) / sizeof(T));
            if (lead_d == span.lead) {
                uint4* to = reinterpret_cast<uint4*>(d - span.lead) + lane;
                int p = 0;
                if (span.w0 == 0)
                    for (; p + 32 * U <= span.w1; p += 32 * U) {
                        uint4 raw[U];
#pragma unroll
                        for (int q = 0; q < U; ++q) raw[q] = from[p + 32 * q];
#pragma unroll
                        for (int q = 0; q < U; ++q) {
                            float v[EPV], y[EPV];
                            Chunk<T>::unpack(raw[q], v);
                            grad.of(v, y);
                            to[p + 32 * q] = Chunk<T>::pack(y);
                        }
                    }
#pragma unroll 1
                for (p += lane; p < chunks; p += 32) {
                    float v[EPV], y[EPV];
                    Chunk<T>::unpack(from[p - lane], v);
                    grad.of(v, y);
                    write_chunk<T, EPV>(d, p * EPV - span.lead, 0, V, y);
                }
            } else {
                for (int c = lane; c < (V + lead_d + EPV - 1) / EPV; c += 32) {
                    float v[EPV], y[EPV];
#pragma unroll
                    for (int r = 0; r < EPV; ++r)
                        v[r] = to_float(l[min(max(c * EPV - lead_d + r, 0), V - 1) + span.lead]);
                    grad.of(v, y);
                    write_chunk<T, EPV>(d, c * EPV - lead_d, 0, V, y);
                }
            }
            __syncwarp();
            res.scatter(need, rec, e, d, rec.label >= 0);
        }
        tc::fence_proxy_async_smem();  // this row's own writes before the next copy
        __syncwarp();
        if (row + kWarpRows * size_t(teams) < rows) issue(row + kWarpRows * size_t(teams), b);
        b ^= 1;
    }
    if (s_aborted) {  // leave with no copy in flight
        asm volatile("cp.async.wait_all;" ::: "memory");
        for (int i = 0; i < kWarpRows; ++i) {
            const unsigned used = n > unsigned(i) ? (n - 1 - i) / kWarpRows : 0;
            for (int t = 0; n > unsigned(i) && t < 1000000 && !tc::mbar_try_wait(full + i, used & 1); ++t) {}
        }
    }
}

template <class T, int NT, int kPass>
void launch_stream(hx_runtime* rt, const DistillArgs& a, uint32_t rows, long chunks)
{
    constexpr int kPerSm = stream_blocks(NT), kSlot = 16 / Chunk<T>::EPV * NT;
    const size_t limit = 233472 / kPerSm - 1024 - 256;  // shared memory of a block
    const size_t fixed = StreamMemory<NT, kSlot>(0, int(a.k)).bytes + 32;
    const int ring = int(std::min<size_t>((limit - fixed) / (size_t(kSlot) * 16 + 16), 64));
    // The ring holds a row's slice from its sums to its gradient, and the next
    // row's with it; the loss alone needs the slice whole only while named
    // logits leave it.  A slot more lets the copies run ahead.
    const int resident = kPass == kFused ? 2 : kPass == kForward && !a.teacher_lse ? 0 : 1;
    auto fits = [&](int s) { return resident * int(((chunks + s - 1) / s + kSlot - 1) / kSlot) + 1 <= ring; };
    int s = 1;
    while (s < 16 && !fits(s)) s *= 2;
    require(resident * int(((chunks + s - 1) / s + kSlot - 1) / kSlot) <= ring && ring >= 1, HX_ERR_UNSUPPORTED,
            "distillation: no room for the row");  // (the slot more is only for speed)
    // few rows: more slices, down to 8 KB, rather than idle SMs
    while (NT == 512 && s < 8 && long(rows) * s * 2 <= rt->sm_count && chunks / (2 * s) >= 512) s *= 2;
    const StreamShape shape{ring, s, __builtin_ctz(unsigned(s))};
    const StreamMemory<NT, kSlot> mem(ring, int(a.k));
    auto kernel = distill_stream_kernel<T, NT, kPass>;
    static thread_local int opted[64] = {};
    if (!opted[rt->device & 63]) {
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(limit)));
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        opted[rt->device & 63] = 1;
    }
    const int teams = resident_teams(rt, kernel, stream_threads(NT), mem.bytes, s);
    launch_rows(kernel, std::min<uint32_t>(rows, uint32_t(teams)) * unsigned(s), stream_threads(NT), s, true, mem.bytes,
                rt->stream, a, rows, shape);
    HX_LAUNCHED(rt);
}

template <class T, int kChunks, int kHeld, int kPass>
void launch_warp(hx_runtime* rt, const DistillArgs& a, uint32_t rows)
{
    const size_t smem = kWarpTeams * WarpMemory<kChunks>(int(a.k)).bytes;
    auto kernel = distill_warp_kernel<T, kChunks, kHeld, kPass>;
    static thread_local int opted[64] = {};
    if (!opted[rt->device & 63]) {
        HX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 131072));
        opted[rt->device & 63] = 1;
    }
    const unsigned blocks =
        std::min((rows + kWarpTeams - 1) / kWarpTeams, unsigned(resident_teams(rt, kernel, 32 * kWarpTeams, smem, 1)));
    launch_rows(kernel, blocks, 32 * kWarpTeams, 1, false, smem, rt->stream, a, rows);
    HX_LAUNCHED(rt);
}

// By the row's bytes: up to 8 KB a warp, 16 KB 128 consumers, 32 KB 256, then 512.  134 MB
// of float32 logits, k 64, tail, loss + gradient in us, the other variant in brackets:
// 7.6 KB 64 (109 by 128), 14 KB 76 (86 by 256), 19 KB 76 (94 by 128), 30 KB 62 (78 by
// 512), 36 KB 76 (78 by 256).  For 16-bit rows of 19 and 36 KB, and for the loss or
// the gradient alone, the smaller block would be 4 to 23 % faster there.
template <class T, int kPass>
void launch_distill(hx_runtime* rt, const DistillArgs& a, uint32_t rows)
{
    const long chunks = row_chunks(a.logits, a.stride, rows, a.vocab, sizeof(T));
    if (chunks <= 256) {
        if (a.k <= 32) launch_warp<T, 256, 1, kPass>(rt, a, rows);
        else launch_warp<T, 256, 8, kPass>(rt, a, rows);
    } else if (chunks <= 512) {
        if (a.k <= 32) launch_warp<T, 512, 1, kPass>(rt, a, rows);
        else launch_warp<T, 512, 8, kPass>(rt, a, rows);
    } else if (chunks <= 1024) {
        launch_stream<T, 128, kPass>(rt, a, rows, chunks);
    } else if (chunks <= 2048) {
        launch_stream<T, 256, kPass>(rt, a, rows, chunks);
    } else {
        launch_stream<T, 512, kPass>(rt, a, rows, chunks);
    }
}

template <class T>
void launch_distill(hx_runtime* rt, const DistillArgs& a, uint32_t rows, bool backward)
{
    if (backward) launch_distill<T, kBackwardPass>(rt, a, rows);
    else if (a.d_logits) launch_distill<T, kFused>(rt, a, rows);
    else launch_distill<T, kForward>(rt, a, rows);
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
    int exponent = 0;
    a.exact_inverse = std::frexp(a.tau, &exponent) == 0.5f;
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
