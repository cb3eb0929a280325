// head_stream.cuh -- rows of logits streamed through shared memory.
//
// A persistent block takes row after row (or, in a cluster, its slice of each).
// One producer warp copies the row's aligned 16-byte chunks with
// cp.async.bulk into a ring of slots, as far ahead as the ring has room, while the
// NT consumer threads work: a slot holds NT chunks, thread t reads chunk t of
// every slot.  The loads of the next rows are in flight through all of a row's
// reductions and barriers, which is what a memory-bound row operator of short
// phases needs: with one row per block and loads straight to registers the
// same arithmetic took 1.4 to 4 times as long.
//
// Every wait is bounded; one that runs out records a code, sets the block's
// abort flag and lets every other wait pass, so that all loops and barriers run
// to their end and the block leaves in order.
#pragma once

#include "head_plan.cuh"
#include "head_rows.cuh"

namespace hx {
namespace head {

struct WaitState {
    int* err;               // the runtime's error word
    volatile int* aborted;  // in shared memory
};
__device__ __forceinline__ void stream_wait(uint64_t* bar, uint32_t parity, const WaitState& w) {
    if (tc::mbar_try_wait(bar, parity)) return;
    const long long t0 = clock64();
    while (!tc::mbar_try_wait(bar, parity)) {
        if (*w.aborted) return;
        if (clock64() - t0 > tc::kWaitCycles) {
            atomicCAS(w.err, 0, kHeadWaitCode);
            *w.aborted = 1;
            return;
        }
    }
}

// Copies `bytes` (a multiple of 16, both ends 16-byte aligned) to this block's
// shared memory, completing on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     tc::smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(tc::smem_u32(bar))
                 : "memory");
}
// Stores 16 bytes to a cluster CTA's shared memory, completing on its barrier.
__device__ __forceinline__ void store_async(uint32_t addr, float4 x, uint32_t bar) {
    asm volatile(
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "f"(x.x),
        "f"(x.y), "f"(x.z), "f"(x.w), "r"(bar)
        : "memory");
}
// A number of each CTA of a cluster, from the same warp of each, to all of them.
struct ClusterExchange {
    float4* slots;   // [2][16]
    uint64_t* bars;  // [2], one arrival each
    int rank, slices;
    unsigned n = 0;
    // lane r gets the number of CTA r, the others `none`
    __device__ __forceinline__ float4 operator()(float4 x, float4 none, const WaitState& ws) {
        const int lane = threadIdx.x & 31;
        uint64_t* bar = bars + exchange_place(n);
        float4* to = slots + exchange_place(n) * 16;
        if (lane == 0) tc::mbar_arrive_expect_tx(bar, 16u * slices);
        __syncwarp();
        if (lane < slices) store_async(tc::cluster_addr(to + rank, lane), x, tc::cluster_addr(bar, lane));
        stream_wait(bar, exchange_parity(n), ws);
        ++n;
        return lane < slices ? to[lane] : none;
    }
};
// A place in the ring: slots in turn, the phase changes with every round.
struct RingCursor {
    int slot;
    uint32_t phase;
    __device__ __forceinline__ void next(int ring) {
        if (++slot == ring) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// A slice of a row in chunks: chunk c holds elements [c EPV - lead, + EPV).
template <class T>
struct Span {
    static constexpr int EPV = Chunk<T>::EPV;
    const T* row;
    int vocab, lead, first, last, w0, w1;  // chunks [first, last), whole ones [w0, w1)
    __device__ __forceinline__ Span(const T* row_, int vocab_, int rank, int log_slices)
        : row(row_), vocab(vocab_), lead(int((reinterpret_cast<uintptr_t>(row_) & 15) / sizeof(T))) {
        const int chunks = (vocab + lead + EPV - 1) / EPV, each = (chunks + (1 << log_slices) - 1) >> log_slices;
        first = min(chunks, rank * each);
        last = min(chunks, first + each);
        w0 = max(first, lead > 0 ? 1 : 0);
        w1 = max(w0, min(last, (vocab + lead) / EPV));
    }
    __device__ __forceinline__ int chunks() const { return last - first; }
    __device__ __forceinline__ bool holds(int i) const { return i + lead >= first * EPV && i + lead < last * EPV; }
    // position of element i in the slice
    __device__ __forceinline__ int position(int i) const { return i + lead - first * EPV; }
    __device__ __forceinline__ bool whole(int c) const { return c >= w0 && c < w1; }
};

// The producer warp: the chunks of rows team, team + teams, ... into the ring's
// slots of kSlot chunks.
template <class T, int kSlot, class SpanOf>
__device__ __forceinline__ void stream_producer(uint8_t* smem, uint64_t* full, uint64_t* empty, int ring, uint32_t rows,
                                                size_t team, size_t teams, SpanOf span_of, const WaitState& ws) {
    constexpr int EPV = Chunk<T>::EPV;
    const int lane = threadIdx.x & 31;
    RingCursor at{0, 1};  // a fresh barrier lets a wait for phase 1 pass
    unsigned filled = 0;
    for (size_t row = team; row < rows; row += teams) {
        const Span<T> span = span_of(row);
        // an element of the row's partial chunks: the first (lanes 0-7), the last (8-15)
        const int r = lane & 7, pc = lane < 8 ? span.first : span.last - 1;
        const bool partial = lane < 16 && r < EPV && span.chunks() > 0 && !span.whole(pc);
        const int pi = pc * EPV + r - span.lead;
        const T px = partial && pi >= 0 && pi < span.vocab ? span.row[pi] : from_float<T>(-INFINITY);
        for (int c0 = span.first; c0 < span.last; c0 += kSlot) {
            stream_wait(empty + at.slot, at.phase, ws);
            T* to = reinterpret_cast<T*>(smem) + at.slot * (kSlot * EPV);
            const int c1 = min(c0 + kSlot, span.last);
            if (partial && pc >= c0 && pc < c1) {
                to[(pc - c0) * EPV + r] = px;
                tc::fence_proxy_async_smem();
            }
            __syncwarp();
            if (lane == 0) {
                const int b0 = max(c0, span.w0), b1 = min(c1, span.w1);
                const uint32_t bytes = b1 > b0 ? uint32_t(b1 - b0) * 16 : 0;
                tc::mbar_arrive_expect_tx(full + at.slot, bytes);
                if (bytes)
                    bulk_load(to + (b0 - c0) * EPV, span.row - span.lead + size_t(b0) * EPV, bytes, full + at.slot);
            }
            at.next(ring);
            ++filled;
        }
    }
    if (*ws.aborted)  // leave with no copy in flight
        for (unsigned i = filled > unsigned(ring) ? filled - ring : 0; i < filled; ++i)
            for (int n = 0; n < 1000000 && !tc::mbar_try_wait(full + i % ring, (i / ring) & 1); ++n) {}
}

}  // namespace head
}  // namespace hx
