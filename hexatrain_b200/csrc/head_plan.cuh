// head_plan.cuh -- how the streaming kernels over rows of logits share out a block:
// plain arithmetic without device code, so that a host program can walk through it.
#pragma once

#include <algorithm>
#include <cstddef>

#ifdef __CUDACC__
#define HX_PLAN_FN __host__ __device__
#else
#define HX_PLAN_FN
#endif

namespace hx {
namespace head {

// ---- the exchange between the CTAs of a cluster (head_stream.cuh) -------------------
// Exchange n uses slots and barrier n % 2; it is phase n / 2 of that barrier.  A
// barrier counts bytes, not senders, and a CTA that is through exchange n sends for
// n + 1 while another may still wait for bytes of n: on one barrier these would
// stand in for those.  No CTA sends for n + 2 before every one has sent for n + 1, which
// it does when it is through n.
HX_PLAN_FN constexpr int exchange_place(unsigned n) { return int(n & 1); }
HX_PLAN_FN constexpr unsigned exchange_parity(unsigned n) { return (n >> 1) & 1; }

// ---- top logits of long rows (top_logits.cu) ---------------------------------------
constexpr int kGroups = 512, kTopRing = 64, kTopSlices = 16;
// Blocks of nt consumer threads on an SM, and row warps of a block.
HX_PLAN_FN constexpr int top_blocks(int nt) { return nt == 128 ? 4 : nt == 256 ? 2 : 1; }
HX_PLAN_FN constexpr int top_row_warps(int nt) { return nt == 128 ? 4 : nt == 256 ? 6 : 8; }

// Entries of a row's list (a power of two): the bound lets a quarter more than k pass,
// nearly twice as many where k is half of the groups.
HX_PLAN_FN constexpr int stream_list(int k) { return k <= 64 ? 128 : k <= 128 ? 256 : 512; }

struct TopShape {
    int ring, slices, log_slices, row_warps;  // row_warps 0: no room
};

// Offsets into a block's dynamic shared memory; a slot holds `slot` 16-byte chunks.
struct TopMemory {
    size_t bars, part, groups, slots, posts, counts, lists, merge, bytes;
    HX_PLAN_FN constexpr TopMemory(int nt, int slot, int ring, int R, int k, int slices)
        : bars(0), part(0), groups(0), slots(0), posts(0), counts(0), lists(0), merge(0), bytes(0) {
        size_t at = size_t(ring) * slot * 16;
        bars = at; at += size_t(2 * ring + 7 * R) * 8;
        at = (at + 15) & ~size_t(15);
        slots = at; at += size_t(R) * 2 * 16 * 16;
        lists = at; at += size_t(R) * stream_list(k) * 8;
        merge = at; at += slices > 1 ? size_t(R) * slices * ((k + 1) & ~1) * 8 : 0;
        groups = at; at += size_t(R) * kGroups * 4;
        part = at; at += size_t(R) * (nt / 32) * 4;
        posts = at; at += size_t(R) * 8;
        counts = at; at += size_t(R) * 4;
        bytes = (at + 15) & ~size_t(15);
    }
};
// Shared memory of a block where `blocks` share an SM.
HX_PLAN_FN constexpr size_t stream_limit(int blocks) { return 233472 / blocks - 1024 - 256; }

// The consumers add row r + 1 before they collect row r, so that the bound of r is
// found meanwhile.  Row r + 1 begins when its warp says so, and that warp says so
// when it is done with its last row: with one row warp that is row r itself,
// which waits for the collection.  One row warp therefore takes row after row.
HX_PLAN_FN constexpr bool top_adds_ahead(int row_warps) { return row_warps >= 2; }

// Shape of a call on rows of up to `chunks` chunks with nt consumer threads.  The ring
// holds two rows' slices and a slot for the copies ahead.  At least three row
// warps, in as few slices as that takes; where the lists of wide records leave no room
// for them, two, in the fewest slices, if need be without the slot ahead; one
// only where nothing else fits.  Three against two in fewer slices, 134 MB: float16
// 82200 wide, k 128, 125 us (225), 42200, k 256, 147 (295); not for short rows or wide
// records of float32: float16 6200, k 200, 629 (520), float32 66200, k 256, 5797 (2434).
inline TopShape top_shape(int nt, int epv, long chunks, int k, long rows, int sm_count) {
    const int slot = 16 / epv * nt, most = top_row_warps(nt), least = 3;
    const size_t limit = stream_limit(top_blocks(nt));
    auto ring_of = [&](int s, int R) {
        const size_t fixed = TopMemory(nt, slot, 0, R, k, s).bytes;
        return fixed < limit ? int(std::min<size_t>((limit - fixed) / (size_t(slot) * 16 + 16), kTopRing)) : 0;
    };
    auto two_rows = [&](int s) { return 2 * int(((chunks + s - 1) / s + slot - 1) / slot); };
    auto fits = [&](int s, int R, int ahead) { return two_rows(s) + ahead <= ring_of(s, R); };
    auto shape = [&](int s, int R) {
        int log = 0;
        while ((1 << log) < s) ++log;
        return TopShape{ring_of(s, R), s, log, R};
    };
    for (int s = 1; s <= kTopSlices; s *= 2) {
        if (!fits(s, least, 1)) continue;
        int R = most;
        while (!fits(s, R, 1)) --R;
        // few rows: more slices, down to 8 KB, rather than idle SMs
        while (nt == 512 && s < 8 && rows * s * 2 <= sm_count && chunks / (2 * s) >= 512 && fits(2 * s, R, 1)) s *= 2;
        return shape(s, R);
    }
    for (int ahead = 1; ahead >= 0; --ahead)
        for (int s = 1; s <= kTopSlices; s *= 2)
            if (fits(s, 2, ahead)) return shape(s, 2);
    for (int s = 1; s <= kTopSlices; s *= 2)
        if (fits(s, 1, 0)) return shape(s, 1);
    return TopShape{0, 1, 0, 0};
}

}  // namespace head
}  // namespace hx
