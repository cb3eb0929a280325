// The plans of csrc/head_plan.cuh walked through on the host: prints what fails, and
// exits with 0 when nothing does.
#include <cstdio>
#include <cstring>
#include <map>
#include <set>
#include <string>
#include <tuple>
#include <vector>

#include "head_plan.cuh"

using namespace hx::head;

// A block of the top-logits kernel over `rows` rows of `need` ring slots each, every
// role as far as its waits let it: the producer fills slots, the consumers add and
// collect rows in the kernel's order, the row warps take every R-th row.  True if
// all of them come to their end.
static bool finishes(int R, bool ahead, int ring, int need, int rows) {
    std::vector<char> formed(rows), summed(rows), bounded(rows), collected(rows);
    int filled = 0, freed = 0;                  // slots, counted through
    std::vector<std::pair<bool, int>> order;    // (add, row)
    for (int r = 0, next = 0; r < rows; ++r) {
        for (; next <= r + (ahead ? 1 : 0) && next < rows; ++next) order.push_back({true, next});
        order.push_back({false, r});
    }
    size_t at = 0;
    std::vector<int> row(R), step(R, 0);
    for (int b = 0; b < R; ++b) row[b] = b;
    for (bool moved = true; moved;) {
        moved = false;
        while (filled < rows * need && filled - freed < ring) ++filled, moved = true;
        while (at < order.size()) {
            const int r = order[at].second;
            if (order[at].first) {
                if (!formed[r] || filled < (r + 1) * need) break;
                summed[r] = 1;
            } else {
                if (!bounded[r]) break;
                freed += need;
                collected[r] = 1;
            }
            ++at;
            moved = true;
        }
        for (int b = 0; b < R; ++b)
            while (row[b] < rows) {
                const int r = row[b];
                if (step[b] == 0) formed[r] = 1, step[b] = 1;
                else if (step[b] == 1 && summed[r]) bounded[r] = 1, step[b] = 2;
                else if (step[b] == 2 && collected[r]) row[b] += R, step[b] = 0;
                else break;
                moved = true;
            }
    }
    bool done = at == order.size();
    for (int b = 0; b < R; ++b) done = done && row[b] >= rows;
    return done;
}

static int top_plans() {
    int bad = 0;
    std::map<std::tuple<int, int, int>, bool> known;
    std::map<int, long> warps;
    auto check = [&](int epv, long V, int lead, int k, long rows) {
        const long chunks = (V + lead + epv - 1) / epv;
        if (chunks <= 32 * (32 / epv) || k > V) return;  // a warp holds the row
        const int nt = chunks <= 1024 ? 128 : chunks <= 2048 ? 256 : 512, slot = 16 / epv * nt;
        const TopShape p = top_shape(nt, epv, chunks, k, rows, 148);
        ++warps[p.row_warps];
        const bool misaligned = epv == 4 && V + lead > 262144;
        if (p.row_warps == 0) {
            if (!(misaligned && k > 224) && ++bad < 20)
                std::printf("no room: %d-byte logits, V %ld, lead %d, k %d\n", 16 / epv, V, lead, k);
            return;
        }
        const size_t bytes = TopMemory(nt, slot, p.ring, p.row_warps, k, p.slices).bytes;
        if (bytes > stream_limit(top_blocks(nt)) && ++bad < 20) std::printf("%zu bytes for V %ld, k %d\n", bytes, V, k);
        const long each = (chunks + p.slices - 1) / p.slices;
        const int need = int((each + slot - 1) / slot);
        auto at = known.find({p.row_warps, p.ring, need});
        bool ok = at != known.end() ? at->second : true;
        if (at == known.end()) {
            for (int n = 1; n <= 3 * p.row_warps + 3; ++n)
                ok = ok && finishes(p.row_warps, top_adds_ahead(p.row_warps), p.ring, need, n);
            known[{p.row_warps, p.ring, need}] = ok;
        }
        if (!ok && ++bad < 20)
            std::printf("does not finish: %d-byte logits, V %ld, lead %d, k %d: %d row warps, ring %d of %d\n", 16 / epv, V,
                        lead, k, p.row_warps, p.ring, need);
        if (p.row_warps < 2 && !misaligned && ++bad < 20)
            std::printf("one row warp: %d-byte logits, V %ld, lead %d, k %d\n", 16 / epv, V, lead, k);
    };
    for (int epv = 4; epv <= 8; epv += 4)
        for (long V = 1; V <= 262144; V += V < 4200 ? 1 : V < 20000 ? 61 : 1021)
            for (int lead = 0; lead < epv; lead += epv - 1)
                for (int k : {1, 32, 64, 65, 100, 128, 129, 200, 213, 224, 254, 255, 256})
                    for (long rows : {1L, 37L, 100000L}) check(epv, V, lead, k, rows);
    for (long V : {2048L, 2049L, 4096L, 4097L, 8192L, 131072L, 131073L, 262140L, 262141L, 262143L, 262144L})
        for (int epv = 4; epv <= 8; epv += 4)
            for (int lead = 0; lead < epv; ++lead)
                for (int k = 1; k <= 256; ++k) check(epv, V, lead, k, 100000);
    for (auto& w : warps) std::printf("%d row warps: %ld shapes\n", w.first, w.second);
    // adding ahead with one row warp would not finish
    if (finishes(1, true, 8, 3, 2) || !finishes(1, true, 8, 3, 1) || !finishes(2, true, 8, 4, 9)) {
        std::printf("the walk does not see what it should\n");
        ++bad;
    }
    return bad;
}

// `kCtas` CTAs of a cluster exchange a number `kTurns` times, in every order in which
// their steps and the arrivals of what they send can come.  `place` and `parity`: the
// barrier of exchange n and the phase that is waited for; the slots are n % 2.  True if
// every CTA reads what was sent for that exchange, and none waits for good.
constexpr int kCtas = 3, kTurns = 4;
struct Cluster {
    signed char turn[kCtas], sent[kCtas];            // exchange, and whether it has sent for it
    signed char slot[kCtas][2][kCtas];               // exchange whose number lies there
    signed char phase[kCtas][2], waits[kCtas][2];    // parity; arrivals still wanted
    signed char bytes[kCtas][2];                     // numbers still wanted
    unsigned short flying[kCtas];                    // by receiver: bits 3 n % 4 ...: sent by whom
};
template <class Place, class Parity>
static bool exchanges(Place place, Parity parity, size_t* states) {
    auto key = [](const Cluster& c) { return std::string(reinterpret_cast<const char*>(&c), sizeof(c)); };
    Cluster first;
    std::memset(&first, 0, sizeof(first));
    std::memset(first.slot, -1, sizeof(first.slot));
    std::memset(first.waits, 1, sizeof(first.waits));
    std::vector<Cluster> todo{first};
    std::set<std::string> seen{key(first)};
    auto settle = [](Cluster& c, int to, int b) {
        if (c.waits[to][b] == 0 && c.bytes[to][b] == 0) c.phase[to][b] ^= 1, c.waits[to][b] = 1;
    };
    while (!todo.empty()) {
        const Cluster at = todo.back();
        todo.pop_back();
        bool moved = false;
        auto go = [&](const Cluster& c) {
            moved = true;
            if (seen.insert(key(c)).second) todo.push_back(c);
        };
        for (int i = 0; i < kCtas; ++i) {
            const int n = at.turn[i];
            if (n == kTurns) continue;
            Cluster c = at;
            if (!at.sent[i]) {  // one arrival, so many bytes wanted; then a number to every CTA
                const int b = place(n);
                --c.waits[i][b];
                c.bytes[i][b] += kCtas;
                settle(c, i, b);
                for (int to = 0; to < kCtas; ++to) c.flying[to] |= 1u << (n % 4 * kCtas + i);
                c.sent[i] = 1;
                go(c);
            } else if (at.phase[i][place(n)] != int(parity(n))) {
                for (int from = 0; from < kCtas; ++from)
                    if (at.slot[i][n % 2][from] != n) return false;
                c.turn[i] = n + 1;
                c.sent[i] = 0;
                go(c);
            }
        }
        for (int to = 0; to < kCtas; ++to)
            for (int bit = 0; bit < 4 * kCtas; ++bit)
                if (at.flying[to] >> bit & 1) {
                    Cluster c = at;
                    const int n = bit / kCtas;
                    c.flying[to] &= ~(1u << bit);
                    c.slot[to][n % 2][bit % kCtas] = n;
                    --c.bytes[to][place(n)];
                    settle(c, to, place(n));
                    go(c);
                }
        if (!moved)
            for (int i = 0; i < kCtas; ++i)
                if (at.turn[i] != kTurns) return false;
    }
    *states = seen.size();
    return true;
}
static int cluster_exchange() {
    size_t states = 0;
    const bool ok = exchanges(exchange_place, exchange_parity, &states);
    std::printf("%zu states\n", states);
    // one barrier for all exchanges lets a CTA read a slot before its number is there
    const bool one = exchanges([](unsigned) { return 0; }, [](unsigned n) { return n & 1; }, &states);
    return !ok || one;
}

int main(int argc, char** argv) {
    const char* what = argc > 1 ? argv[1] : "";
    if (!std::strcmp(what, "top")) return top_plans() != 0;
    if (!std::strcmp(what, "exchange")) return cluster_exchange();
    return 2;
}
