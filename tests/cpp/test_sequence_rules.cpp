// The rules of sequence_rules.h against what they are for, host code only.
#include <cstdio>
#include <vector>

#include "sequence_rules.h"

using namespace seera;

static int bad = 0;

// A block's sums over `waves` waves, `sums` of them, in the order of events that is
// worst for one barrier a sum: `fast` runs alone until the barrier holds it, again
// and again, and the others read as late as they may. Returns the number of parts
// that a wave read of another sum than its own.
template <class NextHalf>
static int stale_reads(int waves, int sums, int fast, NextHalf&& next_half) {
    std::vector<int> part(2 * waves, -1);
    std::vector<int> half(sums);
    for (int k = 0; k < sums; ++k) half[k] = next_half(k);
    int stale = 0;
    auto write = [&](int wave, int k) { part[half[k] * waves + wave] = k; };
    auto read = [&](int k) {
        for (int w = 0; w < waves; ++w) stale += part[half[k] * waves + w] != k;
    };
    // the barrier of sum k opens when all have written k; then `fast` reads k and
    // writes k + 1, before the others read k and write k + 1
    for (int w = 0; w < waves; ++w) write(w, 0);
    for (int k = 0; k < sums; ++k) {
        read(k);
        if (k + 1 < sums) write(fast, k + 1);
        for (int w = 0; w < waves; ++w)
            if (w != fast) read(k);
        for (int w = 0; w < waves; ++w)
            if (w != fast && k + 1 < sums) write(w, k + 1);
    }
    return stale;
}

static void sums_of_a_row() {
    for (int waves : {2, 4, 16})
        for (int fast = 0; fast < waves; ++fast) {
            Halves halves;
            if (stale_reads(waves, 9, fast, [&](int) { return halves.next(); })) ++bad, std::printf("Halves: %d waves, wave %d ahead\n", waves, fast);
            // planted: one half for each kind of sum. Two kinds in turn are right, one alone is not
            if (stale_reads(waves, 9, fast, [](int k) { return k & 1; })) ++bad, std::printf("two kinds in turn\n");
            if (!stale_reads(waves, 9, fast, [](int) { return 0; })) ++bad, std::printf("a planted fixed half is not seen\n");
        }
}

// The rows that a block's threads load, as scan_tiles asks for them: tiles of
// threads * per steps, in a whole tile each step's own row, else the nearest live
// step's; and, with shift 1 (backward, h), the row before it.
static void rows_of_a_walk() {
    // planted: bounds by the segment alone load rows that a length leaves out
    const Walk planted = walk_of(false, 0, 64, 64);
    if (planted.time_of(planted.nearest(40)) < 20) ++bad, std::printf("a planted bound by the segment is not seen\n");
    struct Tile {
        int threads, per;
    };
    for (const Tile tile : {Tile{4, 8}, Tile{32, 4}, Tile{1, 16}, Tile{16, 1}})
        for (int time : {1, 2, 31, 32, 33, 100, 257})
            for (int steps : {time, 32, 64})  // of a segment
                for (int begin = 0; begin < time; begin += steps)
                    for (int n = 0; n <= time; ++n)
                        for (int back = 0; back < 2; ++back) {
                            const int end = begin + steps < time ? begin + steps : time, k = tile.threads * tile.per;
                            const Walk walk = walk_of(back, begin, end, n);
                            for (int u0 = 0; u0 < walk.length(); u0 += k)
                                for (int first = u0; first < u0 + k; first += tile.per)
                                    for (int u = first; u < first + tile.per; ++u) {
                                        const int own = back ? end - 1 - u : begin + u;
                                        const bool inside = own >= begin && own < end && own < n, whole = walk.whole(u0, k);
                                        bool right = walk.live(u) == inside && (!whole || inside);
                                        if (whole || walk.any(first, tile.per)) {
                                            const int at = whole ? own : walk.time_of(walk.nearest(u)), before = whole ? at - 1 : at > 0 ? at - 1 : 0;
                                            right = right && at >= begin && at < end && at < n && (!inside || at == own);
                                            right = right && (!back || (before >= 0 && before < n));
                                        } else {
                                            right = right && !inside;
                                        }
                                        if (!right && bad++ < 5)
                                            std::printf("walk: time %d segment %d..%d n %d back %d u0 %d first %d u %d\n", time, begin, end, n, back, u0, first, u);
                                    }
                        }
}

int main() {
    sums_of_a_row();
    rows_of_a_walk();
    if (!bad) std::puts("all checks passed");
    return bad != 0;
}
