// Host-only exercise of csrc/reader.h for the CPU tests: the warps of a block of the scores' kernel as state machines that take turns in
// a random order, over barriers that count arrivals.  One warp fills accumulators, one fills scales, four readers use both, meet, and store one
// another's lanes.  One wait of one reader (argv[2]: which barrier, 0 accumulators, 1 scales, -1 none) runs out although what it waits
// for comes; after that a wait runs out only where nobody can go on.
// argv[1] = "reader": the rule of the header; "always": a reader that goes on as if nothing had been.  argv[3] = readers that meet and store
// one another's lanes (1: each its own).
// Prints the wrong finite scores, the NaN and the right ones, over many orders.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "reader.h"

struct Barrier {                       // as an mbarrier: a phase ends with its count-th arrival
    int count, pending;
    unsigned phase = 0;
    explicit Barrier(int n) : count(n), pending(n) {}
    void arrive() { if (--pending == 0) { pending = count; phase++; } }
    bool done(unsigned parity) const { return (phase & 1) != parity; }
};

constexpr int kReaders = 4, kBuffers = 2, kSlots = 8, kSteps = 40;

struct Block {
    std::vector<Barrier> ready, spare, judged, used;
    int accumulator[kBuffers], slot[kSlots];                 // the step that they hold
    int met[kReaders] = {};                                  // arrivals at a group's meetings
    Block() : ready(kBuffers, Barrier(1)), spare(kBuffers, Barrier(kReaders)), judged(kSlots, Barrier(1)), used(kSlots, Barrier(kReaders)) {
        for (int& a : accumulator) a = -1;
        for (int& s : slot) s = -1;
    }
};

struct Filler {                        // of accumulators or of scales
    int step = 0;
    bool over = false, gave_up = false;
    bool turn(std::vector<Barrier>& free, std::vector<Barrier>& full, int* content, int n, bool out_of_time) {
        if (over) return false;
        const int b = step % n;
        if (step >= n && !free[b].done((step / n + 1) & 1)) {
            if (out_of_time) over = gave_up = true;
            return out_of_time;
        }
        content[b] = step;
        full[b].arrive();
        over = ++step == kSteps;
        return true;
    }
};

struct Lane { int step; bool nan; };   // what a reader left for its meeting

struct Tally { long wrong = 0, nan = 0, right = 0; };

struct ReaderWarp {
    mascot::Reader reader;
    int step = 0, at = 0;              // at: wait for scales, wait for the accumulator, read, hand back, meet, store, hand back
    bool turn(Block& k, int who, int size, bool always, int deaf_step, int deaf_barrier, bool out_of_time, Lane& mine, const Lane* lanes, Tally& tally) {
        if (step == kSteps) return false;
        const int b = step % kBuffers, q = step % kSlots;
        const auto wait = [&](const Barrier& bar, unsigned parity, bool deaf) {      // true: go on
            if (!reader.ok()) return true;
            if (deaf || (!bar.done(parity) && out_of_time)) { reader.waited(false); return true; }
            return bar.done(parity);
        };
        const auto hand_back = [&](Barrier& bar) {
            if (always) bar.arrive();
            else reader.hand_back([&] { bar.arrive(); });
        };
        const float factor = always && at == 5 ? 1.f : reader.factor(1.f);         // lanes were NaN before, scales of rows were not
        switch (at) {
            case 0: if (!wait(k.judged[q], step / kSlots & 1, step == deaf_step && deaf_barrier == 1)) return false; break;
            case 1: if (!wait(k.ready[b], step / kBuffers & 1, step == deaf_step && deaf_barrier == 0)) return false; break;
            case 2: mine = {k.accumulator[b], std::isnan(factor)}; break;
            case 3: hand_back(k.spare[b]); break;
            case 4: k.met[who / size]++; break;
            case 5:
                if (k.met[who / size] < (step + 1) * size) return false;
                for (int r = who / size * size; r < (who / size + 1) * size; r++) {      // a row of scores: all lanes of the group, this warp's scale
                    const bool nan = lanes[r].nan || std::isnan(factor);
                    if (nan) tally.nan++;
                    else if (lanes[r].step == step && k.slot[q] == step) tally.right++;
                    else tally.wrong++;
                }
                break;
            case 6: hand_back(k.used[q]); break;
        }
        if (++at == 7) { at = 0; step++; }
        return true;
    }
};

int main(int argc, char** argv) {
    if (argc < 4) return 2;
    const bool always = !std::strcmp(argv[1], "always");
    const int deaf_barrier = std::atoi(argv[2]), size = std::atoi(argv[3]);
    Tally tally;
    for (unsigned seed = 0; seed < 400; seed++) {
        std::mt19937 rng(seed);
        Block k;
        Filler products, scales;
        ReaderWarp readers[kReaders];
        Lane lanes[2][kReaders] = {};                            // two meetings' worth, as in the kernel
        const int deaf_step = deaf_barrier < 0 ? -1 : (int)(rng() % kSteps);
        for (int idle = 0;;) {
            bool all = true;
            for (const ReaderWarp& r : readers) all = all && r.step == kSteps;
            if (all) break;
            const bool out_of_time = idle > 200;                 // nobody has gone on for a while: every wait has run out
            if (idle > 100000) { std::printf("stuck\n"); return 1; }
            const int who = (int)(rng() % (kReaders + 2));
            bool went;
            if (who == kReaders) went = products.turn(k.spare, k.ready, k.accumulator, kBuffers, out_of_time);
            else if (who == kReaders + 1) went = scales.turn(k.used, k.judged, k.slot, kSlots, out_of_time);
            else went = readers[who].turn(k, who, size, always, who == 0 ? deaf_step : -1, deaf_barrier, out_of_time, lanes[readers[who].step & 1][who], lanes[readers[who].step & 1], tally);
            idle = went ? 0 : idle + 1;
        }
    }
    std::printf("%ld %ld %ld\n", tally.wrong, tally.nan, tally.right);
    return 0;
}
