// Host run of InFlight (csrc/experts/grouped_tiles.hpp): whatever blocks a loader has given out when its kernel gives up, the waits that it makes end for each block under way
// when its own bytes have landed, and not before, nor by what else arrives on the barriers.
#include "../../csrc/experts/grouped_tiles.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace dccl;

/** Phases that are complete; a wait for a parity ends when the phase of that parity is the last of them. */
struct Barrier {
    unsigned done = 0;
    bool ends(unsigned parity) const { return (done & 1) != parity; }
};

int main() {
    srand(3);
    for (int round = 0; round < 4000; round++) {
        const unsigned stages = 2 + rand() % 5, blocks = rand() % 40, often = 1 + rand() % 6;
        std::vector<Barrier> full(stages), landed(stages);
        std::vector<bool> tail(blocks);
        InFlight loads;
        for (unsigned i = 0; i < blocks; i++) {
            const unsigned s = i % stages;
            if (i >= stages) {          // its stage was free: the block before had landed, and the other CTA had reported it
                full[s].done++;
                if (tail[i - stages]) landed[s].done++;
            }
            tail[i] = rand() % often == 0;
            loads.load(s, tail[i]);
        }
        if (loads.filled != blocks || blocks - loads.oldest(stages) != (blocks < stages ? blocks : stages)) return printf("blocks under way\n"), 1;
        for (unsigned i = loads.oldest(stages); i < blocks; i++) {
            Barrier &waits = (loads.on_landed(i, stages) ? landed : full)[i % stages], &other = (loads.on_landed(i, stages) ? full : landed)[i % stages];
            const unsigned parity = loads.parity(i, stages);
            if (waits.ends(parity)) return printf("ends before anything has landed\n"), 1;
            if (tail[i]) {
                other.done++;           // the other CTA's arrival completes `full`
                if (waits.ends(parity)) return printf("ends by the other CTA's arrival\n"), 1;
            }
            if (loads.on_landed(i, stages) != tail[i]) return printf("the wrong barrier\n"), 1;
            waits.done++;
            if (!waits.ends(parity)) return printf("does not end\n"), 1;
        }
    }
    printf("OK\n");
    return 0;
}
