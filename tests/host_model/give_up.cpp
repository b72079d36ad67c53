// Host run of what a block or pair does about its copies when it has given up (give_up.h), over made-up barriers: arrivals and bytes that are
// outstanding, phases that end when both are none.  Test code only.
#include <vector>

#include "../../openfish_b200/csrc/give_up.h"

namespace {
struct Barrier {
    int phase = 0, arrivals = 1;
    long bytes = 0;
    void settle() {
        if (arrivals == 0 && bytes == 0) ++phase, arrivals = 1;
    }
};
}  // namespace

// A pair of blocks (or one, pair = 0) through a ring of `ring` stages: `read` steps have been copied and read, the first block has issued
// `mine` in all, the other one `theirs`; a copy lands when somebody waits for it.  Returns how many copies are under way at the end, or -1 for a
// wait that would run out, -2 for a step that was announced twice.
extern "C" int copies_left(int ring, int read, int mine, int theirs, int pair) {
    std::vector<Barrier> full(ring);
    std::vector<int> under_way(ring, 0);  // copies into a stage that have not landed
    const long half = 100;
    const int most = mine > theirs ? mine : theirs;
    for (int i = 0; i < most; ++i) {
        Barrier &b = full[i % ring];
        const bool first = i < mine, other = pair && i < theirs;
        if (first) b.arrivals -= 1, b.bytes += pair ? 2 * half : half;
        if (i < read) {
            b.bytes -= pair ? 2 * half : half;
            b.settle();
        } else {
            under_way[i % ring] += first + other;
        }
    }
    int bad = 0;
    land_copies(
        mine, pair ? theirs : mine, ring,
        [&](int stage) {
            if (full[stage].arrivals != 1) bad = -2;
            full[stage].arrivals -= 1;
            full[stage].bytes += half;
        },
        [&](int stage) { full[stage].bytes -= half; },
        [&](int stage, uint32_t parity) {
            Barrier &b = full[stage];
            b.bytes -= half * under_way[stage];
            under_way[stage] = 0;
            b.settle();
            if (b.phase == 0 || (uint32_t)((b.phase - 1) & 1) != parity) bad = bad ? bad : -1;
        });
    if (bad) return bad;
    int left = 0;
    for (int n : under_way) left += n;
    return left;
}
