// CPU check of the pipeline ring (reciprocating-engine_b200/csrc/ring.h)
// against barriers that count their completed phases: for every number of
// stages and fills, a stage is refilled only when its last fill was consumed,
// and the walk back from the end names the last fill of every used stage
// once, by a parity that tells consumed from not yet consumed.
#include <cstdio>
#include <vector>

#include "ring.h"

using reng::Ring;

// An mbarrier's test of a phase's parity: true once the phase of that parity
// that is current or newest is complete.
static bool done(int completed, uint32_t parity) { return (uint32_t)(completed & 1) != parity; }

int main() {
    long long bad = 0, cases = 0;
    for (int stages = 1; stages <= 12; stages++)
        for (int fills = 0; fills <= 5 * stages + 3; fills++)
            for (int behind = 0; behind <= stages && behind <= fills; behind++) {  // fills not consumed at the end
                cases++;
                std::vector<int> filled(stages, 0), consumed(stages, 0);
                std::vector<int> order;  // stage of each fill
                size_t taken = 0;
                Ring ring(stages);
                for (int i = 0; i < fills; i++) {
                    if (ring.full()) {
                        if (done(consumed[ring.stage], ring.phase ^ 1u) != (consumed[ring.stage] == filled[ring.stage])) bad++;
                        while (!done(consumed[ring.stage], ring.phase ^ 1u)) consumed[order[taken++]]++;  // in order
                        if (consumed[ring.stage] != filled[ring.stage]) bad++;
                    } else if (filled[ring.stage] != 0) {
                        bad++;
                    }
                    filled[ring.stage]++;
                    order.push_back(ring.stage);
                    ring.fill();
                }
                while ((int)taken < fills - behind) consumed[order[taken++]]++;
                std::vector<int> named(stages, 0);
                Ring last = ring;
                bool landed = true;
                for (int newest = fills - 1; last.back(); newest--) {
                    named[last.stage]++;
                    if (newest < 0 || last.stage != order[newest]) bad++;
                    const bool ok = done(consumed[last.stage], last.phase);
                    if (ok != (consumed[last.stage] == filled[last.stage])) bad++;
                    landed = landed && ok;
                }
                for (int s = 0; s < stages; s++)
                    if (named[s] != (filled[s] > 0)) bad++;
                if (landed != ((int)taken == fills)) bad++;
            }
    printf("cases %lld bad %lld\n", cases, bad);
    return bad ? 1 : 0;
}
