// Host check of the ring of asynchronous copies (copy_ring.h): barriers with phases, copies that land in any order, and
// consumers that give up at any wait. Whatever the moment, a copy never goes to a stage that still holds one, every wait
// asks for the phase that its copy completes, and after drain() nothing is in flight. Prints "0 failure(s)" on success.
#include "copy_ring.h"

#include <algorithm>
#include <cstdio>
#include <random>
#include <set>

template <unsigned DEPTH>
long long run(std::mt19937& rng, int copies, int step, int give_up_at) {
    struct Stage {
        bool in_flight = false, full = false;
        unsigned phase = 0;  // completed phases
    } stages[DEPTH];
    long long failures = 0;
    mfb::CopyRing<DEPTH> ring;
    auto issue = [&] {
        if (static_cast<int>(ring.issued) == copies) return;
        Stage& s = stages[ring.next()];
        failures += s.in_flight || s.full;
        s.in_flight = true;
        ++ring.issued;
    };
    auto land = [&](Stage& s) {
        if (!s.in_flight) return;
        s.in_flight = false, s.full = true;
        ++s.phase;
    };
    // A parity wait: over once the phase of that parity is completed, which is the stage's latest one.
    auto wait = [&](unsigned at, unsigned parity) {
        Stage& s = stages[at];
        while (rng() % 3) land(stages[rng() % DEPTH]);
        land(s);
        failures += !s.full || ((s.phase - 1) & 1) != parity;
        return true;
    };
    for (unsigned i = 0; i < DEPTH; ++i) issue();
    int waits = 0;
    while (static_cast<int>(ring.consumed) < copies) {
        const unsigned n = static_cast<unsigned>(std::min<int>(step, copies - static_cast<int>(ring.consumed)));
        bool ok = true;
        for (unsigned u = 0; ok && u < n; ++u) ok = waits++ != give_up_at && wait(ring.stage(u), ring.parity(u));
        if (!ok) break;
        for (unsigned u = 0; u < n; ++u) stages[ring.stage(u)].full = false;
        ring.consumed += n;
        for (unsigned u = 0; u < n; ++u) issue();
    }
    failures += !ring.drain(wait);
    for (const Stage& s : stages) failures += s.in_flight;
    return failures;
}

int main() {
    std::mt19937 rng(12345);
    long long failures = 0, checked = 0;
    for (int copies = 0; copies < 40; ++copies)
        for (int step = 1; step <= 2; ++step)
            for (int give_up_at = -1; give_up_at < copies; ++give_up_at, ++checked)
                failures += run<2>(rng, copies, step, give_up_at) + run<4>(rng, copies, step, give_up_at);
    // The full ring: the case that positions alone take for an empty one.
    mfb::CopyRing<4> ring;
    ring.issued = 4;
    std::set<unsigned> seen;
    ring.drain([&](unsigned s, unsigned parity) { return seen.insert(s).second && parity == 0; });
    failures += seen.size() != 4;
    std::printf("%lld checked, %lld failure(s)\n", checked, failures);
    return failures == 0 ? 0 : 1;
}
