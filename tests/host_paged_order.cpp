// The issuer's order of csrc/paged_order.h against a tensor core that finishes a product no sooner than somebody has waited for it, for tests/test_paged_order.py.
#include <stdio.h>
#include <string.h>

#include <set>
#include <string>

#include "../slai_b200/csrc/paged_order.h"

using namespace paged;

extern "C" {
// Parts of units[0 .. parts): the first thing that goes wrong, or "".
const char* host_chunk_products(const int* units, int parts) {
    static std::string why;
    why.clear();
    std::set<uint32_t> qk, pv;  // under way, for all that the issuer knows
    uint32_t u = 0, scores_so_far = 0, outputs_so_far = 0;
    auto bad = [&](const char* what, uint32_t i) {
        if (why.empty()) why = std::string(what) + " " + std::to_string(i);
    };
    for (int k = 0; k < parts; k++) {
        // the queries of a part are there once the rows' threads have taken the outputs of the part before: of its last unit, and so of all
        qk.clear();
        pv.clear();
        const uint32_t first = u;
        chunk_products(
            u, units[k], [&](uint32_t i) { pv.erase(i); },
            [&](uint32_t i) {
                if (i != scores_so_far++) bad("scores out of turn:", i);
                for (uint32_t p : pv)
                    if (p % 2 == i % 2) bad("scores over weights that a product still reads: unit", i);
                for (uint32_t q : qk)
                    if (q % 2 == i % 2) bad("scores over scores that nobody has read: unit", i);
                qk.insert(i);
            },
            [&](uint32_t i) {
                if (i != outputs_so_far++) bad("outputs out of turn:", i);
                // its weights are there: the rows' threads have seen its scores, and before they say so they take the outputs of the part's unit before
                if (!qk.count(i)) bad("weights of scores that were not asked for: unit", i);
                qk.erase(i);
                if (i > first) pv.erase(i - 1);
                if (!pv.empty()) bad("outputs over outputs that nobody has taken: unit", i);
                pv.insert(i);
            });
        u += units[k];
    }
    if (scores_so_far != u || outputs_so_far != u) bad("units left out:", u);
    return why.c_str();
}
}

namespace {
struct Barrier {  // phases begun and completed; a wait knows a phase by its parity alone
    uint32_t done = 0;
    bool over(uint32_t phase) const { return (done & 1) != (phase & 1); }
};
}  // namespace
extern "C" {
// `rounds` fills of a slot whose reader stops after `reads` of them (a wait for the next then gives up, as do all behind it), the last fill being still on its way: how often
// settle() says that all have landed while one has not, or waits for a phase that nobody will complete.
int host_settles_wrongly(int rounds, int reads) {
    SlotFills f;
    Barrier full, empty;
    int asked = 0;
    bool gone = false;
    for (int r = 0; r < rounds; r++) {
        const bool go = f.may_fill([&](uint32_t i) {
            if (gone) return false;
            if (empty.done < (uint32_t)reads && (uint32_t)asked > empty.done) empty.done++;  // the reader has had its last fill
            gone = !empty.over(i);
            return !gone;
        });
        if (!go) continue;
        if (asked > 0) full.done = asked;  // the reader can only have read what had landed
        f.filled();
        asked++;
    }
    int wrong = 0;
    bool waited = false;
    f.settle([&](uint32_t i) {
        waited = true;
        if (full.over(i)) wrong++;       // over although the last is on its way
        full.done = asked;
        if (!full.over(i)) wrong++;      // not over although it has landed
    });
    return wrong + (asked > 0 && !waited);
}
}
