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
