// The planner of a step over a paged cache (csrc/paged_plan.h), for tests/test_paged_plan.py.
#include <string.h>

#include "../slai_b200/csrc/paged_plan.h"

using namespace paged;

struct Host {
    Planner p;
    Config c;
    std::string why;
};

extern "C" {
int host_paged_div(int n, int d) { return n / Div(d); }
// cfg: the nine fields of Config; lanes: {rows, unit, blocks, least, join} twice; returns null and the reason where the configuration is refused
Host* host_paged_create(const int* cfg, const int* lanes, int few, int most, char* why, int len) {
    Config c = {cfg[0], cfg[1], cfg[2], cfg[3], cfg[4], cfg[5], cfg[6], cfg[7], cfg[8]};
    const std::string w = check_config(c);
    strncpy(why, w.c_str(), len - 1);
    why[len - 1] = 0;
    if (!w.empty()) return nullptr;
    Lane l[2];
    for (int i = 0; i < 2; i++) {
        l[i].rows = lanes[5 * i];
        l[i].unit = lanes[5 * i + 1];
        l[i].blocks = lanes[5 * i + 2];
        l[i].least = lanes[5 * i + 3];
        l[i].join = lanes[5 * i + 4];
        l[i].low = i ? l[i].rows / 2 : 0;
        l[i].unit_us[0] = 3.4;
        l[i].unit_us[1] = 2.6;
        l[i].whole_us[0] = l[i].whole_us[1] = 12;
        l[i].cut_us[0] = 25;
        l[i].cut_us[1] = 19;
    }
    Host* h = new Host();
    h->c = c;
    l[0].fixed = 5;
    l[0].each = 0.005;
    l[1].fixed = 13;
    l[1].each = 0.02;
    h->p.init(c, l[0], l[1], few, most);
    return h;
}
void host_paged_destroy(Host* h) { delete h; }
// total ints; offsets of starts, joins, count, rows, dynamic
void host_paged_layout(Host* h, int* out) {
    const Layout& L = h->p.lay();
    const int v[8] = {L.total, L.starts[0], L.starts[1], L.joins[0], L.joins[1], L.count, L.rows, L.dynamic};
    memcpy(out, v, sizeof(v));
}
// out: total ints; step: n_rows, blocks of each lane, used, joins of each lane.  Returns the reason ("" = fine).
const char* host_paged_plan(Host* h, int n, const int* pos0, const int* n_new, const int* tables, long long ld, int* out, int* step) {
    Step s;
    h->why = h->p.plan(n, pos0, n_new, tables, ld, out, &s);
    const int v[6] = {s.n_rows, s.blocks[0], s.blocks[1], s.used, s.joins[0], s.joins[1]};
    memcpy(step, v, sizeof(v));
    return h->why.c_str();
}
}
