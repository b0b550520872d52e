// The host's side of a step over a paged cache: checks of lengths and page tables, and who computes what.  Plain C++ (the tests compile it by itself).
//
// A sequence's rows of the step's attention are (token, query head of the group) pairs, one cache head at a time: rows [R i, R i + R) of them are a
// tile.  A tile's work is its positions, 0 .. the last one its last row sees, in units of `unit` positions; the units of all (tile, cache head) pairs stand
// in one line, tile by tile and head by head, and a block takes an equal share of that line, from somewhere in one pair to somewhere in another.  So
// one long sequence and many short ones keep all SMs equally long.  To begin and end a pair costs a block about as much as PAIR_COST units, which stand in the
// line in front of the pair's own.  A pair that lies on several blocks leaves partial results (two a block at most),
// which a launch behind it joins in the order of their positions.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <string>
#include <vector>

#ifdef __CUDACC__
#define PAGED_HD __host__ __device__ __forceinline__
#else
#define PAGED_HD inline
#endif

namespace paged {

// A divisor 1 .. 2^30 of numbers 0 .. 2^31 - 1: with L = ceil(log2 d) and m = floor(2^(31 + L) / d) + 1, m d is above 2^(31 + L) by at most 2^L, so that
// n m / 2^(31 + L) is above n / d by less than 1 / d.
struct Div {
    int d = 1;
    uint32_t mul = 0;
    int shift = 0;  // L - 1
    Div() = default;
    explicit Div(int by) : d(by) {
        if (by <= 1) return;
        int L = 0;
        while ((1ll << L) < by) L++;
        mul = (uint32_t)(((1ull << (31 + L)) / (uint64_t)by) + 1);
        shift = L - 1;
    }
    PAGED_HD operator int() const { return d; }
};
PAGED_HD int operator/(int n, const Div& by) {
    if (by.d == 1) return n;
#ifdef __CUDA_ARCH__
    return (int)(__umulhi((uint32_t)n, by.mul) >> by.shift);
#else
    return (int)((uint32_t)(((uint64_t)(uint32_t)n * by.mul) >> 32) >> by.shift);
#endif
}
PAGED_HD int operator%(int n, const Div& by) { return n - n / by * by.d; }

constexpr int PAIR_COST = 2;

struct Config {
    int n_q_heads, n_kv_heads, head_size, page_size, n_pages, kv_dtype;
    int max_seqs, max_tokens, max_table;
};

// What a kernel reads.  All offsets are in ints from the start of the device copy.
struct Tile {
    int row0;     // first row (token) of the sequence in q / out
    int pos0;     // position of that token
    int first;    // first packed row of the tile (token first / group, head first % group)
    int rows;     // packed rows of the tile
    int table;    // page table of the sequence
    int units;    // of one cache head
    int line;     // place in the line of the tile's first pair
    int pad;
};
struct Start {  // where a block begins
    int tile, head, unit, count;   // count: places of the line from there to the end of the block's share
    Tile t;                        // tiles[tile]
    int tiles;                     // offset of the tiles
    int units, blocks, me;         // places of the whole line; blocks that share it
};
struct Join {  // a pair that lies on several blocks
    int row0, first, rows, head;  // as in Tile
    int begin, end;               // the blocks; of `begin` the second slot, of the others the first
    int pad[2];
};
struct Row {  // a token of the step
    int pos, slot;  // slot: page * page_size + place in the page
};
static_assert(sizeof(Tile) == 32 && sizeof(Start) == 64 && sizeof(Join) == 32 && sizeof(Row) == 8, "read as words by the kernels");

struct Lane {  // one of the two kinds of kernel
    int rows = 0, unit = 0;    // tile height, positions of a unit
    int low = 0;               // a lower tile height (0: none), for steps that are sooner done so.  What decides, for (rows, low): us of a unit of the block with the most,
    double unit_us[2] = {}, whole_us[2] = {}, cut_us[2] = {};  // and of all else, where pairs are whole and where they are cut
    int blocks = 0;            // most blocks
    int least = 1;             // units a block has at least, if the line allows it
    double fixed = 0, each = 0;  // us of a launch, and of a unit in a launch that fills the GPU: which lane takes the sequences that either could take
    int join = 0;              // units that the join costs: where every pair can have a block, none is cut that is longer than nine eighths of a share by no more than this
};

struct Layout {  // of the device copy, in ints
    int starts[2], joins[2], count, rows, dynamic, total;  // count: numbers of the step's rows and of each lane's joins
};
inline int tiles_cap(const Config& c, const Lane& l) {
    return l.blocks ? (int)std::min<long long>(((long long)c.max_tokens * (c.n_q_heads / c.n_kv_heads)) / (l.low ? l.low : l.rows) + c.max_seqs, 1ll << 30) : 0;
}
inline Layout layout(const Config& c, const Lane (&lanes)[2]) {
    Layout L;
    L.starts[0] = 0;
    L.starts[1] = L.starts[0] + lanes[0].blocks * (int)(sizeof(Start) / 4);
    L.joins[0] = L.starts[1] + lanes[1].blocks * (int)(sizeof(Start) / 4);
    L.joins[1] = L.joins[0] + lanes[0].blocks * (int)(sizeof(Join) / 4);
    L.count = L.joins[1] + lanes[1].blocks * (int)(sizeof(Join) / 4);
    L.rows = L.count + 8;
    L.dynamic = (L.rows + 2 * c.max_tokens + 7) & ~7;
    L.total = L.dynamic + ((c.max_table + 7) & ~7) + (tiles_cap(c, lanes[0]) + tiles_cap(c, lanes[1])) * (int)(sizeof(Tile) / 4);
    return L;
}

struct Step {
    int n_rows = -1;          // -1: there has been no step
    int blocks[2] = {0, 0};   // blocks with work
    int joins[2] = {0, 0};    // pairs on several blocks
    int longest[2] = {0, 0};  // most blocks of one
    int used = 0;             // ints of the dynamic part
};

// Why `c` cannot be served, or "".
inline std::string check_config(const Config& c) {
    auto bad = [](const char* what, long long v) { return std::string(what) + " (" + std::to_string(v) + ")"; };
    if (c.n_kv_heads < 1 || c.n_q_heads < 1 || c.n_q_heads > 65536 || c.n_q_heads % std::max(1, c.n_kv_heads)) return "n_kv_heads must divide n_q_heads (" + std::to_string(c.n_q_heads) + " on " + std::to_string(c.n_kv_heads) + ")";
    if (c.head_size < 1 || c.head_size > 256) return bad("head_size must be 1 .. 256", c.head_size);
    if (c.page_size < 1 || c.page_size > (1 << 20)) return bad("page_size must be 1 .. 2^20", c.page_size);
    if (c.n_pages < 1 || (long long)c.n_pages * c.page_size > 0x7fffffffll) return bad("n_pages must be at least 1 and n_pages * page_size below 2^31", c.n_pages);
    if (c.kv_dtype != 0 && c.kv_dtype != 1) return bad("unknown cache type", c.kv_dtype);
    if (c.max_seqs < 1 || c.max_seqs > (1 << 20)) return bad("max_seqs must be 1 .. 2^20", c.max_seqs);
    if (c.max_tokens < 1 || c.max_tokens > (1 << 24)) return bad("max_tokens must be 1 .. 2^24", c.max_tokens);
    if (c.max_table < 1 || c.max_table > (1 << 28)) return bad("max_table must be 1 .. 2^28", c.max_table);
    if ((long long)c.max_tokens * (c.n_q_heads / c.n_kv_heads) > 0x7fffffffll / 2) return bad("max_tokens * group is too large", c.max_tokens);
    return "";
}

// Whether a layer's strides give every (page, cache head, place) a row of its own: whichever of the three moves least moves by a row at least, the next by all that
// lies within, the last by all that lies within those.
inline bool rows_apart(const Config& c, int64_t page_stride, int64_t head_stride, int64_t pos_stride) {
    struct Dim {
        int64_t stride, n;
    } d[3] = {{page_stride, c.n_pages}, {head_stride, c.n_kv_heads}, {pos_stride, c.page_size}};
    std::sort(d, d + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    __int128 span = c.head_size;  // from a row's first element to the last of all that lie within
    for (const Dim& x : d) {
        if (x.n == 1) continue;
        if (x.stride < span) return false;
        span += (__int128)(x.n - 1) * x.stride;
    }
    return true;
}

class Planner {
  public:
    // Sequences of up to `few` rows (tokens * group) go to lane 0, of more than `most` to lane 1 (it may be absent, blocks 0); those between to where the step
    // takes less time, by the lanes' `fixed` and `each`.
    void init(const Config& c, const Lane& a, const Lane& b, int few, int most) {
        cfg_ = c;
        lanes_[0] = a;
        lanes_[1] = b;
        few_ = b.blocks ? few : 0x7fffffff;
        most_ = std::max(few_, most);
        now_ = few_;
        lay_ = layout(cfg_, lanes_);
        seen_.assign((size_t)c.n_pages, 0);
    }
    const Layout& lay() const { return lay_; }
    const Lane& lane(int i) const { return lanes_[i]; }

    // Sequence b: pos0[b] positions are cached, n_new[b] tokens follow (0: it takes no part); row b of `tables` ([n_seq][ld]) names the pages of positions
    // 0 .. pos0 + n_new - 1 in order.  Writes the device copy to `out` (lay().total ints) and `step`; returns why not, or "" (nothing is written then).
    std::string plan(int n_seq, const int32_t* pos0, const int32_t* n_new, const int32_t* tables, int64_t ld, int32_t* out, Step* step) {
        auto say = [](const char* what, long long b, long long v) { return std::string(what) + " (sequence " + std::to_string(b) + ": " + std::to_string(v) + ")"; };
        if (n_seq < 0 || n_seq > cfg_.max_seqs) return "n_seq must be 0 .. " + std::to_string(cfg_.max_seqs) + " (" + std::to_string(n_seq) + ")";
        if (n_seq > 0 && (!pos0 || !n_new || !tables)) return "lengths and tables are missing";
        const int group = cfg_.n_q_heads / cfg_.n_kv_heads, ps = cfg_.page_size;
        const int before = now_;
        struct Back {  // a step that is refused leaves no trace
            int &now, was;
            bool keep;
            ~Back() {
                if (!keep) now = was;
            }
        } back = {now_, before, false};
        now_ = few_;
        long long tokens = 0;
        for (int b = 0; b < n_seq; b++) tokens += std::max(0, n_new[b]);
        const bool fits = tokens <= cfg_.max_tokens;  // (else it is refused below)
        if (most_ > few_ && fits) {
            double us[2];
            for (int way = 0; way < 2; way++) us[way] = cost(n_seq, pos0, n_new, group, way ? most_ : few_);
            if (us[1] < us[0]) now_ = most_;
        }
        for (int k = 0; k < 2; k++) {
            height_[k] = lanes_[k].rows;
            if (lanes_[k].low && fits && takes(k, 1, n_seq, pos0, n_new, group) < takes(k, 0, n_seq, pos0, n_new, group)) height_[k] = lanes_[k].low;
        }
        long long rows = 0, entries = 0, line[2] = {0, 0};
        for (int b = 0; b < n_seq; b++) {
            if (pos0[b] < 0) return say("a negative number of cached positions", b, pos0[b]);
            if (n_new[b] < 0) return say("a negative number of new tokens", b, n_new[b]);
            if (n_new[b] == 0) continue;
            const long long held = (long long)pos0[b] + n_new[b], pages = (held + ps - 1) / ps;
            if (held > 0x7fffffffll - 1024) return say("too many positions", b, held);
            if (pages > ld) return say("the page table is too narrow", b, ld);
            rows += n_new[b];
            entries += pages;
            if (rows > cfg_.max_tokens) return "more new tokens than max_tokens (" + std::to_string(cfg_.max_tokens) + ")";
            if (entries > cfg_.max_table) return "more pages than max_table (" + std::to_string(cfg_.max_table) + ")";
            const int k = lane_of(n_new[b]);
            for_tiles(b, pos0[b], n_new[b], group, [&](const Tile& t) { line[k] += (long long)(t.units + PAIR_COST) * cfg_.n_kv_heads; });
        }
        if (line[0] > 0x7fffffffll || line[1] > 0x7fffffffll) return "the step's attention is too large";
        // Every page exists; one that gets new tokens belongs to its sequence alone, and to one place of it (pages that are only read may be shared).
        if (++mark_ > 0x3fffffff) {
            std::fill(seen_.begin(), seen_.end(), 0);
            mark_ = 1;
        }
        const int written = 2 * mark_, read = 2 * mark_ + 1;
        for (int pass = 0; pass < 2; pass++)
            for (int b = 0; b < n_seq; b++) {
                if (n_new[b] == 0) continue;
                const int32_t* tab = tables + (int64_t)b * ld;
                const int pages = (int)(((long long)pos0[b] + n_new[b] + ps - 1) / ps), first_new = pos0[b] / ps;
                for (int i = pass ? first_new : 0; i < (pass ? pages : first_new); i++) {
                    const int id = tab[i];
                    if (id < 0 || id >= cfg_.n_pages) return say("no such page", b, id);
                    if (pass && (seen_[id] == read || seen_[id] == written)) return say("a page that gets new tokens is used twice", b, id);
                    seen_[id] = pass ? written : read;
                }
            }
        std::vector<int>& tab_at = tmp_;
        tab_at.assign((size_t)std::max(1, n_seq), 0);
        // -- nothing fails from here on --
        back.keep = true;
        step->n_rows = (int)rows;
        out[lay_.count] = (int)rows;
        int* row = out + lay_.rows;
        int at = lay_.dynamic, r0 = 0;
        for (int b = 0; b < n_seq; b++) {
            if (n_new[b] == 0) continue;
            const int32_t* tab = tables + (int64_t)b * ld;
            const int held = pos0[b] + n_new[b], pages = (held + ps - 1) / ps;
            tab_at[b] = at;
            std::copy(tab, tab + pages, out + at);
            at += pages;
            for (int i = 0; i < n_new[b]; i++) {
                const int p = pos0[b] + i;
                *row++ = p;
                *row++ = tab[p / ps] * ps + p % ps;
            }
        }
        at = (at + 7) & ~7;
        for (int k = 0; k < 2; k++) {
            Tile* tiles = reinterpret_cast<Tile*>(out + at);
            const int tiles_at = at;
            int n = 0, so_far = 0;
            r0 = 0;
            for (int b = 0; b < n_seq; b++) {
                if (n_new[b] > 0 && lane_of(n_new[b]) == k)
                    for_tiles(b, pos0[b], n_new[b], group, [&](Tile t) {
                        t.row0 = r0;
                        t.table = tab_at[b];
                        t.line = so_far;
                        so_far += (t.units + PAIR_COST) * cfg_.n_kv_heads;
                        tiles[n++] = t;
                    });
                r0 += n_new[b];
            }
            at += n * (int)(sizeof(Tile) / 4);
            const long long U = so_far;
            int longest = 0;
            long long pairs = (long long)n * cfg_.n_kv_heads;
            for (int i = 0; i < n; i++) longest = std::max(longest, tiles[i].units);
            const long long share = lanes_[k].blocks ? std::max<long long>(lanes_[k].least, U / lanes_[k].blocks) : 0;
            const bool whole = lanes_[k].join > 0 && pairs <= lanes_[k].blocks && longest <= share + share / 8 + lanes_[k].join;
            const int C = (int)(whole ? pairs : std::min<long long>(lanes_[k].blocks, (U + lanes_[k].least - 1) / std::max(1, lanes_[k].least)));
            step->blocks[k] = C;
            Start* st = reinterpret_cast<Start*>(out + lay_.starts[k]);
            Join* jo = reinterpret_cast<Join*>(out + lay_.joins[k]);
            int tile = 0, joins = 0, known = -1;  // known: the line's place of the last pair in `jo`
            for (int c = 0; c < lanes_[k].blocks; c++) {
                Start s = {};
                if (c < C) {
                    long long lo = U * c / C, hi = U * (c + 1) / C;
                    if (whole) {
                        const Tile& t = tiles[c / cfg_.n_kv_heads];
                        lo = t.line + (long long)(c % cfg_.n_kv_heads) * (t.units + PAIR_COST);
                        hi = lo + t.units + PAIR_COST;
                    }
                    while (lo >= tiles[tile].line + (long long)(tiles[tile].units + PAIR_COST) * cfg_.n_kv_heads) tile++;
                    const int in = (int)(lo - tiles[tile].line), pair = tiles[tile].units + PAIR_COST, skip = std::max(0, PAIR_COST - in % pair);
                    s.tile = tile;
                    s.head = in / pair;
                    s.unit = std::max(0, in % pair - PAIR_COST);
                    s.count = (int)(hi - lo) - skip;  // (none is left where the share ends in front of the pair's first unit)
                    s.t = tiles[tile];
                    s.tiles = tiles_at;
                    s.units = (int)U;
                    s.blocks = C;
                    s.me = c;
                    const int at = tiles[tile].line + s.head * pair;
                    if (s.unit > 0 && at != known) {
                        auto block = [&](long long x) { return (int)(((x + 1) * C - 1) / U); };
                        Join j = {};
                        j.row0 = s.t.row0;
                        j.first = s.t.first;
                        j.rows = s.t.rows;
                        j.head = s.head;
                        j.begin = block(at + PAIR_COST);
                        j.end = block(at + pair - 1);
                        jo[joins++] = j;
                        step->longest[k] = std::max(step->longest[k], j.end - j.begin + 1);
                        known = at;
                    }
                }
                st[c] = s;
            }
            step->joins[k] = out[lay_.count + 1 + k] = joins;
        }
        step->used = at - lay_.dynamic;
        return "";
    }

  private:
    int lane_of(int n_new) const { return (long long)n_new * (cfg_.n_q_heads / cfg_.n_kv_heads) <= now_ ? 0 : 1; }
    // Roughly the us of a step whose sequences of up to `few` rows go to lane 0.
    double cost(int n_seq, const int32_t* pos0, const int32_t* n_new, int group, long long few) const {
        double line[2] = {0, 0};
        for (int b = 0; b < n_seq; b++) {
            if (n_new[b] <= 0 || pos0[b] < 0) continue;
            const long long all = (long long)n_new[b] * group;
            const int k = all <= few ? 0 : 1;
            line[k] += (double)((all + lanes_[k].rows - 1) / lanes_[k].rows) * (((double)pos0[b] + n_new[b]) / lanes_[k].unit + PAIR_COST);
        }
        double us = 0;
        for (int k = 0; k < 2; k++)
            if (line[k] > 0) us += lanes_[k].fixed + lanes_[k].each * line[k] * cfg_.n_kv_heads;
        return us;
    }
    // Roughly the us of lane k's sequences in tiles of its rows, or of its lower height.
    double takes(int k, int lower, int n_seq, const int32_t* pos0, const int32_t* n_new, int group) const {
        const Lane& l = lanes_[k];
        const int height = lower ? l.low : l.rows;
        double line = 0, pairs = 0, longest = 0;
        for (int b = 0; b < n_seq; b++) {
            if (n_new[b] <= 0 || pos0[b] < 0 || lane_of(n_new[b]) != k) continue;
            const int64_t all = (int64_t)n_new[b] * group;
            for (int64_t first = 0; first < all; first += height) {
                const double units = (double)((pos0[b] + (std::min(all, first + height) - 1) / group) / l.unit + 1);
                pairs += 1;
                line += units + PAIR_COST;
                longest = std::max(longest, units);
            }
        }
        if (pairs == 0 || l.blocks == 0) return 0;
        const double share = std::max((double)l.least, line * cfg_.n_kv_heads / l.blocks);
        if (l.join > 0 && pairs * cfg_.n_kv_heads <= l.blocks && longest <= share + share / 8 + l.join) return l.whole_us[lower] + l.unit_us[lower] * longest;
        return l.cut_us[lower] + l.unit_us[lower] * share;
    }
    template <class F>
    void for_tiles(int, int pos0, int n_new, int group, F f) const {
        const int k = lane_of(n_new), all = n_new * group, height = height_[k];
        const Lane& l = lanes_[k];
        for (int first = 0; first < all; first += height) {
            Tile t = {};
            t.pos0 = pos0;
            t.first = first;
            t.rows = std::min(height, all - first);
            const int last = pos0 + (first + t.rows - 1) / group;  // the last position any of its rows sees
            t.units = last / l.unit + 1;
            f(t);
        }
    }
    Config cfg_ = {};
    Lane lanes_[2];
    Layout lay_ = {};
    int few_ = 0, most_ = 0, now_ = 0, mark_ = 0, height_[2] = {0, 0};
    std::vector<int> seen_, tmp_;
};

}  // namespace paged
