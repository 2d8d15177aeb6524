// mxh_shared_plan.h — how attention of a batch with common prefixes shares its
// work out: the integers, on the host and on the device.  Plain C++ without HIP.
//
// A run is what is cut into tiles together: the tokens of a group over the rows
// they have in common, or those of a sequence over the rows of its own.  An item
// is some stages of a tile.
#pragma once

#include "mxh_paged_plan.h"

namespace mxh {

// Whether prefixes are read apart, from what the host knows: as long as the table
// allows, the batch's K and V rows, and the rows of q that a sequence has on average.
// Read with the sequences' own rows, a prefix comes out of the caches for all but the
// first of them; read apart, it takes a plan, a third kernel and 10 us more.
// Apart and not, us, 32/8 heads of 128 (4 KB of K and V a row):
//   single tokens: 4 at 1,200 rows 17 and 11, 8 at 4,500 25 and 21, 12 at 2,200 21.3
//   and 19.5, 6 at 8,200 25.7 and 25.1 (200 MB), 32 at 1,200 22.3 and 22.8 (160 MB), 24
//   at 2,200 23 and 25 (220 MB), 16 at 4,500 26 and 31, 64 at 8,200 (2 GB) and of their
//   own up to 1,000 60 and 158
//   up to 4 tokens each (12 rows of q): 12 at 6,300 30 and 34, 30 45 and 65
//   More rows of q are not read apart, where it takes from a quarter less time to a
//   third more, by how the tiles happen to fill.  Up to 16 (39 rows): 12 at 6,300 49 and
//   53, 30 100 and 102; up to 33 (81): 80 and 84, 181 and 178; up to 64 (152): 116 and
//   153, 302 and 293, 12 at 16,300 257 and 294; up to 90 (204): 176 and 169, 328 and 364;
//   up to 128: 208 and 200, 503 and 527, but 30 at 1,300 (170 MB) 166 and 125
// 16/8 heads of 128: 12 of up to 16 (20 rows of q) at 6,300 36 and 47, 30 71 and 96; 16
// drafted trees of up to 13 at 3,200 (210 MB) 29 and 35, at 16,300 57 and 135, of up to
// 33 (39 rows, not read apart) 124 and 157.
// Heads of 64, 6/2 (512 bytes a row): 64 single tokens at 9,000 (300 MB) 27 and 39, at
// 4,500 (150) 23 and 24, 16 at 16,500 (135) 32 and 24; 16 trees of up to 13 at 3,200
// (26) 21 and 17, at 16,300 (134) 29 and 33.  Of 32, 8/1 (128 bytes): 64 at 31,000 (250
// MB) 31 and 51, at 17,000 (140) 27 and 32, at 9,000 (74) 23 and 21.
constexpr int kSharedRows = 32;         // rows of q of a sequence, on average, at most
constexpr double kSharedBytes = 180e6;  // of K and V at least
inline bool shared_pays(const PagedSize& a, int hd, int n_groups) {
    return n_groups > 0 && (int64_t)a.n_tokens * a.group <= (int64_t)kSharedRows * a.n_seq &&
           (double)a.n_seq * (double)a.table_rows * a.nkv * hd * 4 >= kSharedBytes;
}
// tokens of a batch with prefixes read apart, at most, of those up to a's size
inline int shared_tokens(const PagedSize& a) {
    return (int)std::min<int64_t>(a.n_tokens, (int64_t)kSharedRows * a.n_seq / a.group);
}

// What the host chooses without the lengths: rows of the tiles over prefixes and
// of those over the sequences' own rows, items that the stages of either kind are cut
// into, and how many there can be.  Items over prefixes are one a CU, first: two on a
// CU take nearly twice as long, and the sequences' own rows, which wait for memory,
// fit beside one.  64 single tokens behind 8,000 rows, up to 1,000 of their own (32/8
// heads of 128): one a CU 45 us, 5 for 4 CUs 54, 12 for 4 59; own rows first 60, the
// two in turn 55; either by itself 31.
struct SharedShape {
    int rows_p, rows_s, target_p, target_s;
    int64_t items_p, items_s;
};
inline SharedShape shared_shape(const PagedSize& a, int n_groups) {
    SharedShape s;
    const auto rows = [&](int n) { return (int64_t)((a.n_tokens + n - 1) / n) * a.group > 16 ? 64 : 16; };
    s.rows_s = rows(a.n_seq);
    s.rows_p = n_groups > 0 ? std::max(rows(n_groups), s.rows_s) : s.rows_s;
    s.target_p = most_items(16, a.nkv, a.cus);
    s.target_s = most_items(64, a.nkv, a.cus);
    s.items_p = n_groups > 0 ? s.target_p + a.n_tokens / (s.rows_p / a.group) + n_groups : 0;
    s.items_s = s.target_s + a.n_tokens / (s.rows_s / a.group) + a.n_seq;
    return s;
}

// A run's tiles and the stages of its longest
struct SharedRun {
    uint32_t tiles, stages;
    // (tiles of a prompt have fewer stages the earlier they are: counted in full)
    MXH_HD uint64_t units() const { return (uint64_t)tiles * stages; }
    // Parts that each of its tiles is cut into, of at most `per` stages: as many equal
    // ones as that takes
    MXH_HD uint32_t length(uint32_t per) const {  // of a part
        if (stages <= per) return stages;
        const uint32_t n = (stages + per - 1) / per;
        return (stages + n - 1) / n;
    }
    MXH_HD uint32_t parts(uint32_t per) const {
        if (stages <= per) return 1;
        const uint32_t len = length(per);
        return (stages + len - 1) / len;
    }
};
MXH_HD SharedRun shared_run(uint32_t n, uint32_t keys, int rows, uint32_t tokens) {
    return SharedRun{(n + tokens - 1) / tokens, (keys + (uint32_t)stage_keys(rows) - 1) / (uint32_t)stage_keys(rows)};
}
// stages of an item, so that `units` make no more than target items beside one a tile
MXH_HD uint32_t shared_per(uint64_t units, int target) {
    const double per = ceil((double)units / (double)target);  // (units fit 53 bits; a 64-bit division is slow)
    return per < 2. ? 2 : (uint32_t)per;
}

// One item: tile `tile` of the run's, stages [st0, st1) over the rows of sequence s
struct alignas(16) SharedItem {
    int s, first, n, cached;       // tokens of the run; cached rows (a prefix: its rows)
    int tile, st0, st1, begin;     // begin: first row (a sequence's own rows)
    int slot, slot0, stride, parts;  // the part's; of the tile's parts 0, 1, ...: slot0, slot0 + stride, ...
};

// The parts' floats of `items` tiles of `rows` rows, at most of any batch up to a's
// sizes with `runs` runs; and those items
struct SharedBound {
    int64_t items = 0, rows = 0;
};
inline SharedBound shared_bound(const PagedSize& a, int runs) {
    SharedBound b;
    const int tokens = shared_tokens(a);
    for (const int rows : {16, 64}) {
        if (runs == 0 || (rows == 64 && (int64_t)tokens * a.group <= 16)) continue;
        const int64_t items = most_items(64, a.nkv, a.cus) + tokens / (rows / a.group) + runs;
        b.items = std::max(b.items, items), b.rows = std::max(b.rows, items * rows);
    }
    return b;
}

// The workspace: items, of every token two records (where the parts of its prefix
// and of its own rows are), and the parts of both kinds
struct SharedWork {
    size_t items, records, part_p, part_s, ml_p, ml_s, bytes;
};
inline SharedWork shared_work(const SharedBound& p, const SharedBound& s, int n_tokens, int nkv, int hd) {
    SharedWork w;
    size_t at = 16;  // the number of items of each kind
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 15) / 16 * 16;
        return here;
    };
    w.items = take((size_t)(p.items + s.items) * sizeof(SharedItem));
    w.records = take((size_t)n_tokens * 32);
    w.part_p = take((size_t)p.rows * nkv * hd * 4);
    w.part_s = take((size_t)s.rows * nkv * hd * 4);
    w.ml_p = take((size_t)p.rows * nkv * 8);
    w.ml_s = take((size_t)s.rows * nkv * 8);
    w.bytes = at;
    return w;
}
// ... of this batch
inline SharedWork shared_work(const SharedShape& s, int n_tokens, int nkv, int hd) {
    return shared_work(SharedBound{s.items_p, s.items_p * s.rows_p}, SharedBound{s.items_s, s.items_s * s.rows_s},
                       n_tokens, nkv, hd);
}

}  // namespace mxh
