// mxh_shared_plan.h — how attention of a batch with common prefixes shares its
// work out: the integers, on the host and on the device.  Plain C++ without HIP.
//
// A run is what is cut into tiles together: the tokens of a group over the rows
// they have in common, or those of a sequence over the rows of its own.  An item
// is some stages of a tile.
#pragma once

#include "mxh_paged_plan.h"

namespace mxh {

// What the host chooses without the lengths: rows of the tiles over prefixes and
// of those over the sequences' own rows, items that the stages are cut into,
// and how many there can be of either kind.
struct SharedShape {
    int rows_p, rows_s, target;
    int64_t items_p, items_s;
};
inline SharedShape shared_shape(const PagedSize& a, int n_groups) {
    SharedShape s;
    const auto rows = [&](int n) { return (int64_t)((a.n_tokens + n - 1) / n) * a.group > 16 ? 64 : 16; };
    s.rows_s = rows(a.n_seq);
    s.rows_p = n_groups > 0 ? std::max(rows(n_groups), s.rows_s) : s.rows_s;
    s.target = most_items(64, a.nkv, a.cus);
    s.items_p = n_groups > 0 ? s.target + a.n_tokens / (s.rows_p / a.group) + n_groups : 0;
    s.items_s = s.target + a.n_tokens / (s.rows_s / a.group) + a.n_seq;
    return s;
}

// A run's tiles and the stages of its longest
struct SharedRun {
    uint32_t tiles, stages;
    // (tiles of a prompt have fewer stages the earlier they are: counted in full)
    MXH_HD uint64_t units() const { return (uint64_t)tiles * stages; }
    // parts that each of its tiles is cut into, `per` stages at most each
    MXH_HD uint32_t parts(uint32_t per) const { return stages > per ? (stages + per - 1) / per : 1; }
};
MXH_HD SharedRun shared_run(uint32_t n, uint32_t keys, int rows, uint32_t tokens) {
    return SharedRun{(n + tokens - 1) / tokens, (keys + (uint32_t)stage_keys(rows) - 1) / (uint32_t)stage_keys(rows)};
}
// stages of an item, so that `units` make no more than target items beside one a tile
MXH_HD uint32_t shared_per(uint64_t units, int target) {
    const uint64_t per = (units + (uint64_t)target - 1) / (uint64_t)target;
    return per < 2 ? 2 : (uint32_t)per;
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
    for (const int rows : {16, 64}) {
        if (runs == 0 || (rows == 64 && (int64_t)a.n_tokens * a.group <= 16)) continue;
        const int64_t items = most_items(64, a.nkv, a.cus) + a.n_tokens / (rows / a.group) + runs;
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
