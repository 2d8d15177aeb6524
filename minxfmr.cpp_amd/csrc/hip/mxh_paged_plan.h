// mxh_paged_plan.h — how attention over the paged cache shares its work out:
// the integers of a batch's tiles, stages and items, on the host and, from the
// lengths that are there, in every workgroup.  Plain C++ without HIP.
//
// A tile is T = R / group consecutive tokens of one sequence with the q heads of
// one kv head, R = 16 or 64 rows; a stage is 128 or 64 keys (mxh_paged_attn.hip).
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define MXH_HD __host__ __device__ __forceinline__
#else
#define MXH_HD inline
#endif

namespace mxh {

constexpr int kTreeMax = 64;        // new tokens of a drafted tree (one lane, one mask bit each)
constexpr int kPagedSeqMax = 4096;  // sequences of a batch

// keys of a stage: 32 for every group of waves that share them
constexpr int stage_keys(int rows) { return rows == 64 ? 64 : 128; }
// a tile's cost beside its stages, in stages (64 rows: 3 to 6 are within 5% of one
// another; without it items that cross tiles end late)
constexpr int tile_lead(int rows) { return rows == 16 ? 2 : 4; }

// whether `target` items of a batch of `all` units finish before its whole tiles
// do, the longest of `longest` units (PagedLine)
constexpr bool cut_pays(int rows, float longest, float all, float target) {
    return rows == 64 ? longest * target > 13.f * target + 1.8f * all || longest * target > 7.5f * target + 3.6f * all
                      : longest > 12.f || 2.f * longest * target > all;
}

// A sequence as the plan sees it
struct PagedSeq {
    uint32_t first, n, cached;  // first token row, new tokens, rows before them
    uint32_t tiles, stages;     // stages of its last tile
};

// A tile's stages [st0, st1) that an item takes, `len` units of the line with
// what they hold of its lead
struct PagedPiece {
    uint32_t tile, st0, st1, len;
    int slot;  // of the part in the workspace; -1: the whole tile
};

// The batch as a line of units, cut into items.  Where tiles are cut, the units
// are the stages of all tiles, sequence by sequence, `lead` units before each
// tile's; elsewhere the tiles themselves.  The lead is what a tile costs beside
// its stages (its q, the merge of the waves), so an item that goes on into
// another tile does as many stages less.
//
// A prompt's earlier tiles have fewer stages.  `block` tiles have at most the
// tokens of one stage, so those of block b need no more stages than the cached
// rows and b + 1; the line gives them that many, and all of the sequence's to
// the tiles from the block on where this reaches them (ramp).
//
// Cut or not: with M units the longest tile and U all of them, in us of a head
// group of 128 dims on 256 CUs:
//   R = 64: whole tiles take 4 + 1.07 M while they are few, `target` items of
//   the cut ones (two resident a CU) 18 + 1.95 U / target, half as many 12 + 3.8
//   U / target.  A prompt of 256 at 4,096 cached rows 82 whole, 54 cut; of 1,024
//   150 and 168; of 8 at 500 15.7 and 12.8; 16 drafted trees of up to 33 tokens
//   at up to 8,000 rows 151 and 80, 20 of up to 60 at up to 1,000 33 and 38.
//   Half the items where they would have less than 8 units: a prompt of 64 at
//   4,096 28.5 and 25.2.
//   R = 16: cut unless all tiles are short and there are many: 200 single tokens
//   at up to 300 rows 29 whole, 43 cut, at up to 1,000 83 and 89, at up to 6,000
//   437 and 406; 64 at up to 2,000 61 and 53.
//   (Shorter ones beside the longest: 64 at up to 2,000 40 and 45.)
// Heads of 64 and 32 go by the same numbers, which suit them less where the times
// are short.  Whole and cut, 32/8 heads of 64; 32/8 of 32; 8/1 of 32:
//   whole: a prompt of 1,024 21 and 35; 18 and 27.  200 single tokens at up to 300
//   21 and 35; 17 and 33; and at up to 1,000 34 and 51; 31 and 43 (45 and 34 with
//   the second kernel that the table's width asks for)
//   cut: a prompt of 256 at 4,096 59 and 36; 52 and 32; 52 and 19.  16 trees of up
//   to 33 at up to 8,000 105 and 41; 93 and 36; 93 and 20, 20 of up to 60 at up to
//   1,000 23 and 26; 20 and 22; 18 and 15.  Single tokens: 200 at up to 6,000 229
//   and 172; 170 and 159; 36 and 27, 64 at up to 2,000 23 and 27; 22 and 25; 15 and
//   11, 200 at up to 300 with 8/1 heads of 32 8.5 and 12, one at 8,192 53 and 11; 47
//   and 11; 46 and 11.
struct PagedLine {
    uint32_t t, key_shift, lead, block;  // tokens of a tile; a stage has 1 << key_shift keys
    float inv_t;
    bool tree, cut;
    uint32_t total, per, items;  // units of the batch (they fit 31 bits: paged_shape), of an item; items
    uint32_t all;                // stages and leads of the batch (0: not counted, target == 0)

    MXH_HD PagedLine(int rows, uint32_t tokens, bool drafted, int target)
        : t(tokens), key_shift(rows == 16 ? 7 : 6), lead((uint32_t)tile_lead(rows)), inv_t(1.0f / (float)t),
          tree(drafted), cut(target > 0), total(0), per(1), items(0), all(0) {
        block = (uint32_t)(((float)stage_keys(rows) + 0.5f) * inv_t);
    }
    // The sequence with tokens first .. end - 1 of n_tokens and `cached` rows, as the
    // arrays have them.  Rows past the table's do not exist, so no tile has stages there
    MXH_HD PagedSeq seq(int first, int end, int cached, int n_tokens, uint64_t table_rows) const {
        PagedSeq q;
        end = end < n_tokens ? end : n_tokens;
        q.first = (uint32_t)first;
        q.n = first >= 0 && end > first ? (uint32_t)(end - first) : 0;
        if (tree) q.n = q.n < kTreeMax ? q.n : kTreeMax;
        q.cached = (uint32_t)(cached < 0 ? 0 : cached < 1 << 30 ? cached : 1 << 30);
        // (n up to 2^20: the quotient is off by less than 2^-3 / t, and n + t - 1/2 is
        // at least half a token from a multiple of t)
        q.tiles = (uint32_t)(((float)(q.n + t) - 0.5f) * inv_t);
        const uint64_t own = q.cached + q.n;
        const uint32_t rows = (uint32_t)(own < table_rows ? own : table_rows);
        q.stages = (rows + (1u << key_shift) - 1) >> key_shift;
        return q;
    }
    MXH_HD uint32_t cached_stages(const PagedSeq& q) const { return (q.cached + (1u << key_shift) - 1) >> key_shift; }
    // blocks of tiles with fewer stages than the sequence
    MXH_HD uint32_t ramp(const PagedSeq& q) const {
        const int r = (int)q.stages - (int)cached_stages(q) - 1;  // (below the blocks that q.n fills)
        return tree || r < 0 ? 0 : (uint32_t)r;
    }
    // units of the first b <= ramp blocks
    MXH_HD uint32_t before(const PagedSeq& q, uint32_t b) const {
        return block * (b * (lead + cached_stages(q) + 1) + b * (b - 1) / 2);
    }
    MXH_HD uint32_t units(const PagedSeq& q) const {
        if (!cut) return q.tiles;
        const uint32_t r = ramp(q);  // (block b < r has r - b stages less)
        return q.tiles * (lead + q.stages) - (r > 0 ? block * (r * (r + 1) / 2) : 0);
    }
    // The items of a line that tiles may be cut on: `units` stages and leads, the
    // longest tile's `longest`
    MXH_HD void settle_cut(uint32_t units, bool pays, int rows, int target) {
        all = total = units;
        cut = pays;
        items = (uint32_t)(rows == 64 && (int64_t)units < 8 * (int64_t)target ? target / 2 : target);
        per = cut ? (units + items - 1) / items : 1;
    }
    // ... and of one of whole tiles
    MXH_HD void settle_whole(uint32_t tiles) { total = items = tiles; }
    // Item i's first unit, at or past the total where there is no such item.  The
    // grid has workgroups for as many whole tiles as there can be: where tiles are
    // cut, i times per passes 32 bits long before the last of them
    MXH_HD uint32_t first_unit(uint32_t i) const { return i < items ? i * per : total; }

    // unit x of a sequence: its tile, the units of the tile and those before x
    struct Spot {
        uint32_t tile, units, at;
    };
    MXH_HD Spot spot(const PagedSeq& q, uint32_t x) const {
        if (!cut) return Spot{x, 1, 0};
        const uint32_t r = ramp(q);
        uint32_t b = r, len = lead + q.stages, done = r > 0 ? before(q, r) : 0;
        if (x < done) {
            // the root of before(b) = x, put right by whole blocks
            const float c = (float)(lead + cached_stages(q)) + 0.5f;
            const float root = sqrtf(c * c + 2.0f * (float)x / (float)block) - c;
            b = (uint32_t)(root > 0.f ? root : 0.f);
            b = b < r - 1 ? b : r - 1;
            while (b > 0 && before(q, b) > x) --b;
            while (b + 1 < r && before(q, b + 1) <= x) ++b;
            len = lead + cached_stages(q) + 1 + b, done = before(q, b);
        }
        const uint32_t i = (x - done) / len;
        return Spot{b * block + i, len, x - done - i * len};
    }
    // what item i, with `left` units to go, takes of the tile there
    MXH_HD PagedPiece piece(const PagedSeq& q, const Spot& at, uint32_t left, uint32_t i) const {
        PagedPiece p;
        const uint32_t rest = at.units - at.at, end = at.at + (rest < left ? rest : left);
        p.len = end - at.at;
        p.tile = cut ? at.tile : q.tiles - 1 - at.tile;  // (the most keys first)
        p.st0 = !cut || at.at < lead ? 0 : at.at - lead;
        p.st1 = !cut ? q.stages : end < lead ? 0 : end - lead;
        p.slot = !cut || (p.st0 == 0 && end == at.units) ? -1 : (int)(2 * i + (p.st0 == 0));
        return p;
    }
    // Parts of the tile that is cut for the first time where an item starts there, 0
    // where none is: no stage comes before the lead's end, and a tile's first cut is
    // not a whole item after it
    MXH_HD uint32_t parts(const Spot& at) const {
        const bool first = cut && at.at > lead && at.at <= lead + per;
        return first ? 1 + (at.units - at.at + per - 1) / per : 0;
    }
    // slot of the z-th part of the tile that is cut first where item i starts
    static MXH_HD uint32_t part_slot(uint32_t i, uint32_t z) { return z ? 2 * (i - 1 + z) : 2 * (i - 1) + 1; }
};

// What the host chooses without the lengths: rows of a tile, by the average
// sequence, and how many items there can be; whether tiles are cut the plan
// decides.  16-row tiles re-read the keys where a sequence has several of them,
// 64-row ones leave rows empty: 16 sequences of 2 tokens (8 rows) at up to 4,000
// keys took 25 us with 16 and 31 with 64, of up to 12 tokens 36 and 32; one of 4
// tokens at 8,192 16 and 20, of 27 28 and 24, at 40,000 173 and 69.
// One height for all, so the average costs where sequences differ: 200 single tokens
// at up to 2,000 rows and a prompt of 2,000 226 us (119 and 91 apart), of 500 155
// (119 and 18); a tree of 27 at 40,000 beside 20 single tokens 168 (68 and 16).
// Empty sequences count: that tree in a batch of 16 whose others are empty 167, at
// 8,192 30 (25 by itself).
struct PagedShape {
    int rows, target;  // target: items that stages are cut into, at most; 0: an item is a tile
    int64_t items;     // at most
};
// a launch: sequences and tokens, rows of its table, kv heads, q heads of one, CUs
struct PagedSize {
    int n_seq, n_tokens;
    int64_t table_rows;
    int nkv, group, cus;
};
// items of R-row tiles; stages of a tile, at most
inline int most_items(int rows, int nkv, int cus) { return (rows == 64 ? 2 : 1) * std::max(2, cus / nkv); }
inline int64_t most_stages(int64_t table_rows, int rows) {
    return (table_rows + stage_keys(rows) - 1) / stage_keys(rows);
}
// whether some lengths could make cut tiles worth the second kernel's 4 us: the
// longest tile that the table allows, and `tiles` of one stage
inline bool cut_may_pay(const PagedSize& a, int rows, int64_t tiles) {
    const int64_t stages = most_stages(a.table_rows, rows);
    return stages > 1 && cut_pays(rows, (float)(stages + tile_lead(rows)), (float)(1 + tile_lead(rows)) * (float)tiles,
                                  (float)most_items(rows, a.nkv, a.cus));
}
inline PagedShape paged_shape(const PagedSize& a) {
    PagedShape s;
    s.rows = (int64_t)((a.n_tokens + a.n_seq - 1) / a.n_seq) * a.group > 16 ? 64 : 16;
    const int64_t tiles = a.n_tokens / (s.rows / a.group) + a.n_seq;
    const int64_t tiles_min = std::max(a.n_tokens / (s.rows / a.group), std::min(a.n_seq, a.n_tokens));  // (none empty)
    const bool fits = tiles * (most_stages(a.table_rows, s.rows) + tile_lead(s.rows)) < INT32_MAX;  // (the line's units)
    s.target = fits && cut_may_pay(a, s.rows, tiles_min) ? most_items(s.rows, a.nkv, a.cus) : 0;
    s.items = std::max((int64_t)s.target, tiles);
    return s;
}
// the workspace: two parts an item, word of the cut tiles
inline size_t paged_work_bytes(int rows, int target, int nkv, int hd) {
    return (size_t)2 * target * nkv * rows * (hd + 2) * sizeof(float) + (size_t)target * 16;
}
// ... of any batch up to this n_seq, n_tokens and table_rows
inline size_t paged_work_bound(const PagedSize& a, int hd) {
    size_t most = 0;
    for (const int rows : {16, 64})
        if ((rows == 16 || (int64_t)a.n_tokens * a.group > 16) && cut_may_pay(a, rows, 1))
            most = std::max(most, paged_work_bytes(rows, most_items(rows, a.nkv, a.cus), a.nkv, hd));
    return most;
}

}  // namespace mxh
