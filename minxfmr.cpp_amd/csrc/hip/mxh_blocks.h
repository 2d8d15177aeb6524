// mxh_blocks.h — how the operators over blocks of the paged cache share their
// work out: the integers, on the host.  Plain C++ without HIP.
//
// A block is block_rows rows of a sequence that lie in one page; block b of a
// sequence holds its rows [b block_rows, (b + 1) block_rows).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace mxh {

constexpr int kSelectMax = 1024;      // blocks that a token attends
constexpr int kBlocksMax = 1 << 18;   // blocks of a sequence: a bit each of a token's in LDS
constexpr int kListMax = 1024;        // blocks of a tile's list in LDS
constexpr int kBitBytes = 32768;      // bits of a tile's tokens

struct BlockSize {
    int n_seq, n_tokens;
    int64_t n_blocks;  // of a row of the table
    int nkv, group, n_select, block_rows, cus;
};

// Stages of 128 keys that a token's list has, at most
inline int64_t block_stages(const BlockSize& a) {
    return (std::min<int64_t>(a.n_select, a.n_blocks) * a.block_rows + 127) / 128;
}
// Tokens that share a tile, and its rows.  Tokens of one sequence attend many of the
// same blocks, whose rows are then loaded once for all of them; single tokens of
// sequences (up to two each on average) share nothing and go by themselves, and so do
// all where that makes little work, 46 stages a CU with four for a token's start: in a
// tile they wait for the union of their lists, and for one another's sequences.  All
// by themselves and in tiles, us (32/8 heads of 128; work): 40 tokens of two sequences,
// a stage each 9 and 18 (6); of one sequence 30 of 16 24 and 29 (19), 60 of 16 31 and
// 35 (38), 100 of 16 58 and 45 (63), 120 of 4 27 and 28 (30), 200 of 3.5 46 and 31 (47),
// 8 of 100 38 and 39 (26); of 16 sequences up to 8 each of 16 56 and 65 (45), of 4 up to 30
// 32 and 43 (45).
inline bool block_alone(const BlockSize& a) {
    return a.n_tokens <= 2 * (int64_t)a.n_seq ||
           (int64_t)a.n_tokens * a.nkv * (block_stages(a) + 4) <= 46 * (int64_t)a.cus;
}
// 32 rows where sequences have tokens enough and lists and bits leave room for them: 512
// tokens with 32 of 469 blocks of 64 rows each, of which four tokens together have
// some 63 and eight some 82 (32/8 heads of 128), 114 us, in tiles of 16 rows 126; 100 of
// them 45 and 43, 200 tokens with 7 blocks 31 and 21.
inline int block_tokens_of(const BlockSize& a, int rows) {
    const int64_t words = (a.n_blocks + 31) / 32;
    return (int)std::max<int64_t>(
        1, std::min<int64_t>({rows / a.group, 16, kListMax / a.n_select, kBitBytes / (4 * words)}));
}
inline int block_rows_of_tile(const BlockSize& a) {
    return !block_alone(a) && a.n_tokens > 8 * (int64_t)a.n_seq && block_tokens_of(a, 32) * a.group > 16 ? 32 : 16;
}
inline int block_tokens(const BlockSize& a) {
    return block_alone(a) ? 1 : block_tokens_of(a, block_rows_of_tile(a));
}
inline int64_t block_tiles(const BlockSize& a) {
    const int t = block_tokens(a);
    return (a.n_tokens + t - 1) / t;
}
// Workgroups that share a tile's list, for two a CU: of one token with 2,048 rows for
// each of 8 kv heads of 128 a stage of 128 keys each, 16 workgroups, 9.4 us, 8 11.2, 4
// 13.3 (and 3.9 for joining their parts).  (48 tokens with 1,280, a workgroup each 53
// us, two each 55 and 5)
inline int block_splits(const BlockSize& a) {
    const int64_t items = block_tiles(a) * a.nkv;
    return (int)std::max<int64_t>(1, std::min<int64_t>({2 * (int64_t)a.cus / items, block_stages(a), 64}));
}
// the workspace: parts of the tiles that are split
inline size_t block_part_bytes(int64_t parts, int rows, int nkv, int hd) {
    return (size_t)parts * nkv * rows * (hd + 2) * sizeof(float);
}
inline size_t block_work_bytes(const BlockSize& a, int hd) {
    const int s = block_splits(a);
    return s > 1 ? block_part_bytes(block_tiles(a) * s, block_rows_of_tile(a), a.nkv, hd) : 0;
}
// ... of any batch (splits > 1: splits x items are at most two a CU)
inline size_t block_work_bound(const BlockSize& a, int hd) {
    const int64_t stages = ((int64_t)a.n_select * a.block_rows + 127) / 128;
    return stages < 2 ? 0 : block_part_bytes(std::max<int64_t>(2, 2 * (int64_t)a.cus / a.nkv), 32, a.nkv, hd);
}

// Selecting: scores of a token and kv head (whole tiles of 16 blocks), and tokens whose
// scores the workspace holds at a time
constexpr int64_t kSelectBytes = 256 << 20;
inline int64_t select_row(int64_t n_blocks) { return (n_blocks + 15) / 16 * 16; }
inline int64_t select_tokens(int n_tokens, int64_t n_blocks, int nkv) {
    const int64_t row = select_row(n_blocks) * nkv * 8;
    return std::min<int64_t>(n_tokens, std::max<int64_t>(16, kSelectBytes / row / 16 * 16));
}
inline size_t select_work_bytes(int n_tokens, int64_t n_blocks, int nkv) {
    return (size_t)select_tokens(n_tokens, n_blocks, nkv) * (size_t)(select_row(n_blocks) * nkv) * 8;
}
// ... of any batch up to this n_tokens and n_blocks: tokens come in sixteens, so rows a
// little shorter may fill more of the 256 MB
inline size_t select_work_bound(int n_tokens, int64_t n_blocks, int nkv) {
    const int64_t row = select_row(n_blocks) * nkv * 8;
    return (size_t)std::min<int64_t>(n_tokens * row, std::max<int64_t>(kSelectBytes, 16 * row));
}

}  // namespace mxh
