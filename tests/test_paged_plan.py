"""How attention over the paged cache shares its work out (mxh_paged_plan.h), on the CPU.

The line of units, the items, the pieces of tiles, their slots in the workspace
and the word that the second kernel gets of cut tiles are walked as the
workgroups walk them: every stage of every tile is taken exactly once, every
part lies in the workspace, and the parts that the second kernel would join are
those that were left.  At the documented limits too (4,096 sequences, the widest
tables, 2^20 tokens), where products of indexes pass 32 bits.
"""
from __future__ import annotations

import ctypes as C
import random
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

HDR = Path(__file__).resolve().parent.parent / "minxfmr.cpp_amd" / "csrc" / "hip"
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
SRC = """
#include <vector>
#include "mxh_paged_plan.h"
using namespace mxh;

#define REQUIRE(x) do { if (!(x)) return __LINE__; } while (0)

// what happened: rows of a tile, target, cut, items with work, total
extern "C" int walk(int n_seq, int n_tokens, const int* start, const int* cached, int tree, int64_t table_rows, int nkv,
                    int group, int cus, int64_t* out) {
    const PagedShape sh = paged_shape(PagedSize{n_seq, n_tokens, table_rows, nkv, group, cus});
    const uint32_t T = (uint32_t)(sh.rows / group);
    PagedLine line(sh.rows, T, tree, sh.target);
    std::vector<PagedSeq> seqs;
    uint64_t units = 0, tiles = 0;
    uint32_t longest = 0;
    for (int s = 0; s < n_seq; ++s) {
        const PagedSeq q = line.seq(start[s], start[s + 1], cached[s], n_tokens, (uint64_t)table_rows);
        seqs.push_back(q);
        REQUIRE(q.tiles == (q.n + T - 1) / T);
        tiles += q.tiles;
        if (line.cut && q.tiles > 0) units += line.units(q), longest = std::max(longest, line.lead + q.stages);
    }
    REQUIRE(tiles <= (uint64_t)sh.items && units < 1ull << 31);
    if (line.cut)
        line.settle_cut((uint32_t)units, cut_pays(sh.rows, (float)longest, (float)units, (float)sh.target), sh.rows,
                        sh.target);
    if (!line.cut) line.settle_whole((uint32_t)tiles);
    out[0] = sh.rows, out[1] = sh.target, out[2] = line.cut, out[3] = 0, out[4] = line.total;
    REQUIRE(line.cut || line.total == tiles);

    struct Cut { uint32_t first, rows, parts; };
    struct Part { int s; uint32_t tile, st0, st1; };
    std::vector<Cut> cuts((size_t)sh.target, Cut{0, 0, 0});
    std::vector<Part> slots((size_t)2 * sh.target, Part{-1, 0, 0, 0});
    // every workgroup of the grid (kv heads, y, z)
    const uint32_t grid_y = (uint32_t)std::min<int64_t>(sh.items, 32768);
    const uint64_t grid = (uint64_t)grid_y * ((sh.items + grid_y - 1) / grid_y);
    uint64_t next = 0;  // the first unit that no item has taken yet
    size_t s = 0;
    uint32_t r_unit = 0, tile_now = 0, taken = 0;  // of the sequence; the tile that is open, its stages taken
    for (uint64_t i = 0; i < grid; ++i) {
        uint32_t x = line.first_unit((uint32_t)i);
        if (x >= line.total) continue;
        ++out[3];
        REQUIRE(x == next);
        REQUIRE(!line.cut || i < (uint64_t)sh.target);
        const uint32_t x1 = std::min(x + line.per, line.total);
        next = x1;
        for (bool first = true; x < x1; first = false) {
            while (r_unit >= line.units(seqs[s])) {
                r_unit = 0, tile_now = 0;
                REQUIRE(++s < seqs.size());
            }
            const PagedSeq& q = seqs[s];
            const PagedLine::Spot at = line.spot(q, r_unit);
            const PagedPiece p = line.piece(q, at, x1 - x, (uint32_t)i);
            REQUIRE(p.len > 0 && at.at < at.units && p.tile < q.tiles);
            const uint32_t all = line.cut ? at.units - line.lead : q.stages;  // of the tile
            if (at.at == 0) {
                REQUIRE(at.tile == tile_now);
                taken = 0;
            }
            // the stages that its tokens can attend are all there
            const uint64_t keys = std::min<uint64_t>(q.cached + (tree ? q.n : std::min((p.tile + 1) * T, q.n)), table_rows);
            REQUIRE((uint64_t)all << line.key_shift >= keys && all <= q.stages);
            REQUIRE(p.st0 == taken && p.st1 >= p.st0 && p.st1 <= all);
            taken = p.st1;
            if (at.at + p.len == at.units) {
                REQUIRE(taken == all);
                ++tile_now;
            }
            if (p.slot < 0) {
                REQUIRE(p.st0 == 0 && p.st1 == all);
            } else if (p.st0 < p.st1) {
                REQUIRE(line.cut && p.slot < 2 * sh.target && slots[p.slot].s < 0);
                slots[p.slot] = Part{(int)s, p.tile, p.st0, p.st1};
            }
            if (first && i < (uint64_t)sh.target)
                cuts[i] = Cut{q.first + at.tile * T, std::min(T, q.n - at.tile * T) * (uint32_t)group, line.parts(at)};
            x += p.len, r_unit += p.len;
        }
    }
    REQUIRE(next == line.total);
    // what the second kernel joins is what was left, in order, and all of it
    uint64_t left = 0, joined = 0;
    for (const Part& p : slots) left += p.s >= 0;
    for (int i = 1; i < sh.target; ++i)
        for (uint32_t z = 0, st = 0; z < cuts[i].parts; ++z, ++joined) {
            const uint32_t at = PagedLine::part_slot((uint32_t)i, z);
            REQUIRE(at < slots.size() && slots[at].s >= 0);
            const Part& p = slots[at];
            REQUIRE(p.st0 == st && seqs[p.s].first + p.tile * T == cuts[i].first);
            REQUIRE(cuts[i].rows == std::min(T, seqs[p.s].n - p.tile * T) * (uint32_t)group);
            st = p.st1;
        }
    REQUIRE(left == joined);
    // the workspace holds them, and one for the largest batch does
    const size_t need = paged_work_bytes(sh.rows, sh.target, nkv, 64);
    REQUIRE(need <= paged_work_bound(PagedSize{n_seq, n_tokens, table_rows, nkv, group, cus}, 64));
    return 0;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_plan")
    (d / "plan.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{HDR}", str(d / "plan.cpp"), "-o",
                    str(d / "plan.so")], check=True)
    return C.CDLL(str(d / "plan.so"))


def walk(lib, seqs, *, nkv, group, tree=False, table_rows=None, cus=256, lead=0, tail=0):
    """The walk over sequences (cached rows, new tokens); returns rows of a tile, target, cut, items, total."""
    cached = np.asarray([c for c, _ in seqs], np.int32)
    start = np.concatenate([[lead], lead + np.cumsum([n for _, n in seqs])]).astype(np.int32)
    if table_rows is None:
        table_rows = -(-max(c + n for c, n in seqs) // 16) * 16
    out = (C.c_int64 * 5)()
    line = lib.walk(len(seqs), int(start[-1]) + tail, C.c_void_p(start.ctypes.data), C.c_void_p(cached.ctypes.data), int(tree),
                    C.c_int64(max(table_rows, 16)), nkv, group, cus, out)
    text = SRC.splitlines()[line - 1].strip() if line else ""
    assert line == 0, f"line {line}: {text} {list(out)}"
    return tuple(out)


# 4,096 sequences under the widest tables: (cached rows, new tokens, kv heads, heads of one)
WIDE = {
    "2-tokens-64/8-heads": (524288, 2, 8, 8),
    "forks-32/8-heads": (1 << 20, 1, 8, 4),
    "40/40-heads": (185344, 1, 40, 1),
    "64/64-heads": (131072, 1, 64, 1),
    "128/128-heads": (61440, 1, 128, 1),
    "1024/1024-heads": (62000, 1, 1024, 1),
}


@pytest.mark.parametrize("name", list(WIDE))
def test_no_item_beyond_the_workspace_has_work(lib, name):
    """Many workgroups and long items: an index times an item's units passes 32 bits."""
    cached, new, nkv, group = WIDE[name]
    rows, target, cut, items, total = walk(lib, [(cached, new)] * 4096, nkv=nkv, group=group)
    assert cut and items <= target
    tiles = 4096 * new // (rows // group) + 4096  # (workgroups of a kv head)
    assert (tiles - 1) * -(-total // target) >= 2**32


@pytest.mark.parametrize("seqs,nkv,group,tree", [
    ([(0, 1 << 20)], 8, 4, False),
    ([(1 << 20, 1 << 20)], 1, 8, False),
    ([(0, 256)] * 4096, 8, 4, False),
    ([(300000, 64)] * 4096, 2, 8, True),
    ([(1 << 30, 1)] * 3, 8, 4, False),
    ([(1 << 30, 64)] + [(0, 0)] * 4095, 1, 1, True),
    ([(0, 0)] * 4095 + [((1 << 30) - 1, 3)], 16, 2, False),
])
def test_the_largest_batches(lib, seqs, nkv, group, tree):
    walk(lib, seqs, nkv=nkv, group=group, tree=tree)
    walk(lib, seqs, nkv=nkv, group=group, tree=tree, table_rows=16 * 70)


@pytest.mark.parametrize("cus", [32, 256])
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
def test_every_stage_is_taken_once(lib, tree, cus):
    rng = random.Random(7 + tree)
    seen = set()
    for _ in range(1500):
        n_seq = rng.choice([1, 1, 2, 5, 40, 70, 300])
        most = rng.choice([1, 1, 5, 40, 64 if tree else 900])
        deep = rng.choice([0, 20, 300, 5000, 90000])
        seqs = [(rng.randint(0, deep), rng.randint(0, most)) for _ in range(n_seq)] + [(deep, most)]
        rows = rng.choice([None, None, 16, 1024, 1 << 20])
        r = walk(lib, seqs, nkv=rng.choice([1, 2, 8, 16, 200]), group=rng.randint(1, 8), tree=tree, table_rows=rows, cus=cus,
                 lead=rng.randint(0, 9), tail=rng.randint(0, 3))
        seen.add((r[0], r[1] > 0, r[2]))
    assert {(16, True, 1), (64, True, 1), (64, True, 0), (16, False, 0), (64, False, 0)} <= seen, seen
