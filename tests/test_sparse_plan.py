"""Common prefixes and blocks of rows on the CPU: page bookkeeping, refusals, the integers of the plans.

None of the refused calls gets as far as a GPU; the addresses they name are never read.
"""
from __future__ import annotations

import ctypes as C
import random
import shutil
import subprocess
import weakref
from pathlib import Path

import numpy as np
import pytest

import mxhip
from test_pages import AT, BAD_POOLS, BAD_STEPS, batch, pool

ERR_ARG = -1


# ---- rows that sequences have in the same pages ----------------------------------------------------


def test_common_rows_of_forks():
    p = mxhip.Pages(20, 16, 8)
    a = p.open()
    p.extend(a, 50), p.set_length(a, 50)
    b = p.fork(a)
    assert p.common([a, b]) == 48 and p.common([b]) == 48 and p.common([]) == 0
    p.extend(b, 5)  # copies the last page, which both would write
    p.set_length(b, 55)
    c = p.fork(b)
    assert p.common([a, b, c]) == 48 and p.common([b, c]) == 48
    p.extend(b, 30), p.set_length(b, 85)
    d = p.fork(b)
    assert p.common([b, d]) == 80 and p.common([d, b, c]) == 48 and p.common([a, a]) == 48
    p.set_length(d, 20)
    assert p.common([b, d]) == 16
    e = p.open()
    assert p.common([a, e]) == 0
    p.extend(e, 40), p.set_length(e, 40)
    assert p.common([a, e]) == 0
    p.close()


def test_rows_only_reserved_are_not_common():
    p = mxhip.Pages(20, 16, 8)
    a = p.open()
    p.extend(a, 64)
    b = p.fork(a)
    assert p.common([a, b]) == 0
    p.close()


def test_common_rows_refuse():
    p = mxhip.Pages(20, 16, 8)
    a = p.open()
    for bad in ([a, 1], [-1], [a, 99]):
        with pytest.raises(mxhip.MxhError, match="no sequence"):
            p.common(bad)
    one = np.asarray([a], np.int32)
    assert mxhip.lib.mxh_pages_common(None, one.ctypes.data, 1) == ERR_ARG
    assert mxhip.lib.mxh_pages_common(p.h, None, 1) == ERR_ARG
    assert mxhip.lib.mxh_pages_common(p.h, one.ctypes.data, -1) == ERR_ARG
    assert mxhip.lib.mxh_pages_common(p.h, None, 0) == 0
    p.close()
    with pytest.raises(mxhip.MxhError):
        p.common([a])


# ---- refusals ----------------------------------------------------------------------------------------


def groups(n=1, start=AT, shared=AT):
    return mxhip.KvGroups(n, start, shared)


def blocks(bounds=6 * AT, block_rows=16, n_first=1, n_last=1, n_select=4, layer_stride=0):
    return mxhip.KvBlocks(bounds, block_rows=block_rows, n_first=n_first, n_last=n_last, n_select=n_select,
                          layer_stride=layer_stride)


def shared(pl, layer, b, nh=4, g=None, q=4 * AT, att=5 * AT, work=8 * AT, nbytes=1 << 40):
    mxhip.attention_shared(pl, layer, b, g or groups(), q, nh, att, work, nbytes)


def bounds(pl, layer, b, nh=4, bl=None):
    mxhip.kv_block_bounds(pl, layer, b, bl or blocks())


def select(pl, layer, b, nh=4, bl=None, q=4 * AT, chosen=5 * AT, work=8 * AT, nbytes=1 << 40):
    mxhip.kv_select_blocks(pl, layer, b, bl or blocks(), q, nh, chosen, work, nbytes)


def listed(pl, layer, b, nh=4, bl=None, chosen=7 * AT, q=4 * AT, att=5 * AT, work=8 * AT, nbytes=1 << 40):
    mxhip.attention_blocks(pl, layer, b, bl or blocks(), chosen, q, nh, att, work, nbytes)


CALLS = [shared, bounds, select, listed]


@pytest.mark.parametrize("call", CALLS)
def test_pools_and_batches_are_checked(call):
    for over in BAD_POOLS:
        with pytest.raises(mxhip.MxhError):
            call(pool(**over), 0, batch())
    for over in BAD_STEPS:
        with pytest.raises(mxhip.MxhError):
            call(pool(), 0, batch(**over))
    for layer in (-1, 2):
        with pytest.raises(mxhip.MxhError, match="layer"):
            call(pool(), layer, batch())
    if call is not bounds:
        for nh in (0, -2, 3, 18):
            with pytest.raises(mxhip.MxhError, match="heads"):
                call(pool(), 0, batch(), nh=nh)
    call(pool(), 0, batch(n_tokens=0))  # nothing to do
    if call is not shared:
        call(pool(), 0, batch(n_seq=0))


def test_groups_are_checked():
    for g in (groups(-1), groups(3), groups(1, start=None), groups(1, shared=None)):
        with pytest.raises(mxhip.MxhError, match="groups|array"):
            shared(pool(), 0, batch(), g=g)
    for b in (batch(n_seq=0), batch(n_seq=0, n_tokens=0)):
        shared(pool(), 0, b, g=groups(0, None, None))
        with pytest.raises(mxhip.MxhError, match="1 groups of 0"):
            shared(pool(), 0, b)
    n = C.c_size_t(7)
    f = mxhip.lib.mxh_attention_shared_workspace
    assert f(C.byref(pool()), C.byref(batch()), None, 4, C.byref(n)) == ERR_ARG and n.value == 0
    assert f(C.byref(pool()), C.byref(batch()), C.byref(groups()), 4, None) == ERR_ARG
    assert mxhip.lib.mxh_attention_shared(C.byref(pool()), 0, C.byref(batch()), None, 4 * AT, 4, 5 * AT, 8 * AT,
                                          1 << 40) == ERR_ARG
    assert mxhip.attention_shared_workspace(pool(), batch(n_tokens=0), groups(), 4) == 0


BAD_BLOCKS = [dict(block_rows=8), dict(block_rows=0), dict(block_rows=-16), dict(block_rows=24), dict(block_rows=32),
              dict(n_select=0), dict(n_select=1025), dict(n_select=-1)]
BAD_BOUNDS = [dict(bounds=None), dict(bounds=AT + 8), dict(layer_stride=8), dict(layer_stride=-8),
              dict(layer_stride=8 * 2 * 2 * 64 + 4)]
BAD_BUDGETS = [dict(n_first=-1), dict(n_last=0), dict(n_last=-1), dict(n_first=4), dict(n_first=2, n_last=3),
               dict(n_first=2**31 - 1, n_last=2**31 - 1)]


@pytest.mark.parametrize("call", [bounds, select, listed])
def test_blocks_are_checked(call):
    bad = BAD_BLOCKS + (BAD_BOUNDS if call is not listed else []) + (BAD_BUDGETS if call is select else [])
    for over in bad:
        with pytest.raises(mxhip.MxhError):
            call(pool(), 0, batch(), bl=blocks(**over))
    with pytest.raises(mxhip.MxhError, match="blocks"):
        call(pool(), 0, batch(table_ld=262145))
    with pytest.raises(mxhip.MxhError, match="blocks"):
        call(pool(page_rows=1024), 0, batch(table_ld=2**31 - 1), bl=blocks())


@pytest.mark.parametrize("name", ["mxh_kv_select_workspace", "mxh_attention_blocks_workspace"])
def test_workspace_queries_refuse(name):
    f, n = getattr(mxhip.lib, name), C.c_size_t(7)
    ask = lambda p, b, bl, nh, out: f(p and C.byref(p), b and C.byref(b), bl and C.byref(bl), nh, out)  # noqa: E731
    assert ask(pool(), batch(), None, 4, C.byref(n)) == ERR_ARG and n.value == 0
    assert ask(pool(), None, blocks(), 4, C.byref(n)) == ERR_ARG
    assert ask(None, batch(), blocks(), 4, C.byref(n)) == ERR_ARG
    assert ask(pool(), batch(), blocks(), 3, C.byref(n)) == ERR_ARG
    assert ask(pool(), batch(), blocks(), 4, None) == ERR_ARG
    n.value = 7
    assert ask(pool(), batch(n_tokens=0), blocks(), 4, C.byref(n)) == 0 and n.value == 0


def test_arrays_are_checked():
    for over in (dict(q=None), dict(att=None), dict(q=AT + 4), dict(att=AT + 4), dict(work=AT + 4), dict(att=4 * AT + 16)):
        for call in (shared, listed):
            with pytest.raises(mxhip.MxhError):
                call(pool(), 0, batch(), **over)
    for over in (dict(chosen=None), dict(chosen=7 * AT + 2), dict(chosen=5 * AT + 64)):
        with pytest.raises(mxhip.MxhError, match="chosen"):
            listed(pool(), 0, batch(), **over)
    for over in (dict(q=None), dict(chosen=None), dict(q=4 * AT + 4), dict(chosen=5 * AT + 1), dict(work=None),
                 dict(work=8 * AT + 4), dict(chosen=4 * AT + 64), dict(work=4 * AT), dict(work=5 * AT), dict(nbytes=8)):
        with pytest.raises(mxhip.MxhError):
            select(pool(), 0, batch(), **over)


def test_bounds_overlap_nothing():
    """Of the call's layer: 8 pages of 16 rows, 2 kv heads of 64, so 32 KB of K and of V and 4 KB of bounds."""
    pl, b = pool(), batch()
    size = 2 * pl.n_pages * pl.page_rows * pl.n_kv * pl.head_dim
    own = 2 * 2 * pl.n_pages * pl.n_kv * pl.head_dim
    for at in (pl.k, pl.v):
        for x in (at - own + 16, at, at + size - 16):
            with pytest.raises(mxhip.MxhError, match="bounds overlap"):
                bounds(pl, 0, b, bl=blocks(bounds=x))
        with pytest.raises(mxhip.MxhError, match="bounds overlap"):
            bounds(pl, 1, b, bl=blocks(bounds=at + size - own))
    for over in (dict(chosen=6 * AT + own - 16), dict(work=6 * AT + own - 16), dict(chosen=6 * AT - 16)):
        with pytest.raises(mxhip.MxhError, match="overlaps the bounds"):
            select(pl, 0, b, **over)
    with pytest.raises(mxhip.MxhError, match="overlaps the bounds"):
        select(pl, 1, b, chosen=6 * AT + own)


def test_the_selection_workspace_is_enough_for_shorter_tables_and_fewer_tokens():
    """What the query says of a batch, every call up to its tokens and its table's width takes (and then refuses its
    arrays, so that none gets to a GPU)."""
    rng = random.Random(7)
    wide = [(8, 2048, 2064, 2048, 2048), (8, 512, 8193, 8177, 512), (8, 40, 262144, 70000, 39)]
    for _ in range(300):
        nkv, tokens, ld = rng.choice([1, 2, 8, 40]), int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 18))
        wide.append((nkv, tokens, ld, rng.randint(max(1, ld - 40), ld), rng.randint(max(1, tokens - 40), tokens)))
        wide.append((nkv, tokens, ld, rng.randint(1, ld), rng.randint(1, tokens)))
    for nkv, tokens, ld, less_ld, less_tokens in wide:
        pl = pool(n_kv=nkv)
        enough = mxhip.kv_select_workspace(pl, batch(n_tokens=tokens, table_ld=ld), blocks(), nkv)
        b = batch(n_tokens=less_tokens, table_ld=less_ld)
        assert mxhip.kv_select_workspace(pl, b, blocks(), nkv) <= enough
        with pytest.raises(mxhip.MxhError, match="work overlaps"):
            select(pl, 0, b, nh=nkv, q=1 << 45, chosen=1 << 44, work=1 << 44, nbytes=enough)


def test_descriptions_hold_their_buffers():
    made = []

    def new():
        b = object.__new__(mxhip.DeviceBuffer)  # (no GPU here: an address that is never freed)
        b.ptr, b.nbytes, b.close = AT, 64, lambda: None
        made.append(weakref.ref(b))
        return b

    g, x = mxhip.KvGroups(1, new(), new()), mxhip.KvBlocks(new(), block_rows=16)
    assert (g.start, g.shared, x.bounds) == (AT,) * 3
    assert all(r() is not None for r in made)
    del g, x
    assert all(r() is None for r in made)
    assert mxhip.KvBlocks(None, block_rows=16).bounds is None


# ---- how work is shared out ----------------------------------------------------------------------------

HDR = Path(__file__).resolve().parent.parent / "minxfmr.cpp_amd" / "csrc" / "hip"
SRC = """
#include "mxh_shared_plan.h"
#include "mxh_blocks.h"
using namespace mxh;

#define REQUIRE(x) do { if (!(x)) return __LINE__; } while (0)

// runs of n[r] tokens over keys[r] rows, the first n_groups of them prefixes of `of` tokens in all
extern "C" int shared(int n_seq, int n_tokens, int n_groups, int nkv, int group, int cus, int hd, const int* n,
                      const int* keys, int most_seq, int most_tokens, int most_groups) {
    const PagedSize size{n_seq, n_tokens, 1 << 20, nkv, group, cus};
    const SharedShape s = shared_shape(size, n_groups);
    uint64_t units[2] = {0, 0};
    const auto run = [&](int r) {
        const int rows = r < n_groups ? s.rows_p : s.rows_s;
        return shared_run((uint32_t)n[r], (uint32_t)keys[r], rows, (uint32_t)(rows / group));
    };
    for (int r = 0; r < n_groups + n_seq; ++r) units[r >= n_groups] += run(r).units();
    const uint32_t pers[2] = {shared_per(units[0], s.target_p), shared_per(units[1], s.target_s)};
    int64_t p = 0, o = 0;
    for (int r = 0; r < n_groups + n_seq; ++r) {
        const SharedRun x = run(r);
        const uint32_t per = pers[r >= n_groups], parts = x.parts(per);
        REQUIRE((uint64_t)x.tiles * (uint64_t)((r < n_groups ? s.rows_p : s.rows_s) / group) >= (uint64_t)n[r]);
        REQUIRE(parts >= 1 && (x.stages == 0 || parts <= x.stages));
        uint32_t at = 0;  // a tile's parts cover its stages in order, none empty but of a tile without any
        for (uint32_t z = 0; z < parts; ++z) {
            const uint32_t st0 = z * x.length(per), st1 = std::min((z + 1) * x.length(per), x.stages);
            REQUIRE(st0 == at && (st1 > st0 || x.stages == 0) && st1 - st0 <= per);
            at = st1;
        }
        REQUIRE(at == x.stages);
        (r < n_groups ? p : o) += (int64_t)x.tiles * parts;
    }
    REQUIRE(p <= s.items_p && o <= s.items_s);
    if (!shared_pays(size, hd, n_groups)) return 0;
    const SharedWork w = shared_work(s, n_tokens, nkv, hd);
    const PagedSize most{most_seq, most_tokens, 1 << 20, nkv, group, cus};
    const SharedWork b = shared_work(shared_bound(most, most_groups), shared_bound(most, most_seq), shared_tokens(most),
                                     nkv, hd);
    REQUIRE(w.bytes <= b.bytes);
    return -1;  // (that it pays)
}

extern "C" int blocks(int n_seq, int n_tokens, int64_t n_blocks, int nkv, int group, int n_select, int block_rows,
                      int cus, int hd) {
    const BlockSize a{n_seq, n_tokens, n_blocks, nkv, group, n_select, block_rows, cus};
    const int t = block_tokens(a), s = block_splits(a);
    REQUIRE(t >= 1 && t <= 16 && t * group <= block_rows_of_tile(a) && (int64_t)t * n_select <= kListMax);
    REQUIRE(t * ((n_blocks + 31) / 32) * 4 <= kBitBytes);
    REQUIRE(block_tiles(a) * t >= n_tokens && (block_tiles(a) - 1) * t < n_tokens);
    REQUIRE(s >= 1 && block_work_bytes(a, hd) <= block_work_bound(a, hd));
    const int64_t step = select_tokens(n_tokens, n_blocks, nkv);
    REQUIRE(step >= 1 && step <= n_tokens);
    REQUIRE(select_work_bytes(n_tokens, n_blocks, nkv) <= select_work_bytes(n_tokens + 100, n_blocks, nkv));
    return 0;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-shared",
                    "-fPIC", f"-I{HDR}", "-o", str(d / "plan.so"), str(d / "plan.cpp")], check=True)
    return C.CDLL(str(d / "plan.so"))


def test_items_of_common_prefixes_fit(plan):
    rng, paid = random.Random(3), 0
    for _ in range(3000):
        ns = rng.choice([1, 2, 7, 64, 300, 4096])
        ng = rng.randint(0, min(ns, rng.choice([1, 3, 4096])))
        top = rng.choice([1, 2, 30, 3000 // ns + 1, (1 << 20) // ns])
        n = [rng.randint(0, top) for _ in range(ns)]
        cuts = sorted(rng.sample(range(1, ns), ng - 1)) if ng > 1 else []
        ends = [0] + cuts + [ns] if ng else []
        runs = [sum(n[a:b]) for a, b in zip(ends, ends[1:])] + n
        rows = rng.choice([0, 100, 10000, 1 << 24, 1 << 30])
        keys = [rng.randint(0, rows) for _ in runs]
        tokens = max(sum(n), 1)
        nkv, group = rng.choice([1, 2, 8, 40, 1024]), rng.randint(1, 8)
        arr = lambda x: (C.c_int * len(x))(*x)  # noqa: E731
        rc = plan.shared(ns, tokens, ng, nkv, group, 256, 128, arr(runs), arr(keys), min(4096, ns + rng.randint(0, 9)),
                         min(1 << 20, tokens + rng.randint(0, 99)), min(ns, ng + rng.randint(0, 5)))
        assert rc <= 0, f"line {rc}: {ns} sequences, {ng} groups, {tokens} tokens"
        paid += rc < 0
    assert 300 < paid < 2500


def test_tiles_and_splits_of_lists_fit(plan):
    rng = random.Random(4)
    for _ in range(20000):
        n_tokens = int(2 ** rng.uniform(0, 20))
        a = (rng.randint(1, 4096), n_tokens, int(2 ** rng.uniform(0, 18)), rng.choice([1, 2, 8, 40, 1024]),
             rng.randint(1, 8), int(2 ** rng.uniform(0, 10)), rng.choice([16, 32, 64, 1024]))
        rc = plan.blocks(a[0], a[1], C.c_int64(a[2]), *a[3:], 256, 128)
        assert rc == 0, f"line {rc}: {a}"
