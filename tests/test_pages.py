"""Paged K/V cache: page bookkeeping and the checks of the calls (CPU only).

The bookkeeping is compared with a model that keeps every sequence's rows as
values: what a sequence reads through its table must be what was written to it,
whatever the sequences it was forked from or into did since.  Every refusal
here happens on the host before any GPU is asked for.
"""
from __future__ import annotations

import ctypes as C
import random
import subprocess
import sys
import weakref

import numpy as np
import pytest

import mxhip

ERR_ARG, ERR_OOM = -1, -5


def test_a_sequence_grows_and_shrinks():
    p = mxhip.Pages(4, 16, 2)
    s = p.open()
    assert p.length(s) == 0 and p.free == 4
    assert p.extend(s, 17) == [] and p.free == 2
    p.set_length(s, 17)
    table, cached = p.table([s], 4)
    assert table.tolist() == [[0, 1, -1, -1]] and cached.tolist() == [17]
    p.set_length(s, 16)
    assert p.free == 3
    p.set_length(s, 0)
    assert p.free == 4 and p.table([s], 1)[0].tolist() == [[-1]]
    p.release(s)
    p.close()


def test_rows_reserved_and_not_kept_give_their_pages_back():
    p = mxhip.Pages(8, 16, 2)
    s = p.open()
    p.extend(s, 10)
    p.set_length(s, 10)
    p.extend(s, 64)  # a drafted tree
    assert p.free == 3
    p.set_length(s, 13)  # three tokens kept
    assert p.free == 7 and p.length(s) == 13


def test_fork_shares_and_the_first_writer_copies():
    p = mxhip.Pages(8, 16, 3)
    a = p.open()
    p.extend(a, 20)
    p.set_length(a, 20)
    b = p.fork(a)
    assert p.free == 6 and p.table([b], 2)[0].tolist() == p.table([a], 2)[0].tolist()
    copies = p.extend(b, 1)
    assert copies == [(1, 2)] and p.free == 5
    assert p.table([a], 2)[0].tolist() == [[0, 1]] and p.table([b], 2)[0].tolist() == [[0, 2]]
    assert p.extend(a, 1) == []  # b let go of page 1
    p.release(a)
    assert p.free == 6  # page 0 is b's still
    p.release(b)
    assert p.free == 8


def test_a_fork_leaves_out_rows_that_are_only_reserved():
    p = mxhip.Pages(8, 16, 3)
    a = p.open()
    p.extend(a, 16)
    p.set_length(a, 16)
    p.extend(a, 30)
    b = p.fork(a)
    assert p.table([b], 3)[0].tolist() == [[0, -1, -1]]
    assert p.extend(b, 1) == []  # row 16 starts a page of its own
    with pytest.raises(mxhip.MxhError, match="at most 16"):
        p.set_length(p.fork(a), 17)


def test_too_few_pages_change_nothing():
    p = mxhip.Pages(3, 16, 3)
    a = p.open()
    p.extend(a, 20)
    p.set_length(a, 20)
    b = p.fork(a)
    for rows in (13, 2**31 - 21):  # one new page and the copy; as many rows as there are
        with pytest.raises(mxhip.MxhError, match="free pages"):
            p.extend(b, rows)
    assert p.free == 1 and p.table([b], 2)[0].tolist() == [[0, 1]] and p.length(b) == 20
    assert p.extend(b, 12) == [(1, 2)] and p.free == 0


def test_bookkeeping_refusals():
    p = mxhip.Pages(4, 16, 1)
    s = p.open()
    lib = mxhip.lib
    with pytest.raises(mxhip.MxhError, match="in use"):
        p.open()
    with pytest.raises(mxhip.MxhError, match="in use"):
        p.fork(s)
    for bad in (-1, 1, 99):
        for call in (p.release, p.fork, p.length, lambda q: p.extend(q, 1), lambda q: p.set_length(q, 0),
                     lambda q: p.table([q], 4)):
            with pytest.raises(mxhip.MxhError, match="no sequence"):
                call(bad)
    for rows in (-1, 1):
        with pytest.raises(mxhip.MxhError):
            p.set_length(s, rows)
    with pytest.raises(mxhip.MxhError):
        p.extend(s, -1)
    p.extend(s, 33)
    p.set_length(s, 33)
    with pytest.raises(mxhip.MxhError, match="pages"):
        p.table([s], 2)
    with pytest.raises(mxhip.MxhError):
        p.extend(s, 2**31 - 1)
    p.release(s)
    with pytest.raises(mxhip.MxhError, match="no sequence"):
        p.release(s)
    h = C.c_void_p()
    for args in ((0, 16, 1), (4, 8, 1), (4, 24, 1), (4, 2048, 1), (4, 16, 0), (2**31 - 1, 16, 1)):
        assert lib.mxh_pages_create(*args, C.byref(h)) == ERR_ARG and not h.value
    assert lib.mxh_pages_create(4, 16, 1, None) == ERR_ARG
    assert lib.mxh_pages_free(None) == ERR_ARG and lib.mxh_pages_length(None, 0) == ERR_ARG
    lib.mxh_pages_destroy(None)


@pytest.mark.parametrize("seed", range(6))
def test_random_forks_read_what_they_wrote(seed):
    rng = random.Random(seed)
    n_pages, pr = 24, 16
    p = mxhip.Pages(n_pages, pr, 6)
    pool = np.full(n_pages * pr, -1, np.int64)  # a value a row
    want: dict[int, list[int]] = {}
    value = 0

    def place(seq, r):
        return p.table([seq], 64)[0][0][r // pr] * pr + r % pr

    for _ in range(400):
        act = rng.choice(["open", "fork", "step", "step", "step", "cut", "release"])
        if act == "open" and len(want) < 6:
            want[p.open()] = []
        elif act == "fork" and want and len(want) < 6:
            s = rng.choice(list(want))
            want[p.fork(s)] = list(want[s])
        elif act == "step" and want:
            s, rows = rng.choice(list(want)), rng.randint(0, 40)
            before, length = p.table([s], 64)[0].tolist(), len(want[s])
            try:
                copies = p.extend(s, rows)
            except mxhip.MxhError:
                assert p.table([s], 64)[0].tolist() == before and p.length(s) == length
                continue
            for a, b in copies:
                pool[b * pr:(b + 1) * pr] = pool[a * pr:(a + 1) * pr]
            kept = rng.randint(0, rows)
            for i in range(rows):
                pool[place(s, length + i)] = value
                if i < kept:
                    want[s].append(value)
                value += 1
            if rng.random() < 0.3 and len(want) < 6:  # a fork in the middle of a step
                want[p.fork(s)] = want[s][:length]
            p.set_length(s, length + kept)
        elif act == "cut" and want:
            s = rng.choice(list(want))
            n = rng.randint(0, len(want[s]))
            p.set_length(s, n)
            del want[s][n:]
        elif act == "release" and want:
            s = rng.choice(list(want))
            p.release(s)
            del want[s]
        held = set()
        for s, rows in want.items():
            assert p.length(s) == len(rows)
            assert [int(pool[place(s, r)]) for r in range(len(rows))] == rows
            held |= {x for x in p.table([s], 64)[0][0].tolist() if x >= 0}
        assert p.free == n_pages - len(held)


# ---- checks of the device calls, none of which gets as far as a GPU ----------------------------

AT = 1 << 20  # an address that nothing reads


def pool(**over):
    a = dict(k=AT, v=2 * AT, n_layer=2, n_pages=8, page_rows=16, n_kv=2, head_dim=64, layer_stride=0)
    a.update(over)
    return mxhip.KvPool(a.pop("k"), a.pop("v"), **a)


def batch(**over):
    a = dict(n_seq=2, n_tokens=5, start=AT, cached=AT, table=AT, table_ld=4, parent=None)
    a.update(over)
    return mxhip.KvBatch(**a)


BAD_POOLS = [dict(k=None), dict(v=None), dict(k=AT + 8), dict(head_dim=96), dict(head_dim=0), dict(page_rows=8),
             dict(page_rows=48), dict(page_rows=2048), dict(page_rows=0), dict(n_layer=0), dict(n_pages=0),
             dict(n_pages=-1), dict(n_kv=0), dict(n_pages=2**31 - 1), dict(layer_stride=8),
             dict(layer_stride=8 * 16 * 2 * 64 + 4), dict(layer_stride=-8 * 16 * 2 * 64)]
BAD_STEPS = [dict(n_seq=-1), dict(n_seq=4097), dict(n_tokens=-1), dict(n_tokens=(1 << 20) + 1), dict(start=None),
             dict(cached=None), dict(table=None), dict(table_ld=0)]


def attention(pl, layer, b, nh=4, q=4 * AT, att=5 * AT, work=8 * AT, nbytes=1 << 30):
    mxhip.attention_paged(pl, layer, b, q, nh, att, work, nbytes)


def rope(pl, layer, b, nh=4, qkv=4 * AT, ld=512, bias=None, qn=None, kn=None, eps=1e-6, freq=AT, q=5 * AT):
    mxhip.qk_rope_append(pl, layer, b, qkv, ld, bias, qn, kn, eps, freq, True, nh, q)


@pytest.mark.parametrize("call", [attention, rope], ids=["attention", "rope"])
def test_per_layer_calls_refuse(call):
    for over in BAD_POOLS:
        with pytest.raises(mxhip.MxhError):
            call(pool(**over), 0, batch())
    for over in BAD_STEPS:
        with pytest.raises(mxhip.MxhError):
            call(pool(), 0, batch(**over))
    for layer in (-1, 2):
        with pytest.raises(mxhip.MxhError, match="layer"):
            call(pool(), layer, batch())
    for nh in (0, -2, 3, 18):
        with pytest.raises(mxhip.MxhError, match="heads"):
            call(pool(), 0, batch(), nh=nh)
    for b in (batch(n_seq=0), batch(n_tokens=0)):  # nothing to do
        call(pool(), 0, b)


def test_attention_refuses():
    for over in (dict(q=None), dict(att=None), dict(q=AT + 4), dict(att=AT + 4), dict(work=AT + 4),
                 dict(att=4 * AT + 16)):
        with pytest.raises(mxhip.MxhError):
            attention(pool(), 0, batch(), **over)
    n = C.c_size_t(7)
    assert mxhip.lib.mxh_attention_paged_workspace(C.byref(pool()), C.byref(batch()), 3, C.byref(n)) == ERR_ARG
    assert n.value == 0
    assert mxhip.lib.mxh_attention_paged_workspace(C.byref(pool()), C.byref(batch()), 4, None) == ERR_ARG
    assert mxhip.lib.mxh_attention_paged_workspace(C.byref(pool()), None, 4, C.byref(n)) == ERR_ARG
    assert mxhip.attention_paged_workspace(pool(), batch(n_seq=0), 4) == 0


def test_rope_refuses():
    for over in (dict(qkv=None), dict(q=None), dict(freq=None), dict(qkv=AT + 4), dict(q=AT + 8), dict(bias=AT + 4),
                 dict(qn=AT + 4), dict(kn=AT + 4), dict(freq=AT + 4), dict(ld=508), dict(ld=514), dict(ld=2**33),
                 dict(eps=-1.0), dict(eps=float("nan")), dict(q=4 * AT + 64)):
        with pytest.raises(mxhip.MxhError):
            rope(pool(), 0, batch(), **over)


def test_copies_refuse():
    for over in BAD_POOLS:
        with pytest.raises(mxhip.MxhError):
            mxhip.kv_copy_pages(pool(**over), [0], [1])
    for src, dst in (([-1], [0]), ([0], [8]), ([8], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3])):
        with pytest.raises(mxhip.MxhError):
            mxhip.kv_copy_pages(pool(), src, dst)
    with pytest.raises(ValueError):
        mxhip.kv_copy_pages(pool(), [0, 1], [2])
    mxhip.kv_copy_pages(pool(), [], [])  # nothing to do
    assert mxhip.lib.mxh_kv_copy_pages(C.byref(pool()), None, None, 1) == ERR_ARG
    assert mxhip.lib.mxh_kv_copy_pages(C.byref(pool()), None, None, -1) == ERR_ARG


def test_keeping_refuses():
    keep = mxhip.kv_keep_rows
    for over in BAD_POOLS:
        with pytest.raises(mxhip.MxhError):
            keep(pool(**over), [[0, 1]], [3], [0, 1], [2])
    for table, cached, start, kept in (
            ([[0, 1]], [3], [0, 2], [2, 2]),  # not ascending
            ([[0, 1]], [3], [0, 2], [4, 1]),
            ([[0, 1]], [3], [0, 1], [-1]),
            ([[0, 1]], [3], [0, 1], [29]),  # past the table
            ([[0, 1]], [-1], [0, 1], [2]),
            ([[0, 1]], [2**31 - 1], [0, 1], [2]),
            ([[0, -1]], [3], [0, 1], [20]),  # no such page
            ([[8, 1]], [3], [0, 1], [20]),
            ([[1, 1]], [3], [0, 1], [20]),  # one page in two places
            ([[0, 1], [2, 1]], [14, 14], [0, 2, 4], [0, 3, 0, 3]),  # of two sequences
            ([[0, 1], [2, 3]], [3, 3], [0, 1, 0], [2])):  # keep_start decreases
        with pytest.raises(mxhip.MxhError):
            keep(pool(), table, cached, start, kept)
    with pytest.raises(ValueError):
        keep(pool(), [[0, 1]], [3], [0, 3], [2])
    with pytest.raises(ValueError):
        keep(pool(), [[0, 1]], [3, 4], [0, 1, 1], [2])
    # nothing to move: no GPU needed either
    keep(pool(), [[0, 1]], [3], [0, 3], [0, 1, 2])
    keep(pool(), [[0, 1], [1, 0]], [3, 7], [0, 0, 0], [])


def test_sizes_past_the_limits_are_refused():
    h = C.c_void_p()
    assert mxhip.lib.mxh_pages_create(4, 16, (1 << 20) + 1, C.byref(h)) == ERR_ARG and not h.value
    wide = pool(n_layer=65535, n_kv=512, head_dim=32, n_pages=1, page_rows=16)  # a row of 128 MB
    fits = pool(n_layer=65535, n_kv=32, head_dim=32, n_pages=1, page_rows=16)
    with pytest.raises(mxhip.MxhError, match="unsupported pool"):
        mxhip.kv_copy_pages(wide, [], [])
    mxhip.kv_copy_pages(fits, [], [])


# (starts, kept or None) that begin below zero, fall, or rise past a list that is not there
BAD_STARTS = [([-1, 0], [2]), ([-1, 1], [2]), ([-(1 << 30), 0], [2]), ([-(2**31), 2**31 - 1], [2]),
              ([1 << 30, (1 << 30) + 1, 0], [2]), ([0, 5, 0], None), ([0, 1, 0], None), ([0, 1], None),
              ([0, 2**31 - 1, -(2**31)], [2]), ([3, 3, 2], [2])]


@pytest.mark.parametrize("case", range(len(BAD_STARTS)))
def test_kept_lists_are_read_only_where_their_starts_make_sense(case):
    """In a process of its own: the call is refused, and reads nothing outside its lists on the way."""
    starts, kept = BAD_STARTS[case]
    code = f"""
import ctypes as C, sys
sys.path[:0] = {sys.path!r}
import mxhip
from test_pages import pool
n = {len(starts) - 1}
ints = lambda a: None if a is None else (C.c_int * len(a))(*a)
rc = mxhip.lib.mxh_kv_keep_rows(C.byref(pool()), ints([0, 1] * n), 2, ints([3] * n), ints({starts!r}), ints({kept!r}), n)
sys.exit(0 if rc == {ERR_ARG} else 3)
"""
    assert subprocess.run([sys.executable, "-c", code], timeout=300).returncode == 0


def test_starts_of_kept_lists_need_not_begin_at_zero():
    """A slice of a longer list: the entries before the first start are not looked at."""
    mxhip.kv_keep_rows(pool(), [[0, 1]], [3], [2, 4], [-9, 99, 0, 1])
    assert mxhip.lib.mxh_kv_keep_rows(C.byref(pool()), (C.c_int * 2)(0, 1), 2, (C.c_int * 1)(3), (C.c_int * 2)(0, 0),
                                      None, 1) == 0


def test_pools_and_batches_hold_their_buffers():
    """A buffer that only a pool or a batch was given is not freed under it."""
    def buffer():
        b = object.__new__(mxhip.DeviceBuffer)  # (no GPU here: an address that is never freed)
        b.ptr, b.nbytes, b.close = AT, 64, lambda: None
        return b

    made = []

    def new():
        b = buffer()
        made.append(weakref.ref(b))
        return b

    pl = mxhip.KvPool(new(), new(), n_layer=1, n_pages=1, page_rows=16, n_kv=1, head_dim=32)
    ba = mxhip.KvBatch(1, 1, new(), new(), new(), 1, new())
    assert (pl.k, pl.v, ba.start, ba.cached, ba.table, ba.parent) == (AT,) * 6
    assert all(r() is not None for r in made)
    del pl, ba
    assert all(r() is None for r in made)
    assert mxhip.KvBatch(1, 1, AT, AT, AT, 1).parent is None


def test_closed_bookkeeping_refuses():
    p = mxhip.Pages(4, 16, 1)
    p.close()
    p.close()
    for call in (p.open, lambda: p.free, lambda: p.length(0), lambda: p.fork(0), lambda: p.release(0), lambda: p.extend(0, 1),
                 lambda: p.set_length(0, 0), lambda: p.table([0], 1)):
        with pytest.raises(mxhip.MxhError):
            call()
