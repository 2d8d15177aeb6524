"""Attention of sequences that begin with the same pages (GPU): mxh_attention_shared.

The values expected and their bound are those of attention over the paged cache
(test_paged_gpu.py), which do not depend on what is read once: the sums over the
keys that a row's parts share among them are covered by the bound's L u.  Pages
that members of a group would have had of their own for the common rows hold NaN.

Prefixes are read apart where the table is wide enough for the batch to be large
(180 MB of K and V) and sequences have few tokens on average (32 rows of q): `wide`
cases have such a table, mostly of absent pages.  Others run as attention over the
paged cache.
"""
from __future__ import annotations

import numpy as np
import pytest

import mxhip
from test_graph_capture_gpu import Graph
from test_paged_edges_gpu import check_precision
from test_paged_gpu import FILL, HEADS, Case

pytestmark = pytest.mark.gpu


class Shared(Case):
    """Case whose groups, (first sequence, one past the last, rows in common), have those rows in the same pages."""

    def __init__(self, seqs, groups, *, told=None, starts=None, wide=True, **kw):
        if wide:
            row = 4 * kw["nkv"] * kw["hd"]
            kw["extra_ld"] = kw.get("extra_ld", 0) + -(-180_000_000 // (row * kw["page"] * len(seqs)))
        super().__init__(seqs, **kw)
        self.groups = groups
        width = self.nkv * self.hd
        for a, b, rows in groups:
            p = rows // self.page
            for s in range(a + 1, b):
                for i in range(min(p, seqs[s][0] // self.page)):
                    at = int(self.table[s, i]) * self.page * width
                    self.k[self.layer, at:at + self.page * width] = np.nan
                    self.v[self.layer, at:at + self.page * width] = np.nan
                    self.table[s, i] = self.table[a, i]
        # sequences between the groups make groups of their own, with nothing in common
        first, common = [], []
        for a, b, rows in groups:
            if first and first[-1] != a:
                common.append(0)
                first.append(a)
            if not first:
                first.append(a)
            common.append(rows)
            first.append(b)
        self.starts = np.asarray(first if starts is None else starts, np.int32)
        self.common = np.asarray(common if told is None else told, np.int32)

    def upload(self):
        super().upload()
        b = self.bufs
        n = len(self.common)
        b["g_start"] = mxhip.DeviceBuffer.from_array(self.starts) if n else None
        b["g_shared"] = mxhip.DeviceBuffer.from_array(self.common) if n else None
        self.what = mxhip.KvGroups(n, b["g_start"], b["g_shared"])
        self.work_bytes = mxhip.attention_shared_workspace(self.pool, self.batch, self.what, self.nh)
        if b["work"] is not None:
            b["work"].close()
        b["work"] = mxhip.DeviceBuffer(self.work_bytes)
        # whatever an earlier call left there
        mxhip.memset(b["work"], 0x7f)
        return self

    def attend(self):
        b = self.bufs
        mxhip.attention_shared(self.pool, self.layer, self.batch, self.what, b["q"], self.nh, b["att"], b["work"],
                               self.work_bytes)


# (cached, new) of every sequence, groups; cached rows from the common ones on
GROUPS = {
    "samples": ([(64, 1), (67, 1), (90, 1), (64, 1)], [(0, 4, 64)]),
    "samples-of-a-long-prompt": ([(1300, 1), (1290, 1), (1281, 1)], [(0, 3, 1280)]),
    "two-groups-and-others": ([(40, 1), (200, 1), (210, 1), (700, 1), (5, 1), (640, 1), (650, 1), (900, 1), (0, 1)],
                              [(1, 3, 192), (5, 8, 640)]),
    "a-chat-of-one": ([(320, 1)], [(0, 1, 256)]),
    "questions": ([(256, 70), (256, 9), (270, 130), (256, 1)], [(0, 4, 256)]),
    "empty-among": ([(130, 0), (140, 3), (128, 0), (129, 1), (3, 0)], [(0, 4, 128)]),
    "nothing-in-common": ([(40, 2), (70, 1), (0, 5)], [(0, 3, 0)]),
    "no-groups": ([(40, 2), (200, 1), (0, 5)], []),
    "forty": ([(320 + 3 * s % 50, 1) for s in range(40)], [(0, 40, 320)]),
    "prompts-among-single-tokens": ([(256 + s % 7, 70 if s in (3, 9) else 1) for s in range(34)], [(0, 20, 256), (20, 34, 192)]),
    "few-tokens": ([(640 + s, 2 + s % 5) for s in range(12)], [(0, 5, 640), (7, 12, 576)]),
}
TREES = {
    "trees": ([(128, 7), (130, 12), (190, 64), (128, 1), (64, 16), (95, 33)], [(0, 4, 128)]),
    "trees-of-a-long-prompt": ([(2048, 27), (2050, 5), (2100, 13)], [(0, 3, 2048)]),
    "trees-among-single-tokens": ([(192 + s % 9, 64 if s == 5 else 13 if s in (2, 20) else 1) for s in range(30)],
                                  [(0, 16, 192), (16, 30, 128)]),
    "small-trees": ([(320 + s, 1 + s % 6) for s in range(16)], [(0, 16, 320)]),
}


@pytest.mark.parametrize("wide", [True, False], ids=["wide", "narrow"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", list(GROUPS) + list(TREES))
def test_attention_matches_float64(mxh, name, heads, page, wide):
    nh, nkv, hd = HEADS[heads]
    tree = name in TREES
    seqs, groups = (TREES if tree else GROUPS)[name]
    c = Shared(seqs, groups, nh=nh, nkv=nkv, hd=hd, page=page, tree=tree, lead=2, tail=3, seed=len(name) * 17 + nh,
               extra_ld=2, wide=wide).upload()
    c.check(c.attention())
    c.close()


def test_in_a_layer_of_a_strided_pool(mxh):
    c = Shared([(70, 3), (66, 9)], [(0, 2, 64)], nh=8, nkv=2, hd=64, page=32, layers=3, layer=1, stride=24,
               seed=5).upload()
    c.check(c.attention())
    c.close()


def test_many_sequences_and_groups(mxh):
    """More runs than a workgroup plans one each; many sequences empty, groups of one to nine."""
    rng = np.random.default_rng(8)
    seqs, groups = [], []
    while len(seqs) < 1500:
        n, rows = int(rng.integers(1, 10)), 16 * int(rng.integers(0, 4))
        groups.append((len(seqs), len(seqs) + n, rows))
        seqs += [(rows + int(rng.integers(0, 40)), int(rng.integers(0, 3))) for _ in range(n)]
    c = Shared(seqs, groups, nh=4, nkv=2, hd=32, page=16, seed=8, lead=1, tail=2).upload()
    c.check(c.attention())
    c.close()


def test_more_told_in_common_than_is_cached(mxh):
    """Rows in common end with the shortest cached part of the group's sequences that have tokens, in whole pages."""
    seqs, groups = [(60, 2), (200, 1), (3, 0), (190, 1)], [(0, 4, 48)]
    c = Shared(seqs, groups, told=[2**31 - 1], nh=8, nkv=2, hd=64, page=16, seed=6).upload()
    c.check(c.attention())
    c.close()
    c = Shared([(70, 2), (90, 1)], [(0, 2, 64)], told=[64 + 15], nh=8, nkv=2, hd=64, page=16, seed=6).upload()
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("starts", [[0, 3, 2], [-1, 2, 4], [0, 2, 5], [3, 1, 4], [2**31 - 1, 0, -2**31]])
def test_groups_that_make_no_sense_have_nothing_in_common(mxh, starts):
    seqs = [(64, 2), (70, 1), (80, 3), (64, 1)]
    c = Shared(seqs, [], told=[64, 64], starts=starts, nh=4, nkv=2, hd=64, page=16, seed=7).upload()
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("told", [-5, 0, 15])
def test_less_than_a_page_in_common(mxh, told):
    c = Shared([(64, 2), (70, 1)], [], told=[told], starts=[0, 2], nh=4, nkv=2, hd=64, page=16, seed=7).upload()
    c.check(c.attention())
    c.close()


def test_groups_may_begin_late_and_end_early(mxh):
    seqs = [(30, 2), (64, 2), (70, 1), (9, 3)]
    c = Shared(seqs, [(1, 3, 64)], nh=4, nkv=2, hd=128, page=32, seed=9)
    assert c.starts.tolist() == [1, 3]
    c.upload()
    c.check(c.attention())
    c.close()


def test_starts_that_fall_leave_att_alone(mxh):
    c = Shared([(64, 2), (70, 3), (64, 1)], [(0, 3, 64)], nh=4, nkv=2, hd=64, page=16, seed=7)
    c.start[2] = 1
    c.upload()
    assert np.all(c.attention() == FILL)
    c.close()


def test_absent_rows(mxh):
    """Pages that are not in the pool are nobody's rows; tokens without any rows get zeros."""
    c = Shared([(64, 1), (70, 2), (0, 3)], [(0, 2, 64)], nh=4, nkv=2, hd=64, page=16, seed=3)
    gone = c.table[1, 4]  # (the second sequence's rows 64 to 79)
    c.table[1, 4] = c.n_pages
    c.table[2, 0] = -1
    c.upload()
    got = c.attention()
    c.table[1, 4] = gone
    k, v = (np.array([c.row(x, 1, r) for r in range(64)], np.float64).reshape(64, 2, 64) for x in (c.k, c.v))
    for t in (1, 2):
        for h in range(4):
            sc = k[:, h // 2] @ c.q[t].reshape(4, 64)[h].astype(np.float64) / 8
            p = np.exp(sc - sc.max())
            assert np.all(np.abs(got[t, h] - p @ v[:, h // 2] / p.sum()) <= 1e-4)
    assert np.all(got[3:] == 0)
    c.close()


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
def test_what_is_not_attended_has_no_effect(mxh, tree):
    """Infinities and NaN among the new rows; a token that attends one gets what it makes."""
    seqs, groups = [(64, 40), (80, 21)] + [(64, 1)] * 10, [(0, 12, 64)]
    c = Shared(seqs, groups, nh=8, nkv=2, hd=64, page=16, tree=tree, seed=11)
    assert c.tokens * 4 <= 32 * len(seqs)
    bad = {0: [7, 30, 39], 1: [20, 5]}
    for s, rows in bad.items():
        for i, r in enumerate(rows):
            c.row(c.v, s, seqs[s][0] + r)[i::3] = [np.inf, -np.inf, np.nan][i]
            c.row(c.k, s, seqs[s][0] + r)[i::5] = [-np.inf, np.nan, np.inf][i]
    free = {int(c.start[s]) + i for s, (_, n) in enumerate(seqs) for i in range(n)
            if not set(bad.get(s, [])) & set(c.before(s, i))}
    hit = sorted(set(range(c.tokens)) - free)
    assert len(free) >= 10 and len(hit) >= 3
    c.upload()
    got = c.attention()
    c.check(got, rows=free)
    assert not np.any(np.all(np.isfinite(got[hit]).reshape(len(hit), -1), axis=1))
    c.close()


def test_an_infinity_in_the_prefix_is_everybodys(mxh):
    seqs = [(320, 1), (330, 5), (320, 1)]
    c = Shared(seqs, [(0, 3, 320)], nh=4, nkv=2, hd=64, page=16, seed=12)
    c.row(c.v, 0, 100)[5] = np.inf
    c.row(c.v, 0, 200)[64 + 9] = -np.inf
    c.upload()
    got = c.attention()
    assert np.all(got[:, :2, 5] == np.inf) and np.all(got[:, 2:, 9] == -np.inf)
    got[:, :2, 5] = got[:, 2:, 9] = 0
    assert np.all(np.isfinite(got))
    c.close()


def test_large_scores(mxh):
    """The prefix or the own rows hold all the weight."""
    c = Shared([(320, 2), (400, 9)], [(0, 2, 320)], nh=8, nkv=2, hd=128, page=16, seed=3)
    c.q[::2] *= 40
    for s, r in ((0, 17), (1, 390)):
        c.row(c.k, s, r)[:] *= 8
    c.upload()
    c.check(c.attention())
    c.close()


def test_two_calls_give_the_same_bits_and_agree_with_the_paged_call(mxh):
    c = Shared([(640 + s, 1 + s % 3) for s in range(12)], [(0, 12, 640)], nh=32, nkv=8, hd=128, page=16, seed=4).upload()
    one = c.attention().copy()
    assert np.array_equal(one, c.attention())
    n = mxhip.attention_paged_workspace(c.pool, c.batch, c.nh)
    work = mxhip.DeviceBuffer(max(n, 16))
    mxhip.attention_paged(c.pool, 0, c.batch, c.bufs["q"], c.nh, c.bufs["att"], work, n)
    mxhip.synchronize()
    two = c.bufs["att"].download(np.float32).reshape(one.shape)
    assert np.max(np.abs(one - two)) <= 1e-5
    work.close()
    c.close()


def test_a_recorded_call_follows_lengths_tables_and_groups(mxh):
    seqs, groups = [(128, 1), (140, 1), (200, 1)], [(0, 3, 128)]
    make = lambda s, g, seed, spare=3: Shared(s, g, nh=8, nkv=2, hd=64, page=16, seed=seed, extra_ld=20,  # noqa: E731
                                              spare=spare)
    c = make(seqs, groups, 1, spare=60).upload()
    graph = Graph([c.attend])
    for i, (s, g) in enumerate([(seqs, groups), ([(300, 1), (310, 1), (30, 1)], [(0, 2, 288)]),
                                ([(0, 1), (16, 1), (20, 1)], [(1, 3, 16)]), (seqs, groups)]):
        n = make(s, g, 40 + i)
        assert n.n_pages <= c.n_pages
        n.k, n.v = (np.concatenate([x, np.zeros((1, c.stride - n.stride), np.float16)], 1) for x in (n.k, n.v))
        table = np.full_like(c.table, -1)
        table[:, :min(c.ld, n.ld)] = n.table[:, :min(c.ld, n.ld)]
        (first, end, rows), = g
        starts, common = np.asarray([first, end], np.int32), np.asarray([rows], np.int32)
        for name, a in (("k", n.k), ("v", n.v), ("q", n.q), ("table", table), ("g_start", starts),
                        ("g_shared", common), ("cached", np.asarray([x for x, _ in s], np.int32)),
                        ("att", np.full(c.q.shape, FILL))):
            c.bufs[name].upload(np.ascontiguousarray(a))
        for _ in range(2):
            graph.replay()
            got = c.bufs["att"].download(np.float32).reshape(c.tokens, 8, 64)
            n.check(got)
            eager = c.attention()
            assert np.array_equal(got, eager)
    graph.close()
    c.close()


@pytest.mark.parametrize("ld", [30, 30000])
def test_the_largest_batchs_workspace_is_enough(mxh, ld):
    """Of a batch of n_seq sequences and n_tokens tokens, for all with fewer of either."""
    ns, nt, nh, nkv, hd = 40, 90, 8, 2, 64
    pool = mxhip.KvPool(256, 256, n_layer=1, n_pages=100, page_rows=16, n_kv=nkv, head_dim=hd)
    size = lambda s, t, g: mxhip.attention_shared_workspace(  # noqa: E731
        pool, mxhip.KvBatch(s, t, 256, 256, 256, ld), mxhip.KvGroups(g, 256, 256), nh)
    most = size(ns, nt, 10)
    for s in (1, 2, 7, 39, 40):
        for t in (1, 2, 3, 40, 89, 90):
            for g in (0, 1, 2, 10):
                if g <= s:
                    assert size(s, t, g) <= most
    c = Shared([(64, 1)] * 9 + [(64, 54)], [(0, 10, 64)], nh=nh, nkv=nkv, hd=hd, page=16, seed=1, wide=ld > 30).upload()
    c.bufs["work"].close()
    c.bufs["work"], c.work_bytes = mxhip.DeviceBuffer(most), most
    c.check(c.attention())
    c.close()


def test_a_workspace_that_is_too_small_is_refused(mxh):
    c = Shared([(64, 1), (64, 1)], [(0, 2, 64)], nh=4, nkv=2, hd=64, page=16, seed=1).upload()
    c.work_bytes = 1000
    with pytest.raises(mxhip.MxhError, match="1000 bytes of work"):
        c.attend()
    mxhip.synchronize()
    assert np.all(c.bufs["att"].download(np.float32) == FILL)
    c.close()


@pytest.mark.parametrize("groups", [1, 1365, 4096])
def test_the_most_sequences_and_groups(mxh, groups):
    """4,096 sequences: the plan's lengths, groups and runs fill their place in LDS."""
    n = 4096
    size = n // groups
    ends = [size * g for g in range(groups)] + [n]
    rng = np.random.default_rng(groups)
    seqs = [(16 + int(rng.integers(0, 30)), int(s % 7 != 3)) for s in range(n)]
    c = Shared(seqs, [(a, b, 16) for a, b in zip(ends, ends[1:])], nh=2, nkv=1, hd=32, page=16, seed=groups)
    assert len(c.common) == groups and n * c.ld * 16 * 4 * 32 >= 180e6
    c.upload()
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
@pytest.mark.parametrize("small,large", [(1e-2, 100.0), (1e-5, 1e4), (1e-37, 1e4), (1e33, 1e-6)])
def test_small_q_over_large_k(mxh, heads, small, large):
    """q outside the range of fp16 halves, over prefixes and the rows behind them; every fourth token ordinary."""
    nh, nkv, hd = HEADS[heads]
    for seqs, tree in (([(130, 1), (150, 1), (128, 1)], False), ([(140, 3), (128, 1), (133, 4)], True),
                       ([(128, 2 if s else 20) for s in range(12)], False)):
        c = Shared(seqs, [(0, len(seqs), 128)], nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, seed=19)
        assert c.tokens * nh // nkv <= 32 * len(seqs)
        c.k = np.clip(c.k.astype(np.float32) * large, -65504, 65504).astype(np.float16)
        c.q *= np.float32(small)
        if large > 1:
            c.q[3::4] /= np.float32(small * large)
        c.upload()
        check_precision(c, c.attention())
        c.close()


@pytest.mark.parametrize("whole", [False, True], ids=["a-row", "all-of-the-prefix"])
def test_scores_of_minus_infinity_in_the_prefix(mxh, whole):
    """Nothing of those rows: what is left of the prefix and the rows behind it share the weight."""
    seqs = [(320, 1), (330, 5), (320, 1)]
    c = Shared(seqs, [(0, 3, 320)], nh=4, nkv=2, hd=64, page=16, seed=12)
    gone = range(320) if whole else [100, 319]
    for r in gone:
        c.row(c.k, 0, r)[7] = -np.inf  # (kv head 0)
    q = c.q.reshape(c.tokens, 4, 64)
    q[:, :2, 7] = np.abs(q[:, :2, 7])
    c.upload()
    got = c.attention()
    for s, (n_c, n) in enumerate(seqs):
        k, v = (np.array([c.row(x, s, r) for r in range(n_c + n)], np.float64).reshape(-1, 2, 64) for x in (c.k, c.v))
        for i in range(n):
            t = int(c.start[s]) + i
            for h in range(4):
                sc = k[:n_c + i + 1, h // 2] @ q[t, h].astype(np.float64) / 8
                p = np.exp(sc - sc.max())
                assert np.all(np.abs(got[t, h] - p @ v[:n_c + i + 1, h // 2] / p.sum()) <= 1e-4), (s, i, h)
    c.close()


def test_drafted_trees_end_at_64_tokens(mxh):
    seqs = [(128, 70), (130, 3)] + [(128 + s, 1) for s in range(20)]
    c = Shared(seqs, [(0, 22, 128)], nh=8, nkv=2, hd=64, page=16, tree=True, seed=7)
    assert c.tokens * 4 <= 32 * len(seqs)
    c.upload()
    got = c.attention()
    past = list(range(64, 70))
    assert np.all(got[past] == FILL)
    got[past] = 0
    c.check(got, rows=set(range(c.tokens)) - set(past))
    c.close()
