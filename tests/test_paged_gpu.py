"""Operators over a paged K/V cache (GPU): appending, attention, copies, kept rows.

The expected values are the formulas in float64 on exactly the values that the
kernels read.  Pool rows that no sequence owns hold NaN, outputs start as a
sentinel: a read past a sequence, a write beside a token's row or an output
left unwritten fails.  Bounds (u = 2^-24, half a step of fp32):

- attention: q enters as a pair of fp16 (2^-21 of |q| with its scaling), a
  score is a sum of 2 hd products: |d score| <= D = (2^-21 + 2 hd u) *
  max_j sum_d |q_d k_jd| / sqrt(hd).  A probability is off by 2 D of its value
  (numerator and the sum's shift), by 2^-21 for the exponential and its pair of
  fp16, and the sums over L keys by L u at most, twice (numerator and sum):
  |err| <= (2 D + 2^-20 + 2 L u) sum_j p_j |v_j| + 2^-100.
- rope: bias, norm, weight and rotation round once each to fp32, the rest is in
  double: |err| <= 4 u (|x0| + |x1|) of the pair; k and v in fp16 2^-11 of the
  value (2^-25 below the normal range) on top.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mxhip
from test_graph_capture_gpu import Graph

pytestmark = pytest.mark.gpu

U = 2.0**-24
FILL = np.float32(-77.25)  # outputs before a call


def chain(n):
    return [i - 1 for i in range(n)]


def bush(n, rng):
    return [-1 if i == 0 or rng.random() < 0.15 else int(rng.integers(max(0, i - 5), i)) for i in range(n)]


def path(parent, i):
    at = []
    while i >= 0:
        at.append(i)
        i = parent[i]
    return at


class Case:
    """Sequences (cached rows, new tokens) over a shuffled pool, their parents (None: chains)."""

    def __init__(self, seqs, *, nh, nkv, hd, page, tree=False, lead=0, tail=0, layers=1, layer=0, stride=0, seed=0,
                 spare=3, extra_ld=0):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.nh, self.nkv, self.hd, self.page = seqs, nh, nkv, hd, page
        self.lead, self.layer = lead, layer
        need = [-(-(c + n) // page) for c, n in seqs]
        ids = rng.permutation(sum(need) + spare).astype(np.int32)
        self.ld = max(need + [1]) + extra_ld
        self.table = np.full((len(seqs), self.ld), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.n_pages = len(ids)
        dense = self.n_pages * page * nkv * hd
        self.stride = dense + stride
        shape = (layers, self.stride)
        self.k = np.full(shape, np.nan, np.float16)
        self.v = np.full(shape, np.nan, np.float16)
        self.parents = [bush(n, rng) if tree else None for _, n in seqs]
        self.start = (lead + np.concatenate([[0], np.cumsum([n for _, n in seqs])])).astype(np.int32)
        self.tokens = int(self.start[-1]) + tail
        for s, (c, n) in enumerate(seqs):
            for r in range(c + n):
                self.row(self.k, s, r)[:] = rng.standard_normal(nkv * hd)
                self.row(self.v, s, r)[:] = rng.standard_normal(nkv * hd)
        self.q = (1.5 * rng.standard_normal((self.tokens, nh * hd))).astype(np.float32)
        self.bufs = {}
        self.tree = tree
        self.stride_arg = self.stride if stride else 0

    def row(self, pool, s, r):
        at = (int(self.table[s, r // self.page]) * self.page + r % self.page) * self.nkv * self.hd
        return pool[self.layer, at:at + self.nkv * self.hd]

    def parent_array(self):
        if not self.tree:
            return None
        p = np.full(self.tokens, 12345, np.int32)
        for s in range(len(self.seqs)):
            p[self.start[s]:self.start[s + 1]] = self.parents[s]
        return p

    def before(self, s, i):
        """The new tokens that token i of sequence s follows, itself last."""
        return list(range(i + 1)) if self.parents[s] is None else path(self.parents[s], i)[::-1]

    def upload(self):
        put = lambda a: None if a is None else mxhip.DeviceBuffer.from_array(a)  # noqa: E731
        b = self.bufs = {n: put(getattr(self, n)) for n in ("k", "v", "q", "start", "table")}
        b["cached"] = put(np.asarray([c for c, _ in self.seqs], np.int32))
        b["parent"] = put(self.parent_array())
        self.pool = mxhip.KvPool(b["k"], b["v"], n_layer=self.k.shape[0], n_pages=self.n_pages, page_rows=self.page,
                                 n_kv=self.nkv, head_dim=self.hd, layer_stride=self.stride_arg)
        self.batch = mxhip.KvBatch(len(self.seqs), self.tokens, b["start"], b["cached"], b["table"], self.ld,
                                   b["parent"])
        n = mxhip.attention_paged_workspace(self.pool, self.batch, self.nh)
        b["work"], self.work_bytes = (mxhip.DeviceBuffer(n), n) if n else (None, 0)
        b["att"] = put(np.full((self.tokens, self.nh * self.hd), FILL))
        return self

    def attend(self):
        b = self.bufs
        mxhip.attention_paged(self.pool, self.layer, self.batch, b["q"], self.nh, b["att"], b["work"], self.work_bytes)

    def attention(self):
        self.attend()
        mxhip.synchronize()
        return self.bufs["att"].download(np.float32).reshape(self.tokens, self.nh, self.hd)

    def close(self):
        for b in self.bufs.values():
            if b is not None:
                b.close()

    def check(self, got, rows=None):
        """got against the formula in float64, with the bound above; other token rows untouched."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        group, worst = nh // nkv, 0.0
        inside = np.zeros(self.tokens, bool)
        q = self.q.astype(np.float64).reshape(self.tokens, nh, hd)
        for s, (c, n) in enumerate(self.seqs):
            k = np.array([self.row(self.k, s, r) for r in range(c + n)], np.float64).reshape(-1, nkv, hd)
            v = np.array([self.row(self.v, s, r) for r in range(c + n)], np.float64).reshape(-1, nkv, hd)
            for i in range(n):
                t = int(self.start[s]) + i
                inside[t] = True
                if rows is not None and t not in rows:
                    continue
                at = list(range(c)) + [c + j for j in self.before(s, i)]
                for h in range(nh):
                    kk, vv = k[at, h // group], v[at, h // group]
                    sc = kk @ q[t, h] / np.sqrt(hd)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    want = p @ vv
                    d = (2.0**-21 + 2 * hd * U) * (np.abs(kk) @ np.abs(q[t, h])).max() / np.sqrt(hd)
                    bound = (2 * d + 2.0**-20 + 2 * len(at) * U) * (p @ np.abs(vv)) + 2.0**-100
                    err = np.abs(got[t, h] - want)
                    assert np.all(err <= bound), f"seq {s} token {i} head {h}: {float((err / bound).max()):.3g} x bound"
                    worst = max(worst, float((err / bound).max()))
        assert np.all(got[~inside] == FILL), "rows outside the sequences were written"
        return worst


HEADS = {"g4-d128": (8, 2, 128), "g2-d128": (4, 2, 128), "g3-d64": (6, 2, 64), "g8-d32": (8, 1, 32), "g1-d128": (2, 2, 128),
         "g7-d64": (7, 1, 64), "g5-d32": (10, 2, 32)}
# (cached, new) of every sequence; trees of at most 64 tokens
SETS = {
    "one": [(0, 1)],
    "decode-15": [(15, 1)],
    "decode-16": [(16, 1)],
    "decode-1000": [(1000, 1)],
    "batch": [(0, 1), (31, 1), (32, 1), (33, 1), (500, 1), (127, 1), (128, 1), (1, 1), (129, 1)],
    "empty-among": [(5, 0), (40, 3), (0, 0), (17, 1), (9, 0)],
    "prompt-5": [(0, 5)],
    "prompts": [(0, 70), (33, 130), (200, 1), (0, 17)],
    "prompt-behind-700": [(700, 45)],
}
TREES = {
    "tree-2": [(3, 2)],
    "tree-64": [(100, 64)],
    "tree-no-cache": [(0, 33)],
    "trees": [(30, 7), (0, 12), (513, 64), (2, 1), (64, 16), (95, 33)],
    "tree-behind-2000": [(2000, 27)],
}


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", list(SETS) + list(TREES))
def test_attention_matches_float64(mxh, name, heads, page):
    nh, nkv, hd = HEADS[heads]
    tree = name in TREES
    c = Case((TREES if tree else SETS)[name], nh=nh, nkv=nkv, hd=hd, page=page, tree=tree, lead=2, tail=3,
             seed=len(name) * 31 + nh, extra_ld=2).upload()
    c.check(c.attention())
    c.close()


def test_attention_in_a_layer_of_a_strided_pool(mxh):
    c = Case([(70, 3), (10, 9)], nh=8, nkv=2, hd=64, page=32, layers=3, layer=1, stride=24, seed=5).upload()
    c.check(c.attention())
    c.close()


def test_many_sequences(mxh):
    """More sequences than a wave has lanes, many of them empty."""
    rng = np.random.default_rng(8)
    seqs = [(int(rng.integers(0, 60)), int(rng.integers(0, 3))) for _ in range(333)]
    c = Case(seqs, nh=4, nkv=2, hd=32, page=16, seed=8, lead=1, tail=2).upload()
    c.check(c.attention())
    c.close()


def test_large_scores(mxh):
    """Probabilities from one to nothing: q and k forty times as large in places."""
    c = Case([(300, 9), (1200, 2)], nh=8, nkv=2, hd=128, page=16, seed=3, tree=True)
    c.q[::2] *= 40
    for s, r in ((0, 17), (0, 250), (1, 1100)):
        c.row(c.k, s, r)[:] *= 8
    c.upload()
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
def test_what_is_not_attended_has_no_effect(mxh, tree, heads):
    """Infinities and NaN in rows behind a token and beside its path; a token that attends one gets what it makes."""
    nh, nkv, hd = HEADS[heads]
    clean = Case([(45, 40), (0, 21)], nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, seed=11)
    bad = {0: [7, 30, 39], 1: [20, 5]}
    spoilt = Case([(45, 40), (0, 21)], nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, seed=11)
    values = [np.inf, -np.inf, np.nan]
    for s, rows in bad.items():
        for i, r in enumerate(rows):
            cached = spoilt.seqs[s][0]
            spoilt.row(spoilt.v, s, cached + r)[i::3] = values[i]
            spoilt.row(spoilt.k, s, cached + r)[i::5] = values[(i + 1) % 3]
    clean.upload(), spoilt.upload()
    want, got = clean.attention(), spoilt.attention()
    free, hit = [], []
    for s, (c, n) in enumerate(clean.seqs):
        for i in range(n):
            (hit if set(bad[s]) & set(clean.before(s, i)) else free).append(int(clean.start[s]) + i)
    assert len(free) >= 10 and len(hit) >= 3
    clean.check(want)
    clean.check(got, rows=set(free))
    assert not np.any(np.all(np.isfinite(got[hit]).reshape(len(hit), -1), axis=1))
    clean.close(), spoilt.close()


def test_infinite_values_come_through_where_attended(mxh):
    """V infinities (finite K) at rows that some tokens attend: +-inf or NaN there, finite beside it."""
    c = Case([(20, 12)], nh=4, nkv=2, hd=64, page=16, tree=True, seed=2)
    for r, d, x in ((3, 0, np.inf), (6, 1, -np.inf), (8, 2, np.nan), (9, 0, -np.inf), (2, 70, np.inf)):
        c.row(c.v, 0, 20 + r)[d] = x
    c.upload()
    got = c.attention()
    for i in range(12):
        on = set(c.before(0, i))
        for h in range(4):
            g = h // 2
            for d in range(64):
                col = [float(c.row(c.v, 0, 20 + r)[64 * g + d]) for r in on]
                with np.errstate(invalid="ignore"):
                    want = sum(x for x in col if not np.isfinite(x))
                x = got[i, h, d]
                assert (np.isnan(x) if np.isnan(want) else x == want if np.isinf(want) else np.isfinite(x)), (i, h, d)
    c.close()


@pytest.mark.parametrize("n", [1, 3, 30])
@pytest.mark.parametrize("cached,rows", [(40, 16), (700, 32), (5000, 16)])
def test_infinite_values_among_rows_that_all_attend(mxh, cached, rows, n):
    """V infinities deep in the cached rows are every token's: +-inf in their columns, NaN where both meet."""
    c = Case([(cached, n)], nh=4, nkv=2, hd=64, page=rows, seed=12)
    want = {(0, 5): np.inf, (0, 9): -np.inf, (0, 11): np.nan, (1, 63): np.inf}
    for (g, d), x in want.items():
        for r, y in ((2, np.inf), (cached // 2, -np.inf)) if np.isnan(x) else ((cached // 3, x),):
            c.row(c.v, 0, r)[64 * g + d] = y
    c.upload()
    got = c.attention()
    for h in range(4):
        for d in range(64):
            x, w = got[:, h, d], want.get((h // 2, d), 0.0)
            assert (np.isnan(x) if np.isnan(w) else x == w if np.isinf(w) else np.isfinite(x)).all(), (h, d)
    c.close()


@pytest.mark.parametrize("seqs,tree", [([(300, 1), (20, 2)], False), ([(700, 45)], False), ([(100, 30), (9, 4)], True)])
def test_scores_of_minus_infinity(mxh, seqs, tree):
    """An attended K value of an infinity: nothing of that row where the score is -inf, NaN where it is +inf."""
    c = Case(seqs, nh=4, nkv=2, hd=64, page=16, tree=tree, seed=14)
    for s, (n_c, n) in enumerate(seqs):
        for r in (3, n_c - 1, n_c + n - 1):
            c.row(c.k, s, r)[7 + r % 3] = -np.inf  # (kv head 0)
    q = c.q.reshape(c.tokens, 4, 64)
    q[:, 0, 7:10] = np.abs(q[:, 0, 7:10])  # q head 0: -inf every time; q head 1: by its signs
    c.upload()
    got = c.attention()
    for s, (n_c, n) in enumerate(seqs):
        k, v = (np.array([c.row(x, s, r) for r in range(n_c + n)], np.float64).reshape(-1, 2, 64) for x in (c.k, c.v))
        for i in range(n):
            t, at = int(c.start[s]) + i, list(range(n_c)) + [n_c + j for j in c.before(s, i)]
            for h in range(4):
                sc = k[at, h // 2] @ q[t, h].astype(np.float64) / 8
                if np.any(sc == np.inf):
                    assert np.all(np.isnan(got[t, h])), (s, i, h)
                    continue
                p = np.exp(sc - sc.max())
                want = p @ v[at, h // 2] / p.sum()
                assert np.all(np.abs(got[t, h] - want) <= 1e-4), (s, i, h)
    c.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
def test_q_past_fp16(mxh, heads):
    """q of millions over a K of millionths."""
    nh, nkv, hd = HEADS[heads]
    c = Case([(300, 1), (150, 40), (3, 2)], nh=nh, nkv=nkv, hd=hd, page=16, seed=15)
    c.q *= 2e6
    c.k = (c.k.astype(np.float32) * 1e-5).astype(np.float16)
    c.upload()
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("seqs,tree", [([(300, 1)], False), ([(40, 30), (700, 50)], False), ([(130, 20), (5, 1)], True)])
def test_nan_reaches_the_outputs_that_read_it(mxh, seqs, tree):
    """A NaN in a token's q is its head's; NaN in a cached key is everybody's who attends it, in its kv head."""
    c = Case(seqs, nh=4, nkv=2, hd=128, page=16, tree=tree, seed=31)
    q = c.q.reshape(c.tokens, 4, 128)
    q[0, 1, 77] = np.nan
    last = int(c.start[-1]) - 1
    q[last, 2, :] = np.nan
    s = len(seqs) - 1
    c.row(c.k, s, 3)[5] = np.nan  # kv head 0: q heads 0 and 1 of sequence s
    c.upload()
    got = c.attention()
    for b, (_, n) in enumerate(seqs):
        for i in range(n):
            t = int(c.start[b]) + i
            for h in range(4):
                bad = (t, h) in ((0, 1), (last, 2)) or (b == s and h < 2 and (seqs[s][0] > 3 or 3 in c.before(s, i)))
                assert np.all(np.isnan(got[t, h])) if bad else np.all(np.isfinite(got[t, h])), (b, i, h)
    c.close()


@pytest.mark.parametrize("name", ["decode", "tree", "prompt"])
def test_bad_pages_and_parents_stay_inside(mxh, name):
    """Ids outside the pool and rows past the table are absent; bad parents are roots; trees end at 64 tokens."""
    seqs = {"decode": [(300, 1), (40, 1)], "tree": [(300, 20), (40, 9)], "prompt": [(300, 70), (40, 9)]}[name]
    c = Case(seqs, nh=4, nkv=2, hd=64, page=16, tree=name == "tree", seed=4)
    dropped = {(0, 2): c.n_pages, (0, 5): -1, (0, 9): 2**31 - 1, (1, 0): -2**31}
    for (s, p), x in dropped.items():
        c.table_sent = c.table.copy() if not hasattr(c, "table_sent") else c.table_sent
        c.table_sent[s, p] = x
    if name == "tree":
        c.parents[0][4], c.parents[0][7], c.parents[1][3] = 4, 19, -9
    c.upload()
    c.bufs["table"].upload(c.table_sent)
    got = c.attention()
    if name == "tree":
        c.parents[0][4] = c.parents[0][7] = c.parents[1][3] = -1
    q = c.q.astype(np.float64).reshape(c.tokens, 4, 64)
    for s, (n_c, n) in enumerate(seqs):
        for i in range(n):
            t = int(c.start[s]) + i
            at = [r for r in list(range(n_c)) + [n_c + j for j in c.before(s, i)] if (s, r // 16) not in dropped]
            for h in range(4):
                k = np.array([c.row(c.k, s, r) for r in at], np.float64).reshape(-1, 2, 64)[:, h // 2]
                v = np.array([c.row(c.v, s, r) for r in at], np.float64).reshape(-1, 2, 64)[:, h // 2]
                sc = k @ q[t, h] / 8
                p = np.exp(sc - sc.max())
                p /= p.sum()
                assert np.all(np.abs(got[t, h] - p @ v) <= 1e-4)
    c.close()


def test_a_token_with_no_rows_gets_zeros(mxh):
    c = Case([(20, 2), (10, 1)], nh=4, nkv=2, hd=32, page=16, seed=6).upload()
    c.bufs["table"].upload(np.full((2, c.ld), -1, np.int32))
    assert np.all(c.attention() == 0)
    c.close()


def test_lengths_below_zero_and_trees_past_64(mxh):
    """cached < 0 counts as 0; token rows past the 64th of a drafted tree are left alone."""
    c = Case([(0, 3), (9, 70)], nh=4, nkv=2, hd=32, page=16, seed=6, tree=True).upload()
    c.bufs["cached"].upload(np.asarray([-5, 9], np.int32))
    got = c.attention()
    assert np.all(got[3 + 64:] == FILL)
    got[3 + 64:] = 0
    c.check(got, rows=set(range(3 + 64)))
    c.close()


LOW, HIGH = -2**31, 2**31 - 1


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("start", [[0, LOW, 9], [5, LOW, LOW], [3, 1, 9], [0, HIGH, 9], [HIGH, HIGH, HIGH], [LOW, LOW, HIGH],
                                   [-4, 2, 9], [0, 0, HIGH], [9, 9, 9], [12, 13, 14], [0, 4, HIGH]])
def test_starts_that_make_no_sense_stay_inside(mxh, start, tree):
    """Falling starts attend nothing; a sequence from below 0 has no tokens; ends past n_tokens end there."""
    c = Case([(40, 4), (20, 5)], nh=4, nkv=2, hd=64, page=16, seed=6, tree=tree).upload()
    c.bufs["start"].upload(np.asarray(start, np.int32))
    got = c.attention()
    falls = any(b < a for a, b in zip(start, start[1:]))
    mine = [range(a, min(b, c.tokens)) if a >= 0 and not falls else [] for a, b in zip(start, start[1:])]
    written = sorted(t for r in mine for t in r)
    left = np.all(got == FILL, axis=(1, 2))
    assert [t for t in range(c.tokens) if not left[t]] == written
    qkv, _, _ = rope_inputs(c, 1)
    dq, df = mxhip.DeviceBuffer.from_array(qkv), mxhip.DeviceBuffer.from_array(mxhip.rope_frequencies(1e4, 64))
    out = mxhip.DeviceBuffer.from_array(np.full((c.tokens, 256), FILL))
    mxhip.qk_rope_append(c.pool, 0, c.batch, dq, 512, None, None, None, 1e-6, df, True, 4, out)
    mxhip.synchronize()
    q = out.download(np.float32).reshape(c.tokens, 256)
    if not falls:
        assert [t for t in range(c.tokens) if np.any(q[t] != FILL)] == written
    # only rows of the two sequences' pages may have changed, none before their cached rows
    pool = c.bufs["k"].download(np.uint16).reshape(-1, 128)
    old = c.k.view(np.uint16).reshape(-1, 128)
    for s, (n_c, _) in enumerate(c.seqs):
        for r in range(n_c):
            assert np.array_equal(c.row(pool.reshape(1, -1), s, r), c.row(old.reshape(1, -1), s, r))
    for b in (dq, df, out):
        b.close()
    c.close()


def test_attention_needs_its_work(mxh):
    c = Case([(5000, 1)], nh=8, nkv=2, hd=128, page=16, seed=1).upload()
    if c.work_bytes:
        for work, n in ((None, 0), (c.bufs["work"], c.work_bytes - 1)):
            with pytest.raises(mxhip.MxhError, match="needed"):
                mxhip.attention_paged(c.pool, 0, c.batch, c.bufs["q"], 8, c.bufs["att"], work, n)
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (32, 8, 64), (3, 1, 32)])
def test_the_largest_batchs_work_is_enough(mxh, nh, nkv, hd):
    """Workspaces grow with n_seq, n_tokens and table_ld, and a small batch runs in a large one's."""
    pool = mxhip.KvPool(1 << 20, 1 << 21, n_layer=1, n_pages=4000, page_rows=16, n_kv=nkv, head_dim=hd)
    size = lambda s, t, ld: mxhip.attention_paged_workspace(  # noqa: E731
        pool, mxhip.KvBatch(s, t, 1 << 20, 1 << 20, 1 << 20, ld, None), nh)
    steps = [(1, 4, 64, 4096), (1, 3, 5, 9, 64, 1000, 1 << 20), (1, 3, 5, 9, 30, 40, 70, 600, 4000)]
    for s in steps[0]:
        for t in steps[1]:
            for ld in steps[2]:
                for up in ((4096, t, ld), (s, 1 << 20, ld), (s, t, 4000)):
                    assert size(s, t, ld) <= size(*up), (s, t, ld, up)
    n = size(300, 1000, 70)
    work = mxhip.DeviceBuffer(n)
    for seqs, tree in (([(900, 1)], False), ([(0, 200)] * 5, False), ([(1000, 40), (3, 9)], True), ([(700, 3)] * 20, True),
                       ([(i, 1) for i in range(300)], False)):
        c = Case(seqs, nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, seed=3, extra_ld=1)
        assert c.ld <= 70 and c.tokens <= 1000
        c.upload()
        mxhip.attention_paged(c.pool, 0, c.batch, c.bufs["q"], nh, c.bufs["att"], work, n)
        mxhip.synchronize()
        c.check(c.bufs["att"].download(np.float32).reshape(c.tokens, nh, hd))
        c.close()
    work.close()


def test_graph_follows_the_lengths(mxh):
    """A recorded step replayed on another stream while lengths, tables and q change, eager work between the replays."""
    a = Case([(900, 1), (10, 1), (3000, 1)], nh=8, nkv=2, hd=128, page=16, seed=21).upload()
    b = Case([(1400, 1), (700, 1), (5, 1)], nh=8, nkv=2, hd=128, page=16, seed=22).upload()
    g = Graph([a.attend])
    for _ in range(3):
        mxhip.memset(a.bufs["att"], 0)
        mxhip.synchronize()
        g.replay()
        got = a.bufs["att"].download(np.float32).reshape(a.tokens, 8, 128)
        a.check(got)
        b.check(b.attention())
        # sequence 2 shortened, sequence 0's last page swapped into sequence 1's place
        a.seqs = [(a.seqs[0][0] - 16, 1), (a.seqs[1][0], 1), (a.seqs[2][0] - 700, 1)]
        for s, (c, _) in enumerate(a.seqs):
            a.row(a.k, s, c)[:] = a.rng.standard_normal(256)
        a.q = (1.5 * a.rng.standard_normal(a.q.shape)).astype(np.float32)
        a.bufs["k"].upload(a.k), a.bufs["q"].upload(a.q)
        a.bufs["cached"].upload(np.asarray([c for c, _ in a.seqs], np.int32))
    g.close()
    a.close(), b.close()


# (cached, new), extra table columns: whole tiles under a wide table and under a tight one, tiles cut with
# some, most or all of a prompt's stages behind its cached rows, items that cross many tiles
PLANS = {
    "whole-wide": ([(0, 90)] * 12 + [(30, 5)], 300),
    "whole-tight": ([(0, 90)] * 12 + [(30, 5)], 0),
    "one-long": ([(2500, 40), (0, 130), (7, 90)], 0),
    "long-ramp": ([(900, 300)], 40),
    "all-ramp": ([(0, 1100)], 0),
    "prompt-among-single-tokens": ([(0, 280)] + [(i % 70, 1) for i in range(150)], 60),
    "prompts-over-64": ([(3 * i, 33) for i in range(70)] + [(1500, 20)], 0),
}


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32", "g1-d128"])
@pytest.mark.parametrize("name", list(PLANS))
def test_whole_and_cut_tiles(mxh, name, heads):
    nh, nkv, hd = HEADS[heads]
    seqs, extra = PLANS[name]
    c = Case(seqs, nh=nh, nkv=nkv, hd=hd, page=32, lead=1, tail=2, seed=nh, extra_ld=extra).upload()
    c.check(c.attention())
    c.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
def test_trees_of_many_sequences(mxh, heads):
    """More trees than a wave has lanes, empty ones among them, one behind a long cache; then the most sequences."""
    nh, nkv, hd = HEADS[heads]
    seqs = [(3 * i % 200, i % 20) for i in range(100)] + [(1500, 30)] + [(7, 64), (0, 1)]
    c = Case(seqs, nh=nh, nkv=nkv, hd=hd, page=16, tree=True, lead=2, tail=1, seed=71, extra_ld=3).upload()
    c.check(c.attention())
    c.close()


def test_4096_sequences(mxh):
    c = Case([(i % 37 if i % 500 else 900, 1 - i % 7 // 6) for i in range(4096)], nh=4, nkv=1, hd=32, page=16, lead=1, seed=72,
             extra_ld=1).upload()
    c.check(c.attention())
    qkv, _, _ = rope_inputs(c, 5)
    run_rope(c, qkv, None, [None, None], mxhip.rope_frequencies(1e4, 32), True)
    c.close()


@pytest.mark.parametrize("shared", [False, True])
def test_batches_larger_than_the_caches(mxh, shared):
    """Single tokens over more than 256 MB of rows, apart and of one prompt: each the same as by itself."""
    nh, nkv, hd, page, n, rows = 16, 4, 128, 64, 40, 4000
    rng = np.random.default_rng(61)
    per = rows // page + 1
    kept = 3500 // page if shared else 0
    table = np.arange(n * per, dtype=np.int32).reshape(n, per)
    table[:, :kept] = table[0, :kept]
    cached = np.asarray([rows - 13 * (i % 9) for i in range(n)], np.int32)
    pages = rng.standard_normal((97, page * nkv * hd)).astype(np.float16)  # page p holds pages[p % 97], V those 5 on
    bufs = [mxhip.DeviceBuffer(n * per * pages[0].nbytes) for _ in range(2)]
    for p in range(n * per):
        bufs[0].upload(pages[p % 97], p * pages[0].nbytes), bufs[1].upload(pages[(p + 5) % 97], p * pages[0].nbytes)
    assert 2 * n * rows * nkv * hd * 2 > 256e6
    pool = mxhip.KvPool(*bufs, n_layer=1, n_pages=n * per, page_rows=page, n_kv=nkv, head_dim=hd)
    q = rng.standard_normal((n, nh * hd)).astype(np.float32)
    put = mxhip.DeviceBuffer.from_array
    dev = [put(np.arange(n + 1, dtype=np.int32)), put(cached), put(table), put(q), put(np.zeros_like(q)), put(np.zeros_like(q)),
           put(np.asarray([0, 1], np.int32))]
    batch = mxhip.KvBatch(n, n, dev[0], dev[1], dev[2], per, None)
    size = mxhip.attention_paged_workspace(pool, batch, nh)
    work = mxhip.DeviceBuffer(max(size, 1))
    mxhip.attention_paged(pool, 0, batch, dev[3], nh, dev[4], work, size)
    for i in range(n):
        one = mxhip.KvBatch(1, 1, dev[6], dev[1].ptr + 4 * i, dev[2].ptr + 4 * i * per, per, None)
        mxhip.attention_paged(pool, 0, one, dev[3].ptr + 4 * i * nh * hd, nh, dev[5].ptr + 4 * i * nh * hd, work, size)
    mxhip.synchronize()
    got, alone = (b.download(np.float32).reshape(n, nh, hd) for b in dev[4:6])
    for i in range(0, n, 3):
        r = np.arange(cached[i] + 1)
        p = table[i, r // page]
        k = pages[p % 97].reshape(-1, page, nkv, hd)[r, r % page].astype(np.float64)
        v = pages[(p + 5) % 97].reshape(-1, page, nkv, hd)[r, r % page].astype(np.float64)
        for h in range(nh):
            x, kk, vv = q[i, h * hd:(h + 1) * hd].astype(np.float64), k[:, h // 4], v[:, h // 4]
            sc = kk @ x / np.sqrt(hd)
            e = np.exp(sc - sc.max())
            e /= e.sum()
            d = (2.0**-21 + 2 * hd * U) * (np.abs(kk) @ np.abs(x)).max() / np.sqrt(hd)
            bound = (2 * d + 2.0**-20 + 2 * len(r) * U) * (e @ np.abs(vv))
            for y in (got[i, h], alone[i, h]):
                assert np.all(np.abs(y - e @ vv) <= bound), (i, h)
    for b in [*bufs, *dev, work]:
        b.close()


def test_graph_goes_from_cut_to_whole_tiles(mxh):
    """One recorded call while a sequence's cached rows go from many to none and back."""
    c = Case([(2000, 100), (3, 60), (0, 1)], nh=8, nkv=2, hd=64, page=16, seed=41).upload()
    g = Graph([c.attend])
    for cached in (2000, 0, 777, 2000):
        c.seqs[0] = (cached, 100)
        c.bufs["cached"].upload(np.asarray([cached, 3, 0], np.int32))
        mxhip.memset(c.bufs["att"], 0)
        mxhip.synchronize()
        g.replay()
        c.check(c.bufs["att"].download(np.float32).reshape(c.tokens, 8, 64))
        c.check(c.attention())
    g.close()
    c.close()


# ---- norms, rotation, append -----------------------------------------------------------------


def rope_inputs(c, seed, ld_extra=0, big=False):
    rng = np.random.default_rng(seed)
    width = (c.nh + 2 * c.nkv) * c.hd
    qkv = rng.standard_normal((c.tokens, width + ld_extra)).astype(np.float32)
    if big:
        qkv *= np.exp(rng.uniform(-12, 6, (c.tokens, 1))).astype(np.float32)
    return qkv, rng.standard_normal(width).astype(np.float32), (1 + 0.3 * rng.standard_normal((2, c.hd))).astype(np.float32)


def rope_expected(c, qkv, bias, w, eps, freq, neox):
    """(q, k, v and their bounds) [tokens][heads][hd] in float64; positions by the tokens' paths."""
    nh, nkv, hd = c.nh, c.nkv, c.hd
    x = qkv[:, :(nh + 2 * nkv) * hd].astype(np.float64)
    if bias is not None:
        x = x + bias
    x = x.reshape(c.tokens, -1, hd)
    pos = np.zeros(c.tokens)
    for s, (n_c, n) in enumerate(c.seqs):
        for i in range(n):
            pos[c.start[s] + i] = n_c + len(c.before(s, i)) - 1
    ang = pos[:, None, None] * freq
    cs, sn = np.cos(ang), np.sin(ang)
    out, bound = [], []
    for part, g in ((x[:, :nh], w[0]), (x[:, nh:nh + nkv], w[1])):
        y = part
        if g is not None:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * g
        a, b = (y[..., :hd // 2], y[..., hd // 2:]) if neox else (y[..., 0::2], y[..., 1::2])
        r0, r1, m = a * cs - b * sn, a * sn + b * cs, 4 * U * (np.abs(a) + np.abs(b))
        out.append(np.concatenate([r0, r1], -1) if neox else np.stack([r0, r1], -1).reshape(y.shape))
        bound.append(np.concatenate([m, m], -1) if neox else np.stack([m, m], -1).reshape(y.shape))
    return out + [x[:, nh + nkv:]], bound + [U * np.abs(x[:, nh + nkv:])]


@pytest.mark.parametrize("neox", [False, True], ids=["adjacent", "neox"])
@pytest.mark.parametrize("norm,bias", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", ["one", "empty-among", "prompts", "trees"])
def test_rope_append_matches_float64(mxh, name, heads, norm, bias, neox):
    nh, nkv, hd = HEADS[heads]
    tree = name in TREES
    c = Case((TREES if tree else SETS)[name], nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, lead=1, tail=2, layers=2,
             layer=1, seed=nh, extra_ld=1).upload()
    qkv, b, w = rope_inputs(c, 3, ld_extra=4, big=norm)
    run_rope(c, qkv, b if bias else None, list(w) if norm else [None, None], mxhip.rope_frequencies(1e4, hd), neox)
    c.close()


def run_rope(c, qkv, bias, w, freq, neox, eps=1e-6):
    put = lambda a: None if a is None else mxhip.DeviceBuffer.from_array(a)  # noqa: E731
    bufs = [put(a) for a in (qkv, bias, w[0], w[1], freq, np.full((c.tokens, c.nh * c.hd), FILL))]
    mxhip.qk_rope_append(c.pool, c.layer, c.batch, bufs[0], qkv.shape[1], bufs[1], bufs[2], bufs[3], eps, bufs[4], neox,
                         c.nh, bufs[5])
    mxhip.synchronize()
    q = bufs[5].download(np.float32).reshape(c.tokens, c.nh, c.hd)
    pools = [c.bufs[n].download(np.float16).reshape(c.k.shape) for n in ("k", "v")]
    want, bound = rope_expected(c, qkv, bias, w, eps, freq, neox)
    inside = np.zeros(c.tokens, bool)
    inside[c.start[0]:c.start[-1]] = True
    assert np.all(q[~inside] == FILL)
    assert np.all(np.abs(q[inside] - want[0][inside]) <= bound[0][inside] + 2.0**-140)
    for pool, old, x, m in ((pools[0], c.k, want[1], bound[1]), (pools[1], c.v, want[2], bound[2])):
        left = old.copy()
        for s, (n_c, n) in enumerate(c.seqs):
            for i in range(n):
                t = int(c.start[s]) + i
                got, y = c.row(pool, s, n_c + i).astype(np.float64), x[t].reshape(-1)
                assert np.all(np.abs(got - y) <= (m[t].reshape(-1) + np.abs(y)) * 2.0**-11 + m[t].reshape(-1) + 2.0**-25)
                c.row(left, s, n_c + i)[:] = c.row(pool, s, n_c + i)
        assert np.array_equal(pool.view(np.uint16), left.view(np.uint16)), "other rows were written"
    for b in bufs:
        if b is not None:
            b.close()


def test_rope_far_positions(mxh):
    """Angles of positions up to a million, the fastest pair turning once a token."""
    c = Case([(3, 2)], nh=4, nkv=2, hd=128, page=16, seed=9, extra_ld=70000).upload()
    n = 1 << 20
    table = np.full((1, c.ld), -1, np.int32)
    table[0, n // 16] = c.table[0, 0]
    c.bufs["table"].upload(table), c.bufs["cached"].upload(np.asarray([n + 3], np.int32))
    qkv, _, _ = rope_inputs(c, 1)
    freq = mxhip.rope_frequencies(1e6, 128)
    out = mxhip.DeviceBuffer(4 * c.tokens * 512)
    dq, df = mxhip.DeviceBuffer.from_array(qkv), mxhip.DeviceBuffer.from_array(freq)
    mxhip.qk_rope_append(c.pool, 0, c.batch, dq, 1024, None, None, None, 1e-6, df, True, 4, out)
    mxhip.synchronize()
    c.seqs = [(n + 3, 2)]
    want, bound = rope_expected(c, qkv, None, [None, None], 0, freq, True)
    got = out.download(np.float32).reshape(2, 4, 128)
    assert np.all(np.abs(got - want[0]) <= bound[0] + 2.0**-30 * np.abs(qkv[:, :512].reshape(2, 4, 128)).max())
    k = c.bufs["k"].download(np.float16).reshape(-1, 2, 128)
    at = int(c.table[0, 0]) * 16 + 3
    assert np.all(np.abs(k[at:at + 2] - want[1]) <= np.abs(want[1]) * 2.0**-11 + bound[1] + 2.0**-25)
    for b in (out, dq, df):
        b.close()
    c.close()


def test_rope_without_a_page_still_rotates_q(mxh):
    c = Case([(20, 3)], nh=4, nkv=2, hd=64, page=16, seed=9).upload()
    c.bufs["table"].upload(np.full((1, c.ld), -1, np.int32))
    qkv, _, _ = rope_inputs(c, 1)
    freq = mxhip.rope_frequencies(1e4, 64)
    out = mxhip.DeviceBuffer(4 * 3 * 256)
    dq, df = mxhip.DeviceBuffer.from_array(qkv), mxhip.DeviceBuffer.from_array(freq)
    mxhip.qk_rope_append(c.pool, 0, c.batch, dq, 512, None, None, None, 1e-6, df, False, 4, out)
    mxhip.synchronize()
    want, bound = rope_expected(c, qkv, None, [None, None], 0, freq, False)
    assert np.all(np.abs(out.download(np.float32).reshape(3, 4, 64) - want[0]) <= bound[0])
    assert np.array_equal(c.bufs["k"].download(np.uint16), c.k.view(np.uint16).reshape(-1))
    assert np.array_equal(c.bufs["v"].download(np.uint16), c.v.view(np.uint16).reshape(-1))
    for b in (out, dq, df):
        b.close()
    c.close()


# ---- moving rows --------------------------------------------------------------------------------


def filled(layers, n_pages, page, nkv, hd, stride=0, seed=0):
    rng = np.random.default_rng(seed)
    n = n_pages * page * nkv * hd + stride
    k, v = (rng.integers(0, 65536, (layers, n)).astype(np.uint16) for _ in range(2))
    bufs = [mxhip.DeviceBuffer.from_array(x) for x in (k, v)]
    pool = mxhip.KvPool(*bufs, n_layer=layers, n_pages=n_pages, page_rows=page, n_kv=nkv, head_dim=hd,
                        layer_stride=n if stride else 0)
    return k, v, bufs, pool


@pytest.mark.parametrize("layers,n_pages,page,nkv,hd,pairs,stride",
                         [(1, 2, 16, 1, 32, 1, 0), (3, 40, 16, 2, 64, 13, 8), (2, 1100, 16, 1, 32, 500, 0),
                          (2, 5, 128, 8, 128, 2, 1024), (1, 9, 1024, 3, 32, 4, 0)])
def test_copied_pages(mxh, layers, n_pages, page, nkv, hd, pairs, stride):
    k, v, bufs, pool = filled(layers, n_pages, page, nkv, hd, stride)
    ids = np.random.default_rng(1).permutation(n_pages)[:2 * pairs]
    src, dst = ids[:pairs], ids[pairs:]
    src = np.where(np.arange(pairs) % 3 == 2, src[0], src)  # a page may be copied to several
    mxhip.kv_copy_pages(pool, src, dst)
    mxhip.synchronize()
    n = page * nkv * hd
    for old, b in ((k, bufs[0]), (v, bufs[1])):
        want = old.copy()
        for s, d in zip(src, dst):
            want[:, d * n:(d + 1) * n] = old[:, s * n:(s + 1) * n]
        assert np.array_equal(b.download(np.uint16).reshape(want.shape), want)
        b.close()


def test_copies_larger_than_the_caches(mxh):
    test_copied_pages(mxh, 3, 91, 256, 8, 128, 45, 8)  # 283 MB read and written


@pytest.mark.parametrize("layers,page,nkv,hd,stride,kept", [
    (1, 16, 1, 32, 0, {0: (5, [1])}),
    (3, 16, 2, 64, 16, {0: (14, [0, 3, 4, 9]), 1: (40, []), 2: (0, [2, 3, 4]), 3: (7, [0, 1, 2])}),
    (2, 32, 8, 128, 0, {0: (100, list(range(3, 60))), 1: (31, [63])}),
    (2, 16, 1, 32, 0, {s: (s, list(range(1, 60, 1 + s % 5))) for s in range(40)}),  # several launches
    (1, 16, 1, 32, 0, {0: (3, list(range(1, 701)))}),  # one sequence over launches
])
def test_kept_rows(mxh, layers, page, nkv, hd, stride, kept):
    n_seq = len(kept)
    need = [(c + max(rows + [0])) // page + 1 for c, rows in kept.values()]
    rng = np.random.default_rng(2)
    ids = rng.permutation(sum(need) + 2).astype(np.int32)
    k, v, bufs, pool = filled(layers, len(ids), page, nkv, hd, stride)
    table = np.full((n_seq, max(need)), -7, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    cached = [c for c, _ in kept.values()]
    start = np.concatenate([[0], np.cumsum([len(r) for _, r in kept.values()])])
    keep = np.concatenate([r for _, r in kept.values()])
    mxhip.kv_keep_rows(pool, table, cached, start, keep)
    mxhip.synchronize()
    w = nkv * hd
    for old, b in ((k, bufs[0]), (v, bufs[1])):
        want = old.copy()
        for s, (c, rows) in kept.items():
            for i, r in enumerate(rows):
                to, frm = ((table[s, x // page] * page + x % page) * w for x in (c + i, c + r))
                want[:, to:to + w] = old[:, frm:frm + w]
        assert np.array_equal(b.download(np.uint16).reshape(want.shape), want)
        b.close()


# ---- a run of them together ------------------------------------------------------------------------


def test_a_recorded_step_holds_its_lists(mxh):
    """Append, attention of trees, copy and kept rows in one graph: the host lists may go, device arrays are followed."""
    nh, nkv, hd, page = 8, 2, 128, 16
    c = Case([(30, 20), (100, 9)], nh=nh, nkv=nkv, hd=hd, page=page, tree=True, seed=51, spare=4).upload()
    qkv, b, w = rope_inputs(c, 7)
    freq = mxhip.rope_frequencies(1e4, hd)
    put = mxhip.DeviceBuffer.from_array
    dev = [put(qkv), put(b), put(w[0]), put(w[1]), put(freq)]
    spare = sorted(set(range(c.n_pages)) - set(c.table[c.table >= 0].tolist()))
    src, dst = np.asarray([c.table[0, 0], c.table[1, 3]], np.int32), np.asarray(spare[:2], np.int32)
    cached = np.asarray([30, 100], np.int32)
    keep, keep_start, table = np.asarray([1, 4, 19, 0, 8], np.int32), np.asarray([0, 3, 5], np.int32), c.table.copy()
    g = Graph([lambda: mxhip.qk_rope_append(c.pool, 0, c.batch, dev[0], qkv.shape[1], dev[1], dev[2], dev[3], 1e-6,
                                            dev[4], True, nh, c.bufs["q"]),
               c.attend,
               lambda: mxhip.kv_copy_pages(c.pool, src, dst),
               lambda: mxhip.kv_keep_rows(c.pool, table, cached, keep_start, keep)])
    kept = [(0, [1, 4, 19]), (1, [0, 8])]
    moved = list(zip(src.tolist(), dst.tolist()))
    src[:], dst[:], cached[:], keep[:], keep_start[:], table[:] = 0, 0, 0, 0, 0, -1
    rows = page * nkv * hd
    for r in range(3):
        if r == 2:
            c.parents = [bush(n, c.rng) for _, n in c.seqs]
            c.bufs["parent"].upload(c.parent_array())
        c.bufs["k"].upload(c.k), c.bufs["v"].upload(c.v)
        mxhip.memset(c.bufs["att"], 0)
        mxhip.synchronize()
        g.replay()
        got = c.bufs["att"].download(np.float32).reshape(c.tokens, nh, hd)
        after = [c.bufs[n].download(np.float16) for n in ("k", "v")]
        # the same step eagerly, call by call
        c.bufs["k"].upload(c.k), c.bufs["v"].upload(c.v)
        mxhip.qk_rope_append(c.pool, 0, c.batch, dev[0], qkv.shape[1], dev[1], dev[2], dev[3], 1e-6, dev[4], True, nh,
                             c.bufs["q"])
        assert np.array_equal(c.attention(), got)
        for n, x in zip(("k", "v"), after):
            want = c.bufs[n].download(np.uint16).reshape(1, -1)
            for a, z in moved:
                want[0, z * rows:(z + 1) * rows] = want[0, a * rows:(a + 1) * rows]
            old = want.copy()
            for s, new in kept:
                for i, j in enumerate(new):
                    c.row(want, s, c.seqs[s][0] + i)[:] = c.row(old, s, c.seqs[s][0] + j)
            assert np.array_equal(x.view(np.uint16), want.reshape(-1)), (r, n)
    g.close()
    for x in dev:
        x.close()
    c.close()


def test_offsets_past_32_bits(mxh):
    """Rows more than 2^32 bytes and 2^31 elements into a layer: appended, attended, copied, kept."""
    nh, nkv, hd, page, far = 16, 8, 128, 256, 9000
    n_pages = far + 3
    bufs = [mxhip.DeviceBuffer(n_pages * page * nkv * hd * 2) for _ in range(2)]
    pool = mxhip.KvPool(*bufs, n_layer=1, n_pages=n_pages, page_rows=page, n_kv=nkv, head_dim=hd)
    rng = np.random.default_rng(5)
    pages, row = [far + 1, 2, far], nkv * hd  # of the sequence
    cached, n = 2 * page + 20, 12
    kv = rng.standard_normal((2, 3 * page, row)).astype(np.float16)
    for b, x in zip(bufs, kv):
        for i, p in enumerate(pages):
            b.upload(x[i * page:(i + 1) * page], p * page * row * 2)
    qkv = rng.standard_normal((n, (nh + 2 * nkv) * hd)).astype(np.float32)
    up = mxhip.DeviceBuffer.from_array
    dev = [up(np.asarray(x, np.int32)) for x in ([0, n], [cached], pages)] + [up(qkv), up(np.zeros(hd // 2)),
                                                                            up(np.zeros((2, n, nh * hd), np.float32))]
    batch = mxhip.KvBatch(1, n, *dev[:3], 3)
    q, att = dev[5].ptr, dev[5].ptr + 4 * n * nh * hd
    mxhip.qk_rope_append(pool, 0, batch, dev[3], qkv.shape[1], None, None, None, 1e-6, dev[4], True, nh, q)
    work = mxhip.DeviceBuffer(max(mxhip.attention_paged_workspace(pool, batch, nh), 1))
    mxhip.attention_paged(pool, 0, batch, q, nh, att, work, work.nbytes)
    mxhip.kv_copy_pages(pool, [far], [far + 2])
    mxhip.kv_keep_rows(pool, np.asarray([pages], np.int32), [cached], [0, 3], [1, 5, 11])
    mxhip.synchronize()
    new = qkv[:, nh * hd:].astype(np.float16).reshape(n, 2, row)  # (frequencies 0: nothing turns)
    kv[:, cached:cached + n] = new.transpose(1, 0, 2)
    copied = kv[:, 2 * page:].copy()
    for b, x in zip(bufs, copied):
        assert np.array_equal(b.download(np.float16, page * row, (far + 2) * page * row * 2), x.reshape(-1))
    kept = kv.copy()
    kept[:, cached:cached + 3] = kv[:, cached + np.asarray([1, 5, 11])]
    for b, x in zip(bufs, kept):
        for i, p in enumerate(pages):
            assert np.array_equal(b.download(np.float16, page * row, p * page * row * 2), x[i * page:(i + 1) * page].reshape(-1))
    got = dev[5].download(np.float32).reshape(2, n, nh, hd)[1]
    k, v = (x.astype(np.float64).reshape(-1, nkv, hd) for x in kv)
    for i in range(n):
        for h in range(nh):
            sc = k[:cached + i + 1, h // 2] @ qkv[i, h * hd:(h + 1) * hd].astype(np.float64) / np.sqrt(hd)
            e = np.exp(sc - sc.max())
            assert np.all(np.abs(got[i, h] - e / e.sum() @ v[:cached + i + 1, h // 2]) <= 1e-4)
    for b in [*bufs, *dev, work]:
        b.close()


def test_drafting_forking_and_keeping(mxh):
    """Two steps of two forked sequences over three layers: reserve, copy on write, append, attend, keep the accepted
    paths; then the next step's attention sees exactly the kept rows, at the positions of a chain."""
    nh, nkv, hd, page, layers = 8, 2, 64, 16, 3
    rng = np.random.default_rng(77)
    width, kvd, theta = (nh + 2 * nkv) * hd, nkv * hd, 1e4
    freq = mxhip.rope_frequencies(theta, hd)
    n_pages = 40
    nan = np.full((layers, n_pages * page * kvd), np.nan, np.float16)
    dk, dv = (mxhip.DeviceBuffer.from_array(nan) for _ in range(2))
    pool = mxhip.KvPool(dk, dv, n_layer=layers, n_pages=n_pages, page_rows=page, n_kv=nkv, head_dim=hd)
    book = mxhip.Pages(n_pages, page, 4)
    df = mxhip.DeviceBuffer.from_array(freq)
    rows: dict[int, list] = {}  # sequence -> per row [layers] of (k, v) in float64, rotated, fp16-rounded

    def rotate(x, pos):
        ang = pos * freq
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return np.concatenate([a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)], -1)

    def step(seqs, parents, accept):
        copies = [c for s, p in zip(seqs, parents) for c in book.extend(s, len(p))]
        mxhip.kv_copy_pages(pool, [a for a, _ in copies], [b for _, b in copies])
        table, cached = book.table(seqs, 12)
        start = np.concatenate([[0], np.cumsum([len(p) for p in parents])]).astype(np.int32)
        tokens = int(start[-1])
        tree = any(p != chain(len(p)) for p in parents)
        dev = [mxhip.DeviceBuffer.from_array(x) for x in
               (start, cached, table, np.concatenate(parents).astype(np.int32))]
        batch = mxhip.KvBatch(len(seqs), tokens, dev[0], dev[1], dev[2], 12, dev[3] if tree else None)
        dq, datt = mxhip.DeviceBuffer(4 * tokens * nh * hd), mxhip.DeviceBuffer(4 * tokens * nh * hd)
        work_bytes = mxhip.attention_paged_workspace(pool, batch, nh)
        work = mxhip.DeviceBuffer(work_bytes)
        new = {s: [[None] * layers for _ in p] for s, p in zip(seqs, parents)}
        for layer in range(layers):
            qkv = rng.standard_normal((tokens, width)).astype(np.float32)
            dqkv = mxhip.DeviceBuffer.from_array(qkv)
            mxhip.qk_rope_append(pool, layer, batch, dqkv, width, None, None, None, 1e-6, df, True, nh, dq)
            mxhip.attention_paged(pool, layer, batch, dq, nh, datt, work, work_bytes)
            mxhip.synchronize()
            att = datt.download(np.float32).reshape(tokens, nh, hd)
            x = qkv.astype(np.float64).reshape(tokens, -1, hd)
            for b, (s, p) in enumerate(zip(seqs, parents)):
                for i in range(len(p)):
                    on = path(p, i)[::-1]
                    pos = len(rows[s]) + len(on) - 1
                    t = start[b] + i
                    new[s][i][layer] = (rotate(x[t, nh:nh + nkv], pos).astype(np.float16).astype(np.float64),
                                        x[t, nh + nkv:].astype(np.float16).astype(np.float64))
                    kv = [r[layer] for r in rows[s]] + [new[s][j][layer] for j in on]
                    q = rotate(x[t, :nh], pos)
                    for h in range(nh):
                        k, v = (np.array([r[c][h // (nh // nkv)] for r in kv]) for c in (0, 1))
                        sc = k @ q[h] / np.sqrt(hd)
                        pr = np.exp(sc - sc.max())
                        # k's fp16 rounding may fall the other way: 2^-11 of k in a score and in v
                        assert np.all(np.abs(att[t, h] - pr @ v / pr.sum()) <= 2e-2), (s, i, layer, h)
            dqkv.close()
        keep_start = np.concatenate([[0], np.cumsum([len(a) for a in accept])])
        mxhip.kv_keep_rows(pool, table, cached, keep_start, np.concatenate(accept).astype(np.int32))
        for s, a in zip(seqs, accept):
            rows[s] += [new[s][i] for i in a]
            book.set_length(s, len(rows[s]))
        mxhip.synchronize()
        for b in dev + [dq, datt, work]:
            b.close()

    a = book.open()
    rows[a] = []
    step([a], [chain(21)], [list(range(21))])
    b = book.fork(a)
    rows[b] = list(rows[a])
    step([a, b], [[-1, 0, 0, 1, 2, 4], [-1, -1, 1, 1, 3]], [[0, 2, 4, 5], [1, 3]])
    step([b, a], [[-1, 0, 1, 0], [-1, 0, 0, 2, 1, 3, 5, 5, 7]], [[0, 3], [0, 2, 3, 5, 7]])
    step([a, b], [[-1], [-1]], [[0], [0]])
    # the cache holds exactly the kept rows
    for s in (a, b):
        table, cached = book.table([s], 12)
        assert cached[0] == len(rows[s])
        for buf, c in ((dk, 0), (dv, 1)):
            got = buf.download(np.float16).reshape(layers, -1, nkv, hd).astype(np.float64)
            for r, kv in enumerate(rows[s]):
                for layer in range(layers):
                    x = got[layer, table[0, r // page] * page + r % page]
                    assert np.all(np.abs(x - kv[layer][c]) <= 2.0**-10 * np.abs(kv[layer][c]) + 2.0**-20)
    book.release(a), book.release(b)
    assert book.free == n_pages
    for buf in (dk, dv, df):
        buf.close()
