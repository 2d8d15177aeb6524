"""Long contexts by blocks of rows (GPU): bounds of keys, chosen blocks, attention over them.

- Bounds are the least and greatest of fp16 values: equal bits but for the sign of
  zero.
- Chosen blocks are compared as whole numbers with the definition in float64 (its
  own sums are off by 2^-45 of a score at most; no two different blocks' scores of
  these inputs are that near, which the test checks).
- Attention over chosen rows has the formula and the bound of attention over the
  paged cache (test_paged_gpu.py) for the rows that are listed.
"""
from __future__ import annotations

import numpy as np
import pytest

import mxhip
from test_graph_capture_gpu import Graph
from test_paged_edges_gpu import check_precision
from test_paged_gpu import FILL, HEADS, SETS, TREES, U, Case

pytestmark = pytest.mark.gpu

LEFT = -77  # lists before a call


class Blocks(Case):
    """A Case with blocks of `block` rows."""

    def __init__(self, seqs, *, block, first=1, last=2, select=6, **kw):
        super().__init__(seqs, **kw)
        self.block, self.first, self.last, self.select = block, first, last, select
        self.shape = (self.k.shape[0], self.n_pages, self.page // block, self.nkv, 2, self.hd)
        self.bounds = np.full(self.shape, 9.5, np.float16)
        self.chosen = np.full((self.tokens, self.nkv, select), LEFT, np.int32)

    def place(self, s, b):
        """Page and block of the page."""
        return int(self.table[s, b * self.block // self.page]), b * self.block % self.page // self.block

    def keys(self, s, b, rows):
        """Rows of block b, of `rows` that the sequence has."""
        at = range(b * self.block, min((b + 1) * self.block, rows))
        return np.array([self.row(self.k, s, r) for r in at]).reshape(-1, self.nkv, self.hd)

    def fill_bounds(self):
        """What all rows of the sequences make."""
        for s, (c, n) in enumerate(self.seqs):
            for b in range(-(-(c + n) // self.block)):
                p, x = self.place(s, b)
                k = self.keys(s, b, c + n)
                self.bounds[self.layer, p, x, :, 0] = np.fmin.reduce(k, 0)
                self.bounds[self.layer, p, x, :, 1] = np.fmax.reduce(k, 0)

    def random_lists(self, rng):
        """Sets of blocks in any order: some twice, some of no block, some behind the token's own."""
        for s, (c, n) in enumerate(self.seqs):
            for i in range(n):
                own = (c + i) // self.block
                for g in range(self.nkv):
                    x = rng.integers(-2, own + 4, self.select)
                    if rng.random() < 0.8:
                        x[rng.integers(0, self.select)] = own
                    self.chosen[int(self.start[s]) + i, g] = x

    def upload(self):
        super().upload()
        b = self.bufs
        b["bounds"] = mxhip.DeviceBuffer.from_array(self.bounds)
        b["chosen"] = mxhip.DeviceBuffer.from_array(self.chosen)
        self.what = mxhip.KvBlocks(b["bounds"], block_rows=self.block, n_first=self.first, n_last=self.last,
                                   n_select=self.select)
        n = mxhip.kv_select_workspace(self.pool, self.batch, self.what, self.nh)
        b["s_work"], self.s_bytes = mxhip.DeviceBuffer(max(n, 16)), n
        n = mxhip.attention_blocks_workspace(self.pool, self.batch, self.what, self.nh)
        if b["work"] is not None:
            b["work"].close()
        b["work"], self.work_bytes = mxhip.DeviceBuffer(max(n, 16)), n
        for w in ("work", "s_work"):
            mxhip.memset(b[w], 0x7f)
        return self

    def find_bounds(self):
        mxhip.kv_block_bounds(self.pool, self.layer, self.batch, self.what)

    def choose(self):
        b = self.bufs
        mxhip.kv_select_blocks(self.pool, self.layer, self.batch, self.what, b["q"], self.nh, b["chosen"], b["s_work"],
                               self.s_bytes)

    def attend(self):
        b = self.bufs
        mxhip.attention_blocks(self.pool, self.layer, self.batch, self.what, b["chosen"], b["q"], self.nh, b["att"],
                               b["work"], self.work_bytes)

    def got_bounds(self):
        mxhip.synchronize()
        return self.bufs["bounds"].download(np.float16).reshape(self.shape)

    def got_chosen(self):
        mxhip.synchronize()
        return self.bufs["chosen"].download(np.int32).reshape(self.chosen.shape)

    def check_bounds(self, got):
        want = self.bounds.copy()
        for s, (c, n) in enumerate(self.seqs):
            for b in range(c // self.block, -(-(c + n) // self.block) if n else 0):
                p, x = self.place(s, b)
                k = self.keys(s, b, c + n)
                want[self.layer, p, x, :, 0] = np.fmin.reduce(k, 0)
                want[self.layer, p, x, :, 1] = np.fmax.reduce(k, 0)
        assert np.array_equal(got, want, equal_nan=True)

    def scores(self, s, t, nb):
        """[kv heads, blocks] of a token, in float64; -inf where the page is absent."""
        q = self.q[t].astype(np.float64).reshape(self.nkv, -1, self.hd)
        out = np.full((self.nkv, nb), -np.inf)
        for b in range(nb):
            p, x = self.place(s, b)
            if 0 <= p < self.n_pages:
                bd = self.bounds[self.layer, p, x].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    v = (np.maximum(q, 0) * bd[:, None, 1] + np.minimum(q, 0) * bd[:, None, 0]).sum(-1)
                    out[:, b] = np.where(np.isnan(v).any(1), np.inf, v.max(1))
        return out

    def check_chosen(self, got, near=0):
        want = np.full_like(self.chosen, LEFT)
        for s, (c, n) in enumerate(self.seqs):
            for i in range(min(n, 64) if self.tree else n):
                t, own = int(self.start[s]) + i, (c + i) // self.block
                own = min(own, self.ld * self.page // self.block - 1)
                want[t] = -1
                if own < self.select:
                    want[t, :, :own + 1] = np.arange(own + 1)
                    continue
                k = self.select - self.first - self.last
                score = self.scores(s, t, own + 1)
                for g in range(self.nkv):
                    rivals = np.arange(self.first, own + 1 - self.last)
                    order = rivals[np.argsort(-score[g, rivals], kind="stable")]
                    if 0 < k:
                        a, b = score[g, order[k - 1]], score[g, order[k]]
                        if a != b and abs(a - b) <= 2.0**-40 * abs(a):
                            near -= 1
                    want[t, g] = np.sort(np.concatenate([np.arange(self.first), order[:k],
                                                         np.arange(own + 1 - self.last, own + 1)]))
        assert near >= 0, "scores of these inputs lie next to one another"
        assert np.array_equal(got, want)

    def check_listed(self, got, lists, rows=None):
        """att against float64 over the listed rows, with the bound of the module's docstring."""
        nh, nkv, hd = self.nh, self.nkv, self.hd
        group = nh // nkv
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
                at = np.array(list(range(c)) + [c + j for j in self.before(s, i)])
                for g in range(nkv):
                    on = at[np.isin(at // self.block, lists[t, g])]
                    for h in range(g * group, (g + 1) * group):
                        if on.size == 0:
                            assert np.all(got[t, h] == 0)
                            continue
                        kk, vv = k[on, g], v[on, g]
                        sc = kk @ q[t, h] / np.sqrt(hd)
                        p = np.exp(sc - sc.max())
                        p /= p.sum()
                        d = (2.0**-21 + 2 * hd * U) * (np.abs(kk) @ np.abs(q[t, h])).max() / np.sqrt(hd)
                        bound = (2 * d + 2.0**-20 + 2 * on.size * U) * (p @ np.abs(vv)) + 2.0**-100
                        err = np.abs(got[t, h] - p @ vv)
                        assert np.all(err <= bound), f"seq {s} token {i} head {h}: {float((err / bound).max()):.3g}"
        assert np.all(got[~inside] == FILL), "rows outside the sequences were written"


SIZES = [(16, 16), (64, 32), (128, 64), (256, 128)]  # rows of a page, of a block
LONG = {
    "decode": [(400, 1), (1000, 1), (0, 1), (255, 1), (256, 1), (90, 1)],
    "one": [(2100, 1)],
    "chunks": [(500, 21), (0, 40), (777, 3), (130, 5)],
    "empty-among": [(600, 2), (5, 0), (300, 9)],
    "prompt": [(0, 300)],
}
DRAFTS = {
    "trees": [(530, 7), (600, 64), (64, 16), (950, 33)],
}


def case(name, heads, size, seed=0, cls=Blocks, **kw):
    nh, nkv, hd = HEADS[heads]
    seqs = {**SETS, **TREES, **LONG, **DRAFTS}[name]
    a = dict(nh=nh, nkv=nkv, hd=hd, page=size[0], block=size[1], tree=name in TREES or name in DRAFTS, lead=2, tail=3,
             seed=seed + 13 * len(name) + nh, extra_ld=2)
    return cls(seqs, **{**a, **kw})


@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}-{s[1]}")
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", list(SETS) + list(TREES) + ["chunks"])
def test_bounds(mxh, name, heads, size):
    c = case(name, heads, size).upload()
    c.find_bounds()
    c.check_bounds(c.got_bounds())
    c.close()


def test_bounds_in_a_layer_of_strided_pools(mxh):
    c = Blocks([(70, 3), (10, 90), (64, 1)], block=16, nh=12, nkv=6, hd=64, page=32, layers=3, layer=1, stride=24, seed=5)
    dense = int(np.prod(c.shape[1:]))
    c.upload()
    wide = np.full((3, dense + 40), 9.5, np.float16)
    b = mxhip.DeviceBuffer.from_array(wide)
    c.what = mxhip.KvBlocks(b, block_rows=16, layer_stride=dense + 40)
    c.find_bounds()
    mxhip.synchronize()
    got = b.download(np.float16).reshape(wide.shape)
    assert np.all(got[:, dense:] == 9.5)
    c.check_bounds(got[:, :dense].reshape(c.shape))
    b.close()
    c.close()


def test_bounds_of_many_heads(mxh):
    """Rows of more pieces than a workgroup takes at a time, and of a number that is no power of two."""
    for nkv in (13, 40):
        c = Blocks([(30, 5), (0, 1)], block=32, nh=nkv, nkv=nkv, hd=128, page=32, seed=nkv).upload()
        c.find_bounds()
        c.check_bounds(c.got_bounds())
        c.close()


def test_bounds_pass_nan_over(mxh):
    c = Blocks([(20, 30), (40, 1)], block=16, nh=4, nkv=2, hd=32, page=16, seed=6)
    c.row(c.k, 0, 33)[::3] = np.nan
    c.row(c.k, 0, 34)[::5] = np.inf
    c.row(c.k, 0, 35)[1::5] = -np.inf
    c.upload()
    c.find_bounds()
    c.check_bounds(c.got_bounds())
    c.close()


def test_bounds_of_absent_pages_are_left_out(mxh):
    c = Blocks([(20, 30), (40, 1)], block=16, nh=4, nkv=2, hd=32, page=16, seed=6)
    gone, c.table[0, 2] = c.table[0, 2], c.n_pages
    c.upload()
    c.find_bounds()
    got = c.got_bounds()
    c.table[0, 2] = gone
    assert np.all(got[0, gone] == 9.5)
    got[0, gone, 0, :, 0] = np.fmin.reduce(c.keys(0, 2, 50), 0)
    got[0, gone, 0, :, 1] = np.fmax.reduce(c.keys(0, 2, 50), 0)
    c.check_bounds(got)
    c.close()


@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}-{s[1]}")
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", list(LONG) + list(DRAFTS))
def test_chosen_blocks(mxh, name, heads, size):
    c = case(name, heads, size)
    c.fill_bounds()
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", ["chunks", "empty-among", "prompt", "trees"])
@pytest.mark.parametrize("size", [(16, 16), (128, 64)], ids=lambda s: f"{s[0]}-{s[1]}")
def test_chosen_blocks_in_tiles(mxh, name, heads, size):
    """Rows of the table wide enough that tokens share tiles (1.5 times 64 blocks of a token and kv head a CU)."""
    c = case(name, heads, size, extra_ld=2500 * size[1] // size[0])
    assert 2 * c.tokens * c.nkv * (c.ld * size[0] // size[1] // 64) > 3 * 256
    c.fill_bounds()
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


@pytest.mark.parametrize("first,last,select", [(0, 1, 1), (0, 1, 2), (3, 4, 7), (2, 1, 40), (0, 5, 64), (1, 1, 200)])
def test_budgets(mxh, first, last, select):
    c = Blocks([(3000, 1), (1500, 20), (700, 1)], block=16, first=first, last=last, select=select, nh=8, nkv=2, hd=64,
               page=64, lead=1, seed=select)
    c.fill_bounds()
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


def test_more_blocks_than_a_workgroup_has_threads(mxh):
    """5,000 blocks and 700 chosen ones; rows of the table far wider than the sequence."""
    c = Blocks([(80000, 1), (4000, 2)], block=16, first=1, last=2, select=700, nh=3, nkv=1, hd=32, page=256, seed=2,
               extra_ld=300)
    c.fill_bounds()
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


def test_of_equal_scores_the_earlier_blocks_are_taken(mxh):
    c = Blocks([(960, 9), (640, 1)], block=16, first=1, last=2, select=9, nh=4, nkv=2, hd=64, page=32, seed=3)
    c.fill_bounds()
    for s in (0, 1):
        some = [c.place(s, b) for b in (3, 7, 11, 12, 13, 30, 33)]
        for p, x in some:  # the same bounds, and larger than most
            c.bounds[0, p, x] = c.bounds[0][some[0]] * np.float16(1.5)
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.bounds[:] = 1  # all of them
    c.upload()
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 59, 60]
    c.close()


def test_equal_scores_and_infinities_of_many_rows(mxh):
    c = Blocks([(500, 300)], block=16, first=1, last=2, select=9, nh=8, nkv=8, hd=32, page=32, seed=6)
    c.fill_bounds()
    c.bounds[0, ::3, :, :4] = 1
    c.bounds[0, :, :, 4:6] = 2
    c.bounds[0][c.place(0, 9)][6, 0, 5] = np.inf
    c.bounds[0][c.place(0, 11)][6, 1, 5] = -np.inf
    c.q.reshape(-1, 8, 32)[:, 6, 5] = np.where(np.arange(c.tokens) % 3 == 0, -1, 1)
    c.q.reshape(-1, 8, 32)[:, 7] = 0
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


def test_what_is_no_number_comes_first_and_absent_blocks_last(mxh):
    c = Blocks([(800, 1), (900, 6)], block=16, first=0, last=1, select=4, nh=6, nkv=2, hd=32, page=16, seed=4)
    c.fill_bounds()
    c.bounds[0][c.place(0, 9)][0, 0, 5] = np.nan
    c.bounds[0][c.place(1, 20)][1, 1] = np.inf  # (times zero: no number either)
    c.upload()
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    assert 9 in got[0, 0]
    # all but two of the rivals absent
    c.table[0, 2:50] = c.n_pages + np.arange(48)
    c.upload()
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    assert got[0, 0].tolist() == [0, 1, 2, 50]
    c.close()


def test_a_token_past_the_table_counts_from_its_last_block(mxh):
    c = Blocks([(300, 3)], block=16, first=1, last=2, select=5, nh=4, nkv=2, hd=32, page=32, seed=4)
    c.fill_bounds()
    c.table = np.ascontiguousarray(c.table[:, :7])
    c.ld = 7
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


@pytest.mark.parametrize("new", [1, 40], ids=["few", "many"])
@pytest.mark.parametrize("keys,queries", [(2.0**-19, 1.0), (1.0, 2.0**-140), (2.0**-19, 2.0**100), (2.0**12, 2.0**120)])
def test_small_and_large_values(mxh, new, keys, queries):
    """Bounds and queries of fp16's and fp32's subnormals, and large ones; a few dims of q far above the others."""
    c = Blocks([(1500, new), (900, new)], block=16, first=1, last=2, select=12, nh=8, nkv=2, hd=64, page=64, seed=8,
               extra_ld=0 if new == 1 else 300)
    c.k[:] = (c.k.astype(np.float32) * np.float32(keys)).astype(np.float16)
    c.q *= np.float32(queries)
    c.q.reshape(-1, 64)[:, ::7] *= np.float32(2.0**-16)
    c.fill_bounds()
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


def test_queries_of_infinities_and_nan(mxh):
    """Scores that are no numbers everywhere: the first blocks; of one q head it is the kv head's."""
    c = Blocks([(500, 2)], block=16, first=1, last=1, select=6, nh=4, nkv=2, hd=32, page=16, seed=5)
    c.fill_bounds()
    c.q.reshape(2, 4, 32)[0, 1, 3] = np.nan
    c.q.reshape(2, 4, 32)[1, 2, 0] = np.inf
    c.upload()
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 4, 31]
    c.close()


@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}-{s[1]}")
@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("name", list(SETS) + list(TREES) + list(LONG) + list(DRAFTS))
def test_attention_over_lists(mxh, name, heads, size):
    c = case(name, heads, size, select=5 if size[1] > 32 else 9)
    c.random_lists(c.rng)
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.close()


@pytest.mark.parametrize("select,block", [(1, 16), (2, 64), (64, 16), (300, 16), (1024, 16)])
def test_lists_of_many_lengths(mxh, select, block):
    c = Blocks([(6000, 1), (100, 1), (2500, 30)], block=block, first=0, last=1, select=select, nh=8, nkv=2, hd=64, page=64, lead=1,
               seed=select)
    c.random_lists(c.rng)
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.close()


def test_a_table_of_the_most_blocks(mxh):
    """262,144 blocks a sequence, most of them absent: bits of a list's blocks fill their place in LDS."""
    c = Blocks([(900, 1), (300, 5)], block=16, select=8, nh=4, nkv=2, hd=32, page=16, seed=6, extra_ld=262144 - 57)
    assert c.ld == 262144 and c.table.size < 1 << 20
    c.random_lists(c.rng)
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.close()


def test_all_blocks_listed_is_the_paged_attention(mxh):
    c = Blocks([(300, 1), (0, 64), (700, 9), (511, 1)], block=32, select=24, nh=16, nkv=4, hd=128, page=32, seed=7)
    c.chosen[:] = np.arange(24)[::-1]
    c.upload()
    got = c.attention().copy()
    c.check(got)
    assert np.array_equal(got, c.attention())
    c.close()


def test_a_tile_of_many_sequences(mxh):
    """More than two tokens a sequence on average, so tiles hold several sequences' tokens; many sequences empty."""
    rng = np.random.default_rng(8)
    seqs = [(int(rng.integers(0, 200)), int(rng.choice([0, 0, 1, 2, 5, 12]))) for _ in range(150)]
    c = Blocks(seqs, block=16, select=5, nh=4, nkv=2, hd=32, page=16, seed=8, lead=3, tail=5)
    assert c.tokens > 2 * len(seqs)
    c.random_lists(c.rng)
    c.fill_bounds()
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
def test_what_is_not_listed_or_attended_has_no_effect(mxh, tree):
    """Infinities and NaN in blocks that other tokens list, behind a token and beside its path."""
    c = Blocks([(200, 40), (330, 21), (150, 1)], block=16, select=6, nh=8, nkv=2, hd=64, page=16, tree=tree, seed=11)
    c.random_lists(c.rng)
    bad = {0: [207, 230, 33], 1: [350, 100], 2: [7]}
    for s, rows in bad.items():
        for i, r in enumerate(rows):
            c.row(c.v, s, r)[i::3] = [np.inf, -np.inf, np.nan][i]
            c.row(c.k, s, r)[i::5] = [-np.inf, np.nan, np.inf][i]
    free, hit = set(), []
    for s, (n_c, n) in enumerate(c.seqs):
        for i in range(n):
            t = int(c.start[s]) + i
            at = set(range(n_c)) | {n_c + j for j in c.before(s, i)}
            on = [{r // 16 for r in bad[s] if r in at} & set(c.chosen[t, g].tolist()) for g in range(2)]
            if not on[0] and not on[1]:
                free.add(t)
            hit += [(t, g) for g in range(2) if on[g]]
    assert len(free) >= 20 and len(hit) >= 5
    c.upload()
    got = c.attention()
    c.check_listed(got, c.chosen, rows=free)
    for t, g in hit:
        assert not np.all(np.isfinite(got[t, 4 * g:4 * g + 4]))
    c.close()


def in_tiles(tokens, nkv, select, block):
    """Whether the tokens make 46 stages of 128 keys a CU, four for a token's start among them."""
    return tokens * nkv * (select * block // 128 + 4) > 46 * 256


def thin_lists(c, few=5):
    """Lists with places for more blocks than the few that stand in them: tokens go in tiles where their lists may be
    long (see in_tiles)."""
    c.random_lists(c.rng)
    c.chosen[c.rng.random(c.chosen.shape) < 1 - few / c.select] = -1
    assert in_tiles(c.tokens, c.nkv, c.select, c.block)


def tiles():
    """Cases and the shortest lists, of 64, 128 or 256 blocks, with which they have tiles."""
    for name in ("prompts", "tree-64", "trees", "chunks", "empty-among", "prompt"):
        tokens = sum(n for _, n in {**SETS, **TREES, **LONG, **DRAFTS}[name])
        for heads, (_, nkv, _) in HEADS.items():
            for size in ((256, 128), (64, 16)):
                enough = [s for s in (64, 128, 256) if in_tiles(tokens, nkv, s, size[1])]
                if enough:
                    yield pytest.param(name, heads, size, enough[0], id=f"{name}-{heads}-{size[0]}-{size[1]}")


@pytest.mark.parametrize("name,heads,size,select", tiles())
def test_tiles_of_tokens(mxh, name, heads, size, select):
    """... of one sequence and of several, 16 and 32 rows, whole and split."""
    c = case(name, heads, size, select=select, extra_ld=select * size[1] // size[0])
    thin_lists(c)
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.close()


def test_tiles_of_many_sequences(mxh):
    rng = np.random.default_rng(9)
    seqs = [(int(rng.integers(0, 200)), int(rng.choice([0, 0, 1, 2, 5, 12]))) for _ in range(150)]
    c = Blocks(seqs, block=16, select=100, nh=4, nkv=2, hd=32, page=16, seed=8, lead=3, tail=5, extra_ld=100)
    assert c.tokens > 2 * len(seqs)
    thin_lists(c)
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.close()


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("select", [200, 300])  # tiles of 32 and of 16 rows
def test_in_tiles_what_is_not_listed_or_attended_has_no_effect(mxh, tree, select):
    c = Blocks([(200, 40), (330, 21), (150, 1)], block=16, select=select, nh=32, nkv=8, hd=64, page=16, tree=tree, seed=11,
               extra_ld=300)
    thin_lists(c, few=1)
    bad = {0: [207, 230, 33], 1: [350, 100], 2: [7]}
    for s, rows in bad.items():
        for i, r in enumerate(rows):
            c.row(c.v, s, r)[i::3] = [np.inf, -np.inf, np.nan][i]
            c.row(c.k, s, r)[i::5] = [-np.inf, np.nan, np.inf][i]
    free, hit = set(), []
    for s, (n_c, n) in enumerate(c.seqs):
        for i in range(n):
            t = int(c.start[s]) + i
            at = set(range(n_c)) | {n_c + j for j in c.before(s, i)}
            on = [{r // 16 for r in bad[s] if r in at} & set(c.chosen[t, g].tolist()) for g in range(8)]
            if not any(on):
                free.add(t)
            hit += [(t, g) for g in range(8) if on[g]]
    assert len(free) >= 5 and len(hit) >= 5
    c.upload()
    got = c.attention()
    c.check_listed(got, c.chosen, rows=free)
    for t, g in hit:
        assert not np.all(np.isfinite(got[t, 4 * g:4 * g + 4]))
    c.close()


def test_rows_behind_a_sequence_do_not_matter(mxh):
    """The rest of the last page holds NaN already; of a listed block that is absent nothing is read."""
    c = Blocks([(37, 2), (100, 1)], block=32, select=4, nh=4, nkv=2, hd=128, page=64, seed=12)
    c.chosen[:] = [0, 1, 2, 3]
    gone, c.table[1, 0] = c.table[1, 0], -5
    c.upload()
    got = c.attention()
    c.table[1, 0] = gone
    lists = c.chosen.copy()
    lists[2] = [2, 3, 2, 3]
    c.check_listed(got, lists)
    c.close()


def test_nothing_listed_gives_zeros(mxh):
    for seqs in ([(400, 1), (300, 1)], [(400, 30)]):
        c = Blocks(seqs, block=16, select=64, nh=4, nkv=2, hd=64, page=16, lead=1, seed=12)
        c.chosen[:] = -1
        c.upload()
        got = c.attention()
        assert np.all(got[1:] == 0) and np.all(got[0] == FILL)
        c.close()


def test_large_scores(mxh):
    c = Blocks([(600, 9), (1200, 2)], block=16, select=12, nh=8, nkv=2, hd=128, page=16, seed=3)
    c.q[::2] *= 40
    for s, r in ((0, 17), (0, 250), (1, 1100)):
        c.row(c.k, s, r)[:] *= 8
    c.random_lists(c.rng)
    c.upload()
    c.check_listed(c.attention(), c.chosen)
    c.close()


class Serving:
    """Sequences that grow step by step: append, bounds, selection, attention, as a runtime calls them."""

    def __init__(self, lengths, *, nh=8, nkv=2, hd=64, page=32, block=16, select=6, drafts=1, room=60):
        rng = self.rng = np.random.default_rng(5)
        self.nh, self.nkv, self.hd, self.page, self.block, self.n = nh, nkv, hd, page, block, len(lengths)
        self.drafts, self.ld = drafts, room
        self.book = mxhip.Pages(self.n * room, page, self.n)
        self.seqs = [self.book.open() for _ in lengths]
        width, pages = nkv * hd, self.n * room
        self.k, self.v = (rng.standard_normal((pages, page, width)).astype(np.float16) for _ in range(2))
        self.lengths = list(lengths)
        put = mxhip.DeviceBuffer.from_array
        tokens = self.tokens = self.n * drafts
        b = self.b = {"k": put(self.k), "v": put(self.v),
                      "bounds": put(np.full((pages, page // block, nkv, 2, hd), np.nan, np.float16)),
                      "start": put((drafts * np.arange(self.n + 1)).astype(np.int32)),
                      "cached": put(np.zeros(self.n, np.int32)),
                      "table": put(np.full((self.n, room), -1, np.int32)),
                      "qkv": put(np.zeros((tokens, (nh + 2 * nkv) * hd), np.float32)),
                      "q": put(np.zeros((tokens, nh * hd), np.float32)),
                      "att": put(np.zeros((tokens, nh * hd), np.float32)),
                      "chosen": put(np.zeros((tokens, nkv, select), np.int32)),
                      "freq": put(mxhip.rope_frequencies(1e4, hd))}
        self.pool = mxhip.KvPool(b["k"], b["v"], n_layer=1, n_pages=pages, page_rows=page, n_kv=nkv, head_dim=hd)
        self.batch = mxhip.KvBatch(self.n, tokens, b["start"], b["cached"], b["table"], room)
        self.what = mxhip.KvBlocks(b["bounds"], block_rows=block, n_first=1, n_last=2, n_select=select)
        self.sizes = (mxhip.kv_select_workspace(self.pool, self.batch, self.what, nh),
                      mxhip.attention_blocks_workspace(self.pool, self.batch, self.what, nh))
        b["s_work"], b["work"] = (mxhip.DeviceBuffer(max(x, 16)) for x in self.sizes)
        # what is cached already gets its bounds by a batch of its rows
        for s, n in zip(self.seqs, lengths):
            self.book.extend(s, n)
            self.book.set_length(s, n)
        table, _ = self.book.table(self.seqs, room)
        b["table"].upload(table)
        rows = put(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32))
        zero = put(np.zeros(self.n, np.int32))
        mxhip.kv_block_bounds(self.pool, 0, mxhip.KvBatch(self.n, int(sum(lengths)), rows, zero, b["table"], room),
                              self.what)
        mxhip.synchronize()
        rows.close(), zero.close()

    def step(self):
        b = self.b
        mxhip.qk_rope_append(self.pool, 0, self.batch, b["qkv"], (self.nh + 2 * self.nkv) * self.hd, None, None, None,
                             1e-6, b["freq"], True, self.nh, b["q"])
        mxhip.kv_block_bounds(self.pool, 0, self.batch, self.what)
        mxhip.kv_select_blocks(self.pool, 0, self.batch, self.what, b["q"], self.nh, b["chosen"], b["s_work"],
                               self.sizes[0])
        mxhip.attention_blocks(self.pool, 0, self.batch, self.what, b["chosen"], b["q"], self.nh, b["att"], b["work"],
                               self.sizes[1])

    def begin(self):
        """The next step's rows, lengths and projections on the device."""
        for s in self.seqs:
            assert self.book.extend(s, self.drafts) == []
        table, cached = self.book.table(self.seqs, self.ld)
        self.b["table"].upload(table), self.b["cached"].upload(cached)
        self.b["qkv"].upload(self.rng.standard_normal((self.tokens, (self.nh + 2 * self.nkv) * self.hd)).astype(np.float32))

    def check(self):
        """Bounds, lists and attention against float64 on the pool as it is now."""
        mxhip.synchronize()
        get = lambda n, t: self.b[n].download(t)  # noqa: E731
        seqs = [(self.book.length(s), self.drafts) for s in self.seqs]
        c = Blocks(seqs, block=self.block, first=1, last=2, select=6, nh=self.nh, nkv=self.nkv, hd=self.hd,
                   page=self.page)
        c.table, c.ld = self.book.table(self.seqs, self.ld)[0], self.ld
        c.n_pages, c.stride = self.n * self.ld, self.k.size
        c.k, c.v = (get(n, np.float16).reshape(1, -1) for n in ("k", "v"))
        c.q = get("q", np.float32).reshape(self.tokens, -1)
        c.shape = (1, c.n_pages, self.page // self.block, self.nkv, 2, self.hd)
        c.bounds = np.full(c.shape, np.nan, np.float16)
        c.fill_bounds()
        bounds = get("bounds", np.float16).reshape(c.shape)
        for s, (n_c, n) in enumerate(seqs):
            for x in range(-(-(n_c + n) // self.block)):
                assert np.array_equal(bounds[0][c.place(s, x)], c.bounds[0][c.place(s, x)])
        lists = get("chosen", np.int32).reshape(c.chosen.shape)
        c.check_chosen(lists)
        c.check_listed(get("att", np.float32).reshape(self.tokens, self.nh, self.hd), lists)

    def end(self):
        for s in self.seqs:
            self.book.set_length(s, self.book.length(s) + self.drafts)

    def close(self):
        for x in self.b.values():
            x.close()
        self.book.close()


@pytest.mark.parametrize("drafts", [1, 5])
def test_steps_of_a_runtime(mxh, drafts):
    s = Serving([100, 31, 510, 2, 333], drafts=drafts)
    for _ in range(4):
        s.begin()
        s.step()
        s.check()
        s.end()
    s.close()


def test_a_recorded_step_follows_the_lengths(mxh):
    s = Serving([100, 31, 510, 2, 333])
    s.begin()
    graph = Graph([s.step])
    for i in range(6):
        graph.replay()
        s.check()
        if i == 2:  # eager work between replays
            s.step()
            s.check()
        s.end()
        s.begin()
    graph.close()
    s.close()


def test_kept_rows_get_their_bounds_again(mxh):
    """After drafted rows moved together, a batch that names the rows mends the bounds."""
    s = Serving([100, 31, 510], drafts=9)
    s.begin()
    s.step()
    mxhip.synchronize()
    table, cached = s.book.table(s.seqs, s.ld)
    keep = [[0, 2, 5, 8], [1], [3, 4, 7]]
    mxhip.kv_keep_rows(s.pool, table, cached, np.concatenate([[0], np.cumsum([len(x) for x in keep])]),
                       np.concatenate(keep))
    start = mxhip.DeviceBuffer.from_array(np.asarray([0, 4, 5, 8], np.int32))
    mxhip.kv_block_bounds(s.pool, 0, mxhip.KvBatch(3, 8, start, s.b["cached"], s.b["table"], s.ld), s.what)
    mxhip.synchronize()
    for q, x in zip(s.seqs, keep):
        s.book.set_length(q, s.book.length(q) + len(x))
    s.begin()
    s.step()
    s.check()
    start.close()
    s.close()


def test_workspaces_that_are_too_small_are_refused(mxh):
    c = Blocks([(900, 1)], block=16, select=40, nh=4, nkv=2, hd=64, page=16, seed=1)
    c.chosen[:] = 3
    c.upload()
    assert c.work_bytes > 0 and c.s_bytes > 0
    c.work_bytes, c.s_bytes = c.work_bytes // 1000, c.s_bytes - 1
    with pytest.raises(mxhip.MxhError, match="bytes of work"):
        c.attend()
    with pytest.raises(mxhip.MxhError, match="bytes of work"):
        c.choose()
    mxhip.synchronize()
    assert np.all(c.bufs["att"].download(np.float32) == FILL) and np.all(c.got_chosen() == 3)
    c.close()


@pytest.mark.parametrize("new", [1, 300], ids=["few", "many"])
def test_no_number_comes_before_infinity(mxh, new):
    """A score of +inf is a number: an earlier block with it stands behind a later one whose score is none."""
    for select, want in ((2, [9]), (3, [4, 9]), (4, [4, 6, 9])):
        c = Blocks([(800, new)], block=16, first=0, last=1, select=select, nh=8, nkv=8, hd=32, page=16, seed=4)
        c.fill_bounds()
        c.q[:] = 1
        for b, x in ((4, np.inf), (6, np.inf), (9, np.nan)):
            p, at = c.place(0, b)
            c.bounds[0, p, at, :, 1, 5] = x
        c.upload()
        c.choose()
        got = c.got_chosen()
        for i in range(new):
            assert np.all(got[i] == want + [(800 + i) // 16]), (i, got[i, 0])
        c.close()


@pytest.mark.parametrize("new", [1, 300], ids=["few", "many"])
def test_minus_infinity_comes_before_absent_blocks(mxh, new):
    c = Blocks([(800, new)], block=16, first=0, last=1, select=5, nh=8, nkv=8, hd=32, page=16, seed=4)
    c.fill_bounds()
    c.q[:] = 1
    for b in range(50):
        if b not in (20, 33):
            p, at = c.place(0, b)
            c.bounds[0, p, at, :, 1, 5] = -np.inf
    c.table[0, :6] = c.n_pages
    c.upload()
    c.choose()
    got = c.got_chosen()
    for i in range(16):
        if i < new:
            assert np.all(got[i] == [6, 7, 20, 33, 50]), (i, got[i, 0])
    c.close()


@pytest.mark.parametrize("seqs,nh,extra_ld", [([(300, 1)], 8, 3), ([(300, 12)], 8, 70), ([(300, 40), (70, 40)], 8, 70)],
                         ids=["tokens-alone", "a-tile", "tiles"])
def test_bounds_of_blocks_that_do_not_compete_have_no_effect(mxh, seqs, nh, extra_ld):
    """Behind a sequence and outside its rivals whatever lies there: not even what scores may be off by takes it in
    (with an infinity there all scores would be made again in 64 bits).  That stands in the workspace's rows of
    2 x (blocks of a row of the table, in sixteens) floats, in the second half, one for every 16 blocks."""
    c = Blocks(seqs, block=16, first=1, last=2, select=6, nh=nh, nkv=2, hd=64, page=256, seed=9, extra_ld=extra_ld)
    c.fill_bounds()
    want = c.bounds.copy()
    c.bounds[:] = np.nan
    for s, (n_c, n) in enumerate(seqs):
        p, x = zip(*(c.place(s, b) for b in range(1, (n_c + n - 1) // 16 + 1 - 2)))
        c.bounds[0, p, x] = want[0, p, x]
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    row = (c.ld * 16 + 15) // 16 * 16
    marks = c.bufs["s_work"].download(np.float32)[:c.tokens * c.nkv * 2 * row].reshape(c.tokens, c.nkv, 2, row)[:, :, 1]
    for s, (n_c, n) in enumerate(seqs):
        for i in range(n):
            end = (n_c + i) // 16 + 1 - 2
            if (n_c + i) // 16 >= c.select:
                m = marks[int(c.start[s]) + i, :, :(end + 15) // 16]
                assert np.all((m > 0) & (m < 1e30)), (s, i)
    c.close()


@pytest.mark.parametrize("nh", [8, 32])  # a tile, and tiles enough for four a workgroup
def test_scores_of_more_than_the_workspace_holds(mxh, nh):
    """262,144 blocks a sequence, most of them absent, 8 kv heads: scores of 16 tokens fill the workspace, so that
    three launches use it."""
    c = Blocks([(900, 20), (300, 21)], block=16, select=8, nh=nh, nkv=8, hd=32, page=16, seed=6, extra_ld=262144 - 58,
               lead=1, tail=1)
    assert c.ld == 262144 and 32 < c.tokens <= 48 and 16 * c.ld * c.nkv * 8 == 256 << 20
    c.fill_bounds()
    c.upload()
    for _ in range(2):
        c.choose()
        c.check_chosen(c.got_chosen())
    c.close()


@pytest.mark.parametrize("heads", [(64, 8, 128), (8, 8, 128), (32, 8, 64)], ids=lambda h: "-".join(map(str, h)))
@pytest.mark.parametrize("equal", [False, True], ids=["", "equal-scores"])
def test_many_rows(mxh, heads, equal):
    """More rows of scores than are picked from at a time (8 a CU), where two waves take one."""
    nh, nkv, hd = heads
    c = Blocks([(500, 290), (340, 10)], block=16, select=9, nh=nh, nkv=nkv, hd=hd, page=32, seed=6)
    assert c.tokens * nkv > 8 * 256
    c.fill_bounds()
    if equal:
        c.bounds[0, ::3] = 1
        c.bounds[0][c.place(0, 9)][:, 0, 5] = np.inf
    c.upload()
    c.choose()
    c.check_chosen(c.got_chosen())
    c.close()


@pytest.mark.parametrize("equal", [False, True], ids=["", "equal-scores"])
def test_many_rows_of_more_blocks_than_lds_holds(mxh, equal):
    """4,300 rivals of 2,240 rows of scores: two waves a row, scores left where they are."""
    nkv, hd, tokens, cached, first, last, select = 32, 32, 70, 16 * 4302 + 5, 1, 2, 40
    pages = cached // 16 + 8
    assert tokens * nkv > 8 * 256 and cached // 16 - first - last > 4096
    rng = np.random.default_rng(3)
    table = rng.permutation(pages).astype(np.int32)[None]
    q = rng.standard_normal((tokens, nkv, hd)).astype(np.float32)
    bounds = np.sort(rng.standard_normal((pages, nkv, 2, hd)).astype(np.float16), 2)
    if equal:
        bounds[rng.random(pages) < 0.995] = 1
    put = mxhip.DeviceBuffer.from_array
    b = [put(x) for x in (np.asarray([0, tokens], np.int32), np.asarray([cached], np.int32), table, bounds, q,
                          np.full((tokens, nkv, select), LEFT, np.int32))]
    kv = mxhip.DeviceBuffer(2 * pages * 16 * nkv * hd)  # (no row of it is read)
    pool = mxhip.KvPool(kv, kv, n_layer=1, n_pages=pages, page_rows=16, n_kv=nkv, head_dim=hd)
    batch = mxhip.KvBatch(1, tokens, b[0], b[1], b[2], pages)
    what = mxhip.KvBlocks(b[3], block_rows=16, n_first=first, n_last=last, n_select=select)
    size = mxhip.kv_select_workspace(pool, batch, what, nkv)
    work = mxhip.DeviceBuffer(size)
    mxhip.kv_select_blocks(pool, 0, batch, what, b[4], nkv, b[5], work, size)
    mxhip.synchronize()
    got = b[5].download(np.int32).reshape(tokens, nkv, select)
    least, greatest = bounds[table[0]].astype(np.float64).transpose(2, 1, 3, 0)  # [kv heads, hd, blocks]
    x = q.astype(np.float64).transpose(1, 0, 2)
    score = np.maximum(x, 0) @ greatest + np.minimum(x, 0) @ least
    if equal:  # (blocks of the same bounds: of the first one the score of all, whatever the order of a sum)
        same = np.flatnonzero((bounds[table[0]] == 1).all((1, 2, 3)))
        score[:, :, same] = score[:, :, same[:1]]
    for t in range(tokens):
        own = (cached + t) // 16
        rivals = np.arange(first, own + 1 - last)
        for g in range(nkv):
            s = score[g, t, rivals]
            order = np.argsort(-s, kind="stable")
            k = select - first - last
            a, z = s[order[k - 1]], s[order[k]]
            assert a == z or a - z > 2.0**-40 * abs(a), "scores of these inputs lie next to one another"
            want = [0, *np.sort(rivals[order[:k]]), own - 1, own]
            assert got[t, g].tolist() == want, (t, g)
    for y in [*b, kv, work]:
        y.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
@pytest.mark.parametrize("small,large", [(1e-2, 100.0), (1e-5, 1e4), (1e-37, 1e4), (1e33, 1e-6)])
@pytest.mark.parametrize("tiles", [False, True], ids=["alone", "tiles"])
def test_small_q_over_large_k(mxh, tiles, heads, small, large):
    """q outside the range of fp16 halves, over lists of all blocks; every fourth token ordinary."""
    nh, nkv, hd = HEADS[heads]
    for seqs, tree in (([(150, 33), (300, 1), (0, 2)], False), ([(0, 30), (400, 20)], True)):
        tokens = sum(n for _, n in seqs)
        select = 32 if not tiles else next(s for s in (64, 128, 256, 512, 1024) if in_tiles(tokens, nkv, s, 64))
        c = Blocks(seqs, block=64, select=select, nh=nh, nkv=nkv, hd=hd, page=64, tree=tree, seed=19, extra_ld=select)
        assert in_tiles(tokens, nkv, select, 64) == tiles
        c.chosen[:] = -1
        c.chosen[..., :8] = np.arange(8)[::-1]
        c.k = np.clip(c.k.astype(np.float32) * large, -65504, 65504).astype(np.float16)
        c.q *= np.float32(small)
        if large > 1:
            c.q[3::4] /= np.float32(small * large)
        c.upload()
        check_precision(c, c.attention())
        c.close()


def test_lists_and_attention_in_a_layer_of_strided_pools(mxh):
    c = Blocks([(170, 3), (210, 40), (64, 1)], block=16, select=6, nh=12, nkv=6, hd=64, page=32, layers=3, layer=1,
               stride=24, seed=5)
    c.fill_bounds()
    dense = int(np.prod(c.shape[1:]))
    c.upload()
    wide = np.full((3, dense + 40), np.nan, np.float16)
    wide[1, :dense] = c.bounds[1].reshape(-1)
    b = mxhip.DeviceBuffer.from_array(wide)
    c.what = mxhip.KvBlocks(b, block_rows=16, n_first=1, n_last=2, n_select=6, layer_stride=dense + 40)
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    c.check_listed(c.attention(), got)
    b.close()
    c.close()


@pytest.mark.parametrize("block", [16, 1024])
def test_the_largest_pages(mxh, block):
    c = Blocks([(5000, 1), (1500, 20), (1023, 2), (9000, 1)], block=block, first=1, last=1, select=3, nh=8, nkv=2, hd=64,
               page=1024, seed=3, lead=1, tail=1)
    c.upload()
    c.find_bounds()
    c.check_bounds(c.got_bounds())
    c.fill_bounds()
    c.upload()
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    c.check_listed(c.attention(), got)
    c.close()


@pytest.mark.parametrize("select", [6, 300])
def test_drafted_trees_end_at_64_tokens(mxh, select):
    seqs = [(300, 70), (200, 90), (100, 2)]
    c = Blocks(seqs, block=16, select=select, nh=16, nkv=8, hd=32, page=32, tree=True, seed=7, extra_ld=150)
    assert in_tiles(c.tokens, c.nkv, select, 16) == (select == 300)
    c.fill_bounds()
    c.upload()
    c.choose()
    got = c.got_chosen()
    c.check_chosen(got)
    att = c.attention()
    past = [int(c.start[s]) + i for s, (_, n) in enumerate(seqs) for i in range(64, n)]
    assert np.all(att[past] == FILL) and np.all(got[past] == LEFT)
    att[past] = 0
    c.check_listed(att, got, rows=set(range(c.tokens)) - set(past))
    c.close()
