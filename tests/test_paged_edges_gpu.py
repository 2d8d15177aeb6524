"""Paged attention at the edges of its documented range (GPU).

Expected values are the formula in float64 on the values that the kernels read;
bounds and helpers as in test_paged_gpu.py (u = 2^-24).
"""
from __future__ import annotations

import numpy as np
import pytest

import mxhip
from test_paged_gpu import Case, U, chain, rope_expected, rope_inputs

pytestmark = pytest.mark.gpu


def test_most_sequences_behind_long_tables(mxh):
    """4,096 single tokens of 128 kv heads at 61,440 rows, pages of which most are absent: two items a kv head, and an
    index times an item's units passes 32 bits for the workgroups that have none."""
    n, nh, hd, page, rows = 4096, 128, 32, 1024, 61440
    rng = np.random.default_rng(3)
    kv = rng.standard_normal((2, 2 * page, nh * hd)).astype(np.float16)
    put = mxhip.DeviceBuffer.from_array
    bufs = [put(x) for x in kv]
    table = np.full((n, rows // page + 1), -1, np.int32)
    table[:, 0], table[:, -1] = 0, 1
    q = rng.standard_normal((n, nh * hd)).astype(np.float32)
    dev = [put(np.arange(n + 1, dtype=np.int32)), put(np.full(n, rows, np.int32)), put(table), put(q),
           put(np.zeros_like(q))]
    pool = mxhip.KvPool(*bufs, n_layer=1, n_pages=2, page_rows=page, n_kv=nh, head_dim=hd)
    batch = mxhip.KvBatch(n, n, dev[0], dev[1], dev[2], table.shape[1])
    size = mxhip.attention_paged_workspace(pool, batch, nh)
    work = mxhip.DeviceBuffer(size)
    mxhip.attention_paged(pool, 0, batch, dev[3], nh, dev[4], work, size)
    mxhip.synchronize()
    got = dev[4].download(np.float32).reshape(n, nh, hd)
    k, v = kv[:, :page + 1].astype(np.float64).reshape(2, page + 1, nh, hd)  # (the token's own row begins page 1)
    for t in (0, 1, 63, 64, 2047, 2048, 2049, 3000, 4095):
        x = q[t].astype(np.float64).reshape(nh, hd)
        sc = np.einsum("rhd,hd->hr", k, x) / np.sqrt(hd)
        p = np.exp(sc - sc.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want, size_v = np.einsum("hr,rhd->hd", p, v), np.einsum("hr,rhd->hd", p, np.abs(v))
        d = (2.0**-21 + 2 * hd * U) * np.einsum("rhd,hd->hr", np.abs(k), np.abs(x)).max(-1) / np.sqrt(hd)
        bound = (2 * d[:, None] + 2.0**-20 + 2 * (page + 1) * U) * size_v
        assert np.all(np.abs(got[t] - want) <= bound), t
    for b in [*bufs, *dev, work]:
        b.close()


HEADS = {"g4-d128": (8, 2, 128), "g3-d64": (6, 2, 64), "g8-d32": (8, 1, 32), "g1-d128": (2, 2, 128)}


def check_precision(c, got):
    """got against float64, with what the pairs of fp16 halves promise (q' = q log2(e) / sqrt(hd), in fp32):

    - q' is off by u of itself and its halves by 2^-22 of the row's largest |q'| (rows outside [2^-3, 2^15) are
      scaled by a power of two first; inside, the halves end at 2^-25 absolute, which is no more).  A score's
      products are exact; sums of those that are not zero and of minus the reference round at most once each:
      |d score| <= D = (2^-22 max|q| sum_d |k_d| + (2 z + 4) u max_j sum_d |q_d k_jd|) / sqrt(hd), z products.
    - a probability is off by 2 D of its value (its score, the sum's), 2^-20 for the exponential, its scale and its
      halves, 2 L u for the sums of L keys, and by 2^-31 of the row's largest, where its halves end."""
    group, worst = c.nh // c.nkv, 0.0
    q = c.q.astype(np.float64).reshape(c.tokens, c.nh, c.hd)
    for s, (n_c, n) in enumerate(c.seqs):
        k, v = (np.array([c.row(x, s, r) for r in range(n_c + n)], np.float64).reshape(-1, c.nkv, c.hd) for x in (c.k, c.v))
        for i in range(n):
            t, at = int(c.start[s]) + i, list(range(n_c)) + [n_c + j for j in c.before(s, i)]
            for h in range(c.nh):
                kk, vv, x = k[at, h // group], v[at, h // group], q[t, h]
                sc = kk @ x / np.sqrt(c.hd)
                p = np.exp(sc - sc.max())
                p /= p.sum()
                z = int(((kk != 0) & (x != 0)).sum(1).max())
                d = (2.0**-22 * np.abs(x).max() * np.abs(kk).sum(1).max() +
                     (2 * z + 4) * U * (np.abs(kk) @ np.abs(x)).max()) / np.sqrt(c.hd)
                bound = (2 * d + 2.0**-20 + 2 * len(at) * U) * (p @ np.abs(vv)) + \
                    2.0**-31 * p.max() * np.abs(vv).sum(0) + 2.0**-100
                err = np.abs(got[t, h] - p @ vv)
                assert np.all(err <= bound), (s, i, h, float((err / bound).max()))
                worst = max(worst, float((err / bound).max()))
    return worst


@pytest.mark.parametrize("heads", list(HEADS))
@pytest.mark.parametrize("new,tree", [(1, False), (3, True), (40, False), (40, True)])
def test_q_of_every_size(mxh, heads, new, tree):
    """Scores of up to 6 from one product, of q from 10^-5 up over K down from the largest fp16: two cached keys of
    opposite sign, zeros in the new ones.  Every fifth token has a second, ordinary element that meets no K."""
    nh, nkv, hd = HEADS[heads]
    sizes = [65504.0, 40000.0, 5000.0, 300.0, 20.0, 1.0, 2.0**-5, 2.0**-11, 2.0**-20]
    c = Case([(2, new) for _ in sizes], nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, seed=new + nh)
    q = c.q.reshape(c.tokens, nh, hd)
    keep = c.rng.uniform(0.5, 2, c.tokens)
    y = c.rng.uniform(-6, 6, (c.tokens, nh))
    q[:] = 0
    for s, size in enumerate(sizes):
        for r in range(2 + new):
            row = c.row(c.k, s, r).reshape(nkv, hd)
            row[:] = 0
            if r < 2:
                row[:, 5] = size if r == 0 else -0.75 * size
        q[c.start[s]:c.start[s + 1], :, 5] = y[c.start[s]:c.start[s + 1]] / size * np.sqrt(hd)
    q[::5, :, 9] = keep[::5, None]
    c.upload()
    check_precision(c, c.attention())
    c.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
@pytest.mark.parametrize("small,large", [(1e-2, 100.0), (1e-4, 6e3), (1e-5, 1e4), (1e-7, 1.2e4), (1e-37, 1e4), (1e33, 1e-6)])
def test_small_q_over_large_k(mxh, heads, small, large):
    """Dense rows of q and K of far apart sizes, few and many keys, 16- and 64-row tiles; every fourth token ordinary."""
    nh, nkv, hd = HEADS[heads]
    for seqs, tree in (([(2, 1), (0, 2), (1, 1), (300, 1)], False), ([(1, 40), (150, 33)], False), ([(0, 30), (700, 20)], True)):
        c = Case(seqs, nh=nh, nkv=nkv, hd=hd, page=16, tree=tree, seed=19)
        c.k = np.clip(c.k.astype(np.float32) * large, -65504, 65504).astype(np.float16)
        c.q *= np.float32(small)
        if large > 1:
            c.q[3::4] /= np.float32(small * large)
        c.upload()
        check_precision(c, c.attention())
        c.close()


@pytest.mark.parametrize("below", [5.0, 10.0, 15.0, 18.0, 22.0, 30.0])
@pytest.mark.parametrize("new", [1, 40])
def test_keys_far_below_the_largest(mxh, below, new):
    """One key whose V is zero, 1,000 others `below` nats under it: what the halves of a probability still say of them."""
    c = Case([(1000, new)], nh=8, nkv=2, hd=64, page=16, seed=23)
    q = c.q.reshape(c.tokens, 8, 64)
    q[:] = 0
    q[..., 0] = 8.0
    for r in range(1000 + new):
        row = c.row(c.k, 0, r).reshape(2, 64)
        row[:] = 0
        row[:, 0] = below if r == 333 else 0.0
    c.row(c.v, 0, 333)[:] = 0
    c.upload()
    check_precision(c, c.attention())
    c.close()


@pytest.mark.parametrize("seqs,tree", [([(0, 1), (300, 1)], False), ([(5000, 2)], False), ([(700, 45), (3, 1)], False),
                                       ([(100, 30), (9, 4)], True)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_rows_whose_scores_are_all_minus_infinity(mxh, hd, seqs, tree):
    """They get zeros, as tokens none of whose rows exist do; a q of zero there makes NaN; other heads see nothing."""
    c = Case(seqs, nh=4, nkv=2, hd=hd, page=16, tree=tree, seed=33)
    for s, (n_c, n) in enumerate(seqs):
        for r in range(n_c + n):
            c.row(c.k, s, r)[7] = -np.inf  # (kv head 0)
    q = c.q.reshape(c.tokens, 4, hd)
    q[:, 0, 7] = np.abs(q[:, 0, 7]) + 0.01
    q[:, 1, 7] = 0
    c.upload()
    got = c.attention()
    assert np.all(got[:, 0] == 0)
    assert np.all(np.isnan(got[:, 1]))
    for s, (n_c, n) in enumerate(seqs):
        k, v = (np.array([c.row(x, s, r) for r in range(n_c + n)], np.float64).reshape(-1, 2, hd)[:, 1] for x in (c.k, c.v))
        for i in range(n):
            t, at = int(c.start[s]) + i, list(range(n_c)) + [n_c + j for j in c.before(s, i)]
            for h in (2, 3):
                sc = k[at] @ q[t, h].astype(np.float64) / np.sqrt(hd)
                p = np.exp(sc - sc.max())
                p /= p.sum()
                d = (2.0**-21 + (2 * hd + 4) * U) * (np.abs(k[at]) @ np.abs(q[t, h].astype(np.float64))).max() / np.sqrt(hd)
                bound = (2 * d + 2.0**-20 + 2 * len(at) * U) * (p @ np.abs(v[at])) + 2.0**-31 * np.abs(v[at]).sum(0)
                assert np.all(np.abs(got[t, h] - p @ v[at]) <= bound), (s, i, h)
    c.close()


@pytest.mark.parametrize("heads", ["g4-d128", "g3-d64", "g8-d32"])
def test_long_prompts_beside_drafted_trees_go_in_a_call_of_their_own(mxh, heads):
    """One packed step, two batches over its arrays: trees with parents, then prompts and single tokens without.  Each
    call leaves the other's token rows, and the pool's other rows, alone."""
    nh, nkv, hd = HEADS[heads]
    trees, rest = [(300, 20), (7, 64), (0, 5)], [(40, 100), (900, 1), (0, 130), (63, 1)]
    c = Case(trees + rest, nh=nh, nkv=nkv, hd=hd, page=16, tree=True, lead=1, tail=2, seed=81, extra_ld=1)
    for s in range(len(trees), len(c.seqs)):
        c.parents[s] = chain(c.seqs[s][1])
    c.upload()
    n, b = len(trees), c.bufs
    qkv, bias, w = rope_inputs(c, 4)
    freq = mxhip.rope_frequencies(1e4, hd)
    dev = [mxhip.DeviceBuffer.from_array(x) for x in (qkv, bias, w[0], w[1], freq)]
    first = mxhip.KvBatch(n, c.tokens, b["start"], b["cached"], b["table"], c.ld, b["parent"])
    second = mxhip.KvBatch(len(rest), c.tokens, b["start"].ptr + 4 * n, b["cached"].ptr + 4 * n,
                           b["table"].ptr + 4 * n * c.ld, c.ld)
    mxhip.memset(b["q"], 0)
    for batch in (first, second):
        mxhip.qk_rope_append(c.pool, 0, batch, dev[0], qkv.shape[1], dev[1], dev[2], dev[3], 1e-6, dev[4], True, nh, b["q"])
    mxhip.synchronize()
    q, k, v = (b[x].download(t) for x, t in (("q", np.float32), ("k", np.float16), ("v", np.float16)))
    want, bound = rope_expected(c, qkv, bias, list(w), 1e-6, freq, True)
    inside = slice(int(c.start[0]), int(c.start[-1]))
    c.q = q.reshape(c.tokens, -1)
    assert np.all(np.abs(q.reshape(c.tokens, nh, hd)[inside] - want[0][inside]) <= bound[0][inside] + 2.0**-140)
    assert not c.q[:inside.start].any() and not c.q[inside.stop:].any()
    c.k, c.v = k.reshape(c.k.shape), v.reshape(c.v.shape)
    for s, (n_c, m) in enumerate(c.seqs):
        for i in range(m):
            t = int(c.start[s]) + i
            for pool, x, e in ((c.k, want[1], bound[1]), (c.v, want[2], bound[2])):
                y = x[t].reshape(-1)
                assert np.all(np.abs(c.row(pool, s, n_c + i) - y) <= (np.abs(y) + e[t].reshape(-1)) * 2.0**-11 +
                              e[t].reshape(-1) + 2.0**-25)
    for batch in (first, second):
        size = mxhip.attention_paged_workspace(c.pool, batch, nh)
        assert size <= c.work_bytes  # (the whole step's is enough for its parts)
        mxhip.attention_paged(c.pool, 0, batch, b["q"], nh, b["att"], b["work"], c.work_bytes)
    mxhip.synchronize()
    c.check(b["att"].download(np.float32).reshape(c.tokens, nh, hd))
    for x in dev:
        x.close()
    c.close()


def test_more_items_than_a_grid_axis_takes(mxh):
    """4,096 prompts of 60 tokens of 8/1 heads: 34,816 tiles at most, over two axes of the grid."""
    n, m, nh, hd, page = 4096, 60, 8, 32, 64
    rng = np.random.default_rng(6)
    tokens = n * m
    q = rng.standard_normal((tokens, nh * hd), dtype=np.float32)
    kv = rng.standard_normal((2, n * page, hd), dtype=np.float32).astype(np.float16)
    put = mxhip.DeviceBuffer.from_array
    order = rng.permutation(n).astype(np.int32)
    dev = [put(np.arange(0, tokens + 1, m, dtype=np.int32)), put(np.zeros(n, np.int32)), put(order[:, None]), put(q),
           put(np.full_like(q, -1.5)), put(kv[0]), put(kv[1])]
    pool = mxhip.KvPool(dev[5], dev[6], n_layer=1, n_pages=n, page_rows=page, n_kv=1, head_dim=hd)
    batch = mxhip.KvBatch(n, tokens, dev[0], dev[1], dev[2], 1)
    size = mxhip.attention_paged_workspace(pool, batch, nh)
    work = mxhip.DeviceBuffer(max(size, 1))
    mxhip.attention_paged(pool, 0, batch, dev[3], nh, dev[4], work, size)
    mxhip.synchronize()
    got = dev[4].download(np.float32).reshape(tokens, nh, hd)
    for s in list(range(0, n, 97)) + [n - 1]:
        k, v = (x[order[s] * page:order[s] * page + m].astype(np.float64) for x in kv)
        for i in (0, 7, 8, 33, m - 1):
            t = s * m + i
            x = q[t].reshape(nh, hd).astype(np.float64)
            sc = x @ k[:i + 1].T / np.sqrt(hd)
            p = np.exp(sc - sc.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            d = (2.0**-21 + (2 * hd + 4) * U) * (np.abs(x) @ np.abs(k[:i + 1]).T).max(-1, keepdims=True) / np.sqrt(hd)
            bound = (2 * d + 2.0**-20 + 2 * (i + 1) * U) * (p @ np.abs(v[:i + 1])) + 2.0**-31 * np.abs(v[:i + 1]).sum(0)
            assert np.all(np.abs(got[t] - p @ v[:i + 1]) <= bound), (s, i)
    for b in [*dev, work]:
        b.close()


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
def test_k_and_v_of_a_layer_side_by_side(mxh, tree):
    """One buffer [layer][K, V][page][row]: v begins a layer's K into it and a layer's stride is two of them."""
    nh, nkv, hd, page, layers = 6, 2, 64, 32, 3
    c = Case([(70, 3), (0, 40), (10, 9)], nh=nh, nkv=nkv, hd=hd, page=page, tree=tree, layers=layers, layer=1, seed=91)
    c.upload()
    dense = c.k.shape[1]
    both = np.stack([c.k, c.v], 1)  # [layer][K, V][...]
    buf = mxhip.DeviceBuffer.from_array(both)
    pool = mxhip.KvPool(buf, buf.ptr + 2 * dense, n_layer=layers, n_pages=c.n_pages, page_rows=page, n_kv=nkv, head_dim=hd,
                        layer_stride=2 * dense)
    mxhip.attention_paged(pool, c.layer, c.batch, c.bufs["q"], nh, c.bufs["att"], c.bufs["work"], c.work_bytes)
    mxhip.synchronize()
    c.check(c.bufs["att"].download(np.float32).reshape(c.tokens, nh, hd))
    spare = sorted(set(range(c.n_pages)) - set(c.table[c.table >= 0].tolist()))
    mxhip.kv_copy_pages(pool, c.table[1, :1], spare[:1])
    cached = [n for n, _ in c.seqs]
    mxhip.kv_keep_rows(pool, c.table, cached, [0, 1, 3, 3], [2, 5, 33])
    mxhip.synchronize()
    want = both.view(np.uint16).reshape(layers, 2, c.n_pages, page, nkv * hd).copy()
    want[:, :, spare[0]] = want[:, :, c.table[1, 0]]
    old = want.copy()
    for s, i, kept in ((0, 0, 2), (1, 0, 5), (1, 1, 33)):
        to, frm = cached[s] + i, cached[s] + kept
        want[:, :, c.table[s, to // page], to % page] = old[:, :, c.table[s, frm // page], frm % page]
    assert np.array_equal(buf.download(np.uint16).reshape(want.shape), want)
    buf.close()
    c.close()
