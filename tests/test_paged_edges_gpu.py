"""Paged attention at the edges of its documented range (GPU).

Expected values are the formula in float64 on the values that the kernels read;
bounds and helpers as in test_paged_gpu.py (u = 2^-24).
"""
from __future__ import annotations

import numpy as np
import pytest

import mxhip
from test_paged_gpu import U, Case

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
