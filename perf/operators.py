"""The operators over a paged K/V cache, as measurable cases.

A runtime that serves several sequences keeps K and V in pages, fills them with
a pass that norms, rotates and appends, attends over them for whole prompts,
single tokens and trees of drafted tokens, and moves rows when sequences fork
and when drafted tokens are accepted:

- ``rope``       ``mxh_qk_rope_append``: bias, norms of queries and keys per
                 head, rotary positions, K and V into their cache rows;
- ``attention``  ``mxh_attention_paged``: grouped-head attention of packed
                 tokens, causal or along a drafted tree;
- ``copy``       ``mxh_kv_copy_pages``: pages to other pages, every layer;
- ``keep``       ``mxh_kv_keep_rows``: the accepted rows of drafted tokens
                 moved together behind the cached ones, every layer.

With ``own`` false ``run`` computes the same in elementary torch operations.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

# heads, kv heads, head dim, layers, rotary base, norms of q and k: the benchmark's models, and narrower heads
MODELS = {
    "qwen3-0.6b": (16, 8, 128, 28, 1e6, True),
    "qwen3-8b": (32, 8, 128, 36, 1e6, True),
    "llama3-8b": (32, 8, 128, 32, 5e5, False),
    "h6-kv2-d64": (6, 2, 64, 24, 1e4, False),
    "h8-kv1-d32": (8, 1, 32, 16, 1e4, True),
}
EPS = 1e-6


def listed():
    return [
        # decode: the next token of one chat, where the call's latency counts
        dict(name="rope-1-token", op="rope", model="qwen3-0.6b", n_seq=1, new=1, rows=700, page=16, tree=False,
             neox=True, bias=False, shape=1),
        # speculative decoding: eight chats' drafted trees at long positions
        dict(name="rope-8-trees", op="rope", model="qwen3-8b", n_seq=8, new=33, rows=8000, page=16, tree=True,
             neox=True, bias=False, shape=2),
        # prompts of different lengths packed into one pass, a model with biases and adjacent pairs
        dict(name="rope-prompts", op="rope", model="llama3-8b", n_seq=7, new=1400, rows=300, page=32, tree=False,
             neox=False, bias=True, shape=3),
        # decode: one chat at a short context
        dict(name="attention-1-at-700", op="attention", model="qwen3-0.6b", n_seq=1, new=1, rows=700, page=16,
             tree=False, shared=0, shape=4),
        # speculative decoding: one chat's tree of 27 drafted tokens at a long context
        dict(name="attention-tree-27-at-8192", op="attention", model="qwen3-8b", n_seq=1, new=27, rows=8192, page=16,
             tree=True, shared=0, shape=5),
        # decode: a batch of chats of very different lengths
        dict(name="attention-batch-48", op="attention", model="qwen3-8b", n_seq=48, new=1, rows=16000, page=32,
             tree=False, shared=0, shape=6),
        # prefill: packed prompts, some behind a cached prefix
        dict(name="attention-prompts", op="attention", model="llama3-8b", n_seq=6, new=2100, rows=1500, page=32,
             tree=False, shared=0, shape=7),
        # parallel samples of one prompt, each with its drafted tree: forked sequences share the prompt's pages
        dict(name="attention-forked-trees", op="attention", model="h6-kv2-d64", n_seq=9, new=13, rows=2900, page=64,
             tree=True, shared=2600, shape=8),
        # a fork: the last page that both sequences would write
        dict(name="copy-1-page", op="copy", model="qwen3-0.6b", page=16, pages=64, pairs=1),
        # a prompt's pages duplicated in a large pool
        dict(name="copy-256-pages", op="copy", model="qwen3-8b", page=16, pages=700, pairs=256),
        # one chat's accepted path of its drafted tree
        dict(name="keep-1-path", op="keep", model="qwen3-0.6b", n_seq=1, new=27, rows=700, page=16, kept=4, shape=9),
        # a large batch's accepted paths
        dict(name="keep-64-paths", op="keep", model="qwen3-8b", n_seq=64, new=33, rows=400, page=16, kept=7, shape=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "attention", "attention", "attention", "attention", "copy", "keep"])
    model, page, shape = rng.choice(list(MODELS)), rng.choice([16, 16, 32, 64, 128]), rng.randint(100, 1 << 30)
    if op == "copy":
        pages = rng.randint(8, 300)
        return dict(op=op, model=model, page=rng.choice([16, 32]), pages=pages, pairs=_log(rng, 1, pages // 2))
    if op == "keep":
        new = _log(rng, 2, 64)
        return dict(op=op, model=model, n_seq=_log(rng, 1, 40), new=new, rows=_log(rng, 1, 400), page=page,
                    kept=_log(rng, 1, min(new, 12)), shape=shape)
    kind = rng.choice(["decode", "tree", "tree", "prompt"])
    if kind == "decode":
        n_seq, new = _log(rng, 1, 96), 1
        rows = _log(rng, 1, min(24000, 400000 // n_seq))
    elif kind == "tree":
        n_seq, new = _log(rng, 1, 32), _log(rng, 2, 64)
        rows = _log(rng, 1, min(16000, 200000 // n_seq))
    else:
        n_seq = _log(rng, 1, 12)
        new, rows = _log(rng, 2, 3000 // n_seq), rng.choice([0, _log(rng, 1, 1500)])
    case = dict(op=op, model=model, n_seq=n_seq, new=new, rows=rows, page=page, tree=kind == "tree", shape=shape)
    if op == "rope":
        return dict(case, rows=min(rows, 2000), neox=rng.random() < 0.5, bias=rng.random() < 0.3)
    return dict(case, shared=rng.choice([0, 0, rows // 2]))


# ---- a batch and its pages ----------------------------------------------------------------


def _lengths(case):
    """Cached rows and new tokens of every sequence; the first has the most of both."""
    rng = random.Random(case["shape"])
    cached, new = [], []
    for s in range(case["n_seq"]):
        floor = case.get("shared", 0)
        cached.append(case["rows"] if s == 0 else max(floor, int(case["rows"] * rng.random() ** 1.5)))
        new.append(case["new"] if s == 0 else rng.randint(1, case["new"]) if case["new"] > 1 else 1)
    return cached, new


def _tables(case, cached, new, rng):
    """Page ids of every sequence, pages in no order, the shared prefix's whole pages common; pages in the pool."""
    page, common = case["page"], case.get("shared", 0) // case["page"]
    need = [-(-(c + n) // page) for c, n in zip(cached, new)]
    total = common + sum(n - common for n in need)
    ids = list(range(total + 3))
    rng.shuffle(ids)
    table = np.zeros((len(need), max(need)), np.int32)
    at = common
    for s, n in enumerate(need):
        table[s, :common] = ids[:common]
        table[s, common:n] = ids[at:at + n - common]
        at += n - common
    return table, total + 3


def _tree(n, rng):
    """A drafted tree: each token's parent among the earlier ones (-1: the last cached token), a few branches."""
    return [-1 if i == 0 or rng.random() < 0.1 else max(0, i - 1 - int(4 * rng.random() ** 2)) for i in range(n)]


def _gen(seed, salt):
    return torch.Generator("cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFF)


def _normal(shape, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _pool(layers, pages, page, width, seed):
    g = [_gen(seed, 2), _gen(seed, 3)]
    return [torch.stack([_normal((pages, page, width), x).half() for _ in range(layers)]) for x in g]


def _batch(case, seed):
    """What a serving loop has in hand for a step: the pool of one layer, lengths, tables and parents on the device."""
    nh, nkv, hd, _, _, _ = MODELS[case["model"]]
    rng = random.Random(seed * 7919 + case["shape"])
    cached, new = _lengths(case)
    table, pages = _tables(case, cached, new, rng)
    k, v = _pool(1, pages, case["page"], nkv * hd, seed)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    parent = np.concatenate([_tree(n, rng) for n in new]).astype(np.int32) if case["tree"] else None
    on = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return {"k": k, "v": v, "start": on(start), "cached": on(np.asarray(cached, np.int32)), "table": on(table),
            "parent": on(parent), "host": (cached, new, table, parent), "tokens": int(start[-1]),
            "longest": max(c + n for c, n in zip(cached, new)), "most": max(new)}


def _frequencies(case):
    _, _, hd, _, theta, _ = MODELS[case["model"]]
    return torch.tensor([theta ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device="cuda")


def prepare(case, seed):
    op = case["op"]
    s = {"case": case}
    nh, nkv, hd, layers, _, norm = MODELS[case["model"]]
    if op in ("rope", "attention"):
        s.update(_batch(case, seed))
    if op == "rope":
        width = (nh + 2 * nkv) * hd
        # projections: normal, a few channels eight times as large
        s["qkv"] = _normal((s["tokens"], width), _gen(seed, 4)) * \
            (1 + 7 * (torch.rand(width, generator=_gen(seed, 5), device="cuda") < 1 / 64))
        s["bias"] = 0.5 * _normal((width,), _gen(seed, 6)) if case["bias"] else None
        s["q_norm"] = 1 + 0.2 * _normal((hd,), _gen(seed, 7)) if norm else None
        s["k_norm"] = 1 + 0.2 * _normal((hd,), _gen(seed, 8)) if norm else None
        s["freq"] = _frequencies(case)
        s["q"] = torch.zeros((s["tokens"], nh * hd), device="cuda")
    elif op == "attention":
        s["q"] = 2 * _normal((s["tokens"], nh * hd), _gen(seed, 4))
        s["out"] = torch.zeros_like(s["q"])
    elif op == "copy":
        rng = random.Random(seed)
        ids = rng.sample(range(case["pages"]), 2 * case["pairs"])
        s["src"], s["dst"] = (np.asarray(x, np.int32) for x in (ids[::2], ids[1::2]))
        s["src_gpu"], s["dst_gpu"] = (torch.from_numpy(x).cuda().long() for x in (s["src"], s["dst"]))
        s["k"], s["v"] = _pool(layers, case["pages"], case["page"], nkv * hd, seed)
    else:
        rng = random.Random(seed * 7919 + case["shape"])
        cached, new = _lengths(case)
        table, pages = _tables(case, cached, new, rng)
        kept = [sorted(rng.sample(range(n), min(n, case["kept"]))) for n in new]
        s["table"], s["cached"] = table, np.asarray(cached, np.int32)
        s["keep_start"] = np.concatenate([[0], np.cumsum([len(x) for x in kept])]).astype(np.int32)
        s["keep"] = np.concatenate(kept).astype(np.int32)
        s["gpu"] = [torch.from_numpy(s[x]).cuda().long() for x in ("table", "cached", "keep_start", "keep")]
        s["k"], s["v"] = _pool(layers, pages, case["page"], nkv * hd, seed)
    torch.cuda.synchronize()
    return s


# ---- plain forms --------------------------------------------------------------------------


def _ancestors(s):
    """[n_seq, most, most]: token j is i or one of its ancestors, by powers of the parent relation; also each token's
    sequence and its index there."""
    n, most = s["cached"].numel(), s["most"]
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["start"].long(), token, right=True) - 1
    i = token - s["start"].long()[seq]
    if s["parent"] is None:
        return torch.ones((1, most, most), dtype=torch.bool, device="cuda").tril().expand(n, most, most), seq, i
    one = torch.eye(most, device="cuda").repeat(n, 1, 1)
    p = s["parent"].long()
    has = p >= 0
    one[seq[has], i[has], p[has]] = 1
    return torch.matrix_power(one, 64) > 0, seq, i


def _rotated(x, turn, neox):
    c, sn = turn.cos().float()[:, None], turn.sin().float()[:, None]
    if neox:
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * sn, a * sn + b * c], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rope_plain(s):
    c = s["case"]
    nh, nkv, hd, _, _, _ = MODELS[c["model"]]
    before, seq, i = _ancestors(s)
    turn = (s["cached"].long()[seq] + before[seq, i].sum(-1) - 1).double()[:, None] * s["freq"]
    x = s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]
    x = x.reshape(s["tokens"], nh + 2 * nkv, hd)
    q = _rotated(_normed(x[:, :nh], s["q_norm"]), turn, c["neox"])
    k = _rotated(_normed(x[:, nh:nh + nkv], s["k_norm"]), turn, c["neox"])
    row = s["cached"].long()[seq] + i
    row = s["table"].long()[seq, row // c["page"]] * c["page"] + row % c["page"]
    s["k"].view(-1, nkv * hd)[row] = k.reshape(s["tokens"], -1).half()
    s["v"].view(-1, nkv * hd)[row] = x[:, nh + nkv:].reshape(s["tokens"], -1).half()
    return [q.reshape(s["tokens"], -1), s["k"], s["v"]]


def _attention_plain(s):
    c = s["case"]
    nh, nkv, hd, _, _, _ = MODELS[c["model"]]
    n, most, longest, group = c["n_seq"], s["most"], s["longest"], nh // nkv
    before, seq, i = _ancestors(s)
    row = torch.arange(longest, device="cuda")
    at = s["table"].long()[:, row // c["page"]] * c["page"] + row % c["page"]
    k, v = (s[x].view(-1, nkv, hd)[at].float().transpose(1, 2).contiguous() for x in ("k", "v"))
    q = torch.zeros((n, most, nh, hd), device="cuda")
    q[seq, i] = s["q"].reshape(-1, nh, hd)
    q = q.reshape(n, most, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, group * most, hd)
    score = (q @ k.transpose(2, 3).contiguous() / math.sqrt(hd)).reshape(n, nkv, group, most, longest)
    j = row - s["cached"].long()[:, None]
    seen = before.gather(2, j.clamp(0, most - 1)[:, None].expand(n, most, longest)) & (j < most)[:, None]
    seen = (seen | (j < 0)[:, None])[:, None, None]
    score = score.masked_fill_(~seen, -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    p = (p / p.sum(-1, keepdim=True)).reshape(n, nkv, group * most, longest)
    o = (p @ v).reshape(n, nkv, group, most, hd).permute(0, 3, 1, 2, 4)
    return o[seq, i].reshape(s["tokens"], nh * hd)


def _keep_plain(s):
    table, cached, start, keep = s["gpu"]
    page = s["case"]["page"]
    n = torch.arange(keep.numel(), device="cuda")
    seq = torch.searchsorted(start, n, right=True) - 1
    src, dst = cached[seq] + keep, cached[seq] + n - start[seq]
    src = table[seq, src // page] * page + src % page
    dst = table[seq, dst // page] * page + dst % page
    k, v = (s[x].view(s[x].shape[0], -1, s[x].shape[-1]) for x in ("k", "v"))
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    return [s["k"], s["v"]]


# ---- the framework's calls ----------------------------------------------------------------


def _handles(s):
    """The binding and the descriptions of pool and batch that a program keeps, made on the first pass."""
    if "own" not in s:
        sys.path.insert(0, os.path.abspath("minxfmr.cpp_amd"))
        import mxhip

        mxhip.init(0)
        nh, nkv, hd, _, _, _ = MODELS[s["case"]["model"]]
        k = s["k"]
        pool = mxhip.KvPool(k.data_ptr(), s["v"].data_ptr(), n_layer=k.shape[0], n_pages=k.shape[1],
                            page_rows=k.shape[2], n_kv=nkv, head_dim=hd)
        batch = work = None
        if "start" in s:
            batch = mxhip.KvBatch(s["case"]["n_seq"], s["tokens"], s["start"].data_ptr(), s["cached"].data_ptr(),
                                  s["table"].data_ptr(), s["table"].shape[1],
                                  None if s["parent"] is None else s["parent"].data_ptr())
        if s["case"]["op"] == "attention":
            work = torch.empty(mxhip.attention_paged_workspace(pool, batch, nh), dtype=torch.uint8, device="cuda")
        s["own"] = mxhip, pool, batch, work
    return s["own"]


def _run_own(s):
    mxhip, pool, batch, work = _handles(s)
    c = s["case"]
    nh = MODELS[c["model"]][0]
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if c["op"] == "rope":
        mxhip.qk_rope_append(pool, 0, batch, s["qkv"].data_ptr(), s["qkv"].shape[1], at(s["bias"]), at(s["q_norm"]),
                             at(s["k_norm"]), EPS, s["freq"].data_ptr(), c["neox"], nh, s["q"].data_ptr())
        return [s["q"], s["k"], s["v"]]
    if c["op"] == "attention":
        mxhip.attention_paged(pool, 0, batch, s["q"].data_ptr(), nh, s["out"].data_ptr(), work.data_ptr(),
                              work.numel())
        return s["out"]
    if c["op"] == "copy":
        mxhip.kv_copy_pages(pool, s["src"], s["dst"])
    else:
        mxhip.kv_keep_rows(pool, s["table"], s["cached"], s["keep_start"], s["keep"])
    return [s["k"], s["v"]]


def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op == "rope":
        return _rope_plain(s)
    if op == "attention":
        return _attention_plain(s)
    if op == "copy":
        src, dst = s["src_gpu"], s["dst_gpu"]
        s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
        return [s["k"], s["v"]]
    return _keep_plain(s)


def work(case):
    nh, nkv, hd, layers, _, _ = MODELS[case["model"]]
    row = 4 * nkv * hd  # K and V of a token, fp16
    if case["op"] == "copy":
        return {"bytes": 2 * case["pairs"] * case["page"] * row * layers, "flops": 0}
    cached, new = _lengths(case)
    if case["op"] == "keep":
        return {"bytes": 2 * sum(min(n, case["kept"]) for n in new) * row * layers, "flops": 0}
    tokens = sum(new)
    if case["op"] == "rope":
        return {"bytes": tokens * (4 * (2 * nh + 2 * nkv) * hd + row), "flops": 10 * tokens * (nh + nkv) * hd}
    common = case["shared"] // case["page"] * case["page"]
    rows = common + sum(c + n - common for c, n in zip(cached, new))
    # a drafted token's ancestors are at most the tokens before it
    seen = sum(c * n + n * (n + 1) // 2 for c, n in zip(cached, new))
    return {"bytes": 8 * tokens * nh * hd + rows * row, "flops": 4 * nh * hd * seen}


# ---- 64-bit references ----------------------------------------------------------------------


def _path(parent, i):
    """i and its ancestors; without parents every token up to i."""
    if parent is None:
        return list(range(i + 1))
    at = []
    while i >= 0:
        at.append(i)
        i = int(parent[i])
    return at[::-1]


def _exact_rope(case, seed):
    s = prepare(case, seed)
    nh, nkv, hd, _, theta, norm = MODELS[case["model"]]
    cached, new, table, parent = s["host"]
    x = s["qkv"].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()
    pos, slot, at = [], [], 0
    for q, (c, n) in enumerate(zip(cached, new)):
        for i in range(n):
            depth = i if parent is None else len(_path(parent[at:at + n], i)) - 1
            pos.append(c + depth)
            slot.append(int(table[q, (c + i) // case["page"]]) * case["page"] + (c + i) % case["page"])
        at += n
    pos = torch.tensor(pos, dtype=torch.float64, device="cuda")[:, None, None]
    angle = pos * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    turn = torch.polar(torch.ones_like(angle), angle)

    def rotate(h, w):
        if w is not None:
            h = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
        pair = torch.complex(h[..., :hd // 2], h[..., hd // 2:]) if case["neox"] else \
            torch.view_as_complex(h.reshape(*h.shape[:-1], hd // 2, 2).contiguous())
        pair = pair * turn
        return torch.cat([pair.real, pair.imag], -1) if case["neox"] else torch.view_as_real(pair).flatten(-2)

    q, k, v = x.reshape(len(slot), -1, hd).split([nh, nkv, nkv], 1)
    kk, vv = s["k"].double(), s["v"].double()
    kk.view(-1, nkv * hd)[slot] = rotate(k, s["k_norm"]).reshape(len(slot), -1)
    vv.view(-1, nkv * hd)[slot] = v.reshape(len(slot), -1)
    return [rotate(q, s["q_norm"]).reshape(len(slot), -1), kk, vv]


def _exact_attention(case, seed):
    s = prepare(case, seed)
    nh, nkv, hd, _, _, _ = MODELS[case["model"]]
    cached, new, table, parent = s["host"]
    out = torch.empty((s["tokens"], nh, hd), dtype=torch.float64, device="cuda")
    at = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        pages = torch.from_numpy(table[b, :-(-(c + n) // case["page"])].astype(np.int64)).cuda()
        k, v = (s[x][0, pages].reshape(-1, nkv, hd)[:c + n].double() for x in ("k", "v"))
        hidden = torch.ones((n, c + n), dtype=torch.bool)
        hidden[:, :c] = False
        for i in range(n):
            hidden[i, [c + j for j in _path(None if parent is None else parent[at:at + n], i)]] = False
        hidden = hidden.cuda()
        q = s["q"][at:at + n].double().reshape(n, nh, hd)
        for h in range(nh):
            w = q[:, h] @ k[:, h * nkv // nh].T / math.sqrt(hd)
            out[at:at + n, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[:, h * nkv // nh]
        at += n
    return out.reshape(s["tokens"], nh * hd)


def exact(case, seed):
    if case["op"] == "rope":
        return _exact_rope(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, seed)
    s = prepare(case, seed)
    k, v = (s[x].double() for x in ("k", "v"))
    page = case["page"]
    if case["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b], v[:, b] = s["k"][:, a].double(), s["v"][:, a].double()
        return [k, v]
    for b in range(case["n_seq"]):
        for i, kept in enumerate(s["keep"][s["keep_start"][b]:s["keep_start"][b + 1]].tolist()):
            to, frm = int(s["cached"][b]) + i, int(s["cached"][b]) + kept
            for old, to_pool in ((s["k"], k), (s["v"], v)):
                to_pool[:, int(s["table"][b, to // page]), to % page] = \
                    old[:, int(s["table"][b, frm // page]), frm % page].double()
    return [k, v]
