"""The operators that read less than the whole of a paged K/V cache, as measurable cases.

A runtime that serves many sequences over long contexts need not read every row
for every sequence: what a batch has in common is read once for all of it, and
of a long context each query reads the blocks of rows that promise most:

- ``shared``  ``mxh_attention_shared``: attention of a batch whose sequences
              begin, group by group, with the same pages;
- ``bounds``  ``mxh_kv_block_bounds``: the least and the greatest key of every
              block of rows that a step's tokens were appended to, a value a
              dimension;
- ``select``  ``mxh_kv_select_blocks``: for each token and kv head the blocks
              whose bounds allow the largest scores, besides the first and the
              last ones;
- ``blocks``  ``mxh_attention_blocks``: attention over the chosen blocks.

With ``own`` false ``run`` computes the same in elementary torch operations.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

# heads, kv heads, head dim: the benchmark's models, and narrower heads
MODELS = {
    "qwen3-0.6b": (16, 8, 128),
    "qwen3-8b": (32, 8, 128),
    "llama3-8b": (32, 8, 128),
    "h6-kv2-d64": (6, 2, 64),
    "h8-kv1-d32": (8, 1, 32),
}


def listed():
    return [
        # parallel samples: four answers to one prompt, a token each
        dict(name="shared-4-samples", op="shared", model="qwen3-0.6b", n_seq=4, groups=1, new=1, shared=1000, rows=200,
             page=16, tree=False, shape=1),
        # decode: a batch of chats behind one long system prompt
        dict(name="shared-64-chats", op="shared", model="qwen3-8b", n_seq=64, groups=1, new=1, shared=8000, rows=1000,
             page=32, tree=False, shape=2),
        # speculative decoding: drafted trees of samples of three prompts
        dict(name="shared-trees", op="shared", model="h6-kv2-d64", n_seq=16, groups=3, new=13, shared=2900, rows=400,
             page=64, tree=True, shape=3),
        # questions of different lengths about one document
        dict(name="shared-questions", op="shared", model="llama3-8b", n_seq=12, groups=1, new=400, shared=6000, rows=0,
             page=32, tree=False, shape=4),
        # decode: the next token of one chat, where the call's latency counts
        dict(name="bounds-1-token", op="bounds", model="qwen3-0.6b", n_seq=1, new=1, rows=700, page=64, block=64,
             shape=5),
        # prompts of different lengths, appended in one pass
        dict(name="bounds-prompts", op="bounds", model="qwen3-8b", n_seq=7, new=6000, rows=300, page=32, block=32,
             shape=6),
        # decode: one chat at a long context
        dict(name="select-1-at-60000", op="select", model="qwen3-8b", n_seq=1, new=1, rows=60000, page=64, block=64,
             first=1, last=2, select=32, shape=7),
        # decode: a batch of chats of very different lengths
        dict(name="select-batch-48", op="select", model="llama3-8b", n_seq=48, new=1, rows=16000, page=32, block=32,
             first=1, last=2, select=40, shape=8),
        # prefill: a chunk of a prompt behind a long cached part
        dict(name="select-prompt-512", op="select", model="qwen3-8b", n_seq=1, new=512, rows=30000, page=64, block=64,
             first=1, last=4, select=32, shape=9),
        # the attention that follows each of these
        dict(name="blocks-1-at-60000", op="blocks", model="qwen3-8b", n_seq=1, new=1, rows=60000, page=64, block=64,
             first=1, last=2, select=32, shape=7),
        dict(name="blocks-batch-48", op="blocks", model="llama3-8b", n_seq=48, new=1, rows=16000, page=32, block=32,
             first=1, last=2, select=40, shape=8),
        dict(name="blocks-prompt-512", op="blocks", model="qwen3-8b", n_seq=1, new=512, rows=30000, page=64, block=64,
             first=1, last=4, select=32, shape=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "bounds", "select", "select", "blocks", "blocks"])
    model, page, shape = rng.choice(list(MODELS)), rng.choice([16, 32, 64, 128]), rng.randint(100, 1 << 30)
    if op == "shared":
        kind = rng.choice(["decode", "tree", "prompt"])
        n_seq = _log(rng, 2, {"decode": 64, "tree": 24, "prompt": 10}[kind])
        new = {"decode": 1, "tree": _log(rng, 2, 48), "prompt": _log(rng, 2, 2000 // n_seq)}[kind]
        return dict(op=op, model=model, n_seq=n_seq, groups=rng.randint(1, max(1, n_seq // 2)), new=new,
                    shared=_log(rng, 100, 8000), rows=rng.choice([0, _log(rng, 1, 1000)]), page=page,
                    tree=kind == "tree", shape=shape)
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    kind = rng.choice(["decode", "few", "prompt"])
    if kind == "decode":
        n_seq, new = _log(rng, 1, 48), 1
        rows = _log(rng, 1, min(60000, 400000 // n_seq))
    elif kind == "few":
        n_seq, new = _log(rng, 1, 16), rng.randint(2, 8)
        rows = _log(rng, 1, min(30000, 150000 // n_seq))
    else:
        n_seq = _log(rng, 1, 4)
        new, rows = _log(rng, 9, 400 // n_seq), _log(rng, 1, 20000)
    case = dict(op=op, model=model, n_seq=n_seq, new=new, rows=rows, page=page, block=block, shape=shape)
    if op == "bounds":
        return dict(case, new=_log(rng, 1, 5000 // n_seq), rows=min(rows, 4000))
    first, last = rng.randint(0, 2), rng.randint(1, 4)
    if op == "select":  # (where blocks compete)
        case["rows"] = rows = max(rows, 16 * block)
    return dict(case, first=first, last=last,
                select=first + last + _log(rng, 1, max(2, min(2000, rows // 2 if op == "select" else 2000) // block)))


# ---- a batch and its pages ----------------------------------------------------------------


def _lengths(case):
    """Cached rows and new tokens of every sequence; the first has the most of both."""
    rng = random.Random(case["shape"])
    cached, new = [], []
    for s in range(case["n_seq"]):
        cached.append(case["rows"] if s == 0 else int(case["rows"] * rng.random() ** 1.5))
        new.append(case["new"] if s == 0 else rng.randint(1, case["new"]) if case["new"] > 1 else 1)
    return cached, new


def _groups(case):
    """First sequence of every group and one past the last, rows that each group has in common (whole pages)."""
    rng = random.Random(case["shape"] + 1)
    n = case["groups"]
    first = [0] + sorted(rng.sample(range(1, case["n_seq"]), n - 1)) + [case["n_seq"]]
    shared = [case["shared"] if g == 0 else rng.randint(case["shared"] // 4, case["shared"]) for g in range(n)]
    return first, [x // case["page"] * case["page"] for x in shared]


def _tables(case, need, common, rng):
    """Page ids of every sequence (need[s] of them, common[s] = (group, pages) of those its group's) in no order;
    pages in the pool."""
    sizes = {}
    for g, n in common:
        sizes[g] = n
    total = sum(sizes.values()) + sum(n - c for n, (_, c) in zip(need, common)) + 3
    ids = list(range(total))
    rng.shuffle(ids)
    at, prefix = 0, {}
    for g, n in sizes.items():
        prefix[g] = ids[at:at + n]
        at += n
    table = np.zeros((len(need), max(need)), np.int32)
    for s, (n, (g, c)) in enumerate(zip(need, common)):
        table[s, :c] = prefix[g]
        table[s, c:n] = ids[at:at + n - c]
        at += n - c
    return table, total


def _tree(n, rng):
    """A drafted tree: each token's parent among the earlier ones (-1: the last cached token), a few branches."""
    return [-1 if i == 0 or rng.random() < 0.1 else max(0, i - 1 - int(4 * rng.random() ** 2)) for i in range(n)]


def _gen(seed, salt):
    return torch.Generator("cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFF)


def _normal(shape, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _on(a, kind=np.int32):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a, kind)).cuda()


def _keys(pages, page, nkv, hd, seed):
    """A page's keys lie around a point of its own, as what a context speaks of changes; a few channels are large."""
    g = _gen(seed, 2)
    large = 1 + 5 * (torch.rand((nkv, hd), generator=g, device="cuda") < 1 / 32)
    point = 0.7 * _normal((pages, 1, nkv, hd), g)
    return ((_normal((pages, page, nkv, hd), g) + point) * large).half().reshape(1, pages, page, nkv * hd)


def _least_and_greatest(k, rows, block):
    """[..., rows, width] keys to [..., blocks, 2, width]; rows: whole blocks."""
    k = k.unflatten(-2, (rows // block, block))
    return torch.stack([k.amin(-2), k.amax(-2)], -2)


def prepare(case, seed):
    """What a serving loop has in hand for a step: the pool of one layer, lengths, tables and parents on the device."""
    op = case["op"]
    nh, nkv, hd = MODELS[case["model"]]
    rng = random.Random(seed * 7919 + case["shape"])
    cached, new = _lengths(case)
    common = [(0, 0)] * case["n_seq"]
    s = {"case": case}
    if op == "shared":
        first, shared = _groups(case)
        group = np.repeat(np.arange(case["groups"]), np.diff(first))
        common = [(int(g), shared[g] // case["page"]) for g in group]
        cached = [c + shared[g] for c, g in zip(cached, group)]
        s["group_start"], s["group_shared"], s["group_host"] = _on(first), _on(shared), (first, shared)
    need = [-(-(c + n) // case["page"]) for c, n in zip(cached, new)]
    table, pages = _tables(case, need, common, rng)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    parent = np.concatenate([_tree(n, rng) for n in new]).astype(np.int32) if case.get("tree") else None
    s.update(start=_on(start), cached=_on(cached), table=_on(table), parent=_on(parent), tokens=int(start[-1]),
             most=max(new), longest=max(c + n for c, n in zip(cached, new)), host=(cached, new, table, parent))
    s["k"] = _keys(pages, case["page"], nkv, hd, seed)
    if op in ("shared", "blocks"):
        s["v"] = _normal(s["k"].shape, _gen(seed, 3)).half()
    # a sequence's queries have much in common, a head's more; the large ones of them are the context's questions
    seq = torch.repeat_interleave(torch.arange(case["n_seq"], device="cuda"), _on(new, np.int64))
    like = _normal((case["n_seq"], nh, hd), _gen(seed, 4))[seq]
    s["q"] = (like + 0.6 * _normal((s["tokens"], nh, hd), _gen(seed, 5))).reshape(s["tokens"], nh * hd).contiguous()
    if op in ("shared", "blocks"):
        s["att"] = torch.zeros_like(s["q"])
    if op in ("bounds", "select"):
        block = case["block"]
        s["bounds"] = _least_and_greatest(s["k"].reshape(1, pages, case["page"], nkv, hd).transpose(2, 3), case["page"],
                                          block).transpose(2, 3).contiguous()  # [1, pages, blocks, kv heads, 2, hd]
        if op == "bounds":  # of what the step appended nothing is known yet
            s["bounds"].view(pages, -1)[torch.from_numpy(np.unique(np.concatenate(
                [t[c // case["page"]:n] for t, c, n in zip(table, cached, need)])).astype(np.int64)).cuda()] = 0
    if op == "select":
        s["chosen"] = torch.zeros((s["tokens"], nkv, case["select"]), dtype=torch.int32, device="cuda")
    if op == "blocks":
        own_block, _, _ = _own_blocks(s)
        n = s["longest"] // case["block"] + 1
        liked = 2 * _normal((case["n_seq"], nkv, n), _gen(seed, 6))[seq] + _normal((s["tokens"], nkv, n), _gen(seed, 7))
        s["chosen"] = _chosen(case, liked, own_block)
    torch.cuda.synchronize()
    return s


# ---- plain forms --------------------------------------------------------------------------


def _tokens(s):
    """Each token's sequence and its index there."""
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["start"].long(), token, right=True) - 1
    return seq, token - s["start"].long()[seq]


def _own_blocks(s):
    seq, i = _tokens(s)
    return (s["cached"].long()[seq] + i) // s["case"]["block"], seq, i


def _chosen(case, score, own_block):
    """[tokens, kv heads, blocks] scores to the ascending list of the first, the last and the best blocks, -1 behind."""
    n = score.shape[-1]
    block, last = torch.arange(n, device="cuda"), own_block[:, None, None]
    score = score.masked_fill((block < case["first"]) | (block > last - case["last"]), math.inf)
    score = score.masked_fill(block > last, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :case["select"]]
    best = torch.where(best <= last, best, n).sort(-1).values
    list_ = torch.full((*score.shape[:-1], case["select"]), -1, dtype=torch.int32, device="cuda")
    list_[..., :best.shape[-1]] = torch.where(best < n, best, -1).int()
    return list_


def _ancestors(s):
    """[n_seq, most, most]: token j is i or one of its ancestors, by powers of the parent relation."""
    n, most = s["cached"].numel(), s["most"]
    seq, i = _tokens(s)
    if s["parent"] is None:
        return torch.ones((1, most, most), dtype=torch.bool, device="cuda").tril().expand(n, most, most)
    one = torch.eye(most, device="cuda").repeat(n, 1, 1)
    p = s["parent"].long()
    has = p >= 0
    one[seq[has], i[has], p[has]] = 1
    return torch.matrix_power(one, 64) > 0


def _pool_rows(s, seq, row):
    """The rows of the pool that rows `row` of sequences `seq` are."""
    page = s["case"]["page"]
    last = s["table"].shape[1] - 1
    return s["table"].long()[seq, (row // page).clamp(0, last)] * page + row % page


def _part(q, k, v, seen):
    """Attention of [n, kv heads, group, tokens, hd] over [n, kv heads, rows, hd], seen [n, 1, 1, tokens, rows]: the
    unscaled sums, the largest scores, the sums of exponentials."""
    n, nkv, group, most, hd = q.shape
    score = (q.reshape(n, nkv, group * most, hd) @ k.transpose(2, 3).contiguous() / math.sqrt(hd))
    score = score.reshape(n, nkv, group, most, -1).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top.clamp(min=-1e30)).exp_()
    o = (p.reshape(n, nkv, group * most, -1) @ v).reshape(n, nkv, group, most, hd)
    return o, top, p.sum(-1, keepdim=True)


def _padded(x, rank, at, shape, nkv):
    """[tokens, nh, hd] to [rows of `shape`, kv heads, group, tokens, hd], token t at (rank[t], at[t])."""
    nh, hd = x.shape[1:]
    y = torch.zeros((*shape, nh, hd), device="cuda")
    y[rank, at] = x
    return y.reshape(*shape, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4)


def _packed(parts, rank, at):
    """Back to [tokens, nh, ...]."""
    return [x.permute(0, 3, 1, 2, 4)[rank, at].flatten(1, 2) for x in parts]


def _shared_plain(s):
    c = s["case"]
    nh, nkv, hd = MODELS[c["model"]]
    seq, i = _tokens(s)
    q = s["q"].reshape(-1, nh, hd)
    k, v = (s[x].view(-1, nkv, hd) for x in ("k", "v"))
    first, shared = s["group_start"].long(), s["group_shared"].long()
    # the prefixes, once for all tokens of a group
    group = torch.searchsorted(first, seq, right=True) - 1
    in_group = torch.arange(s["tokens"], device="cuda") - s["start"].long()[first[group]]
    sizes = s["group_host"][0]
    most = max(sum(s["host"][1][a:b]) for a, b in zip(sizes, sizes[1:]))
    row = torch.arange(max(s["group_host"][1]), device="cuda")
    at = _pool_rows(s, first[:-1, None], row)
    gather = lambda x, at: x[at].float().transpose(1, 2).contiguous()  # noqa: E731
    seen = (row < shared[:, None])[:, None, None, None]
    one = _packed(_part(_padded(q, group, in_group, (c["groups"], most), nkv), gather(k, at), gather(v, at), seen),
                  group, in_group)
    # what each sequence has of its own
    begin = shared[torch.searchsorted(first, torch.arange(c["n_seq"], device="cuda"), right=True) - 1]
    row = torch.arange(int(max(a + n - b for a, n, b in zip(*s["host"][:2], _own_from(s)))), device="cuda")
    at = _pool_rows(s, torch.arange(c["n_seq"], device="cuda")[:, None], begin[:, None] + row)
    j = begin[:, None] + row - s["cached"].long()[:, None]
    seen = _ancestors(s).gather(2, j.clamp(0, s["most"] - 1)[:, None].expand(-1, s["most"], -1))
    seen = ((seen & (j < s["most"])[:, None]) | (j < 0)[:, None])[:, None, None]
    two = _packed(_part(_padded(q, seq, i, (c["n_seq"], s["most"]), nkv), gather(k, at), gather(v, at), seen), seq, i)
    top = torch.maximum(one[1], two[1])
    a, b = (one[1] - top).exp(), (two[1] - top).exp()
    return ((a * one[0] + b * two[0]) / (a * one[2] + b * two[2])).reshape(s["tokens"], nh * hd)


def _own_from(s):
    """The row that each sequence's own ones begin at."""
    first, shared = s["group_host"]
    return np.repeat(shared, np.diff(first)).tolist()


def _bounds_plain(s):
    c = s["case"]
    nkv, hd = MODELS[c["model"]][1:]
    block, n_seq = c["block"], c["n_seq"]
    cached, new = s["cached"].long(), s["start"].long().diff()
    b = cached // block
    count = (cached + new - 1) // block - b + 1
    seq = torch.repeat_interleave(torch.arange(n_seq, device="cuda"), count)
    b = b[seq] + torch.arange(seq.numel(), device="cuda") - (count.cumsum(0) - count)[seq]
    row = b[:, None] * block + torch.arange(block, device="cuda")
    k = s["k"].view(-1, nkv, hd)[_pool_rows(s, seq[:, None], row)]
    gone = (row >= (cached + new)[seq, None])[..., None, None]
    least, greatest = k.masked_fill(gone, math.inf).amin(1), k.masked_fill(gone, -math.inf).amax(1)
    to = _pool_rows(s, seq, b * block) // block
    s["bounds"].view(-1, nkv, 2, hd)[to] = torch.stack([least, greatest], 2)
    return s["bounds"]


def _select_plain(s):
    c = s["case"]
    nh, nkv, hd = MODELS[c["model"]]
    last, seq, i = _own_blocks(s)
    block = torch.arange(s["longest"] // c["block"] + 1, device="cuda")
    at = _pool_rows(s, torch.arange(c["n_seq"], device="cuda")[:, None], block * c["block"]) // c["block"]
    bound = s["bounds"].view(-1, nkv, 2, hd)[at].double()  # [n_seq, blocks, kv heads, 2, hd]
    least, greatest = (bound[:, :, :, x].permute(0, 2, 3, 1).contiguous() for x in (0, 1))
    q = torch.zeros((c["n_seq"], s["most"], nh, hd), dtype=torch.float64, device="cuda")
    q[seq, i] = s["q"].reshape(-1, nh, hd).double()
    q = q.reshape(c["n_seq"], s["most"], nkv, -1, hd).permute(0, 2, 3, 1, 4).reshape(c["n_seq"], nkv, -1, hd)
    # the sum of the larger of q x least and q x greatest, in 64 bits: scores next to one another decide
    score = q.clamp(min=0) @ greatest + q.clamp(max=0) @ least
    score = score.reshape(c["n_seq"], nkv, nh // nkv, s["most"], -1).amax(2)
    return _chosen(c, score.permute(0, 2, 1, 3)[seq, i], last)


def _blocks_plain(s):
    c = s["case"]
    nh, nkv, hd = MODELS[c["model"]]
    last, seq, i = _own_blocks(s)
    place = s["cached"].long()[seq] + i
    chosen, block = s["chosen"].long(), c["block"]
    if s["tokens"] * c["select"] * block > 400000:
        # many tokens: every row of the sequences, what was not chosen masked
        n = -(-s["longest"] // block) * block
        row = torch.arange(n, device="cuda")
        at = _pool_rows(s, torch.arange(c["n_seq"], device="cuda")[:, None], row)
        k, v = (s[x].view(-1, nkv, hd)[at].float().transpose(1, 2).contiguous() for x in ("k", "v"))
        has = torch.zeros((s["tokens"], nkv, n // block + 1), dtype=torch.bool, device="cuda")
        has.scatter_(2, torch.where(chosen < 0, n // block, chosen), True)
        seen = torch.zeros((c["n_seq"], s["most"], nkv, n), dtype=torch.bool, device="cuda")
        seen[seq, i] = has[..., :-1].repeat_interleave(block, 2) & (row <= place[:, None])[:, None]
        parts = _part(_padded(s["q"].reshape(-1, nh, hd), seq, i, (c["n_seq"], s["most"]), nkv), k, v,
                      seen.permute(0, 2, 1, 3)[:, :, None])
        o, _, l = _packed(parts, seq, i)
    else:
        # few: the chosen rows of every token and kv head
        row = (chosen[..., None] * block + torch.arange(block, device="cuda")).flatten(2)
        at = _pool_rows(s, seq[:, None, None], row.clamp(min=0))
        head = torch.arange(nkv, device="cuda")[:, None]
        k, v = (s[x].view(-1, nkv, hd)[at, head].float() for x in ("k", "v"))
        seen = ((row >= 0) & (row <= place[:, None, None]))[:, :, None, None]
        o, _, l = _part(s["q"].reshape(s["tokens"], nkv, nh // nkv, 1, hd), k, v, seen)
        o, l = o[:, :, :, 0], l[:, :, :, 0]
    return (o / l).reshape(s["tokens"], nh * hd)


# ---- the framework's calls ----------------------------------------------------------------


def _handles(s):
    """The binding and the descriptions of pool, batch, groups and blocks that a program keeps, made on the first
    pass."""
    if "own" not in s:
        sys.path.insert(0, os.path.abspath("minxfmr.cpp_amd"))
        import mxhip

        mxhip.init(0)
        c, k = s["case"], s["k"]
        nh, nkv, hd = MODELS[c["model"]]
        pool = mxhip.KvPool(k.data_ptr(), s.get("v", k).data_ptr(), n_layer=1, n_pages=k.shape[1], page_rows=k.shape[2],
                            n_kv=nkv, head_dim=hd)
        batch = mxhip.KvBatch(c["n_seq"], s["tokens"], s["start"].data_ptr(), s["cached"].data_ptr(),
                              s["table"].data_ptr(), s["table"].shape[1],
                              None if s["parent"] is None else s["parent"].data_ptr())
        if c["op"] == "shared":
            what = mxhip.KvGroups(c["groups"], s["group_start"].data_ptr(), s["group_shared"].data_ptr())
            size = mxhip.attention_shared_workspace(pool, batch, what, nh)
        else:
            what = mxhip.KvBlocks(s["bounds"].data_ptr() if "bounds" in s else None, block_rows=c["block"],
                                  n_first=c.get("first", 0), n_last=c.get("last", 1), n_select=c.get("select", 1))
            size = 0
            if c["op"] == "select":
                size = mxhip.kv_select_workspace(pool, batch, what, nh)
            elif c["op"] == "blocks":
                size = mxhip.attention_blocks_workspace(pool, batch, what, nh)
        s["own"] = mxhip, pool, batch, what, torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return s["own"]


def _run_own(s):
    mxhip, pool, batch, what, work = _handles(s)
    op, nh = s["case"]["op"], MODELS[s["case"]["model"]][0]
    if op == "shared":
        mxhip.attention_shared(pool, 0, batch, what, s["q"].data_ptr(), nh, s["att"].data_ptr(), work.data_ptr(),
                               work.numel())
        return s["att"]
    if op == "bounds":
        mxhip.kv_block_bounds(pool, 0, batch, what)
        return s["bounds"]
    if op == "select":
        mxhip.kv_select_blocks(pool, 0, batch, what, s["q"].data_ptr(), nh, s["chosen"].data_ptr(), work.data_ptr(),
                               work.numel())
        return s["chosen"]
    mxhip.attention_blocks(pool, 0, batch, what, s["chosen"].data_ptr(), s["q"].data_ptr(), nh, s["att"].data_ptr(),
                           work.data_ptr(), work.numel())
    return s["att"]


def run(s):
    if own:
        return _run_own(s)
    return {"shared": _shared_plain, "bounds": _bounds_plain, "select": _select_plain,
            "blocks": _blocks_plain}[s["case"]["op"]](s)


def work(case):
    nh, nkv, hd = MODELS[case["model"]]
    cached, new = _lengths(case)
    tokens, row = sum(new), 4 * nkv * hd  # K and V of a row, fp16
    if case["op"] == "shared":
        first, shared = _groups(case)
        rows = sum(shared) + sum(cached) + tokens
        # a drafted token's ancestors are at most the tokens before it
        seen = sum((sh + c) * n + n * (n + 1) // 2 for sh, c, n in
                   zip(np.repeat(shared, np.diff(first)).tolist(), cached, new))
        return {"bytes": 8 * tokens * nh * hd + rows * row, "flops": 4 * nh * hd * seen}
    block = case["block"]
    if case["op"] == "bounds":
        blocks = sum((c + n - 1) // block - c // block + 1 for c, n in zip(cached, new))
        rows = sum(c + n - c // block * block for c, n in zip(cached, new))
        return {"bytes": rows * row // 2 + blocks * row, "flops": 2 * rows * nkv * hd}
    own_blocks = [[(c + i) // block for i in range(n)] for c, n in zip(cached, new)]
    if case["op"] == "select":
        # blocks that compete, each one's bounds once for its sequence; nothing is read where all are taken
        compete = [[max(0, b + 1 - case["first"] - case["last"]) if b >= case["select"] else 0 for b in bs]
                   for bs in own_blocks]
        out = 4 * tokens * nkv * case["select"]
        return {"bytes": sum(map(max, compete)) * row + 4 * tokens * nh * hd + out,
                "flops": 4 * nh * hd * sum(map(sum, compete))}
    rows = [[min(case["select"] * block, c + i + 1) for i in range(n)] for c, n in zip(cached, new)]
    # what a sequence's tokens choose is at least what one of them does
    return {"bytes": sum(map(max, rows)) * row + 8 * tokens * nh * hd + 4 * tokens * nkv * case["select"],
            "flops": 4 * nh * hd * sum(map(sum, rows))}


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


def exact(case, seed):
    if case["op"] == "select":
        return None  # whole numbers
    s = prepare(case, seed)
    nh, nkv, hd = MODELS[case["model"]]
    cached, new, table, parent = s["host"]
    page = case["page"]
    if case["op"] == "bounds":
        out, block = s["bounds"].double(), case["block"]
        for b, (c, n) in enumerate(zip(cached, new)):
            for x in range(c // block, (c + n - 1) // block + 1):
                id_, r = int(table[b, x * block // page]), x * block % page
                k = s["k"][0, id_, r:r + min(block, c + n - x * block)].double().reshape(-1, nkv, hd)
                out[0, id_, r // block, :, 0], out[0, id_, r // block, :, 1] = k.min(0).values, k.max(0).values
        return out
    out = torch.empty((s["tokens"], nh, hd), dtype=torch.float64, device="cuda")
    at = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        pages = torch.from_numpy(table[b, :-(-(c + n) // page)].astype(np.int64)).cuda()
        k, v = (s[x][0, pages].reshape(-1, nkv, hd)[:c + n].double() for x in ("k", "v"))
        hidden = torch.ones((n, c + n), dtype=torch.bool)
        hidden[:, :c] = False
        for i in range(n):
            hidden[i, [c + j for j in _path(None if parent is None else parent[at:at + n], i)]] = False
        hidden = hidden.cuda()
        q = s["q"][at:at + n].double().reshape(n, nh, hd)
        for g in range(nkv):
            off = hidden
            if case["op"] == "blocks":
                there = (s["chosen"][at:at + n, g].long()[:, :, None] ==
                         (torch.arange(c + n, device="cuda") // case["block"])).any(1) \
                    if n * (c + n) * case["select"] < 1 << 28 else _there(s["chosen"][at:at + n, g], c + n, case["block"])
                off = hidden | ~there
            for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                w = (q[:, h] @ k[:, g].T / math.sqrt(hd)).masked_fill(off, -math.inf)
                out[at:at + n, h] = torch.softmax(w, -1) @ v[:, g]
        at += n
    return out.reshape(s["tokens"], nh * hd)


def _there(chosen, rows, block):
    """[tokens, rows]: the row's block is among the token's, block by block of the lists."""
    there = torch.zeros((chosen.shape[0], rows // block + 2), dtype=torch.bool, device="cuda")
    for x in range(chosen.shape[1]):
        t = (chosen[:, x] >= 0).nonzero()[:, 0]
        there[t, chosen[t, x].long()] = True
    return there.repeat_interleave(block, 1)[:, :rows]
