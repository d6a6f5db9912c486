"""Speculative decoding and page selection over the paged KV pools, as measured cases.

Five operators of one serving loop:

* ``tree``: attention of a tree of drafted tokens per request over its cached context, each
  node seeing the context, its ancestors and itself (``ops.tree_attention``);
* ``rows``: after verification, the K/V rows of the accepted nodes of every layer move up
  behind the context (``ops.compact_rows``);
* ``pages``: whole pages of every layer copied to other pages, for forks and for
  copy-on-write (``ops.copy_pages``);
* ``bounds``: elementwise minimum and maximum of the keys of full pages
  (``ops.page_bounds``), kept beside the cache;
* ``sparse``: one-token decode over the ``num_pages`` pages per request and KV head whose
  bounds promise the largest scores, plus the page being written (``ops.sparse_attention``).

``run`` computes them with elementary torch operations, or with the package's kernels when
``own`` is set.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HEADS = dict(q_heads=32, kv_heads=8, head_dim=128, page=128)  # the attention of the repository's benchmark
LAYERS = 36                                                   # its layer count


def _ops():
    package = os.path.join(ROOT, "hayate-exp_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from hayate_b200 import ops

    return ops


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one user, a draft of 8 nodes over a short chat: the smallest call, latency counts
        dict(name="tree_one_user", kind="tree", dtype="bf16", batch=1, ctx_lo=1000, ctx_hi=1000,
             nodes_lo=8, nodes_hi=8, mask="tree", lens=1, **HEADS),
        # the benchmark's decode batch (64 requests, 1K-8K cached) with 16 drafted nodes each
        dict(name="tree_decode_batch", kind="tree", dtype="bf16", batch=64, ctx_lo=1024, ctx_hi=8192,
             nodes_lo=16, nodes_hi=16, mask="tree", lens=2, **HEADS),
        # the long-context workload's 32K requests, ragged trees, half precision
        dict(name="tree_long_context", kind="tree", dtype="f16", batch=4, ctx_lo=32000, ctx_hi=32768,
             nodes_lo=33, nodes_hi=64, mask="tree", lens=3, **HEADS),
        # wide drafts, where the products weigh more than the bytes
        dict(name="tree_wide", kind="tree", dtype="bf16", batch=8, ctx_lo=2000, ctx_hi=4096,
             nodes_lo=256, nodes_hi=256, mask="tree", lens=4, **HEADS),
        # one request accepts 4 drafted tokens: 36 layers of a few rows, latency counts
        dict(name="rows_one_user", kind="rows", dtype="bf16", batch=1, layers=LAYERS, style="path",
             base_lo=200, base_hi=200, rows_lo=4, rows_hi=4, tree=24, lens=5, **HEADS),
        # a batch of 64 accepts paths of 6 to 12 nodes of 64-node trees
        dict(name="rows_decode_batch", kind="rows", dtype="bf16", batch=64, layers=LAYERS, style="path",
             base_lo=100, base_hi=192, rows_lo=6, rows_hi=12, tree=64, lens=6, **HEADS),
        # one page of every layer: a request writes into a page it shares
        dict(name="pages_one", kind="pages", dtype="bf16", layers=LAYERS, pool_pages=16, count=1, **HEADS),
        # 64 forks of the benchmark's batch, each with its own copy of the page being written
        dict(name="pages_fork_batch", kind="pages", dtype="bf16", layers=LAYERS, pool_pages=130, count=64, **HEADS),
        # a decode step of 64 requests in which 5 pages fill up, one layer
        dict(name="bounds_decode_step", kind="bounds", dtype="bf16", layers=1, pool_pages=700, count=5, **HEADS),
        # a 32K prefix arrives: every page of 4 layers
        dict(name="bounds_prefix", kind="bounds", dtype="bf16", layers=4, pool_pages=300, count=256, **HEADS),
        # one 32K request reads 32 of its 256 pages
        dict(name="sparse_one_user", kind="sparse", dtype="bf16", batch=1, ctx_lo=32700, ctx_hi=32700,
             num_pages=32, lens=7, **HEADS),
        # 64 requests of about 32K tokens read 16 pages each
        dict(name="sparse_long_batch", kind="sparse", dtype="bf16", batch=64, ctx_lo=24000, ctx_hi=32768,
             num_pages=16, lens=8, **HEADS),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, wide=True):
    # the benchmark's heads, or other sharing ratios and sizes that the pools can have
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([128, 128, 128, 64, 96]) if wide else 128
    return rng.choice([dict(HEADS), dict(q_heads=kv * group, kv_heads=kv, head_dim=dim, page=rng.choice([128, 256]))])


def draw(rng):
    """A case of the listed ones' ranges: batches of 1 to 64, contexts of nothing to 32K tokens."""
    while True:
        kind = rng.choice(["tree", "tree", "sparse", "sparse", "rows", "pages", "bounds"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        lens = rng.randrange(1, 1 << 30)
        if kind == "tree":
            nodes, ctx = _log_int(rng, 1, 256), _log_int(rng, 1, 32768) - 1
            case = dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 64), ctx_lo=rng.choice([ctx, ctx // 3]),
                        ctx_hi=ctx, nodes_lo=rng.choice([nodes, 1]), nodes_hi=nodes,
                        mask=rng.choice(["tree", "tree", "any"]), lens=lens, **_heads(rng))
            most = 140e9 if dtype != "f32" else 12e9
            if work(case)["flops"] > most or work(case)["bytes"] > 1.2e9 or _padded_scores(case) > 1.2e9:
                continue
        elif kind == "sparse":
            ctx = _log_int(rng, 1, 32768) - 1
            case = dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 64), ctx_lo=rng.choice([ctx, ctx // 3]),
                        ctx_hi=ctx, num_pages=_log_int(rng, 1, 64), lens=lens, **_heads(rng))
            if work(case)["bytes"] > 6.0e8 or case["batch"] * ctx > 64 * 32768 * 0.9:
                continue
        elif kind == "rows":
            style = rng.choice(["path", "path", "drop"])
            rows = _log_int(rng, 1, 32) if style == "path" else _log_int(rng, 1, 2000)
            batch = _log_int(rng, 1, 64) if style == "path" else _log_int(rng, 1, 4)
            base = _log_int(rng, 1, 1000) - 1
            case = dict(kind=kind, dtype=dtype, batch=batch, layers=_log_int(rng, 1, LAYERS), style=style,
                        base_lo=base // 2, base_hi=base, rows_lo=rng.choice([rows, 0]), rows_hi=rows,
                        tree=2 * rows + rng.randrange(0, 9), lens=lens, **_heads(rng))
            if not 1e3 < work(case)["bytes"] < 2.5e8 or _pool_bytes(case) > 2.5e9:
                continue
        else:
            layers, count = _log_int(rng, 1, LAYERS), _log_int(rng, 1, 64 if kind == "pages" else 256)
            case = dict(kind=kind, dtype=dtype, layers=layers, pool_pages=2 * count + rng.randrange(1, 20),
                        count=count, **_heads(rng))
            if work(case)["bytes"] > (2.4e9 if kind == "pages" else 2.7e8) or _pool_bytes(case) > 2.5e9:
                continue
        return case


# ------------------------------------------------------------------ what a case's lengths are
def _span(rng, lo, hi, n):
    return [rng.randint(lo, hi) for _ in range(n)]


def _lengths(case):
    """Per request: (cached tokens, drafted nodes), (chunk start, moved rows) or (context, 1)."""
    rng = random.Random(case["lens"])
    if case["kind"] == "tree":
        return (_span(rng, case["ctx_lo"], case["ctx_hi"], case["batch"]),
                _span(rng, case["nodes_lo"], case["nodes_hi"], case["batch"]))
    if case["kind"] == "rows":
        return (_span(rng, case["base_lo"], case["base_hi"], case["batch"]),
                _span(rng, case["rows_lo"], case["rows_hi"], case["batch"]))
    return _span(rng, case["ctx_lo"], case["ctx_hi"], case["batch"]), [1] * case["batch"]


def _bytes(case):
    return 4 if case["dtype"] == "f32" else 2


def _pool_bytes(case):
    if "pool_pages" in case:
        pages = case["pool_pages"]
    else:
        first, more = _lengths(case)
        reach = [a + (case["tree"] if case["kind"] == "rows" else 0) + b for a, b in zip(first, more)]
        pages = sum(-(-max(n, 1) // case["page"]) for n in reach) + 2
    return 2 * case.get("layers", 1) * case["kv_heads"] * pages * case["page"] * case["head_dim"] * _bytes(case)


def _padded_scores(case):
    first, more = _lengths(case)
    return case["batch"] * case["q_heads"] * max(more) * (max(first) + max(more))


def work(case):
    """Each input read once and each output written once; products of visible pairs."""
    eb, dim, hq, hkv = _bytes(case), case["head_dim"], case["q_heads"], case["kv_heads"]
    if case["kind"] == "tree":
        ctx, nodes = _lengths(case)
        keys, rows = sum(ctx) + sum(nodes), sum(nodes)
        words = -(-max(nodes) // 32)
        return {"bytes": 2 * keys * hkv * dim * eb + 2 * rows * hq * dim * eb + rows * words * 4,
                "flops": 4 * hq * dim * sum(c * n + n for c, n in zip(ctx, nodes))}
    if case["kind"] == "rows":
        _, rows = _lengths(case)
        return {"bytes": 2 * 2 * sum(rows) * case["layers"] * hkv * dim * eb + 4 * sum(rows), "flops": 0}
    if case["kind"] == "pages":
        return {"bytes": 2 * 2 * case["count"] * case["page"] * case["layers"] * hkv * dim * eb, "flops": 0}
    if case["kind"] == "bounds":
        rows = case["count"] * case["layers"] * hkv
        return {"bytes": rows * (case["page"] + 2) * dim * eb, "flops": 2 * rows * case["page"] * dim}
    ctx, _ = _lengths(case)
    pages = [-(-(n + 1) // case["page"]) for n in ctx]
    read = [min(n + 1, min(p, case["num_pages"]) * case["page"]) for n, p in zip(ctx, pages)]
    scored = [p if p > case["num_pages"] else 0 for p in pages]
    return {"bytes": 2 * sum(read) * hkv * dim * eb + 2 * sum(scored) * hkv * dim * eb
                     + 2 * case["batch"] * hq * dim * eb + 4 * case["batch"] * hkv * case["num_pages"],
            "flops": 4 * hq * dim * sum(read) + 2 * hq * dim * sum(scored)}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _page_table(reach, page, seed):
    """Random physical pages for requests that reach so many tokens, -1 past each one's last."""
    counts = [-(-max(n, 1) // page) for n in reach]
    ids = np.random.RandomState(seed % (1 << 31)).permutation(sum(counts) + 2)
    table = np.full((len(reach), max(counts)), -1, dtype=np.int32)
    first = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[first:first + n]
        first += n
    return table, sum(counts) + 2


def _tree_words(nodes, words, style, rs):
    """Visibility bits of one request's nodes: bit j of row i says that node i sees node j."""
    sees = np.zeros((nodes, words * 32), dtype=bool)
    if style == "any":  # an arbitrary mask, rows of nothing among them
        sees[:, :nodes] = rs.rand(nodes, nodes) < 0.4
        sees[rs.rand(nodes) < 0.1] = False
    else:               # each node follows an earlier one, or the context
        for i in range(nodes):
            parent = rs.randint(max(-1, i - 9), i) if i else -1
            if parent >= 0:
                sees[i] = sees[parent]
            sees[i, i] = True
    bits = sees.reshape(nodes, words, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)
    return bits.sum(axis=2).astype(np.uint32).view(np.int32)


def prepare(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    hkv, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    rs = np.random.RandomState((seed * 7919 + 1) % (1 << 31))
    state = dict(case)
    if case["kind"] in ("pages", "bounds"):
        capacity = case["pool_pages"] * page
        state["k_pool"] = _normal((case["layers"], 1, hkv, capacity, dim), dtype, gen)
        order = rs.permutation(case["pool_pages"])
        if case["kind"] == "pages":
            state["v_pool"] = _normal((case["layers"], 1, hkv, capacity, dim), dtype, gen)
            state["src"] = _i32(order[:case["count"]])
            state["dst"] = _i32(order[case["count"]:2 * case["count"]])
        else:
            state["k_bounds"] = torch.zeros((case["layers"], hkv, case["pool_pages"], 2, dim), dtype=dtype, device="cuda")
            state["pages"] = _i32(order[:case["count"]])
        return state
    first, more = _lengths(case)
    batch = case["batch"]
    if case["kind"] == "rows":
        tree = [max(case["tree"], 2 * n) for n in more]
        table, pages = _page_table([a + t for a, t in zip(first, tree)], page, seed)
        # the accepted rows: the root (or none), then later nodes that no accepted row lands on;
        # or the older half of a stretch dropped, the younger half moved up
        src = []
        for n, t in zip(more, tree):
            if case["style"] == "drop":
                rows = np.arange(n) + t - n
            else:
                rows = n + np.sort(rs.permutation(t - n)[:n])
                if n and rs.rand() < 0.7:
                    rows[0] = 0
            src.append(rows)
        shape = (case["layers"], 1, hkv, pages * page, dim)
        state["k_pool"], state["v_pool"] = _normal(shape, dtype, gen), _normal(shape, dtype, gen)
        state["page_table"], state["base"] = torch.from_numpy(table).cuda(), _i32(first)
        state["src"] = _i32(np.concatenate(src).astype(np.int32) if sum(more) else [])
        state["src_start"] = _i32(np.concatenate([[0], np.cumsum(more)]))
        state["entry_request"] = torch.repeat_interleave(torch.arange(batch), torch.tensor(more)).cuda()
        return state
    table, pages = _page_table([a + b for a, b in zip(first, more)], page, seed)
    shape = (1, 1, hkv, pages * page, dim)
    state["page_table"], state["cache_lens"] = torch.from_numpy(table).cuda(), _i32(first)
    state["k_pool"], state["v_pool"] = _normal(shape, dtype, gen), _normal(shape, dtype, gen)
    if case["kind"] == "tree":
        words = -(-max(more) // 32)
        state["tree_mask"] = torch.from_numpy(np.concatenate(
            [_tree_words(n, words, case["mask"], rs) for n in more])).cuda()
        start = np.concatenate([[0], np.cumsum(more)])[:-1]
        state["q_start"], state["q_len"] = _i32(start), _i32(more)
        state["token_request"] = torch.repeat_interleave(torch.arange(batch), torch.tensor(more)).cuda()
        state["max_nodes"], state["max_kv"] = max(more), max(a + b for a, b in zip(first, more))
        # the layout an attention layer hands over: [1, N, H, D] memory viewed as [1, H, N, D]
        state["q"] = _normal((1, sum(more), case["q_heads"], dim), dtype, gen).transpose(1, 2)
        return state
    # pages differ in what they are about: keys of a page share a direction, as text does
    topic = torch.randn((1, 1, hkv, pages, 1, dim), generator=gen, device="cuda") * 0.7
    state["k_pool"].view(1, 1, hkv, pages, page, dim).add_(topic.to(dtype))
    keys = state["k_pool"].view(1, hkv, pages, page, dim)
    state["k_bounds"] = torch.stack([keys.amin(dim=3), keys.amax(dim=3)], dim=3).contiguous()
    state["q"] = _normal((batch, 1, case["q_heads"], dim), dtype, gen).transpose(1, 2)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return {"tree": _tree, "rows": _rows, "pages": _pages, "bounds": _bounds, "sparse": _sparse}[state["kind"]](state)


def _softmax_product(scores, visible, values):
    """softmax over the visible keys (a row that sees none gives zeros), times the values."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(dim=-1, keepdim=True)
    return torch.matmul(weights, values) / torch.where(total == 0, 1.0, total)


def _tree(s):
    if own:
        return _ops().tree_attention(s["q"], s["k_pool"], s["v_pool"], 0, s["page_table"], s["cache_lens"],
                                     s["q_start"], s["q_len"], s["tree_mask"], s["page"], s["max_nodes"])
    hkv, dim, page, nodes, kv = s["kv_heads"], s["head_dim"], s["page"], s["max_nodes"], s["max_kv"]
    group, batch = s["q_heads"] // hkv, s["batch"]
    lens, start, count = s["cache_lens"].long(), s["q_start"].long(), s["q_len"].long()
    t = torch.arange(nodes, device=lens.device)
    rows = torch.minimum(start[:, None] + t, start[:, None] + count[:, None] - 1)             # [B, T]
    q = s["q"][0].float().view(hkv, group, -1, dim)[:, :, rows]                               # [Hkv, G, B, T, D]
    q = q.permute(2, 0, 1, 3, 4).reshape(batch, hkv, group * nodes, dim)
    key = torch.arange(kv, device=lens.device)
    end = lens + count
    pos = torch.minimum(key[None], end[:, None] - 1)                                          # [B, K]
    slot = s["page_table"].long().gather(1, pos // page) * page + pos % page
    k = s["k_pool"][0, 0][:, slot].float().transpose(0, 1)                                    # [B, Hkv, K, D]
    v = s["v_pool"][0, 0][:, slot].float().transpose(0, 1)
    words = s["tree_mask"][rows]                                                              # [B, T, W]
    bits = ((words[..., None] >> torch.arange(32, device=lens.device)) & 1).flatten(2).bool()
    node = key[None] - lens[:, None]                                                          # [B, K]
    seen = bits.gather(2, node.clamp(0, nodes - 1)[:, None].expand(-1, nodes, -1))
    visible = (node < 0)[:, None] | (seen & (key[None] < end[:, None])[:, None])              # [B, T, K]
    visible = visible[:, None, None].expand(-1, hkv, group, -1, -1).reshape(batch, hkv, group * nodes, kv)
    out = _softmax_product(torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dim), visible, v)
    out = out.view(batch, hkv * group, nodes, dim)
    request = s["token_request"]
    own_row = torch.arange(request.numel(), device=lens.device) - start[request]
    return out[request, :, own_row].transpose(0, 1)[None].to(s["q"].dtype)


def _rows(s):
    if own:
        _ops().compact_rows(s["k_pool"], s["v_pool"], s["page_table"], s["base"], s["src"], s["src_start"], s["page"])
        return [s["k_pool"], s["v_pool"]]
    request, page, table = s["entry_request"], s["page"], s["page_table"].long()
    index = torch.arange(request.numel(), device=request.device) - s["src_start"].long()[request]
    old = s["base"].long()[request] + s["src"].long()
    new = s["base"].long()[request] + index
    old_slot = table[request, old // page] * page + old % page
    new_slot = table[request, new // page] * page + new % page
    s["k_pool"][:, :, :, new_slot] = s["k_pool"][:, :, :, old_slot]
    s["v_pool"][:, :, :, new_slot] = s["v_pool"][:, :, :, old_slot]
    return [s["k_pool"], s["v_pool"]]


def _pages(s):
    if own:
        _ops().copy_pages(s["k_pool"], s["v_pool"], s["src"], s["dst"], s["page"])
        return [s["k_pool"], s["v_pool"]]
    shape = (s["layers"], s["kv_heads"], s["pool_pages"], s["page"], s["head_dim"])
    k, v = s["k_pool"].view(shape), s["v_pool"].view(shape)
    src, dst = s["src"].long(), s["dst"].long()
    k[:, :, dst] = k[:, :, src]
    v[:, :, dst] = v[:, :, src]
    return [s["k_pool"], s["v_pool"]]


def _bounds(s):
    if own:
        _ops().page_bounds(s["k_pool"], s["k_bounds"], s["pages"], s["page"])
        return s["k_bounds"]
    pages = s["pages"].long()
    keys = s["k_pool"].view(s["layers"], s["kv_heads"], s["pool_pages"], s["page"], s["head_dim"])[:, :, pages]
    s["k_bounds"][:, :, pages] = torch.stack([keys.amin(dim=3), keys.amax(dim=3)], dim=3)
    return s["k_bounds"]


def _sparse(s):
    if own:
        return list(_ops().sparse_attention(s["q"], s["k_pool"], s["v_pool"], s["k_bounds"], 0, s["page_table"],
                                            s["cache_lens"], s["page"], s["num_pages"]))
    hkv, dim, page, take = s["kv_heads"], s["head_dim"], s["page"], s["num_pages"]
    group, batch = s["q_heads"] // hkv, s["batch"]
    q, table = s["q"][:, :, 0].view(batch, hkv, group, dim), s["page_table"].long()
    width = table.shape[1]
    last = s["cache_lens"].long() // page                                                     # [B]
    index = torch.arange(width, device=table.device)
    bounds = s["k_bounds"][0][:, table.clamp(min=0)].double()                                 # [Hkv, B, W, 2, D]
    low, high = bounds[..., 0, :].permute(1, 0, 3, 2), bounds[..., 1, :].permute(1, 0, 3, 2)  # [B, Hkv, D, W]
    # the most that a key of the page can score: the bound on the side of each q's sign. In
    # 64 bits, since scores next to each other decide which page is read; rounded once
    score = torch.matmul(q.double().clamp(min=0), high) + torch.matmul(q.double().clamp(max=0), low)
    score = score.amax(dim=2).float()                                                         # [B, Hkv, W]
    score = torch.where(index > last[:, None, None], -math.inf, score)
    score = torch.where(index == last[:, None, None], math.inf, score)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :take]       # ties: lowest first
    order = torch.where(order > last[:, None, None], width, order).sort(dim=-1).values
    chosen = torch.full((batch, hkv, take), -1, dtype=torch.int32, device=table.device)
    chosen[..., :order.shape[-1]] = torch.where(order == width, -1, order).int()
    pos = (order[..., None] * page + torch.arange(page, device=table.device)).flatten(2)      # [B, Hkv, take * page]
    visible = pos <= s["cache_lens"].long()[:, None, None]
    pos = torch.where(visible, pos, 0)
    slot = table[:, None].expand(-1, hkv, -1).gather(2, pos // page) * page + pos % page
    head = torch.arange(hkv, device=table.device)[None, :, None]
    k, v = s["k_pool"][0, 0][head, slot].float(), s["v_pool"][0, 0][head, slot].float()
    out = _softmax_product(torch.matmul(q.float(), k.transpose(2, 3)) / math.sqrt(dim), visible[:, :, None], v)
    return [out.reshape(batch, hkv * group, 1, dim).to(s["q"].dtype), chosen]


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    hkv, dim, page = case["kv_heads"], case["head_dim"], case["page"]
    if case["kind"] == "bounds":
        bounds = s["k_bounds"].double()
        for p in s["pages"].tolist():
            keys = s["k_pool"][:, 0, :, p * page:(p + 1) * page].double().sort(dim=2).values
            bounds[:, :, p, 0], bounds[:, :, p, 1] = keys[:, :, 0], keys[:, :, -1]
        return bounds
    if case["kind"] in ("rows", "pages"):
        moves = []  # (to, from, tokens)
        if case["kind"] == "pages":
            moves = [(d * page, f * page, page) for f, d in zip(s["src"].tolist(), s["dst"].tolist())]
        else:
            table, src = s["page_table"].tolist(), s["src"].tolist()
            for b, (base, n) in enumerate(zip(*_lengths(case))):
                at = len(moves)
                for i in range(n):
                    new, old = base + i, base + src[at + i]
                    moves.append((table[b][new // page] * page + new % page, table[b][old // page] * page + old % page, 1))
        pools = []
        for pool in (s.pop("k_pool"), s.pop("v_pool")):
            pools.append(pool.double())
            for to, old, n in moves:
                pools[-1][:, :, :, to:to + n] = pool[:, :, :, old:old + n]
        return pools
    group = case["q_heads"] // hkv
    first, more = _lengths(case)
    q = s["q"].double()
    result = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    chosen = np.full((case["batch"], hkv, case.get("num_pages", 1)), -1, dtype=np.int32)

    def attend(rows, keys, values, sees):  # [G, T, D], [K, D], [K, D], [T, K]
        logit = torch.einsum("gtd,kd->gtk", rows, keys) * dim ** -0.5
        logit = logit.masked_fill(~sees, -math.inf)
        weight = torch.softmax(logit, dim=-1).nan_to_num(0.0)
        return torch.einsum("gtk,kd->gtd", weight, values)

    at = 0
    for b, (cached, new) in enumerate(zip(first, more)):
        ids = s["page_table"][b].tolist()
        length = cached + new

        def rows_of(pool, g, wanted):
            return torch.cat([pool[0, 0, g, ids[i] * page:(ids[i] + 1) * page] for i in wanted]).double()

        if case["kind"] == "tree":
            sees = torch.ones((new, length), dtype=torch.bool)
            bits = np.unpackbits(s["tree_mask"][at:at + new].cpu().numpy().view(np.uint8), axis=1, bitorder="little")
            sees[:, cached:] = torch.from_numpy(bits[:, :new].astype(bool))
            sees = sees.cuda()
            wanted = range(-(-length // page))
            for g in range(hkv):
                heads = slice(g * group, (g + 1) * group)
                result[0, heads, at:at + new] = attend(q[0, heads, at:at + new], rows_of(s["k_pool"], g, wanted)[:length],
                                                       rows_of(s["v_pool"], g, wanted)[:length], sees)
            at += new
            continue
        last, take = cached // page, case["num_pages"]
        side = s["k_bounds"][0][:, torch.tensor(ids[:last + 1], device="cuda")].double()      # [Hkv, n, 2, D]
        for g in range(hkv):
            heads = slice(g * group, (g + 1) * group)
            ask = q[b, heads, 0]
            best = torch.where(ask[:, None] >= 0, side[g, None, :, 1], side[g, None, :, 0]).mul_(ask[:, None])
            best = best.sum(-1).amax(0).float().cpu().numpy()
            order = np.lexsort((np.arange(last), -best[:last]))[:take - 1]
            picked = sorted(order.tolist()) + [last]
            chosen[b, g, :len(picked)] = picked
            keys = rows_of(s["k_pool"], g, picked)
            there = keys.shape[0] - page + cached % page + 1
            sees = torch.ones((1, there), dtype=torch.bool, device="cuda")
            result[b, heads] = attend(q[b, heads], keys[:there], rows_of(s["v_pool"], g, picked)[:there], sees)
    return result if case["kind"] == "tree" else [result, None]
