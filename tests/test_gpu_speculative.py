"""Drafted trees, forks and page-sparse decode as an engine uses them: through the page manager
and its batches, layer after layer, and through ``packed_forward``."""

from __future__ import annotations

import math
import types

import numpy as np
import pytest
import torch

from hayate_b200 import PagedKVCacheManager, ops
from hayate_b200 import workloads as W
from hayate_b200.mixed_step import packed_forward

import operators_util as U

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LAYERS = 2


def manager_with(lengths, dtype, seed, extra=4, layers=LAYERS, track=False):
    pages = sum(-(-(n + 300) // 128) for n in lengths) + extra
    m = PagedKVCacheManager(layers, 8, 128, pages * 128, 128, 2 * len(lengths) + 2, dtype, "cuda")
    W.shuffle_free_pages(m, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hs = [m.allocate() for _ in lengths]
    for h, n in zip(hs, lengths):
        W.fill_history(m, h, n, gen)
    if track:
        m.track_page_bounds()
    return m, hs


def rope_tables():
    cos, sin = W.rope_angles(torch.arange(8192, device="cuda"), 128)
    return cos.contiguous(), sin.contiguous()


def projections(total, dtype, seed, layers=LAYERS):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def make(heads):
        return [torch.randn(1, total, heads, 128, generator=gen, device="cuda").to(dtype) for _ in range(layers)]

    ones = torch.ones(128, device="cuda", dtype=dtype)
    return make(32), make(8), make(8), ones


def bounds_are_right(m, handles):
    expect = U.bounds_reference(m.k_cache, m.page_size)
    for h in handles:
        for page in h.pages[: h.length // m.page_size]:
            if not torch.equal(m.k_bounds[:, :, page], expect[:, :, page]):
                return False
    return True


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("track", [False, True], ids=["plain", "bounds"])
def test_tree_step_equals_the_accepted_tokens_one_by_one(dtype, track):
    """Draft, attend, accept: the accepted nodes' rows and the pools are those of decoding the
    accepted tokens one after the other (the same K/V bytes; attention within its bound)."""
    lengths = [1000, 0, 250, 127]
    rng = np.random.RandomState(3)
    trees = [U.random_parents(n, rng, reach=4) for n in (24, 7, 40, 1)]
    paths = []
    for tree in trees:  # the path to the deepest of a few random nodes
        best = []
        for node in rng.randint(0, len(tree), 6):
            path = [int(node)]
            while tree[path[0]] >= 0:
                path.insert(0, tree[path[0]])
            best = max(best, path, key=len)
        paths.append(best)
    paths[3] = []
    m, hs = manager_with(lengths, dtype, 5, track=track)
    ref, rs = manager_with(lengths, dtype, 5)
    cos, sin = rope_tables()
    total = sum(map(len, trees))
    q, k, v, ones = projections(total, dtype, 9)
    batch = m.begin_tree_batch(hs, trees)
    rows = []
    for layer in range(LAYERS):
        rotated = batch.prepare_layer(layer, q[layer], k[layer], v[layer], ones, ones, cos, sin)
        rows.append((rotated, batch.attend_layer(rotated, layer)))
    m.commit_tree(batch, hs, paths)
    m.check_device_errors()
    starts = np.concatenate([[0], np.cumsum([len(t) for t in trees])])
    for step in range(max(map(len, paths))):
        live = [b for b, p in enumerate(paths) if len(p) > step]
        picked = torch.tensor([starts[b] + paths[b][step] for b in live], device="cuda")
        one = ref.begin_batch([rs[b] for b in live], [1] * len(live))
        for layer in range(LAYERS):
            rotated = one.prepare_layer(layer, q[layer][:, picked], k[layer][:, picked], v[layer][:, picked],
                                        ones, ones, cos, sin)
            assert torch.equal(rotated, rows[layer][0][:, :, picked])
            out = one.attend_layer(rotated, layer)
            for at, b in enumerate(live):
                n = lengths[b] + step + 1
                for g in range(8):
                    kk = U.rows_of(ref.k_cache, layer, g, np.asarray(rs[b].pages), n, 128)
                    vv = U.rows_of(ref.v_cache, layer, g, np.asarray(rs[b].pages), n, 128)
                    heads = slice(4 * g, 4 * g + 4)
                    sees = torch.ones((4, n), dtype=torch.bool, device="cuda")
                    exact, bound = U.attention_rows(rotated[0, heads, at].double(), kk, vv, sees, 128 ** -0.5, dtype)
                    for got in (out[0, heads, at], rows[layer][1][0, heads, picked[at]]):
                        assert bool(((got.double() - exact).abs() <= bound).all())
        ref.commit_batch([rs[b] for b in live], [1] * len(live))
    for h, r, path, n in zip(hs, rs, paths, lengths):
        assert h.length == r.length == n + len(path)
        a, b = m.snapshot(h), ref.snapshot(r)
        if h.length:
            assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    if track:
        assert bounds_are_right(m, hs)


def test_tree_step_after_tree_step_and_plain_steps():
    m, hs = manager_with([120, 5], BF16, 1, extra=8, track=True)
    gen = torch.Generator(device="cuda").manual_seed(0)
    rng = np.random.RandomState(1)
    for turn in range(6):
        trees = [U.random_parents(int(n), rng, reach=3) for n in rng.randint(1, 60, 2)]
        batch = m.begin_tree_batch(hs, trees)
        total = sum(map(len, trees))
        q = torch.randn(1, total, 32, 128, generator=gen, device="cuda").to(BF16).transpose(1, 2)
        kv = torch.randn(1, total, 8, 128, generator=gen, device="cuda").to(BF16).transpose(1, 2)
        for layer in range(LAYERS):
            batch.write_layer(layer, kv, kv)
            out = batch.attend_layer(q, layer)
            table = batch.page_table.cpu().numpy()
            ref, bound = U.tree_reference(q, m.k_cache, m.v_cache, layer, table, [h.length for h in hs],
                                          batch.layout.q_start.tolist(), batch.layout.q_len.tolist(),
                                          [U.sees_of_parents(t) for t in trees], 128, 128 ** -0.5)
            assert bool(((out.double() - ref).abs() <= bound).all())
        paths = []
        for tree in trees:
            path = [len(tree) - 1]
            while tree[path[0]] >= 0:
                path.insert(0, tree[path[0]])
            paths.append(path)
        m.commit_tree(batch, hs, paths)
        step = m.begin_batch(hs, 1)
        q1, k1, v1 = W.step_inputs(m, hs, 1, 32, gen)
        for layer in range(LAYERS):
            step.write_attend_layer(layer, k1, v1, q1)
        m.commit_batch(hs, 1)
        assert bounds_are_right(m, hs)
    m.check_device_errors()


def test_forks_decode_apart_from_each_other():
    m, (h,) = manager_with([300], BF16, 2, extra=16, track=True)
    forks = m.fork(h, 3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    everyone = [h] + forks
    snaps = [m.snapshot(x) for x in everyone]
    assert all(torch.equal(s.k, snaps[0].k) and torch.equal(s.v, snaps[0].v) for s in snaps)
    for _ in range(90):  # past the end of the shared page
        batch = m.begin_batch(everyone, 1)
        q, k, v = W.step_inputs(m, everyone, 1, 32, gen)
        for layer in range(LAYERS):
            batch.write_layer(layer, k, v)
        m.commit_batch(everyone, 1)
    after = [m.snapshot(x) for x in everyone]
    for s, old in zip(after, snaps):
        assert torch.equal(s.k[:, :, :300], old.k) and not torch.equal(s.k[:, :, 300:], after[0].k[:, :, 300:]) or s is after[0]
    assert bounds_are_right(m, everyone)
    m.check_device_errors()


@pytest.mark.parametrize("how", ["older batch", "tree as a chain", "older graph batch", "shared"])
def test_bounds_missed_by_a_step_are_made_up_for(how):
    """Pages filled by steps that keep no bounds have them once the next step begins."""
    m, hs = manager_with([250, 120], BF16, 11, extra=8)
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(1, 8, 40, 128, generator=gen, device="cuda").to(BF16)
    if how == "older graph batch":
        static = m.static_decode_batch(2, 2048, 32)
        m.track_page_bounds()
        for at in range(20):
            static.update(hs)
            for layer in range(LAYERS):
                static.batch.write_layer(layer, k[:, :, at:at + 2], k[:, :, at:at + 2])
            m.commit_batch(hs, 1)
    else:
        if how == "tree as a chain":
            m.track_page_bounds()
            batch = m.begin_tree_batch(hs, [[i - 1 for i in range(20)]] * 2)
        else:
            batch = m.begin_batch(hs, [20, 20])
            m.track_page_bounds()
        for layer in range(LAYERS):
            batch.write_layer(layer, k, k)
        m.commit_batch(hs, [20, 20])
        if how == "shared":
            hs = [m.share(h, h.length) for h in hs]
    batch = m.begin_batch(hs, 1)
    assert bounds_are_right(m, hs)
    q, k1, v1 = W.step_inputs(m, hs, 1, 32, gen)
    for layer in range(LAYERS):
        batch.write_layer(layer, k1, v1)
        _, chosen = batch.attend_pages(q, layer, 2)
        expect = U.selection_reference(q, m.k_bounds, layer, batch.page_table.cpu().numpy(), [h.length for h in hs], 128, 2)
        assert np.array_equal(chosen.cpu().numpy(), expect)
    m.check_device_errors()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_page_sparse_decode_through_the_manager(dtype):
    """Bounds kept through prefill, packed, decode, import and shared pages; every step's rows
    are those of the chosen pages, chosen by the definition."""
    m, hs = manager_with([2000, 300, 700], dtype, 6, extra=24, track=True)
    gen = torch.Generator(device="cuda").manual_seed(8)
    shared = m.share(hs[0], 1990)          # ends inside a page that hs[0] still writes
    snap = m.snapshot(hs[1])
    imported = m.allocate_for_request(snap)
    everyone = hs + [shared, imported]
    chunk = [130, 1, 257, 3, 129]          # a packed step that fills pages of several requests
    batch = m.begin_batch(everyone, chunk)
    total = sum(chunk)
    k = torch.randn(1, 8, total, 128, generator=gen, device="cuda").to(dtype)
    v = torch.randn(1, 8, total, 128, generator=gen, device="cuda").to(dtype)
    for layer in range(LAYERS):
        batch.write_layer(layer, k, v)
    m.commit_batch(everyone, chunk)
    assert bounds_are_right(m, everyone)
    for turn in range(140):
        packed = turn % 2 == 1
        batch = m.begin_batch(everyone, [1] * len(everyone) if packed else 1)
        q, k, v = W.step_inputs(m, everyone, 1, 32, gen)
        lens = [h.length for h in everyone]
        for layer in range(LAYERS):
            if packed:
                def flat(x):
                    return x.permute(2, 1, 0, 3)
                batch.write_layer(layer, flat(k), flat(v))
                out, chosen = batch.attend_pages(flat(q), layer, 4)
                assert out.shape == flat(q).shape
                out = out.permute(2, 1, 0, 3)
            else:
                batch.write_layer(layer, k, v)
                out, chosen = batch.attend_pages(q, layer, 4)
            if turn % 23 == 0 or packed and turn % 35 == 0:
                table = batch.page_table.cpu().numpy()
                expect = U.selection_reference(q, m.k_bounds, layer, table, lens, 128, 4)
                assert np.array_equal(chosen.cpu().numpy(), expect)
                ref, bound = U.sparse_reference(q, m.k_cache, m.v_cache, layer, table, lens, expect, 128, 128 ** -0.5)
                assert bool(((out.double() - ref).abs() <= bound).all())
        m.commit_batch(everyone, 1)
    assert bounds_are_right(m, everyone)
    m.check_device_errors()


def test_attend_pages_with_room_for_all_is_plain_attention():
    m, hs = manager_with([600, 90], BF16, 7, track=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    batch = m.begin_batch(hs, 1)
    q, k, v = W.step_inputs(m, hs, 1, 32, gen)
    batch.write_layer(0, k, v)
    out, chosen = batch.attend_pages(q, 0, 8)
    assert chosen[0, 0].tolist() == [0, 1, 2, 3, 4, -1, -1, -1] and chosen[1, 0].tolist() == [0] + [-1] * 7
    plain = batch.attend_layer(q, 0)
    assert (out.float() - plain.float()).abs().max().item() <= 2 ** -7  # two roundings of values below 1
    for bad in (q.expand(2, 32, 2, 128),):
        with pytest.raises(ValueError, match="one token"):
            batch.attend_pages(bad, 0, 4)
    wide = m.begin_batch(hs, 2)
    with pytest.raises(ValueError, match="one token"):
        wide.attend_pages(q, 0, 4)
    tree = m.begin_tree_batch(hs, [[-1], [-1]])
    with pytest.raises(ValueError, match="one token"):
        tree.attend_pages(q.permute(2, 1, 0, 3), 0, 4)


class TinyBlock(torch.nn.Module):
    def __init__(self, hidden):
        super().__init__()
        attn = torch.nn.Module()
        attn.num_heads, attn.num_kv_groups, attn.head_dim = 32, 8, 128
        attn.q_proj = torch.nn.Linear(hidden, 32 * 128, bias=False)
        attn.k_proj = torch.nn.Linear(hidden, 8 * 128, bias=False)
        attn.v_proj = torch.nn.Linear(hidden, 8 * 128, bias=False)
        attn.o_proj = torch.nn.Linear(32 * 128, hidden, bias=False)
        attn.q_norm, attn.k_norm = torch.nn.RMSNorm(128, eps=1e-6), torch.nn.RMSNorm(128, eps=1e-6)
        self.self_attn = attn
        self.input_layernorm, self.post_attention_layernorm = torch.nn.RMSNorm(hidden), torch.nn.RMSNorm(hidden)
        self.mlp = torch.nn.Linear(hidden, hidden, bias=False)


def tiny_model(hidden=256, vocab=500):
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = torch.nn.Module()
        model.embed_tokens = torch.nn.Embedding(vocab, hidden)
        model.layers = torch.nn.ModuleList([TinyBlock(hidden) for _ in range(LAYERS)])
        model.norm, model.out_head = torch.nn.RMSNorm(hidden), torch.nn.Linear(hidden, vocab, bias=False)
    model.to(BF16)
    model.cos, model.sin = rope_tables()
    return model


def test_packed_forward_on_a_tree_scores_like_its_paths():
    """Speculative decoding through ``packed_forward``: a node's scores are those of the forward
    pass over the tokens on its path."""
    model = tiny_model()
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompt = [torch.randint(0, 500, (n,), generator=gen, device="cuda") for n in (200, 31)]
    trees = [[-1, 0, 0, 1, 2, 2], [-1, 0, -1]]
    drafted = torch.randint(0, 500, (9,), generator=gen, device="cuda")
    with torch.inference_mode():
        m = PagedKVCacheManager(LAYERS, 8, 128, 32 * 128, 128, 8, BF16, "cuda")
        hs = [m.allocate() for _ in prompt]
        lens = [len(p) for p in prompt]
        ends = torch.tensor(lens, device="cuda").cumsum(0) - 1
        packed_forward(model, torch.cat(prompt), m.begin_batch(hs, lens), ends)
        m.commit_batch(hs, lens)
        batch = m.begin_tree_batch(hs, trees)
        scores = packed_forward(model, drafted, batch, torch.arange(9, device="cuda")).float()
        at = 0
        for b, tree in enumerate(trees):
            for node in range(len(tree)):
                path = [node]
                while tree[path[0]] >= 0:
                    path.insert(0, tree[path[0]])
                alone = PagedKVCacheManager(LAYERS, 8, 128, 8 * 128, 128, 2, BF16, "cuda")
                h = alone.allocate()
                tokens = torch.cat([prompt[b], drafted[[at + i for i in path]]])
                step = alone.begin_batch([h], [len(tokens)])
                expect = packed_forward(model, tokens, step, torch.tensor([len(tokens) - 1], device="cuda")).float()
                scale = expect.abs().max().item()
                assert (scores[at + node] - expect[0]).abs().max().item() <= 0.05 * scale
            at += len(tree)
        m.commit_tree(batch, hs, [[0, 2, 5], [2]])
        m.check_device_errors()


def test_decode_step_over_chosen_pages_in_a_graph():
    """A static batch with page bounds, captured and replayed while requests cross page ends."""
    model = tiny_model()
    gen = torch.Generator(device="cuda").manual_seed(1)
    lens = [500, 900, 125]
    with torch.inference_mode():
        mgrs = []
        for _ in range(2):
            m = PagedKVCacheManager(LAYERS, 8, 128, 32 * 128, 128, 8, BF16, "cuda")
            m.track_page_bounds()
            hs = [m.allocate() for _ in lens]
            prompt = torch.randint(0, 500, (sum(lens),), generator=gen.manual_seed(1), device="cuda")
            packed_forward(model, prompt, m.begin_batch(hs, lens), torch.tensor([0], device="cuda"))
            m.commit_batch(hs, lens)
            mgrs.append((m, hs))
        (m, hs), (e, es) = mgrs
        static = m.static_decode_batch(4, 2048, 32)
        tokens, rows = torch.zeros(4, dtype=torch.long, device="cuda"), torch.arange(4, device="cuda")
        static.update([])
        packed_forward(model, tokens, static.batch, rows, 3)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scores = packed_forward(model, tokens, static.batch, rows, 3)
        for turn in range(30):
            new = torch.randint(0, 500, (3,), generator=gen, device="cuda")
            static.update(hs)
            tokens[:3] = new
            graph.replay()
            m.commit_batch(hs, 1)
            eager = packed_forward(model, new, e.begin_batch(es, [1] * 3), rows[:3], 3)
            e.commit_batch(es, 1)
            assert torch.equal(scores[:3], eager), turn
        assert bounds_are_right(m, hs) and bounds_are_right(e, es)
        m.check_device_errors()
        e.check_device_errors()
