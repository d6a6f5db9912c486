"""Tree attention, row compaction, page copies, page bounds and page-sparse decode on the
GPU, each against its 64-bit definition (``operators_util``), with the error bounds derived
there; plus the places where such kernels go wrong: empty rows, values that are not finite
in masked places, ragged and empty requests, other strides, streams, captured graphs."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from hayate_b200 import ops

import operators_util as U

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def i32(values):
    return torch.tensor(np.asarray(values, dtype=np.int32), device="cuda")


def error_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


class Tree:
    """A packed tree step over shuffled pages of one or more layers."""

    def __init__(self, lens, counts, dtype, seed=0, hq=32, hkv=8, dim=128, page=128, layers=1, layer=0,
                 sees=None, gap=0):
        rng = np.random.RandomState(seed)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.counts, self.page, self.layer = list(lens), list(counts), page, layer
        self.table, pages = U.page_table([a + b for a, b in zip(lens, counts)], page, seed)
        shape = (layers, 1, hkv, pages * page, dim)
        self.k = torch.randn(shape, generator=gen, device="cuda").to(dtype)
        self.v = torch.randn(shape, generator=gen, device="cuda").to(dtype)
        self.starts = list(np.concatenate([[0], np.cumsum([c + gap for c in counts])])[:-1])
        total = sum(counts) + gap * len(counts)
        self.q = torch.randn((1, max(total, 1), hq, dim), generator=gen, device="cuda").to(dtype).transpose(1, 2)
        self.sees = sees or [U.sees_of_parents(U.random_parents(c, rng)) for c in counts]
        self.words = max(1, -(-max(counts) // 32))
        mask = np.zeros((self.q.shape[2], self.words), dtype=np.int32)
        for s, c, m in zip(self.starts, counts, self.sees):
            if c:
                mask[s:s + c] = U.pack_bits(m, self.words)
        self.mask = torch.from_numpy(mask).cuda()
        self.scale = 1.0 / math.sqrt(dim)

    def args(self):
        return (self.q, self.k, self.v, self.layer, i32(self.table), i32(self.lens), i32(self.starts),
                i32(self.counts), self.mask, self.page, max(max(self.counts), 1))

    def run(self, **kw):
        word = error_word()
        out = ops.tree_attention(*self.args(), error_word=word, **kw)
        torch.cuda.synchronize()
        assert ops.read_device_errors(word) == []
        return out

    def reference(self):
        return U.tree_reference(self.q, self.k, self.v, self.layer, self.table, self.lens, self.starts,
                                self.counts, self.sees, self.page, self.scale)

    def check(self, out=None):
        out = self.run() if out is None else out
        ref, bound = self.reference()
        for s, c in zip(self.starts, self.counts):
            err = (out[0, :, s:s + c].double() - ref[0, :, s:s + c]).abs()
            assert bool((err <= bound[0, :, s:s + c]).all()), (s, c, float((err / bound[0, :, s:s + c]).max()))


TREES = [
    dict(lens=[1], counts=[1]),
    dict(lens=[0], counts=[1]),
    dict(lens=[0, 0], counts=[5, 33]),
    dict(lens=[1000], counts=[8]),
    dict(lens=[127, 128, 129, 255], counts=[1, 2, 31, 32]),
    dict(lens=[300, 0, 2000, 5], counts=[16, 0, 7, 64]),
    dict(lens=[4000, 17], counts=[100, 3]),
    dict(lens=[513], counts=[256]),
    dict(lens=[90, 3000], counts=[257, 40]),
    dict(lens=[700, 64], counts=[13, 21], hq=8, hkv=8),
    dict(lens=[700, 64], counts=[13, 45], hq=6, hkv=2),
    dict(lens=[700, 64], counts=[13, 21], hq=5, hkv=1, page=256),
    dict(lens=[700, 130], counts=[13, 70], hq=8, hkv=2, dim=64),
    dict(lens=[700, 130], counts=[13, 21], hq=8, hkv=2, dim=96, page=256),
    dict(lens=[200, 70], counts=[9, 40], hq=4, hkv=1, dim=256, page=64),
    dict(lens=[200, 70], counts=[9, 4], hq=4, hkv=2, dim=8),
    dict(lens=[200, 70], counts=[9, 4], hq=4, hkv=2, dim=136),
    dict(lens=[9000], counts=[4], layers=3, layer=2),
    dict(lens=[250] * 40, counts=[3] * 40, hq=4, hkv=1),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:60])
def test_tree_attention(case, dtype):
    Tree(dtype=dtype, seed=len(str(case)), **case).check()


SMALL_TREES = [
    dict(lens=[200, 0, 63], counts=[2, 1, 2], hq=4, hkv=2, dim=8, page=64),
    dict(lens=[200, 0, 130], counts=[2, 1, 2], hq=4, hkv=2, dim=136),
    dict(lens=[200, 0, 63], counts=[2, 0, 2], hq=4, hkv=2, dim=256, page=64),
    dict(lens=[2000, 64, 1], counts=[3, 4, 1], hq=4, hkv=2, dim=40),
    dict(lens=[2000, 64, 1], counts=[8, 4, 1], hq=3, hkv=3, dim=200),
    dict(lens=[2000, 64, 1], counts=[4, 3, 1], hq=8, hkv=2, dim=256),
    dict(lens=[2000, 64, 1], counts=[16, 3, 9], hq=1, hkv=1, dim=192),
    dict(lens=[500], counts=[1], hq=128, hkv=1, dim=128),
    dict(lens=[500, 30], counts=[1, 2], hq=600, hkv=1, dim=64),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", SMALL_TREES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:60])
def test_tree_attention_few_rows_and_other_sharing(case, dtype):
    Tree(dtype=dtype, seed=len(str(case)) + 1, **case).check()


@pytest.mark.parametrize("dtype, dim, hq", [(F32, 128, 2), (F32, 256, 2), (BF16, 256, 4), (F16, 40, 2), (F32, 128, 4)], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
def test_few_rows_masked_values_that_are_not_finite(dtype, dim, hq, bad):
    sees = [np.array([[1, 0], [0, 1]], dtype=bool), np.array([[1, 0], [1, 1]], dtype=bool)]
    clean = Tree([100, 127], [2, 2], dtype, seed=2, hq=hq, hkv=2, dim=dim, sees=sees)
    expect = clean.run()
    dirty = Tree([100, 127], [2, 2], dtype, seed=2, hq=hq, hkv=2, dim=dim, sees=sees)
    for b, n in enumerate(dirty.lens):
        for pool in (dirty.k, dirty.v):
            slot = int(dirty.table[b][(n + 1) // 128]) * 128 + (n + 1) % 128
            pool[:, :, :, slot:(slot // 128 + 1) * 128] = bad   # node 1 and all behind it
    out = dirty.run()
    for b in range(2):  # node 0 of both sees no bad value, node 1 sees itself
        assert torch.equal(out[0, :, 2 * b], expect[0, :, 2 * b])
        assert not torch.isfinite(out[0, :, 2 * b + 1].float()).any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_tree_attention_arbitrary_masks_and_empty_rows(dtype):
    rng = np.random.RandomState(5)
    counts = [40, 130, 1, 3]
    sees = [rng.rand(c, c) < 0.3 for c in counts]
    for m in sees:
        m[::3] = False
    t = Tree([0, 0, 0, 50], counts, dtype, seed=3, sees=sees)
    out = t.run()
    t.check(out)
    empty = torch.from_numpy(np.concatenate([~m.any(1) for m in sees[:3]])).cuda()
    assert bool((out[0][:, :empty.numel()][:, empty] == 0).all())


def test_tree_attention_without_mask_is_causal():
    t = Tree([100, 3], [50, 9], BF16, sees=[np.tril(np.ones((c, c), bool)) for c in (50, 9)])
    word = error_word()
    args = list(t.args())
    args[8] = None
    out = ops.tree_attention(*args, error_word=word)
    assert ops.read_device_errors(word) == []
    t.check(out)


@pytest.mark.parametrize("dtype, dim", [(BF16, 128), (F16, 128), (F32, 128), (BF16, 64), (BF16, 256)], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_tree_attention_masked_values_that_are_not_finite(dtype, dim, bad):
    """Rows behind the request's end and nodes that a row does not see do not reach it."""
    lens, counts = [200, 126, 0], [12, 7, 40]
    clean = Tree(lens, counts, dtype, seed=8, dim=dim, hq=8, hkv=2)
    clean_out = clean.run()
    dirty = Tree(lens, counts, dtype, seed=8, dim=dim, hq=8, hkv=2)
    for b, (n, c) in enumerate(zip(lens, counts)):
        for pool in (dirty.k, dirty.v):
            end, last = n + c, int(dirty.table[b][(n + c - 1) // dirty.page])
            pool[:, :, :, last * dirty.page + (end - 1) % dirty.page + 1:(last + 1) * dirty.page] = bad
    assert torch.equal(dirty.run(), clean_out)
    # now a drafted node of each request too: only the rows that see it may differ
    node = 3
    for b, n in enumerate(lens):
        pos = n + node
        slot = int(dirty.table[b][pos // dirty.page]) * dirty.page + pos % dirty.page
        dirty.k[:, :, :, slot] = bad
        dirty.v[:, :, :, slot] = bad
    out = dirty.run()
    for b, (s, c) in enumerate(zip(dirty.starts, counts)):
        see = torch.from_numpy(dirty.sees[b][:, node]).cuda()
        assert torch.equal(out[0, :, s:s + c][:, ~see], clean_out[0, :, s:s + c][:, ~see])
        if bad != -math.inf:
            assert not torch.isfinite(out[0, :, s:s + c][:, see].float()).all()
    # a value alone that is not finite, its key finite: rows that see it get it
    one = Tree(lens, counts, dtype, seed=8, dim=dim, hq=8, hkv=2)
    for b, n in enumerate(lens):
        pos = n + node
        slot = int(one.table[b][pos // one.page]) * one.page + pos % one.page
        one.v[:, :, :, slot, 5] = bad
    out = one.run()
    for b, (s, c) in enumerate(zip(one.starts, counts)):
        see = torch.from_numpy(one.sees[b][:, node]).cuda()
        rows = out[0, :, s:s + c].float()
        assert torch.equal(out[0, :, s:s + c][:, ~see], clean_out[0, :, s:s + c][:, ~see])
        hit = rows[:, see][..., 5]
        assert bool(torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all())
        rest = [d for d in range(dim) if d != 5]
        assert torch.equal(rows[:, see][..., rest], clean_out[0, :, s:s + c].float()[:, see][..., rest])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_tree_attention_leaves_other_rows_alone(dtype):
    t = Tree([100, 30], [5, 20], dtype, gap=3)
    out = torch.full_like(t.q, 7.0)
    t.run(out=out)
    t.check(out)
    assert bool((out[0, :, 5:8] == 7).all()) and bool((out[0, :, 28:] == 7).all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_tree_attention_strides_and_alignment(dtype):
    t = Tree([300, 40], [20, 9], dtype)
    expect = t.run()
    q = t.q
    wide = torch.empty((1, 29, 33, 3 * 128 + 1), dtype=dtype, device="cuda")  # rows on odd elements
    t.q = wide[:, :, 1:, 129:257].transpose(1, 2)
    t.q.copy_(q)
    got = t.run()
    t.check(got)
    t.q = q.contiguous()  # head-major
    out = torch.empty((1, 29, 32, 131), dtype=dtype, device="cuda")[..., 2:130].transpose(1, 2)
    assert torch.equal(t.run(out=out), expect)
    table = torch.full((2, 9), 123456, dtype=torch.int32, device="cuda")  # a view of wider rows
    table[:, :t.table.shape[1]] = i32(t.table)
    args = list(t.args())
    args[4] = table[:, :t.table.shape[1]]
    assert torch.equal(ops.tree_attention(*args), expect)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("hq, hkv, dim", [(4, 4, 128), (8, 4, 64), (8, 1, 128), (16, 1, 96), (64, 2, 128), (6, 2, 128),
                                          (64, 1, 72)], ids=str)
def test_tree_attention_rows_of_q_in_any_layout(dtype, hq, hkv, dim):
    """q whose heads or tokens are next to each other, with room between rows, or off 16-byte
    boundaries; NaN in the rows that no request owns, beside those that one does."""
    tree = Tree([300, 0, 129], [5, 1, 70], dtype, seed=3, hq=hq, hkv=hkv, dim=dim, gap=3)
    owned = np.zeros(tree.q.shape[2], dtype=bool)
    for s, c in zip(tree.starts, tree.counts):
        owned[s:s + c] = True
    tree.q[0, :, torch.from_numpy(~owned).cuda()] = math.nan
    base, n = tree.q, tree.q.shape[2]
    expect = tree.run()
    tree.check(expect)
    rows = torch.from_numpy(owned).cuda()
    layouts = [torch.empty(1, hq, n, dim, dtype=dtype, device="cuda"),                             # heads apart
               torch.empty(1, n, hq, dim + 8, dtype=dtype, device="cuda").transpose(1, 2)[..., :dim],
               torch.empty(1, n, hq, dim + 1, dtype=dtype, device="cuda").transpose(1, 2)[..., 1:],
               torch.empty(1, n, 2 * hq, dim, dtype=dtype, device="cuda").transpose(1, 2)[:, hq:]]
    for q in layouts:
        q.copy_(base)
        tree.q = q
        assert torch.equal(tree.run()[:, :, rows], expect[:, :, rows])


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("dim", [64, 72, 96, 128])
@pytest.mark.parametrize("bad", [math.nan, -math.inf], ids=str)
def test_wide_trees_with_a_node_that_is_not_finite(dtype, dim, bad):
    """Units of more rows than an MMA holds, some whole, some cut: rows that do not see the node
    are those of a clean run, bit for bit, and right; rows that see it are not finite."""
    make = dict(lens=[100, 127, 40, 700] * 12, counts=[70, 90, 65, 130] * 12, dtype=dtype, seed=6, hq=16, hkv=4, dim=dim)
    clean, dirty = Tree(**make), Tree(**make)
    expect = clean.run()
    clean.check(expect)
    for b, n in enumerate(dirty.lens):
        pos = n + 5
        slot = int(dirty.table[b][pos // 128]) * 128 + pos % 128
        dirty.k[:, :, :, slot] = bad
        dirty.v[:, :, :, slot] = bad
    out = dirty.run()
    for s, c, sees in zip(dirty.starts, dirty.counts, dirty.sees):
        hit = torch.from_numpy(np.ascontiguousarray(sees[:, 5])).cuda()
        got, ref = out[0, :, s:s + c], expect[0, :, s:s + c]
        assert torch.equal(got[:, ~hit], ref[:, ~hit])
        assert not torch.isfinite(got[:, hit].float()).any()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_tree_attention_many_requests(dtype):
    """More requests than a warp has lanes, of lengths far apart, some without nodes."""
    rng = np.random.RandomState(4)
    lens = (rng.randint(0, 300, 101) * rng.choice([0, 1, 9], 101)).tolist()
    counts = (rng.randint(1, 6, 101) * rng.choice([0, 1, 1], 101)).tolist()
    Tree(lens, counts, dtype, seed=5, hq=4, hkv=2, dim=64).check()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_tree_attention_bad_metadata_is_flagged_and_contained(dtype):
    t = Tree([300, 200, 50], [6, 5, 4], dtype)
    good = t.run()
    args = list(t.args())
    for index, value, message in [
        (4, i32(np.where(np.arange(t.table.shape[1]) == 1, 10 ** 6, t.table[0])), "page id"),
        (5, -1, "kv length"),
        (5, 2 ** 31 - 3, "kv length"),
        (7, -2, "q_start"),
        (7, 100, "q_start"),
        (6, 12, "q_start"),
    ]:
        bad = list(args)
        bad[index] = args[index].clone()
        bad[index][0] = value
        if index == 4:
            bad[4][0, t.table.shape[1] - 1:] = t.table[0, -1]
        word = error_word()
        out = torch.full_like(t.q, 3.0)
        ops.tree_attention(*bad, out=out, error_word=word)
        assert any(message in m for m in ops.read_device_errors(word)), (index, value)
        assert torch.equal(out[:, :, 6:], good[:, :, 6:])
        if index == 5:
            assert bool((out[:, :, :6] == 0).all())
        elif index in (6, 7):
            assert bool((out[:, :, :6] == 3).all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_tree_attention_streams_and_graphs(dtype):
    """Captured without a warm-up run, replayed on new contents, two graphs at once."""
    a, b = Tree([900, 20], [16, 3], dtype, seed=1), Tree([64, 5000], [1, 30], dtype, seed=2)
    expect = [a.run(), b.run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [a.run(), b.run()]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(outs, expect))
    graphs, results, args = [], [], [list(a.args()), list(b.args())]
    for x in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(ops.tree_attention(*x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for r in results:
            r.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results, expect))
    # the captured launch follows lengths that change on the device
    args[0][5].copy_(i32([400, 10]))
    a.lens = [400, 10]
    graphs[0].replay()
    torch.cuda.synchronize()
    a.check(results[0])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_tree_attention_offsets_past_32_bits(dtype):
    hkv, dim, page = 2, 128, 128
    capacity = (2 ** 31 // (hkv * dim) // page + 40) * page  # over 2^31 elements in one layer
    k = torch.zeros((1, 1, hkv, capacity, dim), dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    pages = capacity // page
    table = np.array([[pages - 1, 3, pages - 20]], dtype=np.int32)
    t = Tree([300], [20], dtype, hq=8, hkv=hkv)
    for i, p in enumerate(table[0]):
        for dst, src in ((k, t.k), (v, t.v)):
            dst[:, :, :, int(p) * page:(int(p) + 1) * page] = src[:, :, :, int(t.table[0][i]) * page:(int(t.table[0][i]) + 1) * page]
    expect = t.run()
    t.k, t.v, t.table = k, v, table
    assert torch.equal(t.run(), expect)


# ---------------------------------------------------------------------------- moves
def pools(layers, heads, pages, page, dim, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (layers, 1, heads, pages * page, dim)
    return [torch.randn(shape, generator=gen, device="cuda").to(dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype, layers, heads, page, dim", [
    (BF16, 3, 8, 128, 128), (F16, 1, 1, 256, 96), (F32, 2, 3, 128, 4), (BF16, 2, 1, 2, 6), (F16, 1, 2, 1, 3),
    (F32, 2, 1, 16, 1),
], ids=str)
def test_copy_pages(dtype, layers, heads, page, dim):
    k, v = pools(layers, heads, 23, page, dim, dtype)
    src, dst = [3, 0, 7, 22, 3], [1, 4, 21, 2, 9]
    expect = []
    for pool in (k, v):
        e = pool.clone()
        view = e.view(layers, heads, 23, page, dim)
        view[:, :, dst] = view[:, :, src].clone()
        expect.append(e)
    word = error_word()
    ops.copy_pages(k, v, i32(src), i32(dst), page, error_word=word)
    assert ops.read_device_errors(word) == []
    assert torch.equal(k, expect[0]) and torch.equal(v, expect[1])


def test_copy_pages_special_entries():
    k, v = pools(2, 2, 12, 128, 128, BF16)
    before = k.clone().view(2, 2, 12, 128, 128)
    word = error_word()
    ops.copy_pages(k, v, i32([]), i32([]), 128, error_word=word)       # nothing to do
    ops.copy_pages(k, v, i32([5]), i32([5]), 128, error_word=word)     # onto itself
    assert ops.read_device_errors(word) == [] and torch.equal(k.view_as(before), before)
    ops.copy_pages(k, v, i32([1, 2]), i32([7, 7]), 128, error_word=word)  # one target twice: the later counts
    assert ops.read_device_errors(word) == []
    assert torch.equal(k.view_as(before)[:, :, 7], before[:, :, 2])
    # entry 0 writes a page that entry 1 reads: skipped, flagged; entry 1 as asked
    ops.copy_pages(k, v, i32([3, 4]), i32([4, 9]), 128, error_word=word)
    assert any("order" in m for m in ops.read_device_errors(word))
    assert torch.equal(k.view_as(before)[:, :, 4], before[:, :, 4]) and torch.equal(k.view_as(before)[:, :, 9], before[:, :, 4])
    word.zero_()
    now = k.clone()
    ops.copy_pages(k, v, i32([-1, 12, 0, 0]), i32([1, 1, -1, 12]), 128, error_word=word)
    assert any("page id" in m for m in ops.read_device_errors(word)) and torch.equal(k, now)


@pytest.mark.parametrize("dtype, layers, heads, page, dim", [
    (BF16, 3, 8, 128, 128), (F16, 2, 1, 256, 96), (F32, 2, 3, 128, 4), (BF16, 2, 1, 2, 6), (F16, 1, 2, 1, 3),
], ids=str)
def test_compact_rows(dtype, layers, heads, page, dim):
    rng = np.random.RandomState(2)
    base = [0, 127, 5, 300, 64, 9]
    reach = [40, 30, 1, 700, 200, 10]
    src = [sorted(rng.permutation(40)[:17].tolist()), [0, 2, 3, 29], [], sorted(rng.permutation(700)[:333].tolist()),
           list(range(200)), [9]]
    table, pages = U.page_table([a + r for a, r in zip(base, reach)], page, 4)
    k, v = pools(layers, heads, pages, page, dim, dtype)
    expect = [U.compact_reference(p, table, base, src, page) for p in (k, v)]
    flat = i32([s for rows in src for s in rows])
    start = i32(np.concatenate([[0], np.cumsum([len(r) for r in src])]))
    word = error_word()
    ops.compact_rows(k, v, i32(table), i32(base), flat, start, page, error_word=word)
    assert ops.read_device_errors(word) == []
    assert torch.equal(k, expect[0]) and torch.equal(v, expect[1])


def test_compact_rows_refuses_what_it_cannot_order():
    table, pages = U.page_table([300, 300], 128, 0)
    k, v = pools(2, 2, pages, 128, 128, BF16)
    for src, message in [([4, 3], "order"), ([2, 2], "order"), ([-1], "order"), ([0, 500], "pages")]:
        before, word = (k.clone(), v.clone()), error_word()
        ops.compact_rows(k, v, i32(table), i32([10, 10]), i32(src + [0, 7]),
                         i32([0, len(src), len(src) + 2]), 128, error_word=word)
        assert any(message in m for m in ops.read_device_errors(word)), src
        keep = [s if 0 <= s < 290 and s >= i and (i == 0 or s > src[i - 1]) else i for i, s in enumerate(src)]
        for pool, old in zip((k, v), before):
            assert torch.equal(pool, U.compact_reference(old, table, [10, 10], [keep, [0, 7]], 128))
    word = error_word()
    now = k.clone()
    ops.compact_rows(k, v, i32(table), i32([10, 10]), i32([5, 6]), i32([0, 9, 2]), 128, error_word=word)
    assert ops.read_device_errors(word) != [] and torch.equal(k, now)


# ---------------------------------------------------------------------------- bounds, selection
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("layers, heads, page, dim", [(3, 8, 128, 128), (1, 1, 256, 64), (2, 3, 128, 96), (1, 2, 64, 256),
                                                      (1, 1, 1, 8), (2, 1, 2, 40)])
def test_page_bounds(dtype, layers, heads, page, dim):
    k = pools(layers, heads, 9, page, dim, dtype)[0]
    expect = U.bounds_reference(k, page)
    got = torch.full_like(expect, 5.0)
    word = error_word()
    ops.page_bounds(k, got, i32([2, -1, 8, 0, -1]), page, error_word=word)
    assert ops.read_device_errors(word) == []
    for p in range(9):
        assert torch.equal(got[:, :, p], expect[:, :, p] if p in (0, 2, 8) else torch.full_like(expect[:, :, p], 5.0))
    got.fill_(5.0)
    ops.page_bounds(k, got, i32([1]), page, layer=layers - 1, error_word=word)
    assert torch.equal(got[-1, :, 1], expect[-1, :, 1]) and bool((got[:-1] == 5).all())
    ops.page_bounds(k, got, i32([]), page, error_word=word)
    assert ops.read_device_errors(word) == []
    ops.page_bounds(k, got, i32([9, -2]), page, error_word=word)
    assert any("page id" in m for m in ops.read_device_errors(word))


def test_page_bounds_not_finite():
    k = pools(1, 2, 3, 128, 128, BF16)[0]
    k[0, 0, 0, 5, 7], k[0, 0, 0, 6, 8], k[0, 0, 1, 130, 9] = math.nan, math.inf, -math.inf
    expect = U.bounds_reference(k, 128)
    got = torch.zeros_like(expect)
    ops.page_bounds(k, got, i32([0, 1, 2]), 128)
    assert torch.equal(got.nan_to_num(nan=1e4), expect.nan_to_num(nan=1e4)) and bool(torch.isnan(got).sum() == 2)


class Sparse:
    def __init__(self, lens, take, dtype, seed=0, hq=32, hkv=8, dim=128, page=128, layers=1, layer=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.take, self.page, self.layer = list(lens), take, page, layer
        self.table, pages = U.page_table([n + 1 for n in lens], page, seed)
        shape = (layers, 1, hkv, pages * page, dim)
        self.k = torch.randn(shape, generator=gen, device="cuda").to(dtype)
        self.v = torch.randn(shape, generator=gen, device="cuda").to(dtype)
        self.q = torch.randn((len(lens), 1, hq, dim), generator=gen, device="cuda").to(dtype).transpose(1, 2)
        self.bounds = U.bounds_reference(self.k, page)
        self.scale = 1.0 / math.sqrt(dim)

    def args(self):
        return (self.q, self.k, self.v, self.bounds, self.layer, i32(self.table), i32(self.lens), self.page, self.take)

    def run(self, **kw):
        word = error_word()
        out, chosen = ops.sparse_attention(*self.args(), error_word=word, **kw)
        torch.cuda.synchronize()
        assert ops.read_device_errors(word) == []
        return out, chosen

    def check(self, out=None, chosen=None):
        if out is None:
            out, chosen = self.run()
        expect = U.selection_reference(self.q, self.bounds, self.layer, self.table, self.lens, self.page, self.take)
        assert np.array_equal(chosen.cpu().numpy(), expect)
        ref, bound = U.sparse_reference(self.q, self.k, self.v, self.layer, self.table, self.lens, expect,
                                        self.page, self.scale)
        err = (out.double() - ref).abs()
        assert bool((err <= bound).all()), float((err / bound).max())


SPARSE = [
    dict(lens=[0], take=1), dict(lens=[0, 127, 128, 129], take=1), dict(lens=[0, 127, 128, 129], take=2),
    dict(lens=[5000, 3, 2047, 2048], take=4), dict(lens=[5000, 3, 2047, 2048], take=16),
    dict(lens=[5000, 3, 700], take=64), dict(lens=[32700], take=32), dict(lens=[4000, 100], take=7, hq=8, hkv=8),
    dict(lens=[4000, 100], take=7, hq=6, hkv=2, page=256), dict(lens=[4000, 100], take=5, hq=8, hkv=1, dim=64),
    dict(lens=[4000, 100], take=5, hq=10, hkv=2, dim=96), dict(lens=[2000, 100], take=5, hq=4, hkv=2, dim=256, page=64),
    dict(lens=[3000] * 33, take=9, hq=4, hkv=1, layers=2, layer=1), dict(lens=[70000, 11], take=3, hq=2, hkv=1, page=64),
    dict(lens=[3000], take=9, hq=48, hkv=2),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("case", SPARSE, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:60])
def test_sparse_attention(case, dtype):
    Sparse(dtype=dtype, seed=len(str(case)), **case).check()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_sparse_attention_ties_and_values_that_are_not_finite(dtype):
    s = Sparse([40 * 128 + 5, 30 * 128], 9, dtype, hq=8, hkv=2)
    s.bounds[:, :, :, 0], s.bounds[:, :, :, 1] = -1.0, 1.0   # every page scores the same
    _, chosen = s.run()
    assert chosen[0, 0].tolist() == list(range(8)) + [40] and chosen[1, 1].tolist() == list(range(8)) + [30]
    s.check()
    s.bounds.zero_()                                            # and zero of either sign
    s.bounds[:, :, int(s.table[0][3]), 1, 0] = -0.0
    s.check()
    s = Sparse([40 * 128 + 5], 5, dtype, hq=8, hkv=2)
    page = int(s.table[0][17])
    s.bounds[0, 0, page, 1, 3] = math.nan                     # ranks first
    s.bounds[0, 1, page, 0] = -math.inf
    s.bounds[0, 1, page, 1] = -math.inf                      # q of both signs: a NaN sum too, or -inf
    s.check()
    # rows behind the request's end
    s = Sparse([40 * 128 + 5, 130], 5, dtype)
    out, _ = s.run()
    for b, n in enumerate(s.lens):
        last = int(s.table[b][n // 128])
        for pool in (s.k, s.v):
            pool[:, :, :, last * 128 + n % 128 + 1:(last + 1) * 128] = math.nan
    assert torch.equal(s.run()[0], out)


def test_sparse_attention_bad_lengths_are_flagged():
    for lens, message in [([-1, 300], "kv length"), ([10 ** 6, 300], "kv length")]:
        s = Sparse([900, 300], 3, BF16)
        out0, chosen0 = s.run()
        args = list(s.args())
        args[6] = i32(lens)
        word = error_word()
        out, chosen = ops.sparse_attention(*args, error_word=word)
        assert any(message in m for m in ops.read_device_errors(word))
        assert torch.equal(out[1], out0[1]) and torch.equal(chosen[1], chosen0[1])
        assert bool((out[0] == 0).all()) and bool((chosen[0] == -1).all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_sparse_attention_strides_streams_and_graphs(dtype):
    s = Sparse([5000, 60, 1300], 6, dtype)
    expect, pages = s.run()
    q = s.q
    wide = torch.empty((3, 33, 2, 259), dtype=dtype, device="cuda")
    s.q = wide[:, 1:, 1:, 129:257]
    s.q.copy_(q)
    out = torch.empty((3, 40, 1, 130), dtype=dtype, device="cuda")[:, 5:37, :, 1:129]
    got, p = s.run(out=out)
    assert torch.equal(p, pages)
    s.check(got, p)
    s.q = q
    graph = torch.cuda.CUDAGraph()
    args = s.args()
    with torch.cuda.graph(graph):
        got, p = ops.sparse_attention(*args)
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, expect) and torch.equal(p, pages)
    args[6].copy_(i32([300, 1290, 4]))
    s.lens = [300, 59, 4]
    args[6].copy_(i32(s.lens))
    graph.replay()
    torch.cuda.synchronize()
    s.check(got, p)


def test_wrappers_check_their_arguments():
    t = Tree([300, 40], [20, 9], BF16)
    args = list(t.args())

    def tree(index, value):
        bad = list(args)
        bad[index] = value
        return ops.tree_attention(*bad)

    for index, value, kind in [
        (0, t.q.float(), ValueError), (0, t.q[0], ValueError), (0, t.q[..., ::2], ValueError),
        (0, t.q[..., :64], ValueError), (4, args[4].long(), ValueError), (4, args[4][:1], ValueError),
        (4, args[4].t().contiguous().t(), ValueError), (5, args[5].long(), TypeError), (6, args[6][:1], ValueError),
        (7, args[7][None], TypeError), (8, args[8].long(), TypeError), (8, args[8][:-1], ValueError),
        (8, args[8].cpu(), RuntimeError), (10, 40, ValueError), (9, 32, RuntimeError), (3, 1, RuntimeError),
    ]:
        with pytest.raises(kind):
            tree(index, value)
    with pytest.raises(ValueError):
        ops.tree_attention(*args, out=torch.empty_like(t.q).float())
    with pytest.raises(RuntimeError):
        ops.tree_attention(*args, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.tree_attention(*args, scale=0.0)
    with pytest.raises(ValueError):
        ops.copy_pages(t.k, t.v, i32([1, 2]), i32([3]), 128)
    with pytest.raises(TypeError):
        ops.copy_pages(t.k, t.v, i32([1]).long(), i32([3]), 128)
    with pytest.raises(ValueError):
        ops.compact_rows(t.k, t.v, args[4], args[5], i32([1]), i32([0, 1]), 128)
    s = Sparse([300, 40], 2, BF16)
    with pytest.raises(ValueError):
        ops.page_bounds(s.k, s.bounds[:, :4], i32([0]), 128)
    sargs = list(s.args())
    for index, value, kind in [(0, s.q.expand(2, 32, 2, 128), ValueError), (3, s.bounds.float(), ValueError),
                               (6, sargs[6].long(), TypeError), (8, 0, ValueError), (7, 64, ValueError)]:
        bad = list(sargs)
        bad[index] = value
        with pytest.raises(kind):
            ops.sparse_attention(*bad)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("seed", range(6))
def test_sparse_attention_scores_that_are_nearly_equal(dtype, seed):
    """Bounds whose scores differ in their last bits only, and exact ties among them: the pages
    taken are those of the sums in 64 bits, whatever order they are summed in."""
    s = Sparse([200 * 128 + 7, 90 * 128], 40, dtype, seed=seed, hq=8, hkv=2)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((1, 2, 1, 2, 128), generator=gen, device="cuda")
    lo, hi = base.amin(dim=3, keepdim=True), base.amax(dim=3, keepdim=True)
    bounds = torch.cat([lo, hi], dim=3).to(dtype).expand(s.bounds.shape).contiguous()
    # one element of each page moves by one step or not at all
    pages = bounds.shape[2]
    where = torch.randint(0, 128, (pages,), generator=gen, device="cuda")
    side = torch.randint(0, 2, (pages,), generator=gen, device="cuda")
    bits = bounds.view(torch.int16)
    moved = torch.randint(0, 2, (pages,), generator=gen, device="cuda").to(torch.int16)
    bits[0, :, torch.arange(pages, device="cuda"), side, where] += moved
    s.bounds = bounds
    s.check()
