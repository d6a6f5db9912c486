"""Page manager side of drafted trees and forks, on the CPU: metadata of a tree batch, accepted
paths moved up behind the context, refusals, forks and copy-on-write of a whole step."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from hayate_b200 import PagedKVCacheManager
from hayate_b200.paged_cache import _tree_metadata

import operators_util as U


def make_manager(pages=12, requests=6, layers=2, heads=2, dim=4):
    m = PagedKVCacheManager(layers, heads, dim, pages * 128, 128, requests, torch.float32, "cpu")
    torch.manual_seed(0)
    m.k_cache.normal_()
    m.v_cache.normal_()
    return m


def grown(m, length):
    h = m.allocate()
    m.reserve(h, length)
    h.length = length
    return h


@pytest.mark.parametrize("sizes", [[1], [5, 1, 40], [64, 33], [200]])
def test_tree_metadata(sizes):
    rng = np.random.RandomState(sum(sizes))
    trees = [U.random_parents(n, rng) for n in sizes]
    depth, mask = _tree_metadata(trees)
    words = -(-max(sizes) // 32)
    assert mask.shape == (sum(sizes), words) and mask.dtype == np.int32
    at = 0
    for tree in trees:
        sees = U.sees_of_parents(tree)
        assert np.array_equal(mask[at:at + len(tree)], U.pack_bits(sees, words))
        assert np.array_equal(depth[at:at + len(tree)], sees.sum(1) - 1)
        at += len(tree)


def test_tree_batch_layout():
    m = make_manager()
    a, b = grown(m, 130), grown(m, 0)
    batch = m.begin_tree_batch([a, b], [[-1, 0, 0, 1], [-1, -1]])
    lay = batch.layout
    assert lay.total_tokens == 6 and lay.q_start.tolist() == [0, 4] and lay.q_len.tolist() == [4, 2]
    assert lay.token_request.tolist() == [0, 0, 0, 0, 1, 1]
    assert lay.token_depth.tolist() == [0, 1, 1, 2, 0, 0]
    assert lay.tree_mask.tolist() == [[1], [3], [5], [11], [1], [2]]
    assert batch.cache_lens.tolist() == [130, 0] and batch.query_len == 4
    assert len(a.pages) == 2 and len(b.pages) == 1


@pytest.mark.parametrize("parents", [[[0]], [[-1, 1]], [[-2]], [[-1, 0, 2]]])
def test_tree_batch_refuses_parents_that_are_no_tree(parents):
    m = make_manager()
    with pytest.raises(ValueError, match="parent"):
        m.begin_tree_batch([grown(m, 10)], parents)


def test_tree_batch_refusals():
    m = make_manager(pages=2)
    h = grown(m, 10)
    with pytest.raises(ValueError, match="empty batch"):
        m.begin_tree_batch([], [])
    with pytest.raises(ValueError, match="one list of parents"):
        m.begin_tree_batch([h], [[-1], [-1]])
    with pytest.raises(ValueError, match="query_len"):
        m.begin_tree_batch([h], [[]])
    with pytest.raises(ValueError, match="twice"):
        m.begin_tree_batch([h, h], [[-1], [-1]])
    with pytest.raises(MemoryError):
        m.begin_tree_batch([h], [[-1] * 300])
    m.release(h)
    with pytest.raises(RuntimeError):
        m.begin_tree_batch([h], [[-1]])


def test_commit_tree_moves_the_accepted_rows_and_grows_the_requests():
    m = make_manager()
    hs = [grown(m, n) for n in (125, 0, 300, 40)]
    trees = [[-1, 0, 0, 1, 2, 4, 4], [-1, -1, 1], [-1, 0, 1], [-1, 0]]
    paths = [[0, 2, 4, 6], [1, 2], [], [0, 1]]
    batch = m.begin_tree_batch(hs, trees)
    table = np.full((4, 3), -1, dtype=np.int64)
    for b, h in enumerate(hs):
        table[b, :len(h.pages)] = h.pages
    expect = [U.compact_reference(p, table, [h.length for h in hs], paths, 128) for p in (m.k_cache, m.v_cache)]
    m.commit_tree(batch, hs, paths)
    assert torch.equal(m.k_cache, expect[0]) and torch.equal(m.v_cache, expect[1])
    assert [h.length for h in hs] == [129, 2, 300, 42]


def test_commit_tree_refusals():
    m = make_manager()
    a, b = grown(m, 125), grown(m, 10)
    batch = m.begin_tree_batch([a, b], [[-1, 0, 0, 1], [-1]])
    before = m.k_cache.clone()
    for paths in ([[1], []], [[0, 3], []], [[0, 1, 2], []], [[0], [1]], [[-1], []], [[4], []], [[0, 0], []]):
        with pytest.raises(ValueError, match="path"):
            m.commit_tree(batch, [a, b], paths)
    with pytest.raises(ValueError, match="one path per request"):
        m.commit_tree(batch, [a, b], [[0]])
    with pytest.raises(ValueError, match="begin_tree_batch"):
        m.commit_tree(m.begin_batch([a], [2]), [a], [[0]])
    assert torch.equal(m.k_cache, before) and a.length == 125
    m.commit_tree(batch, [a, b], [[0, 1, 3], [0]])
    assert a.length == 128 and b.length == 11
    with pytest.raises(RuntimeError, match="changed"):
        m.commit_tree(batch, [a, b], [[0], []])


def test_commit_tree_takes_the_handles_in_their_order():
    """Two requests of one length and one tree: swapped, each would get the other's path."""
    m = make_manager()
    a, b = grown(m, 10), grown(m, 10)
    batch = m.begin_tree_batch([a, b], [[-1, 0, 0]] * 2)
    before = m.k_cache.clone()
    with pytest.raises(ValueError, match="order"):
        m.commit_tree(batch, [b, a], [[0, 2], [0]])
    with pytest.raises(ValueError, match="order"):
        m.commit_tree(batch, [a, a], [[0, 2], [0]])
    assert torch.equal(m.k_cache, before) and a.length == b.length == 10
    m.commit_tree(batch, [a, b], [[0, 2], [0]])
    assert a.length == 12 and b.length == 11


def test_commit_tree_refuses_a_request_whose_pages_changed():
    """The batch's page table is as old as the batch: rows are not moved through a stale one."""
    m = make_manager()
    a, b = grown(m, 126), grown(m, 10)
    batch = m.begin_tree_batch([a], [[-1, 0, 0, 1, 1]])
    m.truncate(a, 126)        # gives the second page back
    with pytest.raises(RuntimeError, match="changed"):
        m.commit_tree(batch, [a], [[0, 2]])
    m.begin_batch([b], 200)   # and another request takes it
    m.reserve(a, 131)
    before = m.k_cache.clone()
    with pytest.raises(RuntimeError, match="changed"):
        m.commit_tree(batch, [a], [[0, 2]])
    assert torch.equal(m.k_cache, before) and a.length == 126


def test_fork_shares_full_pages_and_copies_the_one_being_written():
    m = make_manager()
    h = grown(m, 300)
    free = len(m._free_pages)
    forks = m.fork(h, 3)
    assert len(m._free_pages) == free - 3
    for f in forks:
        assert f.length == 300 and f.pages[:2] == h.pages[:2] and f.pages[2] not in h.pages
        a, b = h.pages[2] * 128, f.pages[2] * 128
        for pool in (m.k_cache, m.v_cache):
            assert torch.equal(pool[:, :, :, a:a + 128], pool[:, :, :, b:b + 128])
    assert len({f.pages[2] for f in forks}) == 3
    assert [m.page_refcount(p) for p in h.pages] == [4, 4, 1]
    # the forks' next step takes no page and copies nothing
    free = list(m._free_pages)
    m.begin_batch([h] + forks, 1)
    assert m._free_pages == free
    m.release(h)
    assert [m.page_refcount(p) for p in forks[0].pages] == [3, 3, 1]


def test_fork_at_a_page_boundary_copies_nothing():
    m = make_manager()
    h = grown(m, 256)
    free = len(m._free_pages)
    forks = m.fork(h, 2)
    assert len(m._free_pages) == free and all(f.pages == h.pages for f in forks)
    empty = m.fork(m.allocate(), 1)
    assert empty[0].length == 0 and empty[0].pages == []


def test_fork_takes_all_or_nothing():
    m = make_manager(pages=5, requests=4)
    h = grown(m, 300)
    with pytest.raises(MemoryError, match="pages"):
        m.fork(h, 3)
    assert len(m._free_pages) == 2 and len(m._free_slots) == 3
    assert all(m.page_refcount(p) == 1 for p in h.pages)
    with pytest.raises(MemoryError, match="requests"):
        m.fork(h, 4)
    with pytest.raises(ValueError):
        m.fork(h, 0)
    m.release(h)
    with pytest.raises(RuntimeError):
        m.fork(h, 1)


def test_a_step_copies_its_shared_pages_together():
    """Three holders of one partial page append in one step: two copies, the last writer keeps it."""
    m = make_manager()
    h = grown(m, 200)
    others = [m.share(h, 200), m.share(h, 150)]
    page = h.pages[1]
    content = m.k_cache[:, :, :, page * 128:(page + 1) * 128].clone()
    calls = []
    copy = m._copy_pages
    m._copy_pages = lambda pairs: (calls.append(list(pairs)), copy(pairs))
    m.begin_batch([h] + others, 1)
    assert [len(c) for c in calls] == [2]
    last = {x.pages[1] for x in [h] + others}
    assert len(last) == 3 and page in last
    for p in last:
        assert torch.equal(m.k_cache[:, :, :, p * 128:(p + 1) * 128], content)


def test_page_bounds_need_a_gpu():
    m = make_manager()
    with pytest.raises(RuntimeError, match="CUDA"):
        m.track_page_bounds()
    h = grown(m, 200)
    m.refresh_page_bounds(h)  # not kept: nothing to do
    batch = m.begin_batch([h], 1)
    with pytest.raises(RuntimeError, match="track_page_bounds"):
        batch.attend_pages(torch.zeros(1, 4, 1, 4), 0, 2)
