"""Chunk attention whose running maximum moves after values are in O, and whose rows see keys
in one part of a tile only: breadth-first trees, stars, masks of one 64-key half, scores that rise
or fall from tile to tile by more than the 2^8 that a maximum may lag. Trees on tensor cores (one and
two row blocks per unit) and on CUDA cores, and decode over chosen pages; each against its
64-bit definition within the bounds derived in ``operators_util``."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import operators_util as U
from test_gpu_operators import BF16, F16, F32, Sparse, Tree

pytestmark = pytest.mark.gpu


def breadth_first(nodes, fan):
    """Every node has `fan` children, numbered level by level."""
    return [(i - 1) // fan if i else -1 for i in range(nodes)]


def late_star(nodes):
    """A tree in draft order whose nodes from 128 on follow node 0, every 8th the context itself."""
    rng = np.random.RandomState(nodes)
    parents = U.random_parents(min(nodes, 128), rng)
    return parents + [-1 if i % 8 == 7 else 0 for i in range(128, nodes)]


def one_half(nodes, half):
    """Rows that see 64 keys of a 128-key tile: nodes 0..63 or 64..127 of each 128, every 8th itself
    and the last node alone."""
    sees = np.zeros((nodes, nodes), dtype=bool)
    sees[:, (np.arange(nodes) // 64) % 2 == half] = True
    sees[np.arange(nodes), np.arange(nodes)] = True
    sees[::8] = False
    sees[::8, -1] = True
    return sees


def shape_scores(case, how):
    """Scores that spread widely (a standard deviation of 16), or rise or fall by 40 nats along each
    request's positions (q has a constant on one axis, k a part that follows the position)."""
    if how == "spread":
        case.q.mul_(16.0)
    if how in ("plain", "spread"):
        return case
    dim = case.q.shape[-1]
    case.q[..., 0] = 8.0
    case.k[..., 0] = 0.0
    counts = getattr(case, "counts", [1] * len(case.lens))
    for b, (n, c) in enumerate(zip(case.lens, counts)):
        pos = np.arange(n + c)
        at = torch.from_numpy(case.table[b][pos // case.page].astype(np.int64) * case.page + pos % case.page).cuda()
        part = torch.from_numpy(pos / max(n + c - 1, 1)).cuda()
        part = part if how == "rising" else 1 - part
        case.k[case.layer, 0][:, at, 0] = (40.0 * dim ** 0.5 / 8.0 * part).to(case.k.dtype)
    return case


SCORES = ["plain", "spread", "rising", "falling"]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("scores", SCORES)
def test_late_nodes_that_see_early_ones_only(dtype, dim, scores):
    """Nodes 128 .. of a wide tree see node 0 and themselves, some only themselves: of the tile before,
    a row sees keys of one half or nothing."""
    trees = [late_star(n) for n in (160, 136, 200, 255)] * 10
    t = Tree([0] * 40, [len(p) for p in trees], dtype, seed=1, hq=8, hkv=2, dim=dim,
             sees=[U.sees_of_parents(p) for p in trees])
    shape_scores(t, scores).check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("hq, hkv, dim", [(8, 2, 128), (8, 2, 64), (4, 1, 96), (2, 2, 128), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("scores", SCORES)
def test_breadth_first_trees(dtype, hq, hkv, dim, scores):
    lens = [0, 10, 64, 127, 1024] * 8
    trees = [breadth_first(n, fan) for n, fan in zip([129, 256, 170, 200, 140, 33, 64, 255] * 5, [2, 3, 8, 64, 4] * 8)]
    t = Tree(lens, [len(p) for p in trees], dtype, seed=2, hq=hq, hkv=hkv, dim=dim,
             sees=[U.sees_of_parents(p) for p in trees])
    shape_scores(t, scores).check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("scores", SCORES)
def test_rows_that_see_one_half_of_a_tile(dtype, dim, half, scores):
    """Contexts of nothing (whole tiles of drafted nodes) and such that end inside a tile."""
    counts = [256, 130, 192, 31, 8] * 8
    lens = [0, 0, 128, 40, 0, 64] * 6 + [4096, 200, 0, 1000]
    t = Tree(lens, counts, dtype, seed=3, hq=8, hkv=2, dim=dim, sees=[one_half(c, half) for c in counts])
    shape_scores(t, scores).check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("scores", SCORES[1:])
@pytest.mark.parametrize("case", [
    dict(lens=[4000, 17, 900], counts=[8, 3, 20], hq=32, hkv=8), dict(lens=[4000, 17, 900], counts=[40, 3, 100], hq=32, hkv=8),
    dict(lens=[2000, 300], counts=[2, 1], hq=4, hkv=2), dict(lens=[2000, 300], counts=[2, 1], hq=4, hkv=2, dim=256),
    dict(lens=[2000, 300], counts=[9, 4], hq=4, hkv=2, dim=40), dict(lens=[2000, 300], counts=[40, 7], hq=4, hkv=2, dim=136),
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:60])
def test_contexts_whose_scores_move(case, dtype, scores):
    shape_scores(Tree(dtype=dtype, seed=4, **case), scores).check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("scores", SCORES[1:])
@pytest.mark.parametrize("case", [
    dict(lens=[5000, 3, 2047, 2048], take=16), dict(lens=[5000, 700, 2047], take=64, hq=8, hkv=2, dim=64),
    dict(lens=[4000, 100], take=9, hq=10, hkv=2, dim=96), dict(lens=[2000, 100], take=12, hq=4, hkv=2, dim=256, page=64),
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:60])
def test_chosen_pages_whose_scores_move(case, dtype, scores):
    s = shape_scores(Sparse(dtype=dtype, seed=5, **case), scores)
    s.bounds = U.bounds_reference(s.k, s.page)
    s.check()
