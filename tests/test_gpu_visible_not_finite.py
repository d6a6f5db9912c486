"""Keys and queries that are not finite where they are seen: the rows are those of the definition,
NaN wherever a score is NaN or +inf, whatever place of a tile the key has; a score of -inf is a key
of no weight."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import operators_util as U
from test_gpu_operators import BF16, F16, F32, Sparse, Tree

pytestmark = pytest.mark.gpu

SHAPES = [dict(hq=8, hkv=2, dim=128), dict(hq=8, hkv=2, dim=64), dict(hq=8, hkv=2, dim=256), dict(hq=4, hkv=2, dim=128)]
PLACES = list(range(16)) + [31, 39, 63, 64, 71, 95, 103, 127]


def slots_of(case, b, positions):
    pos = np.asarray(positions)
    return torch.from_numpy(case.table[b][pos // case.page].astype(np.int64) * case.page + pos % case.page).cuda()


def check_rows(got, ref, bound):
    """NaN where the definition is NaN, within the bound elsewhere."""
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    assert bool(((got.double() - ref).abs() <= bound)[~nan].all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
@pytest.mark.parametrize("nodes", [1, 3, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
def test_a_cached_key(dtype, shape, nodes, bad):
    """One key of every request's context: NaN in all its elements, or infinite in one, which makes
    scores of +inf or -inf by the sign of the row's q."""
    t = Tree([300] * len(PLACES), [nodes] * len(PLACES), dtype, seed=1, **shape)
    for b, place in enumerate(PLACES):
        at = slots_of(t, b, [128 + place])
        if math.isnan(bad):
            t.k[:, :, :, at] = bad
        else:
            t.k[:, :, :, at, 3] = bad
    out = t.run()
    dirty, k = t.k, t.k.clone()
    for b, place in enumerate(PLACES):  # a weight of nothing is taken from a copy without the infinity
        k[:, :, :, slots_of(t, b, [128 + place]), 3] = 0.0
    group = t.q.shape[1] // k.shape[2]
    for b, (s, c, place) in enumerate(zip(t.starts, t.counts, PLACES)):
        rows = slice(s, s + c)
        sees = torch.ones((c, 300 + c), dtype=torch.bool)
        sees[:, 300:] = torch.from_numpy(t.sees[b])
        sees = sees.cuda()
        at = slots_of(t, b, range(300 + c))
        for h in range(t.q.shape[1]):
            q = t.q[0, h, rows].double()
            scores = q @ dirty[t.layer, 0, h // group][at].double().t()
            poor = torch.isnan(scores[:, 128 + place]) | (scores[:, 128 + place] == math.inf)
            seen = sees.clone()
            seen[:, 128 + place] = False
            ref, bound = U.attention_rows(q, k[t.layer, 0, h // group][at].double(), t.v[t.layer, 0, h // group][at].double(),
                                          seen, t.scale, dtype)
            ref[poor] = math.nan
            check_rows(out[0, h, rows], ref, bound)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
@pytest.mark.parametrize("wide", [False, True], ids=["narrow", "wide"])
def test_a_query_that_sees_one_node(dtype, shape, wide):
    """No context, every node sees itself alone: its own value, or NaN if its q is NaN. Weight over
    sum: a product, a quotient and a product in fp32, 3 x 2^-24; in 16 bits the weight rounds to
    1 (off by 7.5e-5 at most) and the quotient back to the value (2^-12 is half the smallest step)."""
    nodes = 128 if wide else 16
    t = Tree([0, 5 * 128], [nodes, 3], dtype, seed=2, sees=[np.eye(nodes, dtype=bool), np.eye(3, dtype=bool)], **shape)
    rows = list(range(0, nodes, 2)) + [7, 15]
    t.q[0, :, rows] = math.nan
    out = t.run()
    group = t.q.shape[1] // t.k.shape[2]
    own = t.v[0, 0][:, slots_of(t, 0, range(nodes))].repeat_interleave(group, 0).clone()
    own[:, rows] = math.nan
    assert torch.equal(torch.isnan(out[0, :, :nodes]), torch.isnan(own))
    fine = ~torch.isnan(own)
    assert bool(((out[0, :, :nodes] - own).abs()[fine] <= 2.0 ** -22 * own.abs()[fine]).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_key_of_a_chosen_page(dtype, dim):
    s = Sparse([300] * len(PLACES), 4, dtype, seed=3, hq=8, hkv=2, dim=dim)
    clean, _ = s.run()
    for b, place in enumerate(PLACES):
        s.k[:, :, 1, slots_of(s, b, [128 + place])] = math.nan
    out, _ = s.run()
    assert torch.equal(out[:, :4], clean[:, :4])   # the other KV head's rows
    assert bool(torch.isnan(out[:, 4:]).all())
