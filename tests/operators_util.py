"""64-bit definitions of the tree, move, bounds and page-selection operators, and the error
bounds their kernels are held to (shared by their CPU and GPU tests)."""

from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def page_table(reach, page, seed, spare=2):
    """Shuffled physical pages for requests that reach so many tokens (-1 past the last) and
    the page count of a pool that holds them."""
    counts = [max(1, -(-n // page)) for n in reach]
    ids = np.random.RandomState(seed).permutation(sum(counts) + spare)
    table = np.full((len(reach), max(counts)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, sum(counts) + spare


def random_parents(nodes, rng, reach=9):
    """A tree in draft order: every node's parent is an earlier node or the context (-1)."""
    return [-1 if i == 0 else int(rng.randint(max(-1, i - reach), i)) for i in range(nodes)]


def sees_of_parents(parents):
    sees = np.zeros((len(parents), len(parents)), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def pack_bits(sees, words):
    """int32 words of a boolean [rows, nodes] matrix: bit j % 32 of word j // 32 is column j."""
    full = np.zeros((sees.shape[0], words * 32), dtype=np.uint64)
    full[:, :sees.shape[1]] = sees
    bits = full.reshape(sees.shape[0], words, 32) << np.arange(32, dtype=np.uint64)
    return bits.sum(axis=2).astype(np.uint32).view(np.int32)


def rows_of(pool, layer, g, table_row, n, page):
    """The first ``n`` rows of a request's cache as [n, D] in 64 bits."""
    pos = np.arange(n)
    slots = torch.from_numpy(table_row[pos // page].astype(np.int64) * page + pos % page).to(pool.device)
    return pool[layer, 0, g].index_select(0, slots).double()


def attention_rows(q, k, v, sees, scale, dtype):
    """(rows, allowed error) of softmax(scale q k^T) v over the keys that ``sees`` shows.

    q [R, D], k/v [K, D], sees [R, K], 64 bits. The bound counts, against A = sum of weight
    times |v|: one rounding of each weight to the storage type (u, none for fp32), fp32
    scores (a sum of D products, each partial sum off by 2^-24 of sum |q k|; an error e of
    a score is a factor exp(2 e) of its weight), 2^-21 for the base-2 exponential and its
    argument (2^-12 where a cubic serves some exponentials of the 16-bit kernels, whose
    relative error is below 7.5e-5), fp32 sums over K keys; plus the output's rounding, and
    for fp16 the absolute half step 2^-25 of weights below its normal range.
    """
    u = HALF_STEP[dtype]
    logits = scale * (q @ k.t())
    logits = torch.where(sees, logits, -math.inf)
    top = logits.amax(dim=1, keepdim=True)
    w = torch.exp(logits - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(dim=1, keepdim=True)
    w = torch.where(total > 0, w / total, torch.zeros_like(w))
    seen_v = torch.where(sees.any(dim=0)[:, None], v, torch.zeros_like(v))
    out = w @ seen_v
    a = w @ seen_v.abs()
    magnitude = scale * (q.abs() @ k.abs().t())
    e = 2 * (q.shape[1] + 4) * 2.0 ** -24 * torch.where(sees, magnitude, torch.zeros_like(magnitude)).amax(dim=1, keepdim=True)
    e = 2 * e + k.shape[0] * 2.0 ** -24 + 2.0 ** -21
    if dtype != torch.float32:
        e = e + 2.0 ** -12 + u
    bound = a * e * 1.01 + out.abs() * u * 1.01 + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * (1 + sees.sum(dim=1, keepdim=True) * seen_v.abs().amax())
    return out, bound


def tree_reference(q, k_pool, v_pool, layer, table, lens, starts, counts, sees, page, scale):
    """[1, H_q, N, D] rows (64 bits) and allowed errors; ``sees[b]`` is request b's [T, T]."""
    hq, hkv = q.shape[1], k_pool.shape[2]
    group = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, (n, start, t) in enumerate(zip(lens, starts, counts)):
        if t == 0:
            continue
        full = torch.ones((t, n + t), dtype=torch.bool)
        full[:, n:] = torch.from_numpy(np.asarray(sees[b]))
        full = full.to(q.device)
        for g in range(hkv):
            k = rows_of(k_pool, layer, g, table[b], n + t, page)
            v = rows_of(v_pool, layer, g, table[b], n + t, page)
            for h in range(g * group, (g + 1) * group):
                o, e = attention_rows(q[0, h, start:start + t].double(), k, v, full, scale, q.dtype)
                out[0, h, start:start + t], bound[0, h, start:start + t] = o, e
    return out, bound


def compact_reference(pool, table, base, src, page):
    """``pool`` with request b's rows base + src[b][i] moved to base + i, one after the other."""
    pool = pool.clone()
    for b, rows in enumerate(src):
        for i, s in enumerate(rows):
            a, z = base[b] + s, base[b] + i
            a = int(table[b][a // page]) * page + a % page
            z = int(table[b][z // page]) * page + z % page
            pool[:, :, :, z] = pool[:, :, :, a]
    return pool


def bounds_reference(k_pool, page):
    """[layers, H_kv, pages, 2, D] minima and maxima of every page's keys."""
    layers, _, heads, capacity, dim = k_pool.shape
    keys = k_pool.view(layers, heads, capacity // page, page, dim)
    return torch.stack([keys.amin(dim=3), keys.amax(dim=3)], dim=3)


def selection_reference(q, k_bounds, layer, table, lens, page, take):
    """[B, H_kv, take] logical pages, ascending, -1 past the last."""
    batch, hq = q.shape[:2]
    hkv = k_bounds.shape[1]
    group = hq // hkv
    chosen = np.full((batch, hkv, take), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        last = n // page
        ids = torch.from_numpy(table[b][:last].astype(np.int64)).to(q.device)
        for g in range(hkv):
            picked = list(range(last))
            if last >= take:
                lo, hi = k_bounds[layer, g, ids, 0].double(), k_bounds[layer, g, ids, 1].double()
                rows = q[b, g * group:(g + 1) * group, 0].double()
                side = torch.where(rows[:, None] >= 0, hi[None], lo[None])
                score = (rows[:, None] * side).sum(-1).float()
                score = torch.where(torch.isnan(score).any(0), math.inf, score.amax(0)).cpu().numpy()
                picked = sorted(np.lexsort((np.arange(last), -score))[:take - 1].tolist())
            chosen[b, g, :len(picked) + 1] = picked + [last]
    return chosen


def sparse_reference(q, k_pool, v_pool, layer, table, lens, chosen, page, scale):
    """[B, H_q, 1, D] rows (64 bits) and allowed errors over the chosen pages."""
    hq, hkv = q.shape[1], k_pool.shape[2]
    group = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, n in enumerate(lens):
        for g in range(hkv):
            picked = [int(p) for p in chosen[b, g] if p >= 0]
            there = (len(picked) - 1) * page + n % page + 1
            row = table[b][picked]
            k = rows_of(k_pool, layer, g, row, there, page)
            v = rows_of(v_pool, layer, g, row, there, page)
            sees = torch.ones((group, there), dtype=torch.bool, device=q.device)
            heads = slice(g * group, (g + 1) * group)
            out[b, heads, 0], bound[b, heads, 0] = attention_rows(q[b, heads, 0].double(), k, v, sees, scale, q.dtype)
    return out, bound
