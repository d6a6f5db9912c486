"""Which pages the manager computes key bounds of, with the kernel call recorded (CPU)."""

from __future__ import annotations

import pytest
import torch

from hayate_b200 import PagedKVCacheManager, paged_cache


@pytest.fixture
def tracked(monkeypatch):
    m = PagedKVCacheManager(2, 1, 8, 40 * 128, 128, 12, torch.float32, "cpu")
    m.k_bounds = torch.zeros((2, 1, m.num_pages, 2, 8))
    calls = []
    monkeypatch.setattr(paged_cache.ops, "page_bounds",
                        lambda k, bounds, pages, size, layer=None, error_word=None: calls.append(pages.tolist()))
    return m, calls


def grown(m, length):
    h = m.allocate()
    m.reserve(h, length)
    h.length = length
    return h


def test_pages_that_requests_share_are_listed_once(tracked):
    """The first step after bounds are turned on: nine requests over one prefix of 5 full pages."""
    m, calls = tracked
    first = grown(m, 5 * 128 + 7)
    everyone = [first] + [m.share(first, 5 * 128) for _ in range(8)] + [grown(m, 300)]
    m.begin_batch(everyone, 1)
    assert len(calls) == 1 and sorted(calls[0]) == sorted(first.pages[:5] + everyone[-1].pages[:2])
    assert [h.bounded for h in everyone] == [5] * 9 + [2]
    m.commit_batch(everyone, 1)
    calls.clear()
    m.begin_batch(everyone, 1)
    assert calls == []
