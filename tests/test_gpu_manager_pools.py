"""The manager on the GPU with pools that the kernels do not take: bookkeeping still works, what
does not is refused before anything changes."""

from __future__ import annotations

import pytest
import torch

from hayate_b200 import PagedKVCacheManager

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.uint8], ids=str)
def test_copy_on_write_of_any_pool_type(dtype):
    """Pools of types that no kernel takes are shared, copied on write and imported all the same."""
    m = PagedKVCacheManager(2, 2, 12, 16 * 128, 128, 6, dtype, "cuda")
    torch.manual_seed(0)
    for pool in (m.k_cache, m.v_cache):
        pool.copy_(torch.randint(0, 200, pool.shape, device="cuda"))
    a = m.allocate()
    m.reserve(a, 300)
    a.length = 300
    before = m.snapshot(a)
    b = m.share(a, 290)
    m.begin_batch([a, b], 1)  # both write into the third page
    assert a.pages[:2] == b.pages[:2] and a.pages[2] != b.pages[2]
    for h, n in ((a, 300), (b, 290)):
        now = m.snapshot(h)
        assert torch.equal(now.k, before.k[:, :, :n]) and torch.equal(now.v, before.v[:, :, :n])
    forks = m.fork(a, 2)
    m.import_cache(forks[0], before)
    assert torch.equal(m.snapshot(forks[1]).k, before.k) and torch.equal(m.snapshot(forks[0]).v, before.v)


@pytest.mark.parametrize("dim, dtype, error", [(100, torch.bfloat16, RuntimeError), (264, torch.float32, RuntimeError),
                                               (128, torch.float64, TypeError)], ids=str)
def test_bounds_of_pools_that_the_kernel_does_not_take_are_refused_at_once(dim, dtype, error):
    """Not by the step that fills the first page: an untracked manager keeps working."""
    m = PagedKVCacheManager(1, 2, dim, 8 * 128, 128, 4, dtype, "cuda")
    with pytest.raises(error):
        m.track_page_bounds()
    assert m.k_bounds is None
    if dtype is not torch.float64:
        h = m.allocate()
        batch = m.begin_batch([h], 130)
        k = torch.ones(1, 2, 130, dim, dtype=dtype, device="cuda")
        batch.write_layer(0, k, k)
        m.commit_batch([h], 130)
        assert bool((m.snapshot(h).k == 1).all())
        m.check_device_errors()
