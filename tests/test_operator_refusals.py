"""What the tree, move, bounds and page-selection entry points refuse on the host (no GPU:
every case returns before any CUDA call)."""

from __future__ import annotations

import pytest
import torch

from hayate_b200 import _lib, ops


def _call(name, defaults, **overrides):
    args = dict(defaults)
    assert set(overrides) <= set(args)
    args.update(overrides)
    lib = _lib.lib()
    rc = getattr(lib, name)(*args.values())
    return rc, lib.hyt_last_error().decode()


S2 = _lib.int64_array([0, 0])
TREE = dict(q=16, qs=S2, k=16, v=16, layers=2, layer=0, capacity=4096, table=16, stride=8, width=8, lens=16,
            q_start=16, q_len=16, mask=16, words=1, out=16, os=S2, batch=2, total=20, hq=32, hkv=8, dim=128,
            page=128, dtype=0, scale=0.1, max_query_len=10, ws=None, ws_bytes=0, err=None, stream=None)
COPY = dict(k=16, v=16, layers=2, heads=8, capacity=4096, dim=128, page=128, dtype=0, src=16, dst=16, count=1,
            err=None, stream=None)
COMPACT = dict(k=16, v=16, layers=2, heads=8, capacity=4096, dim=128, page=128, dtype=0, table=16, stride=8,
               width=8, base=16, src=16, start=16, batch=2, total=3, err=None, stream=None)
BOUNDS = dict(k=16, bounds=16, layers=2, first=0, n=2, heads=8, capacity=4096, dim=128, page=128, dtype=0,
              pages=16, count=1, err=None, stream=None)
SPARSE = dict(q=16, qs=S2, k=16, v=16, bounds=16, layers=2, layer=0, capacity=4096, table=16, stride=8, width=8,
              lens=16, out=16, os=S2, selected=16, batch=2, hq=32, hkv=8, dim=128, page=128, dtype=0, scale=0.1,
              num_pages=4, ws=None, ws_bytes=0, err=None, stream=None)


@pytest.mark.parametrize("bad, code, message", [
    (dict(q=None), -1, "null pointer"), (dict(q_len=None), -1, "null pointer"), (dict(batch=0), -1, "batch"),
    (dict(hq=30), -1, "multiple of num_kv_heads"), (dict(dtype=5), -1, "dtype"), (dict(layer=2), -1, "layer"),
    (dict(max_query_len=0), -1, "query_len"), (dict(total=0), -1, "total_tokens"),
    (dict(max_query_len=33), -1, "fewer bits"), (dict(width=9), -1, "page_table_width"),
    (dict(width=0), -1, "page_table_width"), (dict(scale=0.0), -1, "scale"), (dict(scale=-1.0), -1, "scale"),
    (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"),
    (dict(dim=12), -2, "head_dim"), (dict(dim=264), -2, "head_dim"), (dict(page=32), -2, "page_size"),
    (dict(page=96), -1, "power of two"), (dict(k=8), -1, "aligned"), (dict(), -4, "workspace"),
    (dict(ws=16, ws_bytes=100), -4, "workspace"), (dict(ws=8, ws_bytes=1 << 40), -4, "workspace"),
    (dict(ws=16, ws_bytes=1 << 40, hq=800, max_query_len=1 << 24, mask=None), -2, "rows"),
])
def test_tree_attention_refuses(bad, code, message):
    rc, said = _call("hyt_tree_attention", TREE, **bad)
    assert rc == code and message in said, said


@pytest.mark.parametrize("bad, code, message", [
    (dict(k=None), -1, "null pointer"), (dict(src=None), -1, "null pointer"), (dict(count=-1), -1, "count"),
    (dict(count=65536), -2, "65535"), (dict(page=3), -1, "power of two"), (dict(capacity=100), -1, "multiple"),
    (dict(dtype=9), -1, "dtype"), (dict(heads=0), -1, "heads"), (dict(layers=0), -1, "layer"),
])
def test_copy_pages_refuses(bad, code, message):
    rc, said = _call("hyt_copy_pages", COPY, **bad)
    assert rc == code and message in said, said


def test_moves_of_nothing_launch_nothing():
    assert _call("hyt_copy_pages", COPY, count=0, src=None, dst=None)[0] == 0
    assert _call("hyt_compact_rows", COMPACT, total=0, src=None)[0] == 0
    assert _call("hyt_page_bounds", BOUNDS, count=0, pages=None)[0] == 0


@pytest.mark.parametrize("bad, code, message", [
    (dict(v=None), -1, "null pointer"), (dict(base=None), -1, "null pointer"), (dict(batch=0), -1, "batch"),
    (dict(total=-1), -1, "total_rows"), (dict(width=9), -1, "page_table_width"), (dict(batch=65536), -2, "batch"),
    (dict(page=0), -1, "power of two"),
])
def test_compact_rows_refuses(bad, code, message):
    rc, said = _call("hyt_compact_rows", COMPACT, **bad)
    assert rc == code and message in said, said


@pytest.mark.parametrize("bad, code, message", [
    (dict(bounds=None), -1, "null pointer"), (dict(pages=None), -1, "null pointer"), (dict(first=1), -1, "layers"),
    (dict(n=0), -1, "layers"), (dict(dim=20), -2, "head_dim"), (dict(bounds=24), -1, "aligned"),
    (dict(count=-2), -1, "count"), (dict(count=70000), -2, "65535"),
])
def test_page_bounds_refuses(bad, code, message):
    rc, said = _call("hyt_page_bounds", BOUNDS, **bad)
    assert rc == code and message in said, said


@pytest.mark.parametrize("bad, code, message", [
    (dict(q=None), -1, "null pointer"), (dict(selected=None), -1, "null pointer"), (dict(num_pages=0), -1, "num_pages"),
    (dict(width=9), -1, "page_table_width"), (dict(stride=20000, width=20000), -2, "8192"),
    (dict(scale=0.0), -1, "scale"), (dict(dim=20), -2, "head_dim"), (dict(bounds=24), -1, "aligned"),
    (dict(), -4, "workspace"), (dict(page=32), -2, "page_size"),
    (dict(num_pages=1 << 28), -2, "too large"),
])
def test_sparse_attention_refuses(bad, code, message):
    rc, said = _call("hyt_sparse_attention", SPARSE, **bad)
    assert rc == code and message in said, said


def test_workspace_sizes():
    tree = ops.tree_workspace_bytes(16, 32, 8, 128, torch.bfloat16)
    assert tree > 0 and tree % 256 == 0
    assert ops.sparse_workspace_bytes(4, 32, 8, 128, 16, torch.bfloat16) >= 4 * 8 * 16 * 4
    lib = _lib.lib()
    assert lib.hyt_tree_workspace_bytes(0, 32, 8, 128, 0) == 0
    assert lib.hyt_sparse_workspace_bytes(0, 32, 8, 128, 4, 0) == 0


def test_wrappers_run_on_cuda_tensors_only():
    pool = torch.zeros(1, 1, 2, 256, 64)
    ids = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.tree_attention(q, pool, pool, 0, ids[None], ids, ids, ids, ids[None], 128, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.copy_pages(pool, pool, ids, ids, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.compact_rows(pool, pool, ids[None], ids, ids, ids, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.page_bounds(pool, torch.zeros(1, 2, 2, 2, 64), ids, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.sparse_attention(q, pool, pool, torch.zeros(1, 2, 2, 2, 64), 0, ids[None], ids, 128, 1)
