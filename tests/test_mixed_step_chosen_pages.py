"""Engine ticks over chosen pages (``DecodeGraphs(engine, num_pages=n)``): a decoding request
attends n pages per KV head in every tick, whatever the other requests of the tick do."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from hayate_b200 import PagedKVCacheManager, mixed_step
from hayate_b200.mixed_step import DecodeGraphs, mixed_generate


class Request(SimpleNamespace):
    def __init__(self, prompt_tokens):
        super().__init__(prompt="", prompt_tokens=list(prompt_tokens), tokens=[], is_prefill=True, is_completed=False,
                         paged_cache=None, kv_cache=None)


class Engine:
    """What ``mixed_generate`` uses of an engine; greedy, with the scores of every sampled row kept."""

    def __init__(self, model, manager, chunk=128):
        self.model, self.paged_cache, self.prefill_chunk_size = model, manager, chunk
        self.max_position_embeddings = 4096
        self.requests, self.scores = [], []
        self.scheduler = self.tokenizer = self.sampler = self

    current_batch = ()

    def tick(self):
        return list(self.requests)

    def sample(self, logits, requests):
        self.scores.append([(id(r), row.float().cpu()) for r, row in zip(requests, logits)])
        return logits.argmax(-1)

    def finalize(self, request, token):
        request.tokens.append(int(token))

    def release_request_cache(self, request):
        self.paged_cache.release(request.paged_cache)

    def _store_prompt_prefix(self, request):
        pass


def test_every_tick_passes_the_page_count_to_decoding_requests(monkeypatch):
    """Ticks that no graph serves: decoding rows run with ``num_pages``, prompt chunks without."""
    manager = PagedKVCacheManager(1, 1, 8, 32 * 128, 128, 24, torch.float32, "cpu")
    engine = Engine(None, manager, chunk=4)
    passes = []

    def forward(model, token_ids, batch, rows, num_pages=None):
        passes.append((batch.layout.query_lens, num_pages))
        return torch.zeros(len(rows), 16)

    monkeypatch.setattr(mixed_step, "packed_forward", forward)
    graphs = DecodeGraphs.__new__(DecodeGraphs)
    graphs.engine, graphs.num_pages, graphs.sizes, graphs.kv_buckets = engine, 2, [], []  # no bucket fits
    engine.requests = [Request(range(3)), Request(range(3))]
    mixed_generate(engine, graphs)
    assert passes == [([3, 3], None)]
    passes.clear()
    mixed_generate(engine, graphs)                     # decoding alone
    assert passes == [([1, 1], 2)]
    passes.clear()
    engine.requests += [Request(range(9)) for _ in range(10)]
    mixed_generate(engine, graphs)                     # beside ten prompts
    assert sorted(passes, key=str) == sorted([([1, 1], 2), ([4] * 8, None), ([4] * 2, None)], key=str)
    assert [len(r.tokens) for r in engine.requests] == [3, 3] + [0] * 10
    passes.clear()
    graphs.num_pages = None                            # the whole context: one pass, as ever
    mixed_generate(engine, graphs)
    assert passes == [([4] * 8 + [1, 1], None), ([4] * 2, None)]


def test_a_graph_serves_the_decoding_requests_of_a_mixed_tick(monkeypatch):
    manager = PagedKVCacheManager(1, 1, 8, 32 * 128, 128, 8, torch.float32, "cpu")
    engine = Engine(None, manager, chunk=4)
    passes, served = [], []

    def forward(model, token_ids, batch, rows, num_pages=None):
        passes.append(batch.layout.query_lens)
        return torch.zeros(len(rows), 16)

    monkeypatch.setattr(mixed_step, "packed_forward", forward)
    graphs = SimpleNamespace(num_pages=2, step=lambda decode: served.append(list(decode)) or True)
    engine.requests = [Request(range(3))]
    mixed_generate(engine, graphs)
    engine.requests.append(Request(range(9)))
    passes.clear()
    assert mixed_generate(engine, graphs)
    assert served == [[engine.requests[0]]] and passes == [[4]]


@pytest.mark.gpu
def test_scores_do_not_change_when_a_prompt_joins():
    """One request decodes over 2 of its pages; another's prompt arrives and is read in chunks
    beside it. Its scores are those of the run without the other, bit for bit."""
    from test_gpu_speculative import BF16, LAYERS, tiny_model

    model = tiny_model()
    gen = torch.Generator().manual_seed(3)
    prompt, other = [torch.randint(0, 500, (n,), generator=gen).tolist() for n in (1500, 1200)]
    runs = []
    for joins in (False, True):
        manager = PagedKVCacheManager(LAYERS, 8, 128, 40 * 128, 128, 4, BF16, "cuda")
        engine = Engine(model, manager)
        graphs = DecodeGraphs(engine, sizes=(4,), kv_buckets=(2048,), num_pages=2)
        first = Request(prompt)
        engine.requests = [first]
        with torch.inference_mode():
            while first.is_prefill:
                mixed_generate(engine, graphs)
            for tick in range(16):
                if joins and tick == 4:
                    engine.requests.append(Request(other))
                mixed_generate(engine, graphs)
        manager.check_device_errors()
        assert graphs.graphs
        if joins:
            assert not engine.requests[1].is_prefill and len(engine.requests[1].tokens) > 1
        runs.append([row for step in engine.scores for who, row in step if who == id(first)])
    assert len(runs[0]) == len(runs[1]) == 17
    same = 1 + 4 + 10  # then the other decodes too, and its rows share the launches
    assert all(torch.equal(a, b) for a, b in zip(runs[0][:same], runs[1][:same]))
