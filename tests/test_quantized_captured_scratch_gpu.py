"""Captured decode steps over a cache in 8 bits that go by way of scratch pages (head sizes that the direct kernel does not have):
the captured launches hold for every length up to the longest, over page edges, after other sequences, and in pools of any size."""
import pytest
import torch

from conftest import random_tokens, rel_err

pytestmark = pytest.mark.gpu


def _run(eng, toks, first, steps):
    slots = [eng.alloc_slot() for _ in toks]
    eng.step(slots, [t[:n] for t, n in zip(toks, first)], "none")
    rows = [eng.step(slots, [[t[n + i]] for t, n in zip(toks, first)], "last").cpu() for i in range(steps)]
    for s in slots:
        eng.free_slot(s)
    return torch.stack(rows)


@pytest.mark.parametrize("max_tokens", [512, 16384])          # the pool's pages, and each sequence's own, are the fewer ones
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name, first, steps", [("C", [60, 1], 60), ("D", [120, 30], 110), ("D", [5], 200)])
def test_over_page_edges(name, first, steps, dtype, max_tokens, model_factory):
    from rust_inference_b200.engine.engine import Engine
    model = model_factory(name, std=0.08)
    engines = [Engine.from_pretrained(model.folder, dtype=dtype, cache_dtype="int8", max_tokens=max_tokens, use_graphs=g) for g in (True, False)]
    toks = [random_tokens(n + steps, model.cfg["vocab_size"], seed=40 + n) for n in first]
    got, want = (_run(eng, toks, first, steps) for eng in engines)
    own = len(first) * engines[0].cache.page_table.shape[1]
    view = engines[0].decode_graph(len(first)).workspace._views[("readback_k", torch.float32 if dtype == "float32" else torch.bfloat16)][1]
    assert view.shape[0] == min(own, engines[0].cache.n_pages)
    bound = 1e-3 if dtype == "float32" else 4e-2
    assert rel_err(got, want) <= bound
    assert rel_err(_run(engines[0], toks, first, steps), got) <= bound           # over pages that have been used
    engines[0].check_device_status()
