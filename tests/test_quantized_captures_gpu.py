"""Captured decode steps over a cache in 8 bits: captured again where their kernels would be others, and only there."""
import pytest
import torch

from conftest import TINY, random_tokens, rel_err

pytestmark = pytest.mark.gpu


def _engine(use_graphs, dtype="float32", **sizes):
    from rust_inference_b200 import config_from_dict
    from rust_inference_b200.engine.engine import Engine
    config = config_from_dict(dict(TINY["A"], max_position_embeddings=16384))
    return Engine.from_random(config, seed=5, std=0.08, dtype=dtype, cache_dtype="int8", use_graphs=use_graphs,
                              **dict(dict(max_tokens=32768, n_slots=4), **sizes))


def _decode(eng, lengths, steps, seed=0):
    """Logits of single tokens behind prompts of so many; and which capture each step ran (None: none)."""
    slots = [eng.alloc_slot() for _ in lengths]
    eng.step(slots, [random_tokens(n, 264, seed=seed + b) for b, n in enumerate(lengths)], "none")
    rows, graphs = [], []
    for i in range(steps):
        rows.append(eng.step(slots, [[(7 * i + 11 * b + seed) % 264] for b in range(len(lengths))], "last").cpu())
        if eng.use_graphs:
            graphs.append(eng.decode_graph(len(lengths)).graph)
    for s in slots:
        eng.free_slot(s)
    eng.check_device_status()
    return torch.stack(rows), graphs


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths", [[8185], [4090, 300, 4088]])
def test_from_clusters_to_runs_of_pages(lengths, dtype):
    """The longest sequence grows past what clusters of blocks take: the step is captured with the other kernel, and its scratch
    and counters are as that one needs them, for the steps after it as well."""
    captured, plain = _engine(True, dtype), _engine(False, dtype)
    got, graphs = _decode(captured, lengths, 24)
    want, _ = _decode(plain, lengths, 24)
    kinds = [g for i, g in enumerate(graphs) if g is not None and (i == 0 or g is not graphs[i - 1])]
    assert len(kinds) == 2, len(kinds)
    assert rel_err(got, want) <= (1e-3 if dtype == "float32" else 4e-2)


def test_no_capture_while_the_kernels_stay(monkeypatch):
    from rust_inference_b200.engine import graphs as module
    monkeypatch.setattr(module, "FIRST_REACH", 16)
    eng = _engine(True)
    _, graphs = _decode(eng, [5], 140)
    assert eng.decode_graph(1).reach == 256
    assert len({id(g) for g in graphs if g is not None}) == 1


def test_back_to_short_sequences():
    """After a long sequence a short one has the short one's kernels again."""
    eng = _engine(True)
    short, first = _decode(eng, [40], 8)
    _, long = _decode(eng, [9000], 8, seed=1)
    again, last = _decode(eng, [40], 8)
    one = eng.decode_graph(1)
    assert first[-1] is not long[-1] and last[-1] is not long[-1] and one.reach == 1024
    assert torch.equal(short, again)
