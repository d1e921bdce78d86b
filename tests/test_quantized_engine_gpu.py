"""A whole model over a cache in 8 bits, and scoring, through the public entry points."""
import json
import math
import os
import subprocess
import sys

import pytest
import torch

import plain_impl
import plain_quantized
from conftest import TOL, random_tokens, rel_err

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _engine(model, dtype, cache_dtype="int8", **kw):
    from rust_inference_b200.engine.engine import Engine
    kw.setdefault("max_tokens", 4096)
    return Engine.from_pretrained(model.folder, dtype=dtype, cache_dtype=cache_dtype, **kw)


def _plain_over_8_bits(model, tokens, monkeypatch):
    """The plain implementation with keys and values as a cache in 8 bits holds them, written in one step."""
    n_kv = plain_impl.resolve_config(model.cfg)["num_key_value_heads"]

    def held(x, store_dtype):
        if x.dim() != 3 or x.shape[1] != n_kv:
            return x
        pages = -(-x.shape[0] // 64)
        codes, scales = torch.zeros(pages, n_kv, 64, x.shape[2], dtype=torch.int8), torch.zeros(pages, n_kv, 4)
        plain_quantized.put(codes, scales, x.float(), 0, list(range(pages)))
        return plain_quantized.values(codes, scales, list(range(pages)), x.shape[0])

    with monkeypatch.context() as m:
        m.setattr(plain_impl, "stored", held)
        return model.plain_logits(tokens)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
def test_a_prompt(name, dtype, model_factory, monkeypatch):
    """float32: a key or value near the middle between two codes may round the other way after a float32 sum in another
    order, one step of 1/127 of its block's largest number in about one of 1e5 of them.  bfloat16: its own rounding moves a key by
    more than a step of its code, so that its codes are rounded apart from the plain model's: each of the two is as far from the
    model without codes as that costs, and they may lie on opposite sides."""
    model = model_factory(name, std=0.08)
    toks = random_tokens(150, model.cfg["vocab_size"], seed=4)
    want = _plain_over_8_bits(model, toks, monkeypatch)
    eng = _engine(model, dtype)
    slot = eng.alloc_slot()
    got = eng.step([slot], [toks], "all").cpu()
    apart = 2 * rel_err(want, model.plain_logits(toks))
    assert rel_err(got, want) <= (2e-3 if dtype == "float32" else TOL[dtype] + apart)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "E"])
def test_decoding_with_graphs_and_without(name, dtype, model_factory, monkeypatch):
    """Token by token behind a prompt: both stay as near the plain model as 8 bits allow (three times what the plain model's own
    keys and values in 8 bits cost), and as near each other as two draws of the rounding (sums of products that are cut over K are
    added in any order, and codes follow them)."""
    model = model_factory(name, std=0.08)
    toks = [random_tokens(120, model.cfg["vocab_size"], seed=5 + b) for b in range(2)]
    engines = [_engine(model, dtype, use_graphs=g) for g in (True, False)]
    out = []
    for eng in engines:
        slots = [eng.alloc_slot() for _ in toks]
        eng.step(slots, [toks[0][:37], toks[1][:64]], "none")
        rows = [eng.step(slots, [[toks[0][37 + i]], [toks[1][64 + i]]], "last").cpu() for i in range(50)]
        out.append(torch.stack(rows))
    for b, first in ((0, 37), (1, 64)):
        want = model.plain_logits(toks[b][:first + 50])
        noise = rel_err(_plain_over_8_bits(model, toks[b][:first + 50], monkeypatch), want)
        assert rel_err(out[0][:, b], out[1][:, b]) <= 2 * noise
        assert rel_err(out[0][:, b], want[first:]) <= 3 * noise + (0 if dtype == "float32" else TOL[dtype])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_captured_step_that_is_outgrown(dtype, model_factory, monkeypatch):
    """Captured steps choose their launches for sequences of so many keys, and are captured again when one has more: what comes out
    stays what an engine without captured steps computes (bounds as above), before, at and after the change."""
    from rust_inference_b200.engine import graphs
    monkeypatch.setattr(graphs, "FIRST_REACH", 16)
    model = model_factory("A", std=0.08)
    toks = random_tokens(150, model.cfg["vocab_size"], seed=9)
    engines = [_engine(model, dtype, use_graphs=g) for g in (True, False)]
    out, reached = [], []
    for eng in engines:
        slot = eng.alloc_slot()
        eng.step([slot], [toks[:5]], "none")
        rows = []
        for t in toks[5:]:
            rows.append(eng.step([slot], [[t]], "last").cpu())
            if eng.use_graphs:
                reached.append(eng.decode_graph(1).reach)
        out.append(torch.cat(rows))
    assert reached[0] == 16 and reached[11] == 32 and reached[-1] == 256 and eng is not engines[0]
    want = model.plain_logits(toks)
    noise = rel_err(_plain_over_8_bits(model, toks, monkeypatch), want)
    assert rel_err(out[0], out[1]) <= 2 * noise
    assert rel_err(out[0], want[5:]) <= 3 * noise + (0 if dtype == "float32" else TOL[dtype])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_pages_that_were_used_before(dtype, model_factory):
    model = model_factory("A", std=0.08)
    toks = random_tokens(90, model.cfg["vocab_size"], seed=7)
    fresh, used = _engine(model, dtype, max_tokens=256, n_slots=2), _engine(model, dtype, max_tokens=256, n_slots=2)
    for seed in range(3):
        s = used.alloc_slot()
        used.step([s], [random_tokens(200, model.cfg["vocab_size"], seed=20 + seed)], "none")
        used.free_slot(s)
    got = []
    for eng in (fresh, used):
        s = eng.alloc_slot()
        parts = [eng.step([s], [toks[:50]], "all").cpu()] + [eng.step([s], [[t]], "last").cpu() for t in toks[50:]]
        got.append(torch.cat(parts))
    assert torch.equal(*got)


def test_model_entry_points(model_factory):
    from rust_inference_b200 import Model, SamplerConfig
    model = model_factory("E", std=0.08)
    prompts = [random_tokens(n, model.cfg["vocab_size"], seed=30 + n) for n in (70, 3, 20)]
    wide, small = (Model.load(model.folder, cache_dtype=c, max_tokens_in_cache=2048) for c in (None, "int8"))
    a, b = wide.memory(), small.memory()
    assert b["cache_bytes"] * 2 <= a["cache_bytes"] * 1.02 and b["cache_bytes_per_position"] * 2 <= a["cache_bytes_per_position"] * 1.02
    results = small.generate(prompts, 12, SamplerConfig.plain(temperature=0.0), stop_ids=())
    assert [len(r.tokens) for r in results] == [12] * 3
    again = small.generate(prompts, 12, SamplerConfig.plain(temperature=0.0), stop_ids=())
    assert [r.tokens for r in again] == [r.tokens for r in results]


def test_decoders_of_mixed_layers(tmp_path):
    """A design whose attention lies beside a recurrence, with values of a size of their own: near the model over its usual cache."""
    from lulisun_models import CONFIGS
    from rust_inference_b200 import config_from_dict
    from rust_inference_b200.engine.engine import Engine
    cfg = config_from_dict(CONFIGS["A"])
    toks = random_tokens(100, 64, seed=9)
    out = []
    for cache in (None, "int8"):
        eng = Engine.from_random(cfg, seed=3, std=0.08, dtype="float32", max_tokens=1024, cache_dtype=cache)
        s = eng.alloc_slot()
        first = eng.step([s], [toks[:80]], "all").cpu()
        out.append(torch.cat([first] + [eng.step([s], [[t]], "last").cpu() for t in toks[80:]]))
    assert 1e-6 < rel_err(out[1], out[0]) < 0.1


def test_what_is_refused(model_factory):
    from vadodra_models import CONFIGS
    from rust_inference_b200 import config_from_dict
    from rust_inference_b200.cache.pager import CacheError
    from rust_inference_b200.engine.engine import Engine
    model = model_factory("A", std=0.08)
    with pytest.raises(ValueError, match="cache_dtype"):
        _engine(model, "bfloat16", cache_dtype="int4")
    with pytest.raises(CacheError, match="8 bits"):
        Engine.from_random(config_from_dict(CONFIGS["A"]), dtype="bfloat16", max_tokens=256, cache_dtype="int8")


@pytest.mark.parametrize("cache_dtype", [None, "int8"])
def test_score(cache_dtype, model_factory, monkeypatch):
    from rust_inference_b200 import Model, api
    model = model_factory("B", std=0.08)
    toks = random_tokens(90, model.cfg["vocab_size"], seed=11)
    lib = Model.load(model.folder, dtype="float32", cache_dtype=cache_dtype, max_tokens_in_cache=1024)
    found = lib.score(toks, top=3)
    want = _plain_over_8_bits(model, toks, monkeypatch) if cache_dtype else model.plain_logits(toks)
    logp = torch.log_softmax(want.double(), dim=1)
    # logits within this of the plain ones: each log probability within twice that, entropies likewise
    slack = 2 * float(want.abs().max()) * (2e-3 if cache_dtype else TOL["float32"])
    for n in range(89):
        assert abs(found.logprobs[n] - float(logp[n, toks[n + 1]])) <= slack
        assert abs(found.entropies[n] + float((logp[n].exp() * logp[n]).sum())) <= slack * 8
        assert [i for i, _ in found.top[n]] and abs(found.top[n][0][1] - float(logp[n].max())) <= slack
    assert found.perplexity == pytest.approx(math.exp(-sum(found.logprobs) / 89))
    # in pieces of a few tokens: the same up to the order of sums, and up to what writing in pieces costs
    monkeypatch.setattr(api, "SCORE_LOGITS", 7 * model.cfg["vocab_size"])
    pieces = lib.score(toks)
    assert pieces.top is None
    assert max(abs(a - b) for a, b in zip(pieces.logprobs, found.logprobs)) <= slack * (1 if cache_dtype is None else 50)
    assert lib.engine.cache.pager.free_slot_count() == lib.engine.cache.n_slots
    for bad in ([], [5], [5, model.cfg["vocab_size"]], [5, -1]):
        with pytest.raises(ValueError):
            lib.score(bad)


def test_the_command_line(model_factory):
    model = model_factory("A", std=0.08)
    toks = random_tokens(20, model.cfg["vocab_size"], seed=13)
    args = [sys.executable, os.path.join(ROOT, "bin", "gguf-infer"), "--model", model.folder, "--prompt", ",".join(map(str, toks)),
            "--dtype", "float32", "--cache-dtype", "int8"]
    scored = subprocess.run(args + ["--score", "2"], capture_output=True, text=True, timeout=600)
    assert scored.returncode == 0, scored.stderr[-2000:]
    lines = [l.split() for l in scored.stdout.splitlines()]
    assert [int(l[0]) for l in lines] == toks[1:] and all(len(l) == 5 and ":" in l[3] for l in lines)
    assert "19 tokens, perplexity" in scored.stderr
    run = subprocess.run(args + ["-n", "5", "-t", "0", "--stop-ids", "", "--bench"], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and len(run.stdout.split()) == 5, run.stderr[-2000:]
    assert json.loads([l for l in run.stderr.splitlines() if l.startswith("{")][0])["cache_bytes"] > 0
