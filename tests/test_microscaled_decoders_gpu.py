"""Decoders with matrices in microscaled 4 bits beside the same decoders with those numbers as plain weights, whose products are given the same rows
rounded to 8 bits: what the two differ by is rounding alone, so that a lost bias, a wrong head or a matrix in the wrong place shows."""
import importlib

import pytest
import torch

from conftest import TOL, make_model, random_tokens, rel_err

pytestmark = pytest.mark.gpu


def engines(folder, dtype):
    from rust_inference_b200.engine.engine import Engine
    kw = dict(dtype=dtype, max_tokens=1024, use_graphs=False)
    held = Engine.from_pretrained(folder, weights_dtype="mxfp4", **kw)
    return held, Engine.from_pretrained(folder, **kw)


def numbers_in_eight_bits(eng):
    """Of a token, over all layers: what its products' rows hold."""
    from rust_inference_b200.kernels import microscaled
    parts = [p for _, p in eng.model._named_parts() if p.weights_dtype is not None]
    names = ("w_qkv", "w_o", "w_gate", "w_down") if any(hasattr(p, "w_gate") for p in parts) else ("w_qkv", "w_o", "w_up", "w_down")
    mats = [getattr(p, n, None) for p in parts for n in names]
    return sum(m.k for m in mats if type(m) is microscaled.Matrix)


def round_rows(eng, monkeypatch):
    """The engine's products of the parts that can hold 4 bits take their rows by way of 8."""
    from rust_inference_b200.kernels import linear, microscaled
    takers = {id(w) for _, p in eng.model._named_parts() if p.holds_microscaled for w in vars(p).values() if type(w) is linear.Weight}
    assert takers

    def patched(fn):
        def call(x, w, *args, **kw):
            if id(w) in takers:
                x = microscaled.values(microscaled.quantize(x), x.dtype)
            return fn(x, w, *args, **kw)
        return call

    for name in ("project", "logits", "into_residual", "gated", "activated", "accumulate_split"):
        monkeypatch.setattr(linear, name, patched(getattr(linear, name)))


def run(eng, toks, first):
    """Logits of every position: the first so many tokens in one step, the others one by one."""
    slot = eng.alloc_slot()
    out = [eng.step([slot], [toks[:first]], "all").cpu()]
    out += [eng.step([slot], [[t]], "last").cpu() for t in toks[first:]]
    eng.free_slot(slot)
    eng.check_device_status()
    return torch.cat(out)


def compare(folder, dtype, monkeypatch):
    held, usual = engines(folder, dtype)
    vocab = held.model.spec.vocab_size
    prompts = [random_tokens(7, vocab, seed=s) for s in range(8)]
    got = [run(held, p, 5) for p in prompts]
    unrounded = [run(usual, p, 5) for p in prompts]
    with monkeypatch.context() as m:
        round_rows(usual, m)
        want = [run(usual, p, 5) for p in prompts]
    if dtype == "float32":
        # one number of some 10^5 lies so near to the middle of two that sums in another order put it on the other side, which changes what comes after
        # it: prompts without one agree as any two float32 runs do
        apart = 7 * numbers_in_eight_bits(held) * 1e-5
        assert apart < 0.6
        near = sum(bool(((g - w).abs().amax(dim=1) <= TOL[dtype] * w.abs().amax(dim=1)).all()) for g, w in zip(got, want))
        assert near >= 2, near                     # (each with a chance of 0.54 at least: seven of eight apart once in a hundred such tests at most)
    for g, w, u in zip(got, want, unrounded):
        # either run is as far from the one without 8 bits as these cost
        assert rel_err(g, w) <= TOL[dtype] + 2.0 * rel_err(w, u)
        assert rel_err(w, u) > 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("family", ["vadodra", "redodra"])
def test_decoders_that_do_not_route(family, name, dtype, tmp_path, monkeypatch):
    from rust_inference_b200 import Model, config_from_dict
    cfg = config_from_dict(importlib.import_module(family + "_models").CONFIGS[name])
    m = Model.random(cfg, seed=3, std=0.05, norm_std=0.2, dtype="float32", weights_dtype="mxfp4", max_tokens_in_cache=512)
    compare(m.save_safetensors(str(tmp_path / "copy")), dtype, monkeypatch)


# hidden and feed-forward sizes that are no whole eights (products in bfloat16 then run on other kernels, and leave no sums for the heads), heads of 20 and
# 10 channels, biases
ODD = {"hidden_size": 100, "intermediate_size": 172, "num_attention_heads": 5, "num_key_value_heads": 1, "head_dim": 20}
ODDER = {"hidden_size": 77, "intermediate_size": 131, "num_attention_heads": 3, "num_key_value_heads": 3, "head_dim": 10}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("base,sizes", [("A", ODD), ("B", ODD), ("B", ODDER), ("E", ODDER)])
def test_sizes_that_are_no_whole_eights(base, sizes, dtype, tmp_path, monkeypatch):
    from rust_inference_b200 import Model
    model = make_model(tmp_path, base, std=0.08, overrides=sizes, matrix_dtype=torch.float32)
    folder = Model.load(model.folder, dtype="float32", weights_dtype="mxfp4").save_safetensors(str(tmp_path / "copy"))
    compare(folder, dtype, monkeypatch)
