"""Scratch of steps that bring keys and values of a cache in 8 bits to another type: as large as what the step sees, and the same
results as over the whole pool's pages."""
import math

import pytest
import torch

from conftest import random_tokens
from test_quantized_cache_gpu import DEV, Step

pytestmark = pytest.mark.gpu


def _step(runs, n_kv, hd, v_hd=None, spare=0):
    step = Step(runs + [(64 * spare, 0)], n_kv, hd, v_hd)       # a sequence that is not in the step: pages that nobody sees
    step.arrays([(s + n, 0) for s, n in runs])
    step.fill()
    step.slots = step.slots[:len(runs)]
    step.arrays(runs)
    return step


@pytest.mark.parametrize("limits", [{}, {"window": 50}, {"chunk": 48}], ids=str)
@pytest.mark.parametrize("runs", [[(0, 130), (37, 90), (0, 1), (200, 17)], [(0, 65)], [(300, 1), (64, 1), (5, 1)]])
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype, forms", [
    (8, 2, 64, torch.bfloat16, {}), (28, 4, 128, torch.bfloat16, {}), (6, 2, 24, torch.bfloat16, {}), (4, 1, 96, torch.float32, {}),
    (8, 2, 64, torch.bfloat16, {"softcap": 20.0}), (8, 2, 128, torch.float32, {"softcap": 20.0})])
def test_as_large_as_the_step(n_heads, n_kv, hd, dtype, forms, runs, limits):
    from rust_inference_b200.kernels import attention
    step = _step(runs, n_kv, hd, spare=400)
    assert step.layer.k.shape[0] > 400
    small = _step(runs, n_kv, hd)                                # the same sequences in a pool that is hardly larger than they are
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    found = []
    for one in (step, small):
        ctx = one.context(dtype)
        out = torch.full_like(q, math.nan)
        attention.attention(q, one.layer, out, ctx, n_heads=n_heads, n_kv_heads=n_kv, head_dim=hd, scale=hd ** -0.5, **forms, **limits)
        torch.cuda.synchronize()
        found.append(out)
        held = {name: view.shape[0] for (name, _), (_, view) in ctx.workspace._views.items() if name[:8] in ("widened_", "readback") and "fact" not in name}
        longest = one.page_table.shape[1] if ctx.all_single else -(-one.max_len // 64)
        assert all(n == min(len(runs) * longest, one.layer.k.shape[0]) for n in held.values())
        if forms or hd not in (64, 128):
            assert held
    assert torch.equal(*found)


def test_a_models_prompt_takes_scratch_for_its_own_pages(model_factory):
    from rust_inference_b200 import Model
    model = model_factory("E", std=0.08)
    lib = Model.load(model.folder, cache_dtype="int8", max_tokens_in_cache=1 << 20)
    eng = lib.engine
    slot = eng.alloc_slot()
    eng.step([slot], [random_tokens(1000, model.cfg["vocab_size"], seed=1)], "last")
    layer = eng.cache.layer(0)
    taken = {name: flat.numel() * flat.element_size() for (name, _), flat in eng.workspace._flat.items() if "widened" in name or "readback" in name}
    assert 0 < sum(taken.values()) < layer.k.numel() // 100
    memory = lib.memory()
    assert memory["cache_scratch_bytes"] == 2 * 2 * layer.k.numel()
    assert Model.load(model.folder, max_tokens_in_cache=1024).memory()["cache_scratch_bytes"] == 0


def test_outputs_of_other_shapes_are_refused():
    from rust_inference_b200.kernels import quantized_cache as qc
    from rust_inference_b200.kernels.ops import KernelError
    step = _step([(100, 1), (30, 1)], 2, 64, spare=10)
    pages = {n: [torch.zeros(n, 2, 64, 64, device=DEV, dtype=torch.float16) for _ in range(2)] for n in (2, 4, 5)}
    factors = torch.zeros(2, 2, 2, device=DEV)
    where = (step.page_table, step.seq_slot, step.seq_start, step.seq_len)

    def both(n, **how):
        qc.widen(step.layer, *pages[n], factors, *where, max_len=101, **how)
        qc.read(step.layer, *[p.float() for p in pages[n]], *where, max_len=101, **how)

    both(4, out_pages=2)
    for n, how in ((5, dict(out_pages=2)), (2, dict(out_pages=1)), (4, {})):
        with pytest.raises(KernelError):
            qc.widen(step.layer, *pages[n], factors, *where, max_len=101, **how)
        with pytest.raises(KernelError):
            qc.read(step.layer, *[p.float() for p in pages[n]], *where, max_len=101, **how)
