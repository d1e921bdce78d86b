"""What attention over a cache in 8 bits keeps of a step follows the step: arrays, scratch and sizes that are put in the place of
others."""
import math

import pytest
import torch

from test_quantized_cache_gpu import DEV, Step

pytestmark = pytest.mark.gpu

CALL = dict(n_heads=4, n_kv_heads=2, head_dim=64, scale=0.125)


def _attend(step, ctx, q):
    from rust_inference_b200.kernels import attention
    out = torch.full_like(q, math.nan)
    attention.attention(q, step.layer, out, ctx, **CALL)
    return out


def _moved(runs, new):
    """A step's context after a call for `runs`, then holding the arrays of `new`, and a fresh one of those."""
    step = Step([(max(a[0] + a[1], b[0] + b[1]), 0) for a, b in zip(runs, new)], 2, 64)
    step.fill()
    step.arrays(runs)
    ctx = step.context(torch.float32)
    _attend(step, ctx, torch.randn(step.n_tokens, 4 * 64, device=DEV))
    step.arrays(new)
    return step, ctx, step.context(torch.float32)


@pytest.mark.parametrize("runs, new", [([(70, 1), (130, 1)], [(71, 1), (20, 1)]), ([(70, 1), (130, 1)], [(60, 12), (129, 3)]),
                                       ([(64, 5), (3, 2)], [(100, 1), (90, 1)])])
def test_arrays_in_the_place_of_others(runs, new):
    step, ctx, fresh = _moved(runs, new)
    for name in ("n_tokens", "token_ids", "token_pos", "token_seq", "seq_start", "seq_len", "cu_seqlens", "max_new", "max_len", "all_single"):
        setattr(ctx, name, getattr(fresh, name))
    q = torch.randn(step.n_tokens, 4 * 64, device=DEV)
    assert torch.equal(_attend(step, ctx, q), _attend(step, fresh, q))


@pytest.mark.parametrize("name", ["page_table", "seq_slot"])
def test_pages_and_slots_in_the_place_of_others(name):
    """The two sequences change places."""
    step, ctx, fresh = _moved([(70, 1), (70, 1)], [(70, 1), (70, 1)])
    if name == "seq_slot":
        changed = step.seq_slot.flip(0).contiguous()
    else:
        changed = step.page_table.clone()
        changed[step.slots[0]], changed[step.slots[1]] = step.page_table[step.slots[1]], step.page_table[step.slots[0]]
    setattr(ctx, name, changed)
    q = torch.randn(2, 4 * 64, device=DEV)
    assert torch.equal(_attend(step, ctx, q), _attend(step, fresh, q.flip(0).contiguous()).flip(0))


def test_scratch_in_the_place_of_other():
    from rust_inference_b200.engine.context import Workspace
    from rust_inference_b200.kernels import quantized_cache as qc
    step, ctx, _ = _moved([(300, 1), (130, 1)], [(300, 1), (130, 1)])
    first = qc.step_of(ctx, 4, 2, 64)
    assert qc.step_of(ctx, 4, 2, 64) is first                  # looked at once while nothing changes
    ctx.workspace = Workspace(DEV)
    second = qc.step_of(ctx, 4, 2, 64)
    assert second is not first and second.native != first.native and ctx.workspace.bytes() > 0


def test_sizes_in_the_place_of_others():
    """Which kernels a step runs is asked of the step as it is."""
    from types import SimpleNamespace
    from rust_inference_b200.kernels import attention
    ctx = SimpleNamespace(n_seqs=64, max_new=1, page_table=torch.zeros(64, 8), extras={})
    assert attention.reads_codes(ctx, False, 32, 8)
    ctx.max_new = 100
    assert not attention.reads_codes(ctx, False, 32, 8)
