"""Attention over a cache in 8 bits whose values differ in size from block to block: a row is as near 64 bits as its own roundings
allow, whatever lies in blocks that it does not see or gives no weight to."""
import math

import pytest
import torch

from plain_quantized_bounds import attend_codes, held
from test_quantized_cache_gpu import DEV, Step

pytestmark = pytest.mark.gpu

SHAPES = [(4, 2, 64, torch.float32), (14, 2, 64, torch.bfloat16), (7, 1, 128, torch.bfloat16), (3, 3, 128, torch.float32), (16, 1, 128, torch.float32)]


def _check(step, q, n_heads, dtype, wide=False, **limits):
    from rust_inference_b200.kernels import quantized_cache as qc
    n_kv, hd = step.n_kv, step.hd
    if wide:
        step.max_len = 1 << 24             # as if a sequence might be long: no clusters, and tiles of 16 rows where there are as many
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=dtype, device=DEV)
    scale = 1.0 / math.sqrt(hd)
    span = limits.get("window") or -limits.get("chunk", 0)
    qc.attend_step(q.to(DEV), step.layer, out, qc.step_of(step.context(dtype), n_heads, n_kv, hd), scale, span, 1.0)
    k, v, ks, vs = step.host()
    for b, (start, n) in enumerate(step.runs):
        a, e = step.cu[b], step.cu[b + 1]
        keys, values = (held(c, s, step.pages(b), start + n) for c, s in ((k, ks), (v, vs)))
        want, bound = attend_codes(q[a:e].double().view(n, n_heads, hd), keys, values, start, scale=scale, float32=dtype is torch.float32, **limits)
        off = (out[a:e].cpu().double().view(n, n_heads, hd) - want).abs()
        assert (off <= bound).all(), (b, float((off / bound).max()))


def _step(runs, n_kv, hd):
    step = Step(runs, n_kv, hd)
    step.arrays([(s + n, 0) for s, n in runs])
    step.fill()
    step.arrays(runs)
    return step


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("factor", [1e5, 1e8, 1e15])
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", SHAPES)
def test_blocks_that_only_later_tokens_see(n_heads, n_kv, hd, dtype, factor, wide):
    runs = [(14, 5), (60, 6), (0, 20), (250, 9)]
    step = _step(runs, n_kv, hd)
    for b, (start, n) in enumerate(runs):
        last = (start + n - 1) // 16
        step.layer.v_scale[int(step.pages(b)[last // 4]), :, last % 4] *= factor
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(2)).to(dtype)
    _check(step, q, n_heads, dtype, wide)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("limits", [{"window": 40}, {"chunk": 48}], ids=str)
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", SHAPES)
def test_blocks_that_only_earlier_tokens_see(n_heads, n_kv, hd, dtype, limits, wide):
    runs = [(47, 12), (100, 9), (140, 7)]
    step = _step(runs, n_kv, hd)
    for b, (start, _) in enumerate(runs):
        first = (start - 39) // 16 if "window" in limits else start // 48 * 3
        step.layer.v_scale[int(step.pages(b)[first // 4]), :, first % 4] *= 1e9
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(3)).to(dtype)
    _check(step, q, n_heads, dtype, wide, **limits)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("score, factor", [(-40.0, 1e8), (-16.0, 1e7), (16.0, 1e-7), (0.0, 1e4), (40.0, 1e-20), (-60.0, 1e30)])
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", SHAPES)
def test_a_block_of_other_scores_and_values(n_heads, n_kv, hd, dtype, score, factor, wide):
    """One of the first blocks has keys of about this score and values so many times as large: large ones without weight, large ones
    whose small weight counts, small ones that have all the weight (what a first token often is)."""
    runs = [(300, 1), (170, 3), (1900, 2)]
    step = _step(runs, n_kv, hd)
    g = torch.Generator().manual_seed(4)
    base = torch.randn(n_kv, hd, generator=g)
    q = base[:, None] * (1.0 + 0.02 * torch.arange(n_heads // n_kv)[None, :, None])
    q = (q.reshape(1, -1) + 0.02 * torch.randn(step.n_tokens, n_heads * hd, generator=g)).to(dtype)
    codes = torch.round(127.0 * base / base.abs().amax(dim=1, keepdim=True))
    # (a small remainder where the score is 0)
    k_scale = (abs(score) + 0.1) * math.sqrt(hd) / (codes * base).sum(dim=1)
    for b in range(len(runs)):
        page = int(step.pages(b)[0])
        step.layer.k[page, :, 16:32] = ((1 if score >= 0 else -1) * codes).to(torch.int8).to(DEV)[:, None]
        step.layer.k_scale[page, :, 1] = k_scale.to(DEV)
        step.layer.v_scale[page, :, 1] *= factor
    _check(step, q, n_heads, dtype, wide)
