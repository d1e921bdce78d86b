"""bfloat16 prompts over a cache in 8 bits whose blocks differ in size: rows are as near 64 bits as 16-bit numbers allow, whatever lies in
blocks that they do not see, or give little weight to."""
import math

import pytest
import torch

from plain_quantized_bounds import attend_pages, held
from test_quantized_cache_gpu import DEV, Step

pytestmark = pytest.mark.gpu

SHAPES = [(8, 2, 64), (14, 2, 128)]


def _step(runs, n_kv, hd):
    step = Step(runs, n_kv, hd)
    step.arrays([(s + n, 0) for s, n in runs])
    step.fill()
    step.arrays(runs)
    return step


def _check(step, q, n_heads, some, apart, **limits):
    from rust_inference_b200.kernels import attention
    n_kv, hd = step.n_kv, step.hd
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=torch.bfloat16, device=DEV)
    scale, ctx = 1.0 / math.sqrt(hd), step.context(torch.bfloat16)
    attention.attention(q.to(DEV), step.layer, out, ctx, n_heads=n_heads, n_kv_heads=n_kv, head_dim=hd, scale=scale, **limits)
    assert any(name.startswith("widened") for name, _ in ctx.workspace._flat)
    k, v, ks, vs = step.host()
    for b, (start, n) in enumerate(step.runs):
        keys, values = (held(c, s, step.pages(b), start + n) for c, s in ((k, ks), (v, vs)))
        for t in some(n):
            row, pos = step.cu[b] + t, start + t
            want, bound = attend_pages(q[row:row + 1].double().view(1, n_heads, hd), keys, values, pos, scale=scale, apart=apart(b), **limits)
            off = (out[row].cpu().double().view(1, n_heads, hd) - want).abs()
            assert (off <= bound).all(), (b, t, float((off / bound).max()))


@pytest.mark.parametrize("limits", [{}, {"window": 40}], ids=str)
@pytest.mark.parametrize("what", ["k_scale", "v_scale"])
@pytest.mark.parametrize("factor", [1.0, 1e3, 1e5, 1e12, 1e20])
@pytest.mark.parametrize("n_heads, n_kv, hd", SHAPES)
def test_blocks_that_only_later_tokens_see(n_heads, n_kv, hd, factor, what, limits):
    """One sequence of the three has such a block: its last one, which only its last tokens see."""
    runs = [(0, 130), (37, 90), (0, 140)]
    step = _step(runs, n_kv, hd)
    for t in (step.layer.k_scale, step.layer.v_scale):         # the others within 2^12 of one another
        t.clamp_(0.005, 0.05).nan_to_num_(0.01)
    last = 126 // 16
    scales = getattr(step.layer, what)
    scales[int(step.pages(1)[last // 4]), :, last % 4] *= factor
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(2)).bfloat16()
    # (rows that see a block of keys as large as that have scores beyond any rounding)
    _check(step, q, n_heads, lambda n: (0, 1, n // 2, 70), lambda b: b == 1 and factor > 1e4, **limits)


@pytest.mark.parametrize("score, factor", [(-40.0, 1e8), (-16.0, 1e7), (16.0, 1e-7), (0.0, 1e2), (40.0, 1e-20), (-60.0, 1e30)])
@pytest.mark.parametrize("n_heads, n_kv, hd", SHAPES)
def test_a_block_of_other_scores_and_values(n_heads, n_kv, hd, score, factor):
    runs = [(0, 300), (100, 170)]
    step = _step(runs, n_kv, hd)
    g = torch.Generator().manual_seed(4)
    base = torch.randn(n_kv, hd, generator=g)
    q = base[:, None] * (1.0 + 0.02 * torch.arange(n_heads // n_kv)[None, :, None])
    q = (q.reshape(1, -1) + 0.02 * torch.randn(step.n_tokens, n_heads * hd, generator=g)).bfloat16()
    codes = torch.round(127.0 * base / base.abs().amax(dim=1, keepdim=True))
    k_scale = (abs(score) + 0.1) * math.sqrt(hd) / (codes * base).sum(dim=1)
    for b in range(len(runs)):
        page = int(step.pages(b)[0])
        step.layer.k[page, :, 16:32] = ((1 if score >= 0 else -1) * codes).to(torch.int8).to(DEV)[:, None]
        step.layer.k_scale[page, :, 1] = k_scale.to(DEV)
        step.layer.v_scale[page, :, 1] *= factor
    _check(step, q, n_heads, lambda n: (10, 60, n // 2, n - 1), lambda b: not 1e-3 < factor < 1e3)


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_marked_and_empty_blocks_beside_scales_far_apart(dtype):
    """Blocks of zeros and blocks that are no numbers set no scale, in either type of page."""
    from rust_inference_b200.kernels import attention
    for factor in (1.0, 1e15):
        step = _step([(0, 200), (0, 90)], 2, 64)
        step.layer.v_scale[int(step.pages(0)[0]), :, 0] *= factor
        step.layer.v_scale[int(step.pages(0)[0]), :, 1] = 0.0
        step.layer.k_scale[int(step.pages(0)[0]), :, 2] = 0.0
        step.layer.v_scale[int(step.pages(0)[2]), 1, 0] = math.nan          # positions 128..143 of kv head 1
        q = torch.randn(step.n_tokens, 8 * 64, device=DEV).to(dtype)
        out = torch.empty_like(q)
        attention.attention(q, step.layer, out, step.context(dtype), n_heads=8, n_kv_heads=2, head_dim=64, scale=0.125)
        out = out.view(-1, 8, 64)
        assert out[:128].isfinite().all() and out[128:200, :4].isfinite().all() and out[128:200, 4:].isnan().all() and out[200:].isfinite().all()
