"""Steps over a cache in 8 bits in which sequences bring different numbers of tokens."""
import math

import pytest
import torch

import plain_quantized as plain
from plain_quantized_bounds import attend_codes, held
from test_quantized_cache_gpu import DEV, UNITS, Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("runs, codes", [([(1900 + 3 * i, 1) for i in range(40)] + [(0, 17)], True), ([(1500, 1)] * 12 + [(0, 60), (333, 1)], True),
                                         ([(130, 1), (70, 1), (0, 700)], False)])
@pytest.mark.parametrize("n_heads, n_kv, hd", [(14, 2, 64), (8, 2, 128)])
def test_a_mixed_step(n_heads, n_kv, hd, runs, codes):
    from rust_inference_b200.kernels import attention, quantized_cache
    step = Step(runs, n_kv, hd)
    for t in (step.layer.k_scale, step.layer.v_scale):
        t.uniform_(0.004, 0.016, generator=torch.Generator(DEV).manual_seed(3))
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(10)).bfloat16()
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=torch.bfloat16, device=DEV)
    ctx = step.context(torch.bfloat16)
    ctx.host_starts, ctx.host_counts = [s for s, _ in runs], [n for _, n in runs]
    scale = hd ** -0.5
    attention.attention(q.to(DEV), step.layer, out, ctx, n_heads=n_heads, n_kv_heads=n_kv, head_dim=hd, scale=scale)
    assert any(name.startswith("widened") for name, _ in ctx.workspace._flat) != codes
    assert out.isfinite().all()
    k, v, ks, vs = step.host()
    for b in (0, 5 % len(runs), len(runs) - 2, len(runs) - 1):
        start, n = runs[b]
        keys, values = (held(c, s, step.pages(b), start + n) for c, s in ((k, ks), (v, vs)))
        for t in {0, n // 2, n - 1}:
            row, pos = step.cu[b] + t, start + t
            row_q = q[row:row + 1].double().view(1, n_heads, hd)
            if codes:
                want, bound = attend_codes(row_q, [x[:pos + 1] for x in keys], [x[:pos + 1] for x in values], pos, scale=scale, float32=False)
            else:                               # keys and values in float16 pages on the way
                whole = [(c * s[..., None])[:pos + 1] for c, s in (keys, values)]
                want, bound = plain.attend(row_q, *whole, pos, scale=scale, unit=UNITS[torch.bfloat16][0], step=UNITS[torch.bfloat16][1])
            off = (out[row].cpu().double().view(1, n_heads, hd) - want).abs()
            assert (off <= bound).all(), (b, t, float((off / bound).max()))
