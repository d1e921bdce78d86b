"""Attention straight from 8-bit codes against a bound of the roundings that it makes, with scores large enough to show a query's low
byte; and that the bound sees such a byte go missing (on the CPU, in the oracle)."""
import math

import pytest
import torch

import plain_quantized as plain
from plain_quantized_bounds import attend_codes, held
from test_quantized_cache_gpu import ATTEND, DEV, Step

SHAPES = [(4, 2, 64, torch.bfloat16), (7, 1, 128, torch.bfloat16), (16, 1, 128, torch.bfloat16), (14, 2, 64, torch.float32), (3, 1, 128, torch.float32)]


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("limits", [{}, {"window": 50}, {"chunk": 48}], ids=str)
@pytest.mark.parametrize("scale", [1.0, 0.09])
@pytest.mark.parametrize("runs", ["single", "one", "few", "mixed"])
@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", SHAPES)
def test_within_its_roundings(n_heads, n_kv, hd, dtype, runs, scale, limits, wide):
    from rust_inference_b200.kernels import quantized_cache as qc
    step = Step(ATTEND[runs], n_kv, hd)
    step.arrays([(s + n, 0) for s, n in ATTEND[runs]])
    step.fill()
    step.arrays(ATTEND[runs])
    if wide:
        step.max_len = 1 << 24
    q = torch.randn(step.n_tokens, n_heads * hd, generator=torch.Generator().manual_seed(12)).to(dtype)
    out = torch.full((step.n_tokens, n_heads * hd), math.nan, dtype=dtype, device=DEV)
    span = limits.get("window") or -limits.get("chunk", 0)
    qc.attend_step(q.to(DEV), step.layer, out, qc.step_of(step.context(dtype), n_heads, n_kv, hd), scale, span, 1.0)
    k, v, ks, vs = step.host()
    for b, (start, n) in enumerate(step.runs):
        a, e = step.cu[b], step.cu[b + 1]
        keys, values = (held(c, s, step.pages(b), start + n) for c, s in ((k, ks), (v, vs)))
        want, bound = attend_codes(q[a:e].double().view(n, n_heads, hd), keys, values, start, scale=scale, float32=dtype is torch.float32, **limits)
        off = (out[a:e].cpu().double().view(n, n_heads, hd) - want).abs()
        assert (off <= bound).all(), float((off / bound).max())


def _digits(q, number):
    """q's rows as whole numbers of so many signed bytes, 127 the largest of the highest, lowest byte first, and what a unit is worth."""
    most = 127.0 * 256 ** (number - 1)
    top = q.abs().amax(dim=-1, keepdim=True)
    left, digits = torch.round(q / top * most), []
    for _ in range(number - 1):
        low = torch.remainder(left + 128, 256) - 128
        digits.append(low)
        left = (left - low) / 256
    return digits + [left], top / most


@pytest.mark.parametrize("n_heads, n_kv, hd, dtype", SHAPES)
def test_the_bound_sees_a_lost_byte(n_heads, n_kv, hd, dtype):
    """With all bytes the oracle stays within its bound, without the lowest one it does not, and neither with two of them exchanged."""
    g = torch.Generator().manual_seed(13)
    pages, n = [2, 0, 1], 130
    codes = [torch.zeros(3, n_kv, 64, hd, dtype=torch.int8) for _ in range(2)]
    scales = [torch.zeros(3, n_kv, 4) for _ in range(2)]
    for c, s in zip(codes, scales):
        plain.put(c, s, torch.randn(n, n_kv, hd, generator=g), 0, pages)
    keys, values = (held(c, s, pages, n) for c, s in zip(codes, scales))
    q = torch.randn(2, n_heads, hd, generator=g).to(dtype).double()
    call = dict(scale=1.0, float32=dtype is torch.float32)
    want, bound = attend_codes(q, keys, values, n - 2, **call)
    number = 3 if dtype is torch.float32 else 2
    digits, unit = _digits(q, number)

    def off(parts):
        found = attend_codes(sum(d * 256.0 ** i for i, d in enumerate(parts)) * unit, keys, values, n - 2, **call)[0]
        return float(((found - want).abs() / bound).max())

    assert off(digits) <= 1.0
    assert off([torch.zeros_like(digits[0])] + digits[1:]) > 1.0
    assert off([digits[1], digits[0]] + digits[2:]) > 1.0
