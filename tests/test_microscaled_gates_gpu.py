"""Gated and activated products with matrices in microscaled 4 bits, at the numbers where an epilogue can go wrong: NaN, infinities, both sides of an
activation's pieces, and every constant of a gate.

Tolerances.  Gate and up are off by (K / 32 + 16) 2^-23 of what is added up, as any such product (tests/test_microscaled_gpu.py), which the epilogue's
slope multiplies; the epilogue's own arithmetic is counted below, where it is bounded.  A code of 8 bits is half a step off what it stands for: 2^-4 of
it, or 2^-10 times 2^e, which is at most the block's largest / 224."""
import math

import pytest
import torch

import plain_microscaled as plain
from test_microscaled_gpu import DEV, HALF_STEP, check_status, context, exact_product, spread

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.fixture(params=["pairs of SMs", "single SMs"])
def one_kernel(request):
    from rust_inference_b200.kernels import microscaled
    microscaled.set_pairs(1 if request.param == "pairs of SMs" else 1 << 30)
    yield
    microscaled.set_pairs()


FORMS = {"silu": None, "bounded": dict(alpha=1.702, limit=1.5, shift=1.0), "gelu": dict(alpha=1.5957691216057308, cubic=0.044715, mult=0.5),
         "bounded silu": dict(limit=1.5)}


def form_of(name):
    from rust_inference_b200.kernels import ops
    return None if FORMS[name] is None else ops.gate_form(device=DEV, **FORMS[name])


def rows_near(got, want, off):
    """Whether `got`, read back from 8 bits, is the nearest there is to something within `off` of `want`."""
    m, n = want.shape
    largest = torch.nn.functional.pad(want.abs() + off, (0, -n % 32)).view(m, -1, 32).amax(dim=2, keepdim=True).expand(-1, -1, 32).reshape(m, -1)[:, :n]
    return ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * largest / 224) + 1.1 * off).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("m", [3, 130, 300])
def test_a_nan_in_either_factor_of_a_gate(one_kernel, m, form):
    """A NaN of the gate's or of the up matrix, or of a token, is not clamped to a number, in any type of result, and touches no other number."""
    from rust_inference_b200.kernels import linear, microscaled
    k, n = 160, 260
    x, wg, wu = spread(m, k, 1, wide=0.5), spread(n, k, 2, wide=0.5) / 12, spread(n, k, 3, wide=0.5) / 12
    x[1, 7], x[2, k - 1] = math.nan, -math.inf
    wg[5, 0], wu[200, 3], wg[259, 100] = math.nan, math.nan, math.inf
    held = [microscaled.Matrix.of(w.to(DEV)) for w in (wg, wu)]
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[1:3] = True
    bad[:, [5, 200, 259]] = True
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.zeros(m, n, dtype=dtype, device=DEV)
        linear.gated(x.to(DEV), *held, out, context(dtype), form=form_of(form))
        assert torch.equal(torch.isnan(out).cpu(), bad) and torch.isfinite(out.cpu()[~bad]).all()
    rows = microscaled.Rows(m, n)
    linear.gated(x.to(DEV), *held, rows, context(), form=form_of(form))
    blocks = torch.nn.functional.pad(bad, (0, -n % 32)).view(m, -1, 32).any(dim=2, keepdim=True).expand(-1, -1, 32).reshape(m, -1)[:, :n]
    assert torch.equal(torch.isnan(microscaled.values(rows)).cpu(), blocks)
    check_status()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("m", [1, 130])
def test_a_nan_in_either_factor_of_a_plain_gate(m, form):
    """The same of products with matrices in the run dtype, whose gate is the same function."""
    from rust_inference_b200.kernels import linear
    k, n = 64, 136
    x, wg, wu = spread(m, k, 1, wide=0.5), spread(n, k, 2, wide=0.5) / 8, spread(n, k, 3, wide=0.5) / 8
    wg[5, 0], wu[100, 3] = math.nan, math.nan
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[:, [5, 100]] = True
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.zeros(m, n, dtype=dtype, device=DEV)
        linear.gated(x.to(DEV, dtype), *(linear.Weight(w.to(DEV, dtype)) for w in (wg, wu)), out, context(dtype), form=form_of(form))
        assert torch.equal(torch.isnan(out).cpu(), bad)
    check_status()


@pytest.mark.parametrize("form", ["silu", "gelu", "steep"])
@pytest.mark.parametrize("m", [2, 130, 300])
def test_an_infinite_gate(one_kernel, m, form):
    """Sums beyond float32's numbers: an infinite gate times a factor is infinite, whichever kernel computes it and whatever it writes."""
    from rust_inference_b200.kernels import linear, microscaled, ops
    k, n = 64, 160
    x = torch.ones(m, k)
    x[1] = 2.0 ** 100
    wg, wu = torch.ones(n, k), torch.ones(n, k) * 2.0 ** -90
    wg[40] = 2.0 ** 100                                    # token 1: 64 2^200
    f = ops.gate_form(alpha=1.702, device=DEV) if form == "steep" else form_of(form)
    held = [microscaled.Matrix.of(w.to(DEV)) for w in (wg, wu)]
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.zeros(m, n, dtype=dtype, device=DEV)
        linear.gated(x.to(DEV), *held, out, context(dtype), form=f)
        assert float(out[1, 40]) == INF and torch.isfinite(out[0]).all() and torch.isfinite(out[1, :40]).all() and torch.isfinite(out[1, 41:]).all()
    rows = microscaled.Rows(m, n)
    linear.gated(x.to(DEV), *held, rows, context(), form=f)
    got = torch.isnan(microscaled.values(rows)).cpu()
    assert got[1, 32:64].all() and not got[0].any() and not got[1, :32].any() and not got[1, 64:].any()
    check_status()
