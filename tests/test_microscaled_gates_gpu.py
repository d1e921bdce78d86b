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


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("m", [8, 700])
def test_a_nan_in_either_factor_of_a_wide_plain_gate(m, form):
    """In bfloat16, one token tile and many (on pairs of SMs too)."""
    from rust_inference_b200.kernels import linear, tcgen05
    k, n = 256, 1024
    x, wg, wu = (spread(r, k, s, torch.bfloat16, 0.3).to(DEV) / math.sqrt(16) for r, s in ((m, 1), (n, 2), (n, 3)))
    wg[5, 0], wu[1000, 3] = math.nan, math.nan
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[:, [5, 1000]] = True
    for always in (False, True):
        tcgen05.set_pairs(1, always=True) if always else tcgen05.set_pairs(0)
        try:
            out = torch.zeros(m, n, dtype=torch.bfloat16, device=DEV)
            linear.gated(x, linear.Weight(wg), linear.Weight(wu), out, context(), form=form_of(form))
        finally:
            tcgen05.set_pairs()
        assert torch.equal(torch.isnan(out), bad)
    check_status()


@pytest.mark.parametrize("form", FORMS)
def test_a_nan_in_either_factor_of_the_experts_gates(form):
    """The experts' products, on the tensor cores (bfloat16) and without them."""
    from rust_inference_b200.kernels import ops, tcgen05
    experts, n, k, tokens = 3, 40, 64, 30
    x = spread(tokens, k, 1, wide=0.3).to(DEV)
    wg, wu = ((spread(experts * n, k, s, wide=0.3) / 8).view(experts, n, k).to(DEV) for s in (2, 3))
    wg[1, 5, 0], wu[2, 33, 3] = math.nan, math.nan
    ids = (torch.arange(tokens, dtype=torch.int32, device=DEV) % experts)[:, None].contiguous()
    bad = torch.zeros(tokens, n, dtype=torch.bool, device=DEV)                      # by token
    bad[1::3, 5] = True
    bad[2::3, 33] = True
    for dtype, cores in ((torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)):
        rows = tcgen05.GROUPED_TILE_ROWS if cores else ops.moe_tile_rows()
        offsets, order, tiles, n_tiles, place = (torch.zeros(c, dtype=torch.int32, device=DEV)
                                                 for c in (experts + 1, tokens, 2 * (-(-tokens // rows) + experts), 1, tokens))
        ops.moe_arrange(ids, tokens, experts, rows, offsets, order, tiles, n_tiles, place)
        out = torch.zeros(tokens, n, dtype=dtype, device=DEV)
        mats = [w.to(dtype).contiguous() for w in (wg, wu)]
        if cores:
            xs = x.to(dtype)[order.long()].contiguous()
            tcgen05.grouped_gemm(xs, *mats, out, offsets, tiles, n_tiles, n_pairs=tokens, gate_form=form_of(form))
            got = torch.isnan(out)[place.long()]
        else:
            ops.moe_grouped_simt(x.to(dtype), *mats, out, offsets, order, tiles, n_tiles, n_pairs=tokens, top=1, gate_form=form_of(form))
            got = torch.isnan(out)
        assert torch.equal(got, bad)
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


@pytest.mark.parametrize("m,n,k", [(1, 300, 640), (16, 130, 333), (100, 256, 512), (300, 390, 1000)])
def test_a_gelu_gate_with_a_factor(one_kernel, m, n, k):
    """Every constant of a gate but the limit: out = mult g sigmoid(alpha g (1 + cubic g^2)) u."""
    from rust_inference_b200.kernels import linear, microscaled
    x, wg, wu = spread(m, k, 3 * m + k, wide=0.5), spread(n, k, n + k, wide=0.5) * 2 / math.sqrt(k), spread(n, k, n + k + 1, wide=0.5) / math.sqrt(k)
    f = form_of("gelu")
    g, gm = exact_product(x, wg)
    u, um = exact_product(x, wu)
    want = plain.gate(g, u, f)
    eg, eu = ((k / 32 + 16) * 2.0 ** -23 * v for v in (gm, um))
    # the slope of the gate is below 1.13, half of that here; the exponential's argument a has three roundings and its result 2 + 1.2 |a| units in the
    # last place, which a term that it leaves counts: (1.2 + 2) |a| + 2, and 6 for the division and the products
    a = (f[0] * g * (1 + f[3] * g * g)).abs()
    off = 0.6 * eg * (u.abs() + eu) + 0.5 * g.abs() * eu + (4 * a.clamp(max=120) + 16) * 2.0 ** -23 * want.abs() + 1e-30
    held = [microscaled.Matrix.of(w.to(DEV)) for w in (wg, wu)]
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m, n), math.nan, dtype=dtype, device=DEV)
        linear.gated(x.to(DEV), *held, out, context(dtype), form=f)
        assert ((out.double() - want).abs() <= off + HALF_STEP[dtype] * want.abs() * 1.01).all()
    rows = microscaled.Rows(m, n)
    linear.gated(x.to(DEV), *held, rows, context(), form=f)
    assert rows_near(microscaled.values(rows).double(), want, off)
    check_status()


@pytest.mark.parametrize("learned", [(0.3, -0.7), (-2.0, 1.5), None])
@pytest.mark.parametrize("m", [1, 16, 130, 300])
def test_an_activation_on_both_sides_of_its_pieces(one_kernel, m, learned):
    """act(z) = a_p z^2 + l z above zero, a_n (e^z - 1 - z) + l z below, with a_p = softplus(p), a_n = 1/2 + softplus(q), l = 1/2 (None: the square of
    relu), for z from -20 to 20, most of them near zero."""
    from rust_inference_b200.kernels import linear, microscaled, ops
    k, n = 500, 390
    x, w = spread(m, k, m, wide=0.5), spread(n, k, 78, wide=0.7) / 40
    if learned is None:
        form, ap, an, lin = torch.tensor(ops.RELU_SQUARED_FORM, device=DEV), 1.0, 0.0, 0.0
    else:
        p, q = (float(torch.tensor(v)) for v in learned)
        form, ap, an, lin = torch.tensor(learned, device=DEV), math.log1p(math.exp(p)), 0.5 + math.log1p(math.exp(q)), 0.5
    z, mass = exact_product(x, w)
    below = z < 0
    if m > 1:
        assert (z > 1).any() and (z < -1).any() and (z.abs() < 0.25).any() and ((z < -0.25) & (z > -1)).any()
    t = torch.expm1(z.clamp(max=0)) - z.clamp(max=0)
    curved = torch.where(below, an * t, ap * z * z)
    want = curved + lin * z
    dz = (k / 32 + 16) * 2.0 ** -23 * mass
    slope = torch.where(below, torch.full_like(z, an + lin), 2 * ap * (z.abs() + dz) + lin) + an + lin
    # constants off by 2^-22 (softplus), four roundings of each term; where the result is rounded to 8 or 16 bits, e^z - 1 - z from five terms above -1/4
    # (2e-5 of it) and as a difference below: its terms are at most 1 + |z|, off by 2^-22 of that
    off = slope * dz + 2.0 ** -21 * (curved.abs() + (lin * z).abs()) + 2.0 ** -22 * an * z.abs() * below
    quick = off + an * (2e-5 * t + torch.where(z < -0.2, 2.0 ** -21 * (1 + z.abs()), 0.0 * z)) * below
    held = microscaled.Matrix.of(w.to(DEV))
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m, n), math.nan, dtype=dtype, device=DEV)
        linear.activated(x.to(DEV), held, out, context(dtype), form)
        assert ((out.double() - want).abs() <= (off if dtype is torch.float32 else quick) + HALF_STEP[dtype] * want.abs() * 1.01).all()
    rows = microscaled.Rows(m, n)
    linear.activated(x.to(DEV), held, rows, context(), form)
    assert rows_near(microscaled.values(rows).double(), want, quick)
    check_status()
