"""The root-mean-square norm into microscaled 8 bits where float32 runs out of numbers: results below 2^-126, factors that bring a vanishing quotient
back, roots at either end.  What is held is as near to the norm in 64 bits as the nearest number, but for the one rounding to 24 bits
(2^-22 of it, as in tests/test_microscaled_gpu.py), which numbers below 2^-126 have fewer of: 2^-149."""
import pytest
import torch

import plain_microscaled as plain
from test_microscaled_gpu import DEV, gen

pytestmark = pytest.mark.gpu


def check(x, w, eps, branch=None):
    from rust_inference_b200.kernels import microscaled
    n, k = x.shape
    _, y = plain.rmsnorm(x, branch, w, eps)
    near = plain.nearest(y, plain.EIGHT)                     # (a block with a NaN: 32 of them)
    none = torch.isnan(near)
    assert not none.all()
    rows = microscaled.Rows(n, k)
    microscaled.rmsnorm(x.to(DEV), w.to(DEV), eps, rows, branch=None if branch is None else branch.to(DEV))
    got = microscaled.values(rows).double().cpu()
    assert torch.equal(torch.isnan(got), none)
    assert ((got - y).abs() <= (near - y).abs() + 2.0 ** -22 * y.abs() + 2.0 ** -149)[~none].all()
    return y


SHAPES = [(1, 32), (3, 896), (2, 1333), (400, 264), (320, 9003)]


@pytest.mark.parametrize("up", [-118, -122, -126, -127, -130, -134])
@pytest.mark.parametrize("n,k", SHAPES)
def test_results_near_the_smallest_numbers(n, k, up):
    """Weights that bring whole blocks below 2^-118, where the exponent is the type's least, and below 2^-126, where float32's numbers thin out."""
    g = gen(n * k - up)
    y = check(torch.randn(n, k, generator=g), (1 + 0.2 * torch.randn(k, generator=g)) * 2.0 ** up, 1e-5)
    assert 0 < y.abs().max() < 2.0 ** (up + 5)


@pytest.mark.parametrize("n,k", SHAPES)
def test_large_weights_on_numbers_far_below_the_root(n, k):
    """x / root is below 2^-126 (and below 2^-149, which float32 has nothing for) for all of a row but its first block; the weight brings it back."""
    g = gen(n + k)
    for far, up in ((-70, 60), (-70, 75), (-84, 40), (-90, 100), (-62, 1)):
        x = torch.randn(n, k, generator=g) * 2.0 ** far
        x[:, :8] = torch.randn(n, 8, generator=g) * 2.0 ** 62
        w = torch.randn(k, generator=g) * 2.0 ** up
        w[:8] = 1.0
        check(x, w, 0.0)


@pytest.mark.parametrize("n,k", SHAPES)
def test_roots_at_either_end(n, k):
    """Rows whose root is beyond 2^126, so that its inverse is no normal float32 (some of their numbers are infinite: those become NaN, the others 0), and
    rows whose root is below 2^-126, so that it is infinite."""
    g = gen(n - k)
    w = 1 + 0.2 * torch.randn(k, generator=g)
    for scale in (2.0 ** 125.5, 2.0 ** 120, 2.0 ** -120, 2.0 ** -128, 2.0 ** -140):
        check((torch.randn(n, k, generator=g).clamp(-5, 5) * 1.5) * scale / 2.0, w, 0.0)
    x = torch.randn(n, k, generator=g) * 2.0 ** -128
    check(x, w, 0.0, branch=(torch.randn(n, k, generator=g) * 2.0 ** -128).bfloat16())


def test_rows_of_zeros_and_negative_zeros():
    x = torch.zeros(3, 160)
    x[1] = -0.0
    x[2, 40] = 2.0 ** -149
    check(x, torch.full((160,), 2.0 ** 20), 1e-6)
