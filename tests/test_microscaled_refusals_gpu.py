"""Refusals of the microscaled operators that need tensors on a device: results that share memory with what is read."""
import pytest
import torch

from test_microscaled_gpu import DEV, check_status, context

pytestmark = pytest.mark.gpu


def rows_in(room, at, n, k):
    """Rows over a buffer's bytes from `at` on: the codes, and the exponents in a buffer of their own."""
    from rust_inference_b200.kernels import microscaled
    a, b = microscaled.Rows.sizes(n, k)
    return microscaled.Rows(n, k, codes=room[at:at + a], exponents=torch.zeros(b, dtype=torch.uint8, device=DEV))


def test_results_that_share_memory_with_what_is_read():
    from rust_inference_b200.kernels import linear, microscaled, ops
    m, n = 6, 256
    room = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV)
    x, other = rows_in(room, 0, m, n), rows_in(room, 128, m, n)
    far = rows_in(room, m * n, m, n)
    w = microscaled.Matrix.of(torch.ones(n, n, device=DEV))
    ctx = context()
    plain = room[:m * n * 4].view(torch.float32).view(m, n)
    inside = w.codes.view(-1)[:m * n * 2].view(torch.bfloat16).view(m, n)
    bias = torch.zeros(m * n, device=DEV)
    calls = [lambda: linear.project(x, w, other, ctx), lambda: linear.gated(x, w, w, other, ctx), lambda: linear.project(x, w, plain, ctx),
             lambda: linear.into_residual(x, w, plain, ctx), lambda: linear.project(far, w, inside, ctx),
             lambda: linear.project(far, w, bias.view(m, n), ctx, bias=bias[7:7 + n]), lambda: microscaled.values(x, torch.float32, out=plain),
             lambda: microscaled.quantize(plain, x), lambda: microscaled.rmsnorm(plain, bias[:n], 1e-5, x),
             lambda: microscaled.rmsnorm(torch.ones(m, n, device=DEV), bias[:n], 1e-5, x, total=plain),
             lambda: microscaled.Rows(m, n, codes=room, exponents=room[128:])]
    for i, call in enumerate(calls):
        with pytest.raises(ops.KernelError, match="apart"):
            call()
            pytest.fail(f"call {i} was not refused")
    assert not room.any()
    # neighbours are no trouble
    linear.project(x, w, far, ctx)
    assert not microscaled.values(x).any()
    check_status()
