"""Matrices in 4 bits and rows in 8 where a tensor is wanted, and tensors where they are: refused with a KernelError, not with what Python makes of a missing
attribute.  Nothing here reaches a device."""
import copy

import pytest
import torch

from rust_inference_b200.kernels import linear, microscaled, ops
from rust_inference_b200.kernels.ops import KernelError


def made(cls, n, k):
    """A `Matrix` or `Rows` without buffers."""
    held = cls.__new__(cls)
    held.n, held.k, held.spans, held.device = n, k, -(-k // 128), torch.device("cuda:0")
    return held


def test_products_that_mix_the_kinds():
    x, w = torch.ones(3, 64, dtype=torch.bfloat16), linear.Weight(torch.ones(40, 64, dtype=torch.bfloat16))
    rows, held, out = made(microscaled.Rows, 3, 64), made(microscaled.Matrix, 40, 64), torch.empty(3, 40, dtype=torch.bfloat16)
    f32 = torch.empty(3, 40)
    for call in (lambda: linear.project(rows, w, out, None), lambda: linear.logits(rows, w, f32, None), lambda: linear.into_residual(rows, w, f32, None),
                 lambda: linear.gated(rows, w, w, out, None), lambda: linear.activated(rows, w, out, None, torch.ones(4)),
                 lambda: linear.accumulate_split(rows, w, f32, None), lambda: linear.wants_split(rows, w), lambda: linear.gated(x, w, held, out, None),
                 lambda: linear.gated(x.float(), linear.Weight(w.t.float()), held, f32, None), lambda: linear.gated(x, held, w, out, None),
                 lambda: linear.project(x.float(), linear.Weight(w.t.float()), made(microscaled.Rows, 3, 40), None), lambda: linear.Weight(held)):
        with pytest.raises(KernelError):
            call()


def test_operators_that_want_the_other_kind():
    x, rows, held = torch.ones(3, 64), made(microscaled.Rows, 3, 64), made(microscaled.Matrix, 40, 64)
    for call in (lambda: microscaled.values(x), lambda: microscaled.values(None), lambda: microscaled.quantize(rows), lambda: microscaled.quantize(x, x),
                 lambda: microscaled.rmsnorm(x, torch.ones(64), 1e-5, x), lambda: microscaled.rmsnorm(x, torch.ones(64), 1e-5, held),
                 lambda: microscaled.Matrix.of(rows), lambda: microscaled.Matrix.of(held), lambda: microscaled.product(x, torch.ones(40, 64), x, None),
                 lambda: ops.rmsnorm(rows, torch.ones(64), 1e-5, x), lambda: ops.rmsnorm(x, torch.ones(64), 1e-5, rows)):
        with pytest.raises(KernelError):
            call()


def test_a_norm_of_chosen_rows():
    """As many rows as there are, in another order: not the rows in 8 bits of all of them."""
    from rust_inference_b200.parts.norm import RMSNorm
    norm = RMSNorm(eps=1e-5, hidden_size=64, dtype=torch.bfloat16, device="cpu")
    norm.set_tensors({"weight": torch.ones(64)})
    with pytest.raises(KernelError, match="choice"):
        norm.forward(torch.ones(3, 64), made(microscaled.Rows, 3, 64), rows=torch.tensor([2, 1, 0], dtype=torch.int32))


def test_codes_of_other_shapes():
    codes, exponents = torch.zeros(4, 6, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    for c, e in ((codes[0, 0], exponents), (codes[0], exponents), (codes[None], exponents), (codes, exponents[0]), (codes.int(), exponents), (codes[:0], exponents[:0])):
        with pytest.raises(KernelError, match="codes uint8"):
            microscaled.Matrix.of_codes(c, e, 12)


def test_they_are_asked_for_attributes_like_any_object():
    for held in (made(microscaled.Rows, 3, 64), made(microscaled.Matrix, 40, 64)):
        assert held.shape == (held.n, held.k) and not hasattr(held, "dtype") and getattr(held, "is_cuda", 5) == 5
        with pytest.raises(AttributeError, match="is_cuda"):
            held.is_cuda
        assert copy.copy(held).shape == held.shape
