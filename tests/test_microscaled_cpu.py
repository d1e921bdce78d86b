"""Weights in microscaled 4 bits: names, refusals and choices that need no GPU."""
import pytest
import torch

import plain_microscaled as plain
from conftest import TINY
from rust_inference_b200 import config_from_dict
from rust_inference_b200.cli import CliError, parse_args
from rust_inference_b200.config.registry import get_architecture
from rust_inference_b200.engine.engine import resolve_weights_dtype
from rust_inference_b200.engine.model import DecoderModel
from rust_inference_b200.kernels import build, linear, microscaled
from rust_inference_b200.kernels.ops import KernelError


def _spec(name):
    c = config_from_dict(TINY[name])
    return get_architecture(c.architecture).build_spec(c)


def test_names():
    assert resolve_weights_dtype(None) is None and resolve_weights_dtype("same") is None and resolve_weights_dtype("mxfp4") == "mxfp4"
    for bad in ("int4", "fp4", torch.int8, 4):
        with pytest.raises(ValueError, match="mxfp4"):
            resolve_weights_dtype(bad)
    a = parse_args(["-m", ".", "-p", "1", "--weights-dtype", "mxfp4"])
    assert a["weights_dtype"] == "mxfp4" and parse_args(["-m", ".", "-p", "1"])["weights_dtype"] is None
    with pytest.raises(CliError, match="Invalid --weights-dtype"):
        parse_args(["-m", ".", "-p", "1", "--weights-dtype", "int4"])


def test_which_parts_hold_their_matrices_in_4_bits():
    for name in TINY:
        m = DecoderModel(_spec(name), dtype=torch.bfloat16, device="cpu", weights_dtype="mxfp4")
        for layer in m.layers:
            assert {role for role, part in layer.parts.items() if part.weights_dtype} == {"mixer", "feed_forward"}
        assert m.embedding.weights_dtype is None and m.head.weights_dtype is None
        plain_model = DecoderModel(_spec(name), dtype=torch.bfloat16, device="cpu")
        assert all(p.weights_dtype is None for _, p in plain_model._named_parts())
        held = m.weight_bytes(False)
        assert held < plain_model.weight_bytes(False)
    with pytest.raises(ValueError, match="mxfp4"):
        DecoderModel(_spec("A"), dtype=torch.bfloat16, device="cpu", weights_dtype="int8")


def test_weight_bytes():
    """128 numbers of a row: 64 bytes of codes and four exponents."""
    m = DecoderModel(_spec("A"), dtype=torch.bfloat16, device="cpu", weights_dtype="mxfp4")
    c = TINY["A"]
    q, kv, h, i = 256, 128, c["hidden_size"], c["intermediate_size"]
    spans = lambda k: -(-k // 128)  # noqa: E731
    layer = 68 * ((q + 2 * kv) * spans(h) + h * spans(q) + 2 * i * spans(h) + h * spans(i)) + 2 * 4 * h
    assert m.weight_bytes() == c["num_hidden_layers"] * layer + 4 * h + 2 * c["vocab_size"] * h


def test_a_decoder_that_routes_is_refused():
    import lulisun_models
    config = config_from_dict(lulisun_models.CONFIGS["A"])
    spec = get_architecture(config.architecture).build_spec(config)
    assert DecoderModel(spec, dtype=torch.bfloat16, device="cpu").routed
    with pytest.raises(ValueError, match="route"):
        DecoderModel(spec, dtype=torch.bfloat16, device="cpu", weights_dtype="mxfp4")


def test_there_is_no_path_on_the_host():
    t = torch.ones(4, 64)
    for call in (lambda: microscaled.Matrix.of(t), lambda: microscaled.quantize(t), lambda: microscaled.Rows(4, 64, "cpu"),
                 lambda: microscaled.Rows(4, 64, codes=torch.zeros(512, dtype=torch.uint8), exponents=torch.zeros(512, dtype=torch.uint8)),
                 lambda: microscaled.Matrix.of_codes(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 64),
                 lambda: microscaled.Matrix.of(torch.ones(4)), lambda: microscaled.Matrix.of(torch.ones(4, 0))):
        with pytest.raises(KernelError):
            call()


def test_the_extension_refuses_what_it_cannot_take():
    calls = build.load_extension("native_calls")
    for fn, count in (("mx_hold", 2), ("mx_matrix", 3), ("mx_values", 2), ("mx_rmsnorm", 6), ("mx_product", 10)):
        with pytest.raises((RuntimeError, TypeError)):
            getattr(calls, fn)(*[None] * count)
        with pytest.raises(RuntimeError):
            getattr(calls, fn)()
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="current device"):
        calls.mx_hold(x, 0)
    with pytest.raises(RuntimeError, match="current device"):
        calls.mx_rmsnorm(x, None, x, None, 1e-5, 0)


def test_sizes_of_rows():
    assert microscaled.Rows.sizes(1, 1) == (128, 512) and microscaled.Rows.sizes(129, 129) == (129 * 256, 2 * 2 * 512)
    assert not linear.is_microscaled(linear.Weight(torch.ones(2, 2)))


def test_the_plain_numbers():
    """The oracle's own numbers: both types' lists, ties, and the exponent's rule."""
    assert plain.EIGHT[-1] == 448.0 and plain.EIGHT[1] == 2.0 ** -9 and len(plain.EIGHT) == 127
    x = torch.zeros(1, 32)
    x[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    assert plain.nearest(x, plain.FOUR)[0, :8].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    x[0, 0] = 6.5                                             # beyond 6: numbers are even ones now
    assert plain.nearest(x, plain.FOUR)[0, :4].tolist() == [6.0, 0.0, 1.0, 1.0]
    assert plain.nearest(torch.full((1, 5), 1e-45), plain.EIGHT).abs().max() == 0
