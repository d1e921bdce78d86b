"""A model whose matrices are held in microscaled 4 bits, on another device than the current one: what brings them to 4 bits and back are kernels, which run
where the model lies.  The devices are stood in for; nothing here needs a GPU."""
import contextlib
import types

import pytest
import torch

from conftest import TINY
from rust_inference_b200 import config_from_dict
from rust_inference_b200.config.registry import get_architecture
from rust_inference_b200.engine.model import DecoderModel
from rust_inference_b200.kernels import linear, microscaled


@pytest.fixture
def devices(monkeypatch):
    """The devices that are current, the innermost last."""
    stack = [torch.device("cuda:0")]

    @contextlib.contextmanager
    def device(d):
        stack.append(torch.device(d))
        yield
        stack.pop()

    monkeypatch.setattr(torch.cuda, "device", device)
    return stack


@pytest.mark.parametrize("name", ["A", "E"])
def test_loading_and_reading_back_where_the_model_lies(name, devices, monkeypatch):
    config = config_from_dict(TINY[name])
    model = DecoderModel(get_architecture(config.architecture).build_spec(config), dtype=torch.float32, device="cpu", weights_dtype="mxfp4")
    model.device = torch.device("cuda:1")
    seen = []

    class Held(types.SimpleNamespace):
        pass

    def of(t):
        seen.append(("held", devices[-1]))
        return Held(t=t, n=t.shape[0], k=t.shape[1])

    def plain(w, dtype):
        seen.append(("read", devices[-1]))
        return w.t

    monkeypatch.setattr(microscaled.Matrix, "of", of)
    monkeypatch.setattr(linear, "plain", plain)
    monkeypatch.setattr(model, "_to", lambda t, dtype: t.to(dtype))
    tensors = {n: torch.randn(ts.shape) for n, ts in model.declared_tensors().items()}

    def arriving():
        for item in tensors.items():
            seen.append(("arrives", devices[-1]))        # (made on the device, or brought to another type there)
            yield item

    model.load(arriving())
    back = model.state_dict()
    assert {what for what, _ in seen} == {"held", "read", "arrives"} and {d for _, d in seen} == {torch.device("cuda:1")}
    assert devices == [torch.device("cuda:0")]
    assert all(torch.equal(back[n], t) for n, t in tensors.items())


def test_on_the_host_no_device_is_asked_for(devices):
    config = config_from_dict(TINY["A"])
    model = DecoderModel(get_architecture(config.architecture).build_spec(config), dtype=torch.float32, device="cpu")
    tensors = {n: torch.randn(ts.shape) for n, ts in model.declared_tensors().items()}

    def arriving():
        for item in tensors.items():
            assert len(devices) == 1
            yield item

    model.load(arriving())
    assert set(model.state_dict()) == set(tensors)
