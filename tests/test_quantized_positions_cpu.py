"""Which position encodings lead into a cache in 8 bits (no GPU): those whose way into it is as much their own as their usual one."""
import pytest
import torch

from rust_inference_b200.cache.pager import CacheError
from rust_inference_b200.cache.sequence_cache import SequenceCache
from rust_inference_b200.parts.attention import GQAttention
from rust_inference_b200.parts.registry import lookup, register, unregister
from rust_inference_b200.parts.spec import PartSpec


def _layer(kind, **params):
    return GQAttention(n_heads=4, n_kv_heads=2, head_dim=64, qkv_bias=False, position=PartSpec(kind, params), hidden_size=128,
                       dtype=torch.float32, device=torch.device("cpu"))


def _rope(kind):
    return _layer(kind, head_dim=64, base=1e4)


@pytest.fixture
def registered():
    names = []

    def add(name, cls):
        register("position", name)(cls)
        names.append(name)
    yield add
    for name in names:
        unregister("position", name)


def test_the_librarys_own():
    assert _rope("rope").quantizable and _layer("unrotated").quantizable


@pytest.mark.parametrize("method", ["apply_and_store", "apply_and_store_from_accumulators"])
def test_one_that_changes_its_usual_way_alone(method, registered):
    """It would be passed by: the layer is refused instead."""
    base = lookup("position", "rope")
    registered("toy_rope", type("Toy", (base,), {method: lambda self, *a, **k: getattr(base, method)(self, *a, **k)}))
    layer = _rope("toy_rope")
    assert not layer.quantizable and not layer.cache_request().quantizable
    with pytest.raises(CacheError, match="8 bits"):
        SequenceCache([layer.cache_request()], max_tokens=64, max_seq_len=64, dtype=torch.float32, device="cpu", kv_dtype=torch.int8)
    # ... and one derived from it
    registered("toy_rope_2", type("Toy2", (lookup("position", "toy_rope"),), {}))
    assert not _rope("toy_rope_2").quantizable


def test_one_that_changes_its_usual_way_in_place():
    layer = _rope("rope")
    layer.position.apply_and_store = lambda *a, **k: None
    assert not layer.quantizable


def test_ones_that_have_a_way_of_their_own(registered):
    base = lookup("position", "rope")

    class Toy(base):
        def apply_and_store(self, *args, **kw):
            super().apply_and_store(*args, **kw)

        def apply_and_quantize(self, *args, **kw):
            super().apply_and_quantize(*args, **kw)

    class Tables(base):
        def prepare(self, max_positions):               # other angles, on either way
            super().prepare(max_positions)

    registered("toy_rope", Toy)
    registered("toy_tables", Tables)
    assert _rope("toy_rope").quantizable and _rope("toy_tables").quantizable


def test_one_that_has_none(registered):
    from rust_inference_b200.parts.base import PositionEncoding

    class Bare(PositionEncoding):
        kind = "bare"

        def apply_and_store(self, *args, **kw):
            pass

    registered("bare", Bare)
    assert not _layer("bare").quantizable
