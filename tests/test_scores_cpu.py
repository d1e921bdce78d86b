"""What scoring a text decides on the host (no GPU)."""
import math
from types import SimpleNamespace

import pytest

from rust_inference_b200.api import Model, TokenScores


def test_perplexity():
    assert TokenScores([-1.0, -3.0], [0.5, 0.5], None).perplexity == pytest.approx(math.exp(2.0))
    assert TokenScores([-2000.0], [0.0], None).perplexity == math.inf          # beyond what a float holds
    assert TokenScores([-math.inf, -1.0], [0.0, 0.0], None).perplexity == math.inf
    assert math.isnan(TokenScores([math.nan, -1.0], [0.0, 0.0], None).perplexity)


@pytest.mark.parametrize("top", [-1, 65, 101])
def test_alternatives_are_looked_at_before_the_model_runs(top):
    def nothing(*args, **kw):
        raise AssertionError("the text has been run")

    engine = SimpleNamespace(model=SimpleNamespace(spec=SimpleNamespace(vocab_size=100)), alloc_slot=nothing, step=nothing, free_slot=nothing)
    with pytest.raises(ValueError, match="alternatives"):
        Model(engine).score([1, 2, 3], top=top)
