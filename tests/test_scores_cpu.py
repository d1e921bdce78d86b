"""What scoring a text decides on the host (no GPU)."""
import math

import pytest

from rust_inference_b200.api import TokenScores


def test_perplexity():
    assert TokenScores([-1.0, -3.0], [0.5, 0.5], None).perplexity == pytest.approx(math.exp(2.0))
    assert TokenScores([-2000.0], [0.0], None).perplexity == math.inf          # beyond what a float holds
    assert TokenScores([-math.inf, -1.0], [0.0, 0.0], None).perplexity == math.inf
    assert math.isnan(TokenScores([math.nan, -1.0], [0.0, 0.0], None).perplexity)
