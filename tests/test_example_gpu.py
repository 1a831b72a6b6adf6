"""The streaming layer example: it trains, and what it serves from the cache is what it computes on
whole rows, up to e4m3's rounding of keys and values."""

import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.parametrize("prompt,new", [(150, 20), (64, 1), (333, 0)])
def test_streaming_layer(prompt, new):
    import streaming_layer

    got = streaming_layer.main(["--steps", "12", "--prompt", str(prompt), "--new", str(new)])
    assert got["last_loss"] < got["first_loss"]
    # e4m3 keeps 4 significant bits: a relative rounding of 2^-4 at most, 2^-5 / sqrt(3) = 1.8% rms, of
    # keys (through the scores) and of values; bf16 elsewhere adds less than 1%.
    assert got["served_against_whole"] < 0.06
    assert got["status"] == 0
