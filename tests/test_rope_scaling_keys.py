"""A scaling that names no factor is refused: taken as 1 it would leave the positions unscaled without a
word (a misspelt key, say)."""
import pytest

from femtotron_b200.ops import rotary

EXTRA = {"llama3": {"low_freq_factor": 1.0, "high_freq_factor": 4.0}}


@pytest.mark.parametrize("kind", [k for k in rotary.SCALINGS if k != "default"])
@pytest.mark.parametrize("given", [{}, {"factor": None}, {"factr": 4.0}, {"scale": 4.0}])
def test_no_factor(kind, given):
    sc = {"rope_type": kind, "original_max_position_embeddings": 2048, **EXTRA.get(kind, {}), **given}
    with pytest.raises(ValueError, match="factor"):
        rotary.inv_frequencies(64, 10000.0, sc)
    rotary.inv_frequencies(64, 10000.0, {**sc, "factor": 4.0})


@pytest.mark.parametrize("missing", ["low_freq_factor", "high_freq_factor"])
def test_llama3_names_its_bounds(missing):
    sc = {"rope_type": "llama3", "factor": 4.0, "original_max_position_embeddings": 2048, **EXTRA["llama3"]}
    del sc[missing]
    with pytest.raises(ValueError, match=missing):
        rotary.inv_frequencies(64, 10000.0, sc)


def test_default_needs_none():
    assert rotary.inv_frequencies(64, 10000.0, {"rope_type": "default", "rope_theta": 10000.0})[1] == 1.0
