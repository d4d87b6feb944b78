"""rotary.rotary_turns where a scaling's formula has no value: refused, as the other
arguments are."""

from __future__ import annotations

import pytest

from pth_flash_attn import rotary


def test_factors_within_one_position():
    """sqrt(1 + ln(factor) / ln(original_max_position)) has no value for 1."""
    kw = dict(scaling="factors", factors=[1.0] * 4, factor=2.0, original_max_position=1, device="cpu")
    with pytest.raises(ValueError, match="attention_scale"):
        rotary.rotary_turns(8, **kw)
    assert rotary.rotary_turns(8, **kw, attention_scale=1.5)[1] == 1.5
    assert rotary.rotary_turns(8, **{**kw, "factor": 1.0})[1] == 1.0


@pytest.mark.parametrize("kw", [
    {"scaling": "linear", "factor": 1e-300}, {"base": 1e-300, "scaling": "none"},
    {"scaling": "base", "factor": 1e300, "base": 1e300},
    {"scaling": "factors", "factors": [1e-300] * 32}])
def test_frequencies_beyond_a_double(kw):
    with pytest.raises(ValueError, match="finite"):
        rotary.rotary_turns(64, device="cpu", **kw)
