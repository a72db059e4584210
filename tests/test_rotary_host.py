"""Rotary's refusals of numbers at the ends of float64."""
import math

import pytest

from prismkv_amd import Rotary

LLAMA3 = dict(rope_type="llama3", factor=8, low_freq_factor=1, high_freq_factor=4, original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=4, original_max_position_embeddings=8192)
ENDS = (math.inf, -math.inf, math.nan, 0.0, -1.0, 5e-324, 1e-300, 1e300)


@pytest.mark.parametrize("base", ENDS)
def test_bases(base):
    try:
        rotary = Rotary(128, base=base, device="cpu")
    except ValueError:
        return
    assert rotary.frequencies.isfinite().all()


@pytest.mark.parametrize("scaling,name", [(s, name) for s in (LLAMA3, YARN, dict(rope_type="linear", factor=2))
                                          for name in [*s, "beta_fast", "beta_slow", "attention_factor"]
                                          if name != "rope_type" and (name in s or s is YARN)])
@pytest.mark.parametrize("value", ENDS)
def test_scalings(scaling, name, value):
    try:
        rotary = Rotary(128, scaling={**scaling, name: value}, device="cpu")
    except ValueError:
        return
    assert rotary.frequencies.isfinite().all() and math.isfinite(rotary.amplitude)
