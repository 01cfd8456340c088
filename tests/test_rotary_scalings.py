"""Scalings of rotary frequencies that mean nothing are refused, not turned into frequencies."""

import math

import pytest
import torch

from nano_vllm_ascend_b200 import rotary_frequencies

INF, NAN = math.inf, math.nan
YARN = dict(type="yarn", factor=4.0, original_max_position=4096)
WAVE = dict(type="wavelength", factor=4.0, original_max_position=4096, low_freq_factor=1.0, high_freq_factor=4.0)


@pytest.mark.parametrize("scaling,text", [
    (dict(YARN, original_max_position=0), "original_max_position 0"),
    (dict(YARN, original_max_position=INF), "original_max_position inf"),
    (dict(YARN, beta_slow=0), "beta_slow 0"), (dict(YARN, beta_fast=1, beta_slow=32), "above beta_fast 1"),
    (dict(YARN, beta_slow=NAN), "beta_slow nan"), (dict(YARN, factor=INF), "not finite"),
    (dict(WAVE, original_max_position=-5), "original_max_position -5"),
    (dict(WAVE, original_max_position=NAN), "original_max_position nan"),
    (dict(type="linear", factor=INF), "not finite"), (dict(type="ntk", factor=INF), "not finite")])
def test_scalings_refuse(scaling, text):
    with pytest.raises(ValueError, match=text):
        rotary_frequencies(64, 1e4, scaling)


def test_an_infinite_base_is_refused():
    with pytest.raises(ValueError, match="base inf"):
        rotary_frequencies(64, INF)


def test_a_ramp_of_no_width_is_a_step():
    inv, _ = rotary_frequencies(64, 1e4, dict(YARN, beta_fast=8, beta_slow=8))
    plain, _ = rotary_frequencies(64, 1e4)
    ratio = inv / plain
    assert torch.isfinite(inv).all() and bool((ratio[:-1] >= ratio[1:] - 1e-12).all())
    assert math.isclose(float(ratio[0]), 1) and math.isclose(float(ratio[-1]), 0.25)
