"""CPU checks of the token choice's oracle: how near it says that min_p's bar is."""

import math

import numpy as np
import pytest

import conftest  # noqa: F401  (paths)
from oracle import sample_oracle as S


def test_the_distance_from_the_bar_is_in_temperatures():
    """The same row at other scales, with its temperature: the same margin."""
    x = np.random.default_rng(0).standard_normal(500) / 4
    want = S.sample(x, 0.4, temperature=0.3, min_p=0.3)
    assert want[2] > 1e-6
    for scale in (1e-41, 1e-30, 2.0 ** 20, 1e30):
        got = S.sample(x * scale, 0.4, temperature=0.3 * scale, min_p=0.3)
        assert got[0] == want[0] and got[2] == pytest.approx(want[2], rel=1e-3), scale


def test_a_logit_at_the_bar_is_not_sure():
    x = np.array([0.0, math.log(0.25), -5.0])
    assert S.sample(x, 0.0, min_p=0.25)[2] == 0.0
    # far above the temperature the bar is no better than its own float64
    y = np.array([1e6, 1e6 - 1e-10, 0.0])
    assert S.sample(y, 0.0, temperature=1e-10, min_p=math.exp(-1))[2] == 0.0
    # as large as the largest: always kept
    assert S.sample(np.array([2.0, 2.0]), 0.1, min_p=0.5)[2] == pytest.approx(0.4)
