"""Settings of ``sample_tokens`` given as numbers, checked before anything reaches the device."""

import math

import pytest

from inferkernellab_b200 import sampling


def _top_k(value):
    return sampling._number(value, "top_k", 0, lambda v: 0 <= v < 2 ** 31)


def test_top_k_is_a_whole_number():
    assert [_top_k(v) for v in (None, 0, 40, 40.0, 2 ** 31 - 1)] == [0, 0, 40, 40, 2 ** 31 - 1]
    for bad in (0.5, 2.5, math.nan, math.inf, -math.inf):  # 0.5 would turn the filter off
        with pytest.raises(ValueError, match="whole"):
            _top_k(bad)
    for bad in (-1, 2 ** 31, 10 ** 400):
        with pytest.raises(ValueError, match="out of range"):
            _top_k(bad)
