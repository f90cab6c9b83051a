"""The factor on cos and sin of a yarn table: 0.1 ln(factor) + 1 above a factor of 1, and 1 up to it (a context that is
not stretched keeps its scores)."""
import math

import pytest

from atomflow_amd import kv


@pytest.mark.parametrize("factor,want", [
    (1e-9, 1.0), (1e-5, 1.0), (0.25, 1.0), (1.0, 1.0), (1.5, 0.1 * math.log(1.5) + 1), (16.0, 0.1 * math.log(16) + 1)])
def test_factor(factor, want):
    got = kv.rope_frequencies(128, 500000.0, "yarn", factor, 8192)[1]
    assert abs(got - want) < 1e-15
    assert kv.rope_frequencies(128, 500000.0, "yarn", factor, 8192, attention_factor=0.75)[1] == 0.75
