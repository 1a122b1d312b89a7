"""The factor of the values that a yarn scaling turns."""
import math

import pytest

from trit_b200 import Rotary


@pytest.mark.parametrize("factor, want", [(0.25, 1.0), (1.0, 1.0), (2.0, 0.1 * math.log(2.0) + 1), (64.0, 0.1 * math.log(64.0) + 1)])
def test_factor(factor, want):
    assert abs(Rotary(64, scaling="yarn", factor=factor, trained=4096).frequencies()[1] - want) <= want * 2.0**-24
    assert Rotary(64, scaling="yarn", factor=factor, trained=4096, attention_factor=0.5).frequencies()[1] == 0.5
