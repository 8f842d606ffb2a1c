"""What both ramps of stretched frequencies promise, whatever the context: pairs that turn `high` times and more over it stay,
those that turn `low` times and less are stretched by the whole factor, and none lies outside the two."""
import math

import numpy as np
import pytest


@pytest.mark.parametrize("scaling", ["turns", "index"])
@pytest.mark.parametrize("n", [2, 16, 128])
@pytest.mark.parametrize("base", [1.5, 1e4, 5e6])
@pytest.mark.parametrize("context", [3, 100, 300, 4096, 131072, 1e9])
@pytest.mark.parametrize("low,high", [(1.0, 32.0), (32.0, 64.0), (0.3, 4.0)])
def test_ends_of_the_ramp(lia, scaling, n, base, context, low, high):
    factor = 8.0
    plain = lia.rope_frequencies(n, base)
    f = lia.rope_frequencies(n, base, scaling, factor=factor, context=context, low=low, high=high)
    turns = context * plain / (2 * math.pi)
    ratio = f / plain
    # (frequencies and turns are within a few units of 2^-53; one on an end itself may fall to either side)
    assert np.abs(ratio[turns >= high * (1 + 1e-9)] - 1).max(initial=0.0) < 1e-12
    assert np.abs(ratio[turns <= low * (1 - 1e-9)] * factor - 1).max(initial=0.0) < 1e-12
    assert (ratio <= 1 + 1e-12).all() and (ratio * factor >= 1 - 1e-12).all()
    assert (np.diff(ratio) <= 1e-12).all()


def test_short_contexts_stretch_every_pair(lia):
    """No pair turns even `low` times over 100 positions."""
    plain = lia.rope_frequencies(128, 1e4)
    f = lia.rope_frequencies(128, 1e4, "index", factor=8.0, context=100, low=32.0, high=64.0)
    assert np.abs(f * 8 / plain - 1).max() < 1e-12
