"""The gain that YaRN has of itself, on the CPU: 1 + 0.1 ln(factor) for contexts that
are stretched, 1 where the factor does not stretch them, as the published rule has it."""
import math

import numpy as np

from test_rope_turns import LINEAR, YARN, driver, made  # noqa: F401


def test_gain(driver):  # noqa: F811
    factors = [8.0, 1.5, 1.0, 0.99, 0.5, 0.3]
    got = made(driver, [(8, 1e4, YARN, f, 4096, 1.0, 32.0, 0.0, None) for f in factors])
    for f, (gain, _) in zip(factors, got):
        want = 1 + 0.1 * math.log(float(np.float32(f))) if f > 1 else 1.0
        assert gain == np.float32(want), f
    given = made(driver, [(8, 1e4, YARN, 0.5, 4096, 1.0, 32.0, -0.7, None), (8, 1e4, LINEAR, 0.5, 0, 0.0, 0.0, 0.0, None)])
    assert [np.float32(g) for g, _ in given] == [np.float32(-0.7), 1]
