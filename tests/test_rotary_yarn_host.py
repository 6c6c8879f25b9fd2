"""What yarn's definition covers: contexts that get longer, and a first pair
that turns no less often than the last one."""
import math

import pytest

import oi2

YARN = {"type": "yarn", "factor": 16.0, "original_len": 4096, "beta_fast": 32.0, "beta_slow": 1.0}


@pytest.mark.parametrize("kw", [{"factor": 0.999}, {"factor": 0.25}, {"factor": 1e-6}, {"beta_fast": 0.999}, {"beta_fast": 0.5},
                                {"beta_slow": 40.0}])
def test_refused(kw):
    with pytest.raises(ValueError, match="yarn"):
        oi2.rotary_frequencies(64, 1e4, {**YARN, **kw})
    with pytest.raises(ValueError):
        oi2.Rotary(64, 1e4, scaling={**YARN, **kw}, device="cpu")


def test_magnitude_never_shrinks():
    plain, _ = oi2.rotary_frequencies(64, 1e4)
    f, m = oi2.rotary_frequencies(64, 1e4, {**YARN, "factor": 1.0})
    assert m == 1.0 and all(abs(a - b) <= 1e-15 * a for a, b in zip(plain, f))
    for factor in (1.5, 4.0, 64.0):
        f, m = oi2.rotary_frequencies(64, 1e4, {**YARN, "factor": factor})
        assert abs(m - (0.1 * math.log(factor) + 1)) < 1e-15 and m > 1
        assert all(a / factor * (1 - 1e-15) <= b <= a for a, b in zip(plain, f))
