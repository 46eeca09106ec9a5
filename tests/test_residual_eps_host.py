"""``eps`` reaches the kernels as a float32: a value that would become an
infinity there (rstd 0) or a zero (NaN for a constant row) is refused."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from namitorch_amd import functional as F


@pytest.mark.parametrize("eps", [1e39, 3.5e38, 1e300, 1e-46, 5e-324, 2.0 ** -150])
def test_values_that_float32_does_not_hold(eps):
    with pytest.raises(ValueError, match="eps must be finite and nonnegative as a float32"):
        F._epsilon(eps)


@pytest.mark.parametrize("eps", [0.0, 0, -0.0, 2.0 ** -149, 1e-40, 1e-12, 1e-5, 1, np.float32(1e-6), 3e38,
                                 float(np.finfo(np.float32).max)])
def test_values_that_it_holds(eps):
    taken = F._epsilon(eps)
    assert taken == eps
    narrowed = ctypes.c_float(taken).value
    assert math.isfinite(narrowed) and (narrowed == 0.0) == (eps == 0)
