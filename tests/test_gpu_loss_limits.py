"""The linear cross entropy where values leave the middle of their range."""

from __future__ import annotations

import numpy as np
import pytest

import test_gpu_loss as base
from namitorch_amd import functional as F

pytestmark = pytest.mark.gpu

# Powers of two by which the operands' logits come to 1.5 * 2**(a + b), and at most 1.25 of it for other classes:
# float32 holds these logits, and lse, without rounding, as the others' exponentials are zero beside the largest's.
FAR = [("bfloat16", 63, 64), ("bfloat16", 20, 20), ("bfloat16", 5, 5), ("float16", 15, 14), ("float16", 5, 5),
       ("float32", 60, 62), ("float32", 20, 20), ("float32", 5, 5)]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype, a, b", FAR)
@pytest.mark.parametrize("rows", [2, 6, 70, 300])
def test_far_logits_are_exact(rows, dtype, a, b, sign):
    """The loss is the distance of two exact logits, and dz a difference of ones: zero where the target is the largest.
    What is left to round are the mean's factor and a gradient's own rounding; with `sign` all logits lie below zero."""
    classes, width = 300, 8
    rng = base._rng(21, rows, a, b)
    levels = np.full(classes, 1.0 if sign > 0 else 1.75)
    levels[rng.permutation(classes)[:100]] = 1.25 if sign > 0 else 1.875
    largest = int(rng.integers(0, classes))
    levels[largest] = 1.5
    x, weight = np.zeros((rows, width)), np.zeros((classes, width))
    x[:, 3], weight[:, 3] = 2.0 ** a, sign * levels * 2.0 ** b
    weight[:, 5] = rng.integers(-4, 5, classes)                 # meets zeros alone
    target = rng.integers(0, classes, rows)
    target[::2] = largest
    tx, tw, at = base._tensor(x, dtype), base._tensor(weight, dtype), base._targets(target)
    loss, lse = F.linear_cross_entropy_forward(tx, tw, at, reduction="none")
    top = 2.0 ** a * weight[largest, 3]
    assert np.all(lse.numpy() == top)
    assert np.array_equal(loss.numpy().astype(np.float64), top - 2.0 ** a * weight[target, 3])
    dx, dw = F.linear_cross_entropy_backward(1.0, tx, tw, at, lse)
    dz = np.zeros((rows, classes))
    dz[:, largest] = 1.0
    dz[np.arange(rows), target] -= 1.0
    for got, exact in ((dx, dz @ weight / rows), (dw, dz.T @ x / rows)):
        # The sums are whole multiples of a power of two; 1 / rows and its product round once each, then the result.
        assert np.all(np.abs(base._values(got) - exact) <= (base.HALF_ULP[dtype] + 3 * base.E) * np.abs(exact))
