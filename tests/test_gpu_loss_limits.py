"""The linear cross entropy where values leave the middle of their range."""

from __future__ import annotations

import numpy as np
import pytest

import namitorch_amd as nt
import test_gpu_loss as base
from namitorch_amd import functional as F

pytestmark = pytest.mark.gpu

DEV, DTYPES = base.DEV, base.DTYPES


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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 2.0 ** 17])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_row_gradient_that_is_not_finite(value, size, dtype):
    """It reaches its own row and the weight's gradient; the other rows' are what they are without it."""
    rows = 50
    x, weight, target = base._problem(base._rng(22), rows, 300, 64, dtype)
    # Float16 then holds the results of all three sizes, with digits to see.
    by_weight, by_x = (256.0, 1 / 256.0) if size < 1.0 else (1 / 64.0, 1 / 64.0)
    x, weight = base._tensor(base._values(x) * by_x, dtype), base._tensor(base._values(weight) * by_weight, dtype)
    target = np.where(target < 0, 3, target)
    grad = (size * (0.5 + base._rng(23).random(rows))).astype(np.float32)
    at = base._targets(target)
    _, lse = F.linear_cross_entropy_forward(x, weight, at)
    held = grad.copy()
    held[1] = value
    dx, dw = F.linear_cross_entropy_backward(nt.Tensor(held, device=DEV), x, weight, at, lse, reduction="none")
    assert not np.any(np.isfinite(dx.numpy()[1])) and not np.any(np.isfinite(dw.numpy()))
    rest = np.arange(rows) != 1
    without = base._targets(np.where(rest, target, -100))
    _, dw = F.linear_cross_entropy_backward(nt.Tensor(held, device=DEV), x, weight, without, lse, reduction="none")
    base._check_backward(nt.Tensor(dx.numpy()[rest]), dw, grad[rest].astype(np.float64), base._values(x)[rest],
                         base._values(weight), target[rest], base._values(lse)[rest], dtype, reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_of_no_class_takes_no_digits_from_others(dtype):
    """Its gradient is NaN whatever it is multiplied by, and the other rows' what they are without it."""
    rows = 50
    x, weight, target = base._problem(base._rng(26), rows, 300, 64, dtype)
    target = np.where(target < 0, 3, target)
    grad = (0.5 + base._rng(27).random(rows)).astype(np.float32)
    _, lse = F.linear_cross_entropy_forward(x, weight, base._targets(target))
    rest = np.arange(rows) != 1
    held, outside = grad.copy(), np.where(rest, target, 300)
    held[1] = 2.0 ** 60
    given = nt.Tensor(held, device=DEV)
    dx, dw = F.linear_cross_entropy_backward(given, x, weight, base._targets(outside), lse, reduction="none")
    assert np.isnan(dx.numpy()[1]).all() and np.isnan(dw.numpy()).all()
    without = base._targets(np.where(rest, target, -100))
    _, dw = F.linear_cross_entropy_backward(given, x, weight, without, lse, reduction="none")
    base._check_backward(nt.Tensor(dx.numpy()[rest]), dw, grad[rest].astype(np.float64), base._values(x)[rest],
                         base._values(weight), target[rest], base._values(lse)[rest], dtype, reduction="none")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("exponent", [-122, -60, 60, 100])
def test_row_gradients_at_the_ends_of_the_range(exponent, dtype):
    """A product of a row's gradient and a probability may lie where the dtype has few digits, or none; the weight's
    gradient does not, as x is large, and is as precise as others.  Large gradients meet a small x."""
    rows, classes, width = 60, 300, 64
    rng = base._rng(24, exponent + 200)
    x, weight, target = base._problem(rng, rows, classes, width, dtype)
    by = 2.0 ** (20 if exponent < 0 else -20)
    x, weight = base._tensor(base._values(x) * by, dtype), base._tensor(base._values(weight) / by, dtype)
    grad = (2.0 ** exponent * (0.5 + rng.random(rows))).astype(np.float32)
    at = base._targets(target)
    _, lse = F.linear_cross_entropy_forward(x, weight, at)
    dx, dw = F.linear_cross_entropy_backward(nt.Tensor(grad, device=DEV), x, weight, at, lse, reduction="none")
    base._check_backward(dx, dw, grad.astype(np.float64), base._values(x), base._values(weight), target,
                         base._values(lse), dtype, reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("rows", [1, 70])
def test_no_row_counts_under_a_gradient_that_is_not_finite(rows, grad, dtype):
    """Rows that do not count give no gradient, whatever the loss's own is."""
    x, weight, _ = base._problem(base._rng(25, rows), rows, 50, 24, dtype)
    at = base._targets(np.full(rows, -100))
    lse = nt.Tensor(np.zeros(rows, np.float32), device=DEV)
    for reduction in ("mean", "sum"):
        for given in (float(grad), nt.Tensor(np.float32(grad), device=DEV)):
            dx, dw = F.linear_cross_entropy_backward(given, x, weight, at, lse, reduction=reduction)
            assert not np.any(dx.numpy()) and not np.any(dw.numpy())
    each = nt.Tensor(np.full(rows, grad, np.float32), device=DEV)
    dx, dw = F.linear_cross_entropy_backward(each, x, weight, at, lse, reduction="none")
    assert not np.any(dx.numpy()) and not np.any(dw.numpy())
