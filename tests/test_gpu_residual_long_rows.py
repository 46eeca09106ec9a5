"""Rows of 2^20 and more elements, with bounds that do not grow with them.

A lane adds its share of a row in 64 bits, which leaves float32 nothing to
lose, and rounds it once; six exchanges join the lanes of a wave and four
additions the waves: a float32 chain of eleven, twelve with some slack,
whatever the width.  Values of one sign are what a longer chain shows in."""

from __future__ import annotations

import numpy as np
import pytest
import test_gpu_residual as base

from namitorch_amd import functional as F

pytestmark = pytest.mark.gpu

LONG = (1 << 20) + 5


@pytest.fixture(autouse=True)
def short_chains(monkeypatch):
    monkeypatch.setattr(base, "_chain", lambda count: 12)


@pytest.mark.parametrize("width", [LONG, 1 << 24])
def test_constant_rows(width):
    """The mean is the value, the output the bias."""
    x = base._tensor(np.full((1, width), np.float32(0.1)), "float32")
    y, mean, rstd = F.layer_norm_forward(x, width)
    base._check_forward(np.full((1, width), np.float64(np.float32(0.1))), np.zeros((1, width)), y, mean, rstd, None, None,
                        "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("level", [0.0, 3.0, 1000.0])
def test_norm(level, dtype):
    rng = base._rng(40, int(level))
    x = base._tensor(level + rng.standard_normal((2, LONG)), dtype)
    w, b = base._tensor(1 + 0.3 * rng.standard_normal(LONG), "float32"), base._tensor(rng.standard_normal(LONG), "float32")
    y, mean, rstd = F.layer_norm_forward(x, LONG, w, b)
    base._check_forward(base._values(x), np.zeros((2, LONG)), y, mean, rstd, base._values(w), base._values(b), dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("level", [0.0, 2.0])
def test_gradients(level, dtype):
    rng = base._rng(41, int(level))
    x = base._tensor(rng.standard_normal((2, LONG)), dtype)
    dy = base._tensor(level + 0.1 * rng.standard_normal((2, LONG)), dtype)
    w = base._tensor(1 + 0.01 * rng.standard_normal(LONG), "float32")
    _, mean, rstd = F.layer_norm_forward(x, LONG, w)
    dx, dw, _ = F.layer_norm_backward(dy, x, mean, rstd, w)
    expected, allowed = base._backward_bounds(*(base._values(v) for v in (dy, x, mean, rstd, w)))
    base._near(dx, expected[0], allowed[0], dtype, "grad_input")
    base._near(dw, expected[1], allowed[1], "float32", "grad_weight")


def test_edge():
    rng = base._rng(42)
    x, r = (base._tensor(0.5 + 0.1 * rng.standard_normal((2, LONG)), "float32") for _ in range(2))
    call = dict(p=0.1, seed=17, offset=4)
    y, total, mean, rstd = F.dropout_add_layer_norm_forward(x, r, LONG, **call)
    t, t_error = base._total(base._values(x), base._values(r), 0.1, 17, 4)
    base._near(total, t, t_error, "float32", "total")
    base._check_forward(t, t_error, y, mean, rstd, None, None, "float32")
    dy = base._tensor(2 + 0.1 * rng.standard_normal((2, LONG)), "float32")
    dx, dr, _, _ = F.dropout_add_layer_norm_backward(dy, None, total, mean, rstd, **call)
    expected, allowed = base._backward_bounds(*(base._values(v) for v in (dy, total, mean, rstd)), None)
    base._near(dr, expected[0], allowed[0], "float32", "grad_residual")
    factor = base.residual.mask((2, LONG), 0.1, 17, 4)
    base._near(dx, expected[0] * factor, (allowed[0] + 2 * base.E * np.abs(expected[0])) * factor, "float32", "grad_input")
