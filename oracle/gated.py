"""The edge after a block that is normalized on both sides, in 64 bits, from
its formulas: ``total = scale residual + gate N(x; u, k)``, ``y = N(total; w, b)``.

Arrays are two-dimensional (rows, width); a gate has one row, one for each run
of equally many rows, or one for each row.  Results are float64."""

from __future__ import annotations

import numpy as np


def _wide(gate, rows):
    """The gate's row of each row."""
    gate = np.ones((1, 1)) if gate is None else np.asarray(gate, dtype=np.float64)
    return np.repeat(gate, rows // len(gate), axis=0)


def norm(x, weight, bias, eps: float, rms: bool):
    """(N(x), mean, rstd) of rows; the mean is zero where there is none."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        mean = np.zeros(len(x)) if rms else x.mean(axis=1)
        away = x - mean[:, None]
        rstd = 1.0 / np.sqrt(np.square(away).mean(axis=1) + eps)
        y = away * rstd[:, None]
        if weight is not None:
            y = y * weight
        return (y if bias is None else y + bias), mean, rstd


def forward(x, residual, u, k, gate, w, b, scale, eps, rms):
    """(y, total, inner mean, inner rstd, mean, rstd)."""
    n, inner_mean, inner_rstd = norm(x, u, k, eps, rms)
    total = scale * np.asarray(residual, dtype=np.float64) + _wide(gate, len(n)) * n
    y, mean, rstd = norm(total, w, b, eps, rms)
    return y, total, inner_mean, inner_rstd, mean, rstd


def _norm_back(dy, x, mean, rstd, weight, rms):
    """(dx, normalized x) with the statistics as given."""
    h = (x - mean[:, None]) * rstd[:, None]
    g = dy if weight is None else dy * weight
    inner = g - h * (g * h).mean(axis=1, keepdims=True)
    if not rms:
        inner = inner - g.mean(axis=1, keepdims=True)
    return inner * rstd[:, None], h


def backward(dy, dtotal, x, total, inner_mean, inner_rstd, mean, rstd, u, k, gate, w, scale, rms):
    """(dx, dresidual, du, dk, dgate, dw, db, dt)."""
    rows, width = x.shape
    dt, h = _norm_back(dy, total, mean, rstd, w, rms)
    if dtotal is not None:
        dt = dt + dtotal
    wide = _wide(gate, rows)
    dn = dt * wide
    dx, i = _norm_back(dn, x, inner_mean, inner_rstd, u, rms)
    n = i * (1.0 if u is None else u) + (0.0 if k is None else k)
    dgate = None
    if gate is not None:
        dgate = (dt * n).reshape(len(gate), rows // len(gate), width).sum(axis=1)
    return dx, scale * dt, (dn * i).sum(axis=0), dn.sum(axis=0), dgate, (dy * h).sum(axis=0), dy.sum(axis=0), dt
