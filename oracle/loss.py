"""Softmax cross entropy of a linear layer in 64 bits, from its formulas.

Inputs are the values the device arrays hold (float arrays of any width);
results are float64, not rounded to a storage dtype."""

from __future__ import annotations

import numpy as np


def counted(target, ignored: int = -100) -> np.ndarray:
    return np.asarray(target) != ignored


def logits(x, weight) -> np.ndarray:
    return np.asarray(x, dtype=np.float64) @ np.asarray(weight, dtype=np.float64).T


def forward(x, weight, target, ignored: int = -100, reduction: str = "mean"):
    """(loss, lse): lse and each row's loss are zero where the target is `ignored`."""
    target = np.asarray(target)
    there = counted(target, ignored)
    rows, classes = len(target), np.shape(weight)[0]
    lse, each = np.zeros(rows), np.zeros(rows)
    z = logits(np.asarray(x)[there], weight)
    most = z.max(axis=1, keepdims=True)
    lse[there] = np.log(np.exp(z - most).sum(axis=1)) + most[:, 0]
    index = target[there]
    inside = (index >= 0) & (index < classes)
    own = z[np.arange(len(index)), np.where(inside, index, 0)]
    each[there] = np.where(inside, lse[there] - own, np.nan)
    if reduction == "none":
        return each, lse
    total = each.sum()
    return (total / max(1, there.sum()) if reduction == "mean" else total), lse


def row_gradients(grad_loss, target, ignored: int = -100, reduction: str = "mean") -> np.ndarray:
    """The gradient of each row's loss."""
    there = counted(target, ignored)
    grad = np.broadcast_to(np.asarray(grad_loss, dtype=np.float64), there.shape)
    if reduction == "mean":
        grad = grad / max(1, there.sum())
    return np.where(there, grad, 0.0)


def backward(grad_loss, x, weight, target, lse, ignored: int = -100, reduction: str = "mean"):
    """(dx, dweight, dz) with lse as given."""
    target = np.asarray(target)
    there = counted(target, ignored)
    grad = row_gradients(grad_loss, target, ignored, reduction)
    x, weight = np.asarray(x, dtype=np.float64), np.asarray(weight, dtype=np.float64)
    dz = np.zeros((len(target), weight.shape[0]))
    part = np.exp(logits(x[there], weight) - np.asarray(lse, dtype=np.float64)[there, None])
    index = target[there]
    inside = (index >= 0) & (index < weight.shape[0])
    part[np.flatnonzero(inside), index[inside]] -= 1.0
    part *= np.where(inside, grad[there], np.nan)[:, None]
    dz[there] = part
    return dz @ weight, dz[there].T @ x[there], dz
