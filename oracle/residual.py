"""Layer norm, dropout and the residual edge in 64 bits, from their formulas.

Inputs are the values the device arrays hold (float arrays of any width);
results are float64, not rounded to a storage dtype."""

from __future__ import annotations

import numpy as np

_WORD = np.uint64(0xFFFFFFFF)
_SHIFT = np.uint64(32)


def philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): four 32-bit words
    per counter.  `counter`: four words (arrays of equal shape or scalars),
    `key`: two integers."""
    a, b, c, d = (np.asarray(word, dtype=np.uint64) for word in counter)
    k0, k1 = key
    for _ in range(10):
        left, right = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = ((right >> _SHIFT) ^ b ^ np.uint64(k0), right & _WORD,
                      (left >> _SHIFT) ^ d ^ np.uint64(k1), left & _WORD)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return a, b, c, d


def numbers(indices, seed: int, offset: int) -> np.ndarray:
    """The 16-bit number of each element index."""
    indices = np.asarray(indices, dtype=np.uint64)
    group = indices >> np.uint64(3)
    words = philox((group & _WORD, group >> _SHIFT, offset & 0xFFFFFFFF, offset >> 32),
                   (seed & 0xFFFFFFFF, seed >> 32))
    place = (indices & np.uint64(7)).astype(np.int64)
    stacked = np.stack([np.broadcast_to(word, indices.shape) for word in words])
    word = np.take_along_axis(stacked, (place // 2)[None], axis=0)[0]
    return ((word >> (np.uint64(16) * (place % 2).astype(np.uint64))) & np.uint64(0xFFFF)).astype(np.int64)


def mask(shape, p: float, seed: int, offset: int, first: int = 0) -> np.ndarray:
    """Factor of each element (0 where dropped) of a tensor of `shape` whose
    first element has flat index `first`."""
    threshold = round(p * 65536)
    count = int(np.prod(shape, dtype=np.int64))
    kept = numbers(np.arange(count, dtype=np.uint64) + np.uint64(first), seed, offset) >= threshold
    factor = 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0
    return np.where(kept, factor, 0.0).reshape(shape)


def dropout(x, p: float, seed: int, offset: int, first: int = 0) -> np.ndarray:
    factors = mask(np.shape(x), p, seed, offset, first)
    with np.errstate(invalid="ignore"):
        return np.where(factors == 0.0, 0.0, np.asarray(x, dtype=np.float64) * factors)


def layer_norm(x, weight, bias, eps: float):
    """(y, mean, rstd) of the rows of a 2-d array."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        mean = x.mean(axis=1)
        rstd = 1.0 / np.sqrt(np.square(x - mean[:, None]).mean(axis=1) + eps)
        y = (x - mean[:, None]) * rstd[:, None]
        if weight is not None:
            y = y * np.asarray(weight, dtype=np.float64)
        if bias is not None:
            y = y + np.asarray(bias, dtype=np.float64)
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight):
    """(dx, dweight, dbias) of the rows of 2-d arrays, with the statistics as given."""
    dy, x = np.asarray(dy, dtype=np.float64), np.asarray(x, dtype=np.float64)
    mean, rstd = (np.asarray(v, dtype=np.float64)[:, None] for v in (mean, rstd))
    with np.errstate(invalid="ignore"):
        h = (x - mean) * rstd
        g = dy if weight is None else dy * np.asarray(weight, dtype=np.float64)
        dx = rstd * (g - g.mean(axis=1, keepdims=True) - h * (g * h).mean(axis=1, keepdims=True))
        return dx, (dy * h).sum(axis=0), dy.sum(axis=0)
