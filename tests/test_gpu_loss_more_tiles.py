"""The linear cross entropy at sizes of each choice of tiles, element by element against 64 bits with the bounds of
test_gpu_loss_tiles.py; test_loss_rules_host.py asserts that the choices are those that stand here."""

from __future__ import annotations

import pytest

import test_gpu_loss_tiles as base

pytestmark = pytest.mark.gpu

# rows, classes, width, the logits' tile, the gradients'.
TILES = [
    (64, 50001, 264, "few", "few"),             # up to 64 rows
    (300, 3001, 520, "few", "middle"),          # small logits for want of tiles
    (65, 50001, 136, "tall", "middle"),
    (128, 150001, 1000, "tall", "middle"),      # as the next, of half a large tile's rows
    (129, 150001, 1000, "tall", "large"),       # large gradients of 129 to 256 rows
    (200, 131501, 1000, "tall", "large"),
    (300, 12001, 264, "middle", "middle"),
    (513, 25003, 264, "large", "middle"),       # the last rows and classes fill no tile
    (513, 25003, 2056, "large", "large"),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, classes, width, logits, grads", TILES)
def test_tiles(rows, classes, width, logits, grads, dtype):
    base.test_tiles(rows, classes, width, dtype)
