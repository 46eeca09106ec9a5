"""How the linear cross entropy is cut into pieces and tiles, without a GPU: nt_tiles.hpp built by the host compiler.
The sizes of the GPU tests have the pieces, tiles and splits that they are there for."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

import test_gpu_loss_more_tiles
import test_gpu_loss_pieces

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    source = Path(__file__).resolve().parent / "host" / "tiles_test.cpp"
    binary = tmp_path_factory.mktemp("tiles") / "tiles_test"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", str(source), "-o", str(binary)], check=True)

    def run(*arguments):
        result = subprocess.run([str(binary), *map(str, arguments)], capture_output=True, text=True)
        assert result.returncode == 0, result.stdout + result.stderr
        return result.stdout.split()

    return run


def _plan(program, dtype, rows, classes, width, backward):
    """(pieces, the logits' tile, the gradients', splits of dx and of dW)."""
    pieces, logits, grads, of_input, of_weight = program(rows, classes, width, 3 if dtype == "float32" else 1, int(backward))
    return int(pieces), logits, grads, int(of_input), int(of_weight)


def test_sizes_of_every_magnitude(program):
    assert "passed" in program()


@pytest.mark.parametrize("dtype, rows, classes, width, forward, backward", test_gpu_loss_pieces.PIECES)
def test_pieces(program, dtype, rows, classes, width, forward, backward):
    assert _plan(program, dtype, rows, classes, width, False)[0] == forward
    assert _plan(program, dtype, rows, classes, width, True)[0] == backward


def test_pieces_of_many_rows_and_of_split_weights(program):
    *problem, forward = test_gpu_loss_pieces.MANY_ROWS
    assert _plan(program, *problem, False)[0] == forward
    assert sum(_plan(program, *case[:4], True)[4] > 1 for case in test_gpu_loss_pieces.PIECES) >= 2


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, classes, width, logits, grads", test_gpu_loss_more_tiles.TILES)
def test_tiles(program, rows, classes, width, logits, grads, dtype):
    assert _plan(program, dtype, rows, classes, width, False)[1] == logits
    assert _plan(program, dtype, rows, classes, width, True)[:3] == (1, logits, grads)


def test_every_choice_of_tiles_is_there():
    assert {case[3] for case in test_gpu_loss_more_tiles.TILES} == {"large", "middle", "tall", "few"}
    assert {case[4] for case in test_gpu_loss_more_tiles.TILES} == {"large", "middle", "few"}
