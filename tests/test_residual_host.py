"""Layer norm and dropout without a GPU: the generator's published answers,
the 64-bit oracle's gradients against differences, and what the functional
entry points refuse before any device is asked."""

from __future__ import annotations

import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import namitorch_amd as nt
from namitorch_amd import functional as F
from oracle import residual


# Known answers of Philox4x32-10 published with the paper: (counter, key, output).
KNOWN = [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
]


@pytest.mark.parametrize("counter, key, answer", KNOWN)
def test_philox_known_answers(counter, key, answer):
    assert tuple(int(word) for word in residual.philox(counter, key)) == answer


def test_numbers_place_halves_of_words():
    seed, offset = 0x299F31D0A4093822, 0x0370734413198A2E
    group = 0x85A308D3243F6A88 & ((1 << 61) - 1)
    words = [int(w) for w in residual.philox((group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32),
                                             (seed & 0xFFFFFFFF, seed >> 32))]
    got = residual.numbers(np.uint64(group) * np.uint64(8) + np.arange(8, dtype=np.uint64), seed, offset)
    assert got.tolist() == [half for word in words for half in (word & 0xFFFF, word >> 16)]


def test_masks_of_other_seeds_and_offsets_are_unrelated():
    base = residual.mask((4096,), 0.5, 7, 3) != 0
    for other in ((8, 3), (7, 4), (7 + (1 << 32), 3), (7, 3 + (1 << 32))):
        same = (residual.mask((4096,), 0.5, *other) != 0) == base
        # Agreement of independent fair bits: 2048 +- 32 (one standard deviation); six of them.
        assert abs(int(same.sum()) - 2048) < 192


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_dropped_share(p):
    n = 1 << 18
    dropped = int((residual.mask((n,), p, 11, 5) == 0).sum())
    assert abs(dropped - n * p) < 6 * math.sqrt(n * p * (1 - p)) + n / 65536


def test_oracle_gradient_against_differences():
    """Central differences of sum(dy * layer_norm(x)): their own error is the third derivative's step^2 and the
    rounding of the function over the step, both below 1e-7 here."""
    rng = np.random.Generator(np.random.PCG64(3))
    x, dy = rng.standard_normal((3, 7)), rng.standard_normal((3, 7))
    w, b = 1 + 0.3 * rng.standard_normal(7), rng.standard_normal(7)
    eps, step = 1e-5, 1e-5
    _, mean, rstd = residual.layer_norm(x, w, b, eps)
    dx, dw, db = residual.layer_norm_backward(dy, x, mean, rstd, w)

    def slope(array, gradient):
        found = np.empty(array.shape)
        for index in np.ndindex(array.shape):
            kept = array[index]
            values = []
            for moved in (kept + step, kept - step):
                array[index] = moved
                values.append((dy * residual.layer_norm(x, w, b, eps)[0]).sum())
            array[index] = kept
            found[index] = (values[0] - values[1]) / (2 * step)
        assert np.allclose(found, gradient, rtol=0, atol=1e-7)

    slope(x, dx)
    slope(w, dw)
    slope(b, db)


def test_host_tensors_are_refused():
    x = nt.Tensor(np.zeros((2, 4), np.float32))
    s = nt.Tensor(np.zeros(2, np.float32))
    for call in (lambda: F.layer_norm(x, 4), lambda: F.layer_norm_forward(x, 4),
                 lambda: F.layer_norm_backward(x, x, s, s), lambda: F.dropout(x, seed=1),
                 lambda: F.dropout_backward(x, seed=1), lambda: F.dropout_add_layer_norm(x, x, 4),
                 lambda: F.dropout_add_layer_norm_backward(x, None, x, s, s)):
        with pytest.raises(RuntimeError, match="only on HIP devices"):
            call()


def test_arrays_are_refused():
    with pytest.raises(TypeError, match="input must be a NamiTorch Tensor, got ndarray"):
        F.layer_norm(np.zeros((2, 4), np.float32), 4)
    with pytest.raises(TypeError, match="out must be a tuple of 3"):
        F.layer_norm_forward(nt.Tensor(np.zeros((2, 4), np.float32)), 4, out=(None,))


@pytest.mark.parametrize("p, threshold", [(0.0, 0), (0.1, 6554), (0.5, 32768), (1.0, 65536), (1e-6, 0), (1 - 1e-6, 65536)])
def test_threshold_is_the_nearest_multiple(p, threshold):
    assert F._threshold(p) == threshold


def test_scalar_arguments():
    for bad in (-0.1, 1.5, math.nan, math.inf):
        with pytest.raises(ValueError, match="p must be between 0 and 1"):
            F._threshold(bad)
    for bad in ("0.1", True, None):
        with pytest.raises(TypeError, match="p must be a real number"):
            F._threshold(bad)
    for bad in (-1, 1 << 64):
        with pytest.raises(ValueError, match=r"seed must be in \[0, 2\*\*64\)"):
            F._counter(bad, "seed")
    for bad in (1.0, True, None):
        with pytest.raises(TypeError, match="seed must be an integer"):
            F._counter(bad, "seed")
    for bad in (-1e-5, math.inf, math.nan):
        with pytest.raises(ValueError, match="eps must be finite and nonnegative"):
            F._epsilon(bad)
    assert F._counter(np.uint64((1 << 64) - 1), "seed") == (1 << 64) - 1


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_generator_header_on_the_host(tmp_path):
    source = Path(__file__).resolve().parent / "host" / "philox_test.cpp"
    binary = tmp_path / "philox_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(source), "-o", str(binary)], check=True)
    result = subprocess.run([str(binary)], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout + result.stderr
