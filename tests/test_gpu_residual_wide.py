"""Ragged and unaligned rows of 8193 to 16384 elements, the widest that stay
in registers: three groups a lane over 512 lanes (16-bit forward, up to
12288) and two over 1024.  Few rows, whose launch also sums columns, and more
than 512, where workgroups take several rows and write partial sums."""

from __future__ import annotations

import pytest
import test_gpu_residual as base

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [8193, 8195, 10240, 12281, 12288, 12289, 14002, 16376, 16383])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_few_rows(width, p, dtype):
    base.test_layer_norm(3, width, dtype, "float32")
    base.test_layer_norm_backward(3, width, dtype, "float32")
    base.test_edge(3, width, p, dtype, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [8195, 12289, 16383])
def test_many_rows(width, dtype):
    base.test_edge_of_many_rows(530, width, dtype, "float32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width, shift", [(8200, 1), (12288, 3), (16384, 1), (16384, 5)])
def test_unaligned_rows(width, shift, dtype):
    base.test_unaligned_arrays(3, width, shift, dtype)
    base.test_unaligned_arrays(530, width, shift, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [8192, 8193, 12288, 12289, 16383, 16384])
def test_mask_of_unaligned_edges(width, dtype):
    base.test_edge_has_the_mask_of_dropout(3, width, dtype)
    base.test_edge_has_the_mask_of_dropout(515, width, dtype)
