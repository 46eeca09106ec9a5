"""Layer norm, dropout and the residual edge on the device against the 64-bit
oracle, elementwise.

Bounds.  Values are rounded once to the result's dtype (relative half ulp u;
half of the smallest subnormal below).  Before that every operation is float32
with unit roundoff e = 2**-24, and a float32 sum of n terms in any order whose
longest chain of additions has length k is off by at most k e sum|terms|
(higher orders are below the slack of k).  A row's sum has chains of at most
`_chain(width)`: each lane adds its share, then lanes and waves are joined.
The errors of mean, rstd, h and the products carry through the formulas as
written at each bound."""

from __future__ import annotations

import gc

import numpy as np
import pytest
import torch

import namitorch_amd as nt
from namitorch_amd import _native, functional as F
from oracle import residual

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E = 2.0 ** -24
HALF_ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}
PAIRS = [("float32", "float32"), ("float16", "float16"), ("float16", "float32"), ("bfloat16", "bfloat16"),
         ("bfloat16", "float32")]
# Widths around the 8-element chunks, the wave and workgroup tilings, and past the widest register tiling.
SHAPES = [(1, 1), (1, 8), (5, 3), (7, 9), (4, 64), (3, 100), (2, 768), (33, 96), (257, 40), (9, 511), (3, 1001),
          (1, 2048), (5, 2050), (2, 4096), (3, 4104), (2, 5120), (3, 8192), (2, 8191), (1, 16384), (2, 20003)]


def _chain(count):
    return count / 64 + 80


def _rng(*key):
    return np.random.Generator(np.random.PCG64(list(key)))


def _tensor(values, dtype, shift=0):
    """A device Tensor of `values`; with `shift`, `shift` elements into its allocation (so not 16-byte aligned)."""
    made = nt.Tensor(np.asarray(values, dtype=np.float32), dtype=dtype, device=DEV)
    if not shift:
        return made
    room = nt.DeviceArray.empty((made.numel() + shift,), dtype, DEV)
    view = room.narrow(shift, made.numel(), made.shape)
    view.copy_from(made._data)
    return nt.Tensor._from_storage(view)


def _inputs(rng, rows, width, dtype, weight_dtype, shift=0, bias=True):
    x = rng.standard_normal((rows, width)) + 0.5 * rng.standard_normal(width)
    w = 1 + 0.3 * rng.standard_normal(width)
    b = 0.2 * rng.standard_normal(width)
    return (_tensor(x, dtype, shift), _tensor(w, weight_dtype, shift), _tensor(b, weight_dtype, shift) if bias else None)


def _values(tensor):
    return None if tensor is None else tensor.numpy().astype(np.float64)


def _near(got, expected, allowed, dtype, what=""):
    got = got.numpy().astype(np.float64).reshape(expected.shape)
    assert np.array_equal(np.isnan(got), np.isnan(expected)), what
    fine = np.isfinite(expected)
    bound = HALF_ULP[dtype] * (np.abs(expected) + allowed) + TINY[dtype] + allowed
    off = np.abs(got - expected)[fine]
    worst = off - np.broadcast_to(bound, expected.shape)[fine]
    assert worst.size == 0 or worst.max() <= 0, (what, off.max(), worst.max())


def _check_forward(t, t_error, y, mean, rstd, w, b, dtype, eps=1e-5):
    """Statistics and output of rows `t` known in 64 bits, computed by the device with errors up to `t_error`."""
    k = _chain(t.shape[1])
    expected, m, r = residual.layer_norm(t, w, b, eps)
    level = np.abs(t).mean(axis=1)
    mean_error = k * E * level + t_error.mean(axis=1) + E * np.abs(m)
    centred = np.abs(t - m[:, None])
    centred_error = t_error + mean_error[:, None] + E * (centred + t_error + mean_error[:, None])
    # var: squares of values off by centred_error, a sum, a product; rstd: half of var's relative error.
    var = np.square(centred).mean(axis=1)
    var_error = (2 * centred * centred_error + centred_error ** 2).mean(axis=1) + (k + 3) * E * var
    rstd_error = r * (0.5 * var_error * r * r * 1.5 + 4 * E)
    scale = np.abs(w) if w is not None else 1.0
    h = centred * r[:, None]
    h_error = centred_error * r[:, None] + (centred + centred_error) * rstd_error[:, None] + E * h
    allowed = scale * h_error + 2 * E * (scale * (h + h_error) + (np.abs(b) if b is not None else 0.0))
    _near(y, expected, allowed, dtype, "output")
    if mean is not None:
        _near(mean, m, mean_error, "float32", "mean")
        _near(rstd, r, rstd_error, "float32", "rstd")


def _backward_bounds(dy, x, mean, rstd, w):
    """(dx, dw, db, allowed errors of each before rounding)."""
    rows, width = x.shape
    dx, dw, db = residual.layer_norm_backward(dy, x, mean, rstd, w)
    mean, rstd = mean[:, None], rstd[:, None]
    h = np.abs((x - mean) * rstd)
    h_error = 2 * E * h
    g = np.abs(dy * (1.0 if w is None else w))
    k = _chain(width) + 3
    level_error = k * E * g.mean(axis=1, keepdims=True)
    along = (g * h).mean(axis=1, keepdims=True)
    along_error = (k + 4) * E * along
    allowed = rstd * (E * g + level_error + h * along_error + h_error * along)
    allowed = allowed + 4 * E * rstd * (g + g.mean(axis=1, keepdims=True) + h * along)
    k = rows / 64 + 400
    magnitude = np.abs(dy)
    return (dx, dw, db), (allowed, (k + 3) * E * (magnitude * h).sum(axis=0), k * E * magnitude.sum(axis=0))


@pytest.mark.parametrize("dtype, weight_dtype", PAIRS)
@pytest.mark.parametrize("rows, width", SHAPES)
def test_layer_norm(rows, width, dtype, weight_dtype):
    rng = _rng(1, rows, width)
    x, w, b = _inputs(rng, rows, width, dtype, weight_dtype)
    y, mean, rstd = F.layer_norm_forward(x, width, w, b)
    assert (y.dtype, mean.shape, rstd.shape) == (x.dtype, (rows,), (rows,))
    _check_forward(_values(x), np.zeros((rows, width)), y, mean, rstd, _values(w), _values(b), dtype)
    assert np.array_equal(F.layer_norm(x, (width,), w, b).bits(), y.bits())


@pytest.mark.parametrize("dtype, weight_dtype", PAIRS)
@pytest.mark.parametrize("rows, width", SHAPES + [(700, 24), (1500, 768), (300, 2056)])
def test_layer_norm_backward(rows, width, dtype, weight_dtype):
    rng = _rng(2, rows, width)
    x, w, b = _inputs(rng, rows, width, dtype, weight_dtype)
    dy = _tensor(0.1 * rng.standard_normal((rows, width)), dtype)
    _, mean, rstd = F.layer_norm_forward(x, width, w, b)
    made = F.layer_norm_backward(dy, x, mean, rstd, w, b)
    expected, allowed = _backward_bounds(_values(dy), _values(x), _values(mean), _values(rstd), _values(w))
    for got, want, bound, kind, what in zip(made, expected, allowed, (dtype, weight_dtype, weight_dtype),
                                            ("grad_input", "grad_weight", "grad_bias")):
        _near(got, want, bound, kind, what)
    again = F.layer_norm_backward(dy, x, mean, rstd, w, b)
    assert all(np.array_equal(a.bits(), c.bits()) for a, c in zip(made, again))      # a fixed order of sums


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, width, shift", [(5, 768, 1), (6, 33, 3), (3, 4096, 5), (70, 1000, 2), (2, 20000, 1)])
def test_unaligned_arrays(rows, width, shift, dtype):
    rng = _rng(3, rows, width)
    x, w, b = _inputs(rng, rows, width, dtype, "float32", shift)
    dy = _tensor(rng.standard_normal((rows, width)), dtype, shift)
    # Results `shift` elements into their allocations too, with room after them that stays as it was.
    room = [nt.DeviceArray.zeros((rows * width + 64,), dtype, DEV) for _ in range(2)]
    outs = [nt.Tensor._from_storage(array.narrow(shift, rows * width, (rows, width))) for array in room]
    y, mean, rstd = F.layer_norm_forward(x, width, w, b, out=(outs[0], None, None))
    _check_forward(_values(x), np.zeros((rows, width)), y, mean, rstd, _values(w), _values(b), dtype)
    dx, dw, db = F.layer_norm_backward(dy, x, mean, rstd, w, b, out=(outs[1], None, None))
    expected, allowed = _backward_bounds(_values(dy), _values(x), _values(mean), _values(rstd), _values(w))
    for got, want, bound, kind in zip((dx, dw, db), expected, allowed, (dtype, "float32", "float32")):
        _near(got, want, bound, kind)
    for array in room:
        bits = array.raw_bits()
        assert not bits[:shift].any() and not bits[shift + rows * width:].any()


@pytest.mark.parametrize("parts", ["none", "weight", "bias"])
def test_absent_parameters(parts):
    rng = _rng(4)
    x, w, b = _inputs(rng, 6, 200, "bfloat16", "float32")
    w, b = (w if parts == "weight" else None), (b if parts == "bias" else None)
    dy = _tensor(rng.standard_normal((6, 200)), "bfloat16")
    y, mean, rstd = F.layer_norm_forward(x, 200, w, b)
    _check_forward(_values(x), np.zeros((6, 200)), y, mean, rstd, _values(w), _values(b), "bfloat16")
    dx, dw, db = F.layer_norm_backward(dy, x, mean, rstd, w, b)
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    expected, allowed = _backward_bounds(_values(dy), _values(x), _values(mean), _values(rstd), _values(w))
    for got, want, bound, kind in zip((dx, dw, db), expected, allowed, ("bfloat16", "float32", "float32")):
        if got is not None:
            _near(got, want, bound, kind)


def test_several_normalized_dimensions():
    rng = _rng(5)
    x = _tensor(rng.standard_normal((3, 2, 4, 6)), "float32")
    w, b = _tensor(rng.standard_normal((4, 6)), "float32"), _tensor(rng.standard_normal((4, 6)), "float32")
    y, mean, rstd = F.layer_norm_forward(x, (4, 6), w, b)
    assert mean.shape == (3, 2) and y.shape == x.shape
    flat = _values(x).reshape(6, 24)
    _check_forward(flat, np.zeros(flat.shape), y, mean, rstd, _values(w).ravel(), _values(b).ravel(), "float32")
    dx, dw, db = F.layer_norm_backward(x, x, mean, rstd, w, b)
    assert dx.shape == x.shape and dw.shape == db.shape == (4, 6)
    expected, allowed = _backward_bounds(flat, flat, _values(mean).ravel(), _values(rstd).ravel(), _values(w).ravel())
    for got, want, bound in zip((dx, dw, db), expected, allowed):
        _near(got, want, bound, "float32")


@pytest.mark.parametrize("edge", [False, True])
def test_no_rows(edge):
    x = nt.Tensor(np.zeros((0, 40), np.float32), dtype="bfloat16", device=DEV)
    w, b = _tensor(np.ones(40), "float32"), _tensor(np.ones(40), "float32")
    if edge:
        y, total, mean, rstd = F.dropout_add_layer_norm_forward(x, x, 40, w, b, 0.1)
        *_, dw, db = F.dropout_add_layer_norm_backward(x, None, x, mean, rstd, w, b, 0.1)
    else:
        y, mean, rstd = F.layer_norm_forward(x, 40, w, b)
        _, dw, db = F.layer_norm_backward(x, x, mean, rstd, w, b)
    assert y.shape == (0, 40) and mean.shape == (0,)
    assert not dw.numpy().any() and not db.numpy().any()
    assert F.dropout(x, 0.5, seed=1).shape == (0, 40)


@pytest.mark.parametrize("width", [96, 1001, 4096, 20003])
def test_large_mean(width):
    """Rows far from zero: the variance is of centred values (E[x^2] - E[x]^2 would lose all of it)."""
    rng = _rng(6, width)
    x = _tensor(1000 + rng.standard_normal((4, width)), "float32")
    y, mean, rstd = F.layer_norm_forward(x, width)
    _check_forward(_values(x), np.zeros((4, width)), y, mean, rstd, None, None, "float32")


@pytest.mark.parametrize("width", [40, 768, 4096, 20003])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_non_finite_rows_stay_apart(width, dtype):
    rng = _rng(7, width)
    values = rng.standard_normal((6, width))
    values[1, width // 2], values[3, 0], values[4, width - 1] = np.nan, np.inf, -np.inf
    x = _tensor(values, dtype)
    y, mean, rstd = F.layer_norm_forward(x, width)
    got = y.numpy()
    assert np.isnan(got[[1, 3, 4]]).all() and np.isfinite(got[[0, 2, 5]]).all()
    clean = values.copy()
    clean[[1, 3, 4]] = 0
    assert np.array_equal(F.layer_norm(_tensor(clean, dtype), width).bits()[[0, 2, 5]], y.bits()[[0, 2, 5]])


def test_constant_rows():
    """No variance: rstd = 1 / sqrt(eps), the output is the bias."""
    x = _tensor(np.full((3, 72), 2.5), "float16")
    b = _tensor(np.linspace(-1, 1, 72), "float16")
    y, mean, rstd = F.layer_norm_forward(x, 72, None, b, 1e-5)
    assert np.array_equal(y.bits(), np.tile(b.bits(), (3, 1))) and (mean.numpy() == 2.5).all()
    assert np.allclose(rstd.numpy(), 1e-5 ** -0.5, rtol=4 * E)


@pytest.mark.parametrize("width", [24, 768])
def test_gradient_against_differences(width):
    """The device's gradients against central differences of the device's own float32 forward pass, summed in 64 bits.
    With step s the function's rounding gives (width e sum|dy|) / s, the third derivative s**2 terms."""
    rng = _rng(8, width)
    x, w, b = (v.numpy().astype(np.float64) for v in _inputs(rng, 2, width, "float32", "float32"))
    dy = rng.standard_normal((2, width)).astype(np.float32).astype(np.float64)
    tx, tw, tb = (_tensor(v, "float32") for v in (x, w, b))
    _, mean, rstd = F.layer_norm_forward(tx, width, tw, tb)
    grads = F.layer_norm_backward(_tensor(dy, "float32"), tx, mean, rstd, tw, tb)
    step = 2.0 ** -6
    for position, array in enumerate((x, w, b)):
        direction = rng.standard_normal(array.shape).astype(np.float32).astype(np.float64)
        sums = []
        for sign in (1, -1):
            moved = [x, w, b]
            moved[position] = (array + sign * step * direction).astype(np.float32)
            out = F.layer_norm(_tensor(moved[0], "float32"), width, _tensor(moved[1], "float32"),
                               _tensor(moved[2], "float32"))
            sums.append((dy * out.numpy().astype(np.float64)).sum())
        slope = (sums[0] - sums[1]) / (2 * step)
        along = (grads[position].numpy().astype(np.float64) * direction).sum()
        # Rounding of moved inputs and outputs: values below 8, each off by a few e, over the step; then the cubic term.
        allowed = 40 * E * 8 * np.abs(dy).sum() / step + 4 * step ** 2 * np.abs(dy).sum()
        assert abs(slope - along) <= allowed, (position, slope, along, allowed)


# ---- dropout --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("count, shift", [(1, 0), (7, 0), (8, 0), (9, 1), (2047, 0), (2048, 3), (40013, 0), (1 << 20, 1)])
def test_dropout(count, shift, dtype):
    rng = _rng(9, count)
    x = _tensor(rng.standard_normal(count), dtype, shift)
    seed, offset = int(rng.integers(1 << 63)) * 2 + 1, int(rng.integers(1 << 63))
    for p in (0.1, 0.5):
        y = F.dropout(x, p, seed=seed, offset=offset)
        expected = residual.dropout(_values(x), p, seed, offset)
        assert np.array_equal(y.numpy() == 0, expected == 0)
        _near(y, expected, 2 * E * np.abs(expected), dtype)
        assert np.array_equal(F.dropout_backward(x, p, seed=seed, offset=offset).bits(), y.bits())
    assert F.dropout(x, 0.0, seed=seed) is x and F.dropout(x, 0.5, False, seed=seed) is x
    assert not F.dropout(x, 1.0, seed=seed).numpy().any()
    copy = nt.Tensor(np.zeros(count, np.float32), dtype=dtype, device=DEV)
    assert F.dropout(x, 0.0, seed=seed, out=copy) is copy and np.array_equal(copy.bits(), x.bits())
    version = x._version
    assert F.dropout(x, 0.5, seed=seed, offset=offset, out=x) is x and np.array_equal(x.bits(), y.bits())
    assert x._version == version + 1


def test_dropped_non_finite_values_are_zero():
    values = np.resize([np.nan, np.inf, -np.inf, 1.0, -0.0], 4000)
    for dtype in ("float32", "float16", "bfloat16"):
        y = F.dropout(_tensor(values, dtype), 0.5, seed=3, offset=4).numpy()
        expected = residual.dropout(values, 0.5, 3, 4)
        assert np.array_equal(y, expected, equal_nan=True)


def test_dropout_far_into_a_tensor():
    """Element indices past 2**35: group counters past 32 bits."""
    count = (1 << 35) + 4099
    if torch.cuda.mem_get_info()[0] < 2 * count + (8 << 30):
        pytest.skip("needs 77 GB of device memory")
    storage = nt.DeviceArray.empty((count,), "bfloat16", DEV)
    storage.fill_bits(0x3F80)                               # ones
    x = nt.Tensor._from_storage(storage)
    seed, offset = 12345, 678
    F.dropout(x, 0.25, seed=seed, offset=offset, out=x)
    for first, size in ((0, 4096), ((1 << 32) - 100, 4096), ((1 << 35) - 2048, 2048 + 4099)):
        got = nt.Tensor._from_storage(x._data.narrow(first, size)).numpy()
        expected = residual.dropout(np.ones(size), 0.25, seed, offset, first)
        assert np.array_equal(got == 0, expected == 0)
        _near(nt.Tensor(got, device=DEV), expected, HALF_ULP["bfloat16"] * expected, "float32")
    del x, storage
    nt.runtime.empty_cache(0)


# ---- the edge -------------------------------------------------------------------------------------
def _total(x, r, p, seed, offset):
    """(64-bit total, bound on the float32 total's error)."""
    dropped = residual.dropout(x, p, seed, offset) if p else x
    return dropped + r, 3 * E * (np.abs(dropped) + np.abs(r))


@pytest.mark.parametrize("dtype, weight_dtype", PAIRS)
@pytest.mark.parametrize("rows, width", SHAPES)
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_edge(rows, width, p, dtype, weight_dtype):
    rng = _rng(10, rows, width)
    r, w, b = _inputs(rng, rows, width, dtype, weight_dtype)
    x = _tensor(0.5 * rng.standard_normal((rows, width)), dtype)
    call = dict(p=p, seed=99, offset=rows)
    y, total, mean, rstd = F.dropout_add_layer_norm_forward(x, r, width, w, b, **call)
    t, t_error = _total(_values(x), _values(r), p, 99, rows)
    _near(total, t, t_error, dtype, "total")
    _check_forward(t, t_error, y, mean, rstd, _values(w), _values(b), dtype)
    y2, total2 = F.dropout_add_layer_norm(x, r, width, w, b, **call)
    assert np.array_equal(y2.bits(), y.bits()) and np.array_equal(total2.bits(), total.bits())

    dy = _tensor(0.1 * rng.standard_normal((rows, width)), dtype)
    dt = _tensor(0.1 * rng.standard_normal((rows, width)), dtype)
    expected, allowed = _backward_bounds(_values(dy), _values(total), _values(mean), _values(rstd), _values(w))
    for passed in (dt, None):
        dx, dr, dw, db = F.dropout_add_layer_norm_backward(dy, passed, total, mean, rstd, w, b, **call)
        more = 0.0 if passed is None else _values(dt)
        want, bound = expected[0] + more, allowed[0] + E * (np.abs(expected[0]) + np.abs(more))
        _near(dr, want, bound, dtype, "grad_residual")
        factor = residual.mask((rows, width), p, 99, rows) if p else np.ones((rows, width))
        _near(dx, want * factor, (bound + 2 * E * np.abs(want)) * factor, dtype, "grad_input")
        for got, want, bound in zip((dw, db), expected[1:], allowed[1:]):
            _near(got, want, bound, weight_dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows, width", [(37, 33), (20, 1001), (6, 2056), (3, 8191), (2, 16390)])
def test_edge_has_the_mask_of_dropout(rows, width, dtype):
    """One mask for one (seed, offset), whatever the width and alignment: the edge of zeros plus dropout."""
    x = _tensor(np.ones((rows, width)), dtype, 1)
    zero = _tensor(np.zeros((rows, width)), dtype, 3)
    _, total = F.dropout_add_layer_norm(x, zero, width, p=0.3, seed=5, offset=6)
    assert np.array_equal(total.bits(), F.dropout(x, 0.3, seed=5, offset=6).bits())
    mean, rstd = (_tensor(np.full(rows, v), "float32") for v in (0.0, 1.0))
    dx, dr, _, _ = F.dropout_add_layer_norm_backward(zero, x, x, mean, rstd, p=0.3, seed=5, offset=6)
    assert np.array_equal(dr.bits(), x.bits()) and np.array_equal(dx.bits(), total.bits())


def test_edge_drops_every_element():
    rng = _rng(11)
    r, w, b = _inputs(rng, 3, 50, "float32", "float32")
    y, total = F.dropout_add_layer_norm(_tensor(np.full((3, 50), np.nan), "float32"), r, 50, w, b, p=1.0, seed=1)
    assert np.array_equal(total.bits(), r.bits()) and np.array_equal(y.bits(), F.layer_norm(r, 50, w, b).bits())


# ---- rows past 32-bit offsets, streams, refusals ------------------------------------------------------
def test_more_than_2_to_the_32_elements():
    """The last rows of a tensor of 2**32 + elements."""
    width, rows = 4096, (1 << 20) + 3
    if torch.cuda.mem_get_info()[0] < 6 * 2 * rows * width:
        pytest.skip("needs 52 GB of device memory")
    rng = _rng(12)
    storage = nt.DeviceArray.zeros((rows, width), "bfloat16", DEV)
    tail = _tensor(rng.standard_normal((3, width)), "bfloat16")
    storage.narrow((rows - 3) * width, 3 * width, (3, width)).copy_from(tail._data)
    x = nt.Tensor._from_storage(storage)
    w = _tensor(1 + rng.standard_normal(width), "float32")
    y, total, mean, rstd = F.dropout_add_layer_norm_forward(x, x, width, w, None, 0.1, seed=3, offset=2)
    last = lambda v, n: nt.Tensor._from_storage(v._data.narrow((rows - 3) * n, 3 * n, (3, n) if n > 1 else (3,)))  # noqa: E731
    values = _values(tail)
    t = residual.dropout(values, 0.1, 3, 2, (rows - 3) * width) + values
    _near(last(total, width), t, 4 * E * np.abs(t) + 4 * E * np.abs(values), "bfloat16")
    _check_forward(t, 4 * E * (np.abs(t) + np.abs(values)), last(y, width), last(mean, 1), last(rstd, 1), _values(w),
                   None, "bfloat16")
    dx, dr, dw, db = F.dropout_add_layer_norm_backward(y, None, total, mean, rstd, w, None, 0.1, seed=3, offset=2)
    t3, m3, r3 = (_values(last(v, n)) for v, n in ((total, width), (mean, 1), (rstd, 1)))
    expected, allowed = _backward_bounds(_values(last(y, width)), t3, m3, r3, _values(w))
    _near(last(dr, width), expected[0], allowed[0], "bfloat16")
    # The other rows are zero: they add nothing to the weight's gradient.
    _near(dw, expected[1], allowed[1] * (rows / 64 + 400) / 400, "float32")
    del x, y, total, dx, dr, storage
    nt.runtime.empty_cache(0)


def test_another_stream():
    rng = _rng(13)
    x, w, b = _inputs(rng, 64, 768, "bfloat16", "float32")
    expected = F.layer_norm(x, 768, w, b).bits()
    torch.cuda.synchronize()
    side = nt.runtime.Stream(0)
    with nt.runtime.stream(side):
        y, mean, rstd = F.layer_norm_forward(x, 768, w, b)
        grads = [F.layer_norm_backward(y, x, mean, rstd, w, b) for _ in range(3)]    # one workspace after another
        assert np.array_equal(y.bits(), expected)
        assert all(np.array_equal(g[1].bits(), grads[0][1].bits()) for g in grads)


def test_refusals():
    x, w, b = _inputs(_rng(14), 4, 64, "bfloat16", "float32")
    y, mean, rstd = F.layer_norm_forward(x, 64, w, b)
    short, double = _tensor(np.zeros(63), "float32"), nt.Tensor(np.zeros((4, 64)), dtype="float64", device=DEV)
    wide = _tensor(np.zeros((4, 64)), "float32")
    host = nt.Tensor(np.ones(64, np.float32))
    stat = _tensor(np.zeros(3), "float32")
    leaf = nt.Parameter(np.zeros((4, 64), np.float32), dtype="bfloat16", device=DEV)
    cases = [
        (TypeError, "input must be float16, bfloat16 or float32", lambda: F.layer_norm(double, 64)),
        (ValueError, "trailing dimensions", lambda: F.layer_norm(x, 63)),
        (ValueError, "trailing dimensions", lambda: F.layer_norm(x, ())),
        (ValueError, "at least one element", lambda: F.layer_norm(_tensor(np.zeros((3, 0)), "float32"), 0)),
        (ValueError, "weight has shape", lambda: F.layer_norm(x, 64, short)),
        (TypeError, "weight must be bfloat16 or float32", lambda: F.layer_norm(x, 64, _tensor(np.ones(64), "float16"))),
        (TypeError, "one dtype", lambda: F.layer_norm(x, 64, w, _tensor(np.ones(64), "bfloat16"))),
        (RuntimeError, "different devices", lambda: F.layer_norm(x, 64, host)),
        (ValueError, "eps must be", lambda: F.layer_norm(x, 64, eps=-1.0)),
        (TypeError, "mean must be float32", lambda: F.layer_norm_backward(x, x, _tensor(np.zeros(4), "bfloat16"), rstd)),
        (ValueError, "mean has shape", lambda: F.layer_norm_backward(x, x, stat, rstd)),
        (ValueError, "rstd has shape", lambda: F.layer_norm_backward(x, x, mean, stat)),
        (TypeError, "grad_output has dtype", lambda: F.layer_norm_backward(wide, x, mean, rstd)),
        (ValueError, "residual has shape", lambda: F.dropout_add_layer_norm(x, _tensor(np.zeros((1, 64)), "bfloat16"), 64)),
        (ValueError, "p must be", lambda: F.dropout(x, 1.1, seed=1)),
        (TypeError, "training must be", lambda: F.dropout(x, 0.5, 1, seed=1)),
        (TypeError, "out: output has dtype", lambda: F.layer_norm(x, 64, out=wide)),
        (ValueError, "out: output has shape", lambda: F.dropout(x, seed=1, out=short)),
        (RuntimeError, "requires_grad", lambda: F.dropout(x, seed=1, out=leaf)),
        (ValueError, "no such parameter", lambda: F.layer_norm_backward(x, x, mean, rstd, w, None, out=(None, None, w))),
        (ValueError, "overlaps", lambda: F.layer_norm(x, 64, out=x)),
        (ValueError, "overlaps", lambda: F.dropout_add_layer_norm(x, y, 64, out=(y, None))),
    ]
    before = x.bits(), y.bits(), w.bits()
    for kind, message, call in cases:
        with pytest.raises(kind, match=message):
            call()
    overlapping = nt.Tensor._from_storage(x._data.reshape((256,)).narrow(8, 248))
    with pytest.raises(ValueError, match="overlaps"):
        F.dropout(nt.Tensor._from_storage(x._data.reshape((256,)).narrow(0, 248)), seed=1, out=overlapping)
    assert all(np.array_equal(a, c) for a, c in zip(before, (x.bits(), y.bits(), w.bits())))


def test_capture():
    """Captured with every result given, the forward calls replay with the inputs of the time; what allocates or
    draws a mask is refused and queues nothing."""
    x, w, b = _inputs(_rng(15), 8, 256, "float32", "float32")
    x2 = _tensor(_rng(16).standard_normal((8, 256)), "float32")
    y, mean, rstd = F.layer_norm_forward(x, 256, w, b)
    out, edge_out = nt.Tensor(np.zeros((8, 256), np.float32), device=DEV), [
        nt.Tensor(np.zeros((8, 256), np.float32), device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    gc.disable()                                         # no finalizer may run HIP calls mid-capture
    try:
        with torch.cuda.graph(graph):
            F.layer_norm(x, 256, w, b, out=out)
            F.dropout_add_layer_norm(x, out, 256, w, b, out=tuple(edge_out))
            for call in (lambda: F.layer_norm(x, 256), lambda: F.dropout(x, seed=1, out=out),
                         lambda: F.layer_norm_backward(x, x, mean, rstd, w, b),
                         lambda: F.dropout_add_layer_norm(x, x, 256, p=0.5, out=tuple(edge_out))):
                with pytest.raises(RuntimeError, match="capture"):
                    call()
    finally:
        gc.enable()
    for values in (x.numpy(), x2.numpy(), x.numpy()[::-1].copy()):
        x.copy_(values)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        expected = F.layer_norm(x, 256, w, b)
        e_out, e_total = F.dropout_add_layer_norm(x, expected, 256, w, b)
        assert np.array_equal(out.bits(), expected.bits())
        assert np.array_equal(edge_out[0].bits(), e_out.bits()) and np.array_equal(edge_out[1].bits(), e_total.bits())


def test_results_feed_a_step():
    """The weights' gradients go where a training loop puts them."""
    x, w, b = _inputs(_rng(17), 16, 96, "float32", "float32")
    params = [nt.Parameter(w, device=DEV), nt.Parameter(b, device=DEV)]
    optimizer = nt.optim.AdamW(params, lr=1e-2)
    before = [p.numpy() for p in params]
    y, mean, rstd = F.layer_norm_forward(x, 96, *params)
    _, dw, db = F.layer_norm_backward(y, x, mean, rstd, *params)
    nt.accumulate_grads(params, [dw, db])
    nt.amp.fused_step(optimizer, None, max_norm=1.0)
    for parameter, old, gradient in zip(params, before, (dw, db)):
        moved = old - parameter.numpy()
        assert (np.sign(moved) == np.sign(gradient.numpy()))[np.abs(gradient.numpy()) > 1e-3].all()


# ---- launch shapes: few and many rows, every tiling, both dropout paths -----------------------------------
MANY = [(512, 768), (513, 768), (600, 5), (2000, 33), (1100, 1001), (520, 4096), (514, 8200), (520, 1531), (4099, 16)]


@pytest.mark.parametrize("dtype, weight_dtype", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("rows, width", MANY)
def test_edge_of_many_rows(rows, width, dtype, weight_dtype):
    """Past 512 rows the weight's gradient goes through partial sums; up to there the launch sums columns."""
    rng = _rng(20, rows, width)
    t, w, b = _inputs(rng, rows, width, dtype, weight_dtype)
    dy, dt = (_tensor(0.1 * rng.standard_normal((rows, width)), dtype) for _ in range(2))
    _, mean, rstd = F.layer_norm_forward(t, width, w, b)
    call = dict(p=0.25, seed=width, offset=rows)
    dx, dr, dw, db = F.dropout_add_layer_norm_backward(dy, dt, t, mean, rstd, w, b, **call)
    expected, allowed = _backward_bounds(_values(dy), _values(t), _values(mean), _values(rstd), _values(w))
    want, more = expected[0] + _values(dt), np.abs(expected[0]) + np.abs(_values(dt))
    _near(dr, want, allowed[0] + E * more, dtype, "grad_residual")
    factor = residual.mask((rows, width), 0.25, width, rows)
    _near(dx, want * factor, (allowed[0] + E * more + 2 * E * np.abs(want)) * factor, dtype, "grad_input")
    _near(dw, expected[1], allowed[1], weight_dtype, "grad_weight")
    _near(db, expected[2], allowed[2], weight_dtype, "grad_bias")
    x = _tensor(0.5 * rng.standard_normal((rows, width)), dtype)
    y, total, mean, rstd = F.dropout_add_layer_norm_forward(x, dy, width, w, b, **call)
    t, t_error = _total(_values(x), _values(dy), 0.25, width, rows)
    _near(total, t, t_error, dtype, "total")
    _check_forward(t, t_error, y, mean, rstd, _values(w), _values(b), dtype)


@pytest.mark.parametrize("width", list(range(1, 34)) + [63, 65, 127, 129, 255, 257, 383, 385, 513, 767, 1023, 1025, 1537])
def test_every_tiling(width):
    rng = _rng(21, width)
    for rows in (3, 700):
        x, w, b = _inputs(rng, rows, width, "bfloat16", "float32")
        dy = _tensor(rng.standard_normal((rows, width)), "bfloat16")
        y, mean, rstd = F.layer_norm_forward(x, width, w, b)
        _check_forward(_values(x), np.zeros((rows, width)), y, mean, rstd, _values(w), _values(b), "bfloat16")
        made = F.layer_norm_backward(dy, x, mean, rstd, w, b)
        expected, allowed = _backward_bounds(_values(dy), _values(x), _values(mean), _values(rstd), _values(w))
        for got, want, bound, kind in zip(made, expected, allowed, ("bfloat16", "float32", "float32")):
            _near(got, want, bound, kind)


@pytest.mark.parametrize("shift", [0, 1])
def test_dropout_of_a_large_tensor(shift):
    """Past 96 MiB, where a 16-bit input is read around the caches."""
    count = (52 << 20) + 5
    room = nt.DeviceArray.empty((count + shift,), "bfloat16", DEV)
    room.fill_bits(0x4040)                                  # 3.0
    x = nt.Tensor._from_storage(room.narrow(shift, count))
    y = F.dropout(x, 0.1, seed=8, offset=9)
    for first, size in ((0, 5000), (count // 2 + 3, 5000), (count - 5000, 5000)):
        got = nt.Tensor._from_storage(y._data.narrow(first, size))
        expected = residual.dropout(np.full(size, 3.0), 0.1, 8, 9, first)
        assert np.array_equal(got.numpy() == 0, expected == 0)
        _near(got, expected, 2 * E * np.abs(expected), "bfloat16")


def test_one_row_without_leading_dimensions():
    x, w, b = _inputs(_rng(22), 1, 96, "float32", "float32")
    flat = nt.Tensor._from_storage(x._data.reshape((96,)))
    y, mean, rstd = F.layer_norm_forward(flat, 96, w, b)
    assert y.shape == (96,) and mean.shape == rstd.shape == ()
    assert np.array_equal(y.bits(), F.layer_norm(x, 96, w, b).bits()[0])
    dx, dw, db = F.layer_norm_backward(flat, flat, mean, rstd, w, b)
    assert dx.shape == dw.shape == (96,) and np.array_equal(db.bits(), flat.bits())


def test_deferred_transforms_are_seen():
    """A gradient whose unscaling is still pending is read as the unscaled values; written as `out`, it holds what the
    call wrote."""
    rng = _rng(23)
    parameter = nt.Parameter(rng.standard_normal((4, 40)).astype(np.float32), device=DEV)
    optimizer = nt.optim.AdamW([parameter], lr=1e-3)
    scaler = nt.GradScaler(init_scale=1024.0)
    scaled = rng.standard_normal((4, 40)).astype(np.float32)
    for write in (False, True):
        scaler.scale(nt.Tensor(np.float32(1.0), device=DEV))
        parameter.grad = nt.Tensor(scaled, device=DEV)
        assert scaler.unscale_(optimizer)
        if write:
            y = F.layer_norm(nt.Tensor(scaled, device=DEV), 40, out=parameter.grad)
            assert y is parameter.grad
            assert np.array_equal(y.bits(), F.layer_norm(nt.Tensor(scaled, device=DEV), 40).bits())
        else:
            y = F.dropout(parameter.grad, 0.5, seed=1)
            expected = F.dropout(nt.Tensor(scaled / np.float32(1024), device=DEV), 0.5, seed=1)
            assert np.array_equal(y.bits(), expected.bits())
        scaler.step(optimizer)
        scaler.update()


def test_library_refusals():
    """The C entries' own checks (a caller without this package's Python layer)."""
    call = _native.call
    x = torch.zeros(64, device=DEV)
    p, out = x.data_ptr(), torch.zeros(64, device=DEV).data_ptr()
    F32, F64 = _native.NT_F32, _native.NT_F64
    cases = [
        (TypeError, "float32, float16 or bfloat16", ("nt_dropout", 0, p, F64, out, 8, 1, 0, 0, None)),
        (ValueError, "0..65536", ("nt_dropout", 0, p, F32, out, 8, 65537, 0, 0, None)),
        (ValueError, "NULL", ("nt_dropout", 0, p, F32, None, 8, 1, 0, 0, None)),
        (ValueError, "not aligned", ("nt_dropout", 0, p + 2, F32, out, 8, 1, 0, 0, None)),
        (ValueError, "overlaps", ("nt_dropout", 0, p, F32, p + 4, 8, 1, 0, 0, None)),
        (ValueError, "1..2\\*\\*24", ("nt_layer_norm", 0, p, F32, None, None, F32, 1e-5, out, None, None, 1, 0, None)),
        (ValueError, "1..2\\*\\*24", ("nt_layer_norm", 0, p, F32, None, None, F32, 1e-5, out, None, None, 1,
                                      (1 << 24) + 1, None)),
        (ValueError, "too many", ("nt_layer_norm", 0, p, F32, None, None, F32, 1e-5, out, None, None, 1 << 60, 8, None)),
        (ValueError, "together", ("nt_layer_norm", 0, p, F32, None, None, F32, 1e-5, out, p + 128, None, 1, 8, None)),
        (TypeError, "weight and bias", ("nt_layer_norm", 0, p, F32, p + 64, None, _native.NT_F16, 1e-5, out, None,
                                        None, 1, 8, None)),
        (ValueError, "NULL", ("nt_layer_norm_backward", 0, p, p, F32, None, None, None, F32, out, None, None, 1, 8, None)),
        (ValueError, "overlaps", ("nt_dropout_add_layer_norm", 0, p, p, F32, None, None, F32, 1e-5, 0, 0, 0, out, out,
                                  None, None, 1, 8, None)),
        (ValueError, "0..65536", ("nt_dropout_add_layer_norm_backward", 0, p, None, p, F32, p, p, None, F32, 1 << 20, 0,
                                  0, out, out + 64, None, None, 1, 8, None)),
    ]
    for kind, message, arguments in cases:
        with pytest.raises(kind, match=message):
            call(*arguments)
    call("nt_dropout", 0, None, F32, None, 0, 1, 0, 0, None)
    call("nt_layer_norm", 0, None, F32, None, None, F32, 1e-5, None, None, None, 0, 8, None)
    assert _native.load().nt_last_error() == b""
