"""The linear cross entropy on the device against the 64-bit oracle.

Bounds.  e = 2**-24, u the half ulp of the operands' dtype.  Products of 16-bit
values are exact in float32.  A logit is a float32 sum of `width` products in
some order, in steps that the matrix cores may truncate instead of round: off
by at most 2 width e sum|x w|.  Float32 operands are three bfloat16 parts: six
products a pair, each as above, and parts below 2**-23 of |x w| left out.  An
exponential of d is off by (2 |d| + 4) e (its argument's two roundings, its
own), sums of them by their chains (at most 32 terms of a tile, 16 lanes'
shares of the tiles, their join).  A result that is stored is rounded once, dz
once before (its products are then those of rounded values)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import namitorch_amd as nt
from namitorch_amd import functional as F
from oracle import loss as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E = 2.0 ** -24
HALF_ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}
DTYPES = ["float32", "float16", "bfloat16"]
# (rows, classes, width): single ones, around the tiles' edges, ragged widths and vocabularies.
SHAPES = [(1, 1, 1), (1, 300, 8), (2, 37, 5), (3, 257, 64), (4, 1000, 96), (5, 1000, 100), (17, 129, 72), (33, 700, 40),
          (64, 512, 128), (65, 513, 136), (130, 515, 200), (129, 1031, 264), (200, 64, 1000), (257, 777, 65),
          (300, 300, 321), (513, 1025, 32)]


def _rng(*key):
    return np.random.Generator(np.random.PCG64(list(key)))


def _tensor(values, dtype, shift=0):
    """A device Tensor of `values`; with `shift`, that many elements into its allocation."""
    made = nt.Tensor(np.asarray(values, dtype=np.float32), dtype=dtype, device=DEV)
    if not shift:
        return made
    room = nt.DeviceArray.empty((made.numel() + shift,), dtype, DEV)
    view = room.narrow(shift, made.numel(), made.shape)
    view.copy_from(made._data)
    return nt.Tensor._from_storage(view)


def _targets(values, dtype=np.int64):
    return nt.Tensor(np.asarray(values).astype(dtype), device=DEV)


def _values(tensor):
    return tensor.numpy().astype(np.float64)


def _problem(rng, rows, classes, width, dtype, shift=0, ignored=-100):
    weight = rng.standard_normal((classes, width)) * 2.0 / np.sqrt(width)
    target = rng.integers(0, classes, rows)
    x = rng.standard_normal((rows, width)) + rng.uniform(0, 3, (rows, 1)) * weight[target]
    if rows > 2:
        target[rng.random(rows) < 0.2] = ignored
    return _tensor(x, dtype, shift), _tensor(weight, dtype, shift), target


def _logit_error(x, weight, dtype):
    """(logits, bound of their error)."""
    width, magnitude = x.shape[1], np.abs(x) @ np.abs(weight).T
    share = 2 * width * E if dtype != "float32" else 12 * width * E + 2.0 ** -23
    return oracle.logits(x, weight), share * magnitude


def _check_forward(loss, lse, x, weight, target, dtype, ignored=-100, reduction="mean"):
    expected, expected_lse = oracle.forward(x, weight, target, ignored, "none")
    z, z_error = _logit_error(x, weight, dtype)
    classes = weight.shape[0]
    there = oracle.counted(target, ignored)
    error = z_error.max(axis=1) + (classes / 1024 + 200) * E + 4 * E * np.abs(expected_lse)
    error = np.where(there, error, 0.0)
    if lse is not None:
        assert np.all(np.abs(_values(lse) - expected_lse) <= error)
    known = np.where(there, np.asarray(target), 0)
    bad = there & ((known < 0) | (known >= classes))
    place = np.where(bad, 0, known)
    each_error = np.where(there, error + z_error[np.arange(len(known)), place] + 2 * E * np.abs(expected), 0.0)
    if reduction == "none":
        got = _values(loss)
        assert np.array_equal(np.isnan(got), bad)
        assert np.all(np.abs(got - expected)[~bad] <= each_error[~bad])
        return
    total, allowed = expected.sum(), each_error.sum()
    if reduction == "mean":
        total, allowed = total / max(1, there.sum()), allowed / max(1, there.sum())
    got = float(loss.numpy())
    if bad.any():
        assert np.isnan(got)
    else:
        assert abs(got - total) <= allowed + 2 * E * abs(total), (got, total)


def _check_backward(dx, dw, grad, x, weight, target, lse, dtype, ignored=-100, reduction="mean"):
    """Elementwise against the worst case, and as a whole against independent roundings of dz: the root mean square of
    those is below u / sqrt(3) of each term.  What is stored below the smallest normal value is off by up to half the
    smallest subnormal, however small it is: the norm of those errors is at most TINY sqrt(elements)."""
    expected_dx, expected_dw, dz = oracle.backward(grad, x, weight, target, lse, ignored, reduction)
    there = oracle.counted(target, ignored)
    u = HALF_ULP[dtype]
    z, z_error = _logit_error(np.where(there[:, None], x, 0.0), weight, dtype)
    g = np.abs(oracle.row_gradients(grad, target, ignored, reduction))[:, None]
    distance = np.abs(z - np.where(there, lse, 0.0)[:, None])
    p = np.where(there[:, None], np.exp(np.where(there[:, None], z - lse[:, None], -1.0)), 0.0)
    # Before its rounding: p's error, the subtraction's, the weight's and product's (three roundings).
    before = g * p * (np.exp(z_error) - 1 + (2 * distance + 4) * E) + E * np.abs(dz) * 4
    # A float16 dz is scaled so that the largest g is 2**14 at least; below that lie its subnormals.
    least = g.max() * 2.0 ** -14 * TINY["float16"] if dtype == "float16" else 0.0
    dz_error = before + (u * (np.abs(dz) + before) if dtype != "float32" else 2 * E * np.abs(dz)) + least
    dz_error = np.where(there[:, None], dz_error, 0.0)
    rows, classes = dz.shape
    steps = 2.0 if dtype != "float32" else 12.0
    xs = np.where(there[:, None], x, 0.0)
    for got, exact, error, sizes, count in (
            (dx, expected_dx, dz_error @ np.abs(weight), np.abs(dz) @ np.abs(weight), classes),
            (dw, expected_dw, dz_error.T @ np.abs(xs), np.abs(dz).T @ np.abs(xs), rows)):
        allowed = error + (steps * (count + 64) * E + 2.0 ** -22) * (sizes + error)
        off = np.abs(_values(got) - exact)
        bound = allowed + u * (np.abs(exact) + allowed) + TINY[dtype]
        assert np.all(off <= bound), (off.max(), (off - bound).max())
    for got, exact, squares in ((dx, expected_dx, np.square(dz) @ np.square(weight)),
                                (dw, expected_dw, np.square(dz).T @ np.square(xs))):
        if exact.size < 4096 or dtype == "float32":
            continue
        allowed = u * np.sqrt(squares.sum() / 3) + u * np.sqrt(np.square(exact).sum() / 3)
        allowed += TINY[dtype] * np.sqrt(exact.size)
        assert np.sqrt(np.square(_values(got) - exact).sum()) <= 1.2 * allowed
    assert not np.any(_values(dx)[~there])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, classes, width", SHAPES)
def test_forward(rows, classes, width, dtype):
    x, weight, target = _problem(_rng(1, rows, classes, width), rows, classes, width, dtype)
    for reduction in ("mean", "none", "sum"):
        loss, lse = F.linear_cross_entropy_forward(x, weight, _targets(target), reduction=reduction)
        assert (loss.dtype, lse.dtype, lse.shape) == (nt.float32, nt.float32, (rows,))
        _check_forward(loss, lse, _values(x), _values(weight), target, dtype, reduction=reduction)
        alone = F.linear_cross_entropy(x, weight, _targets(target, np.int32), reduction=reduction)
        assert np.array_equal(alone.bits(), loss.bits())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, classes, width", SHAPES)
def test_backward(rows, classes, width, dtype):
    rng = _rng(2, rows, classes, width)
    x, weight, target = _problem(rng, rows, classes, width, dtype)
    at = _targets(target)
    _, lse = F.linear_cross_entropy_forward(x, weight, at)
    for reduction in ("mean", "none", "sum"):
        grad = 1.0 if reduction != "none" else nt.Tensor(rng.standard_normal(rows).astype(np.float32), device=DEV)
        dx, dw = F.linear_cross_entropy_backward(grad, x, weight, at, lse, reduction=reduction)
        assert (dx.shape, dw.shape, dx.dtype, dw.dtype) == (x.shape, weight.shape, x.dtype, x.dtype)
        _check_backward(dx, dw, grad if reduction != "none" else _values(grad), _values(x), _values(weight), target,
                        _values(lse), dtype, reduction=reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, width, shift", [(40, 64, 1), (40, 64, 4), (40, 72, 3), (3, 61, 1), (2, 64, 1)])
def test_unaligned_arrays(rows, width, shift, dtype):
    """The same numbers from arrays that start anywhere, written to arrays that start anywhere."""
    x, weight, target = _problem(_rng(3, rows, width), rows, 301, width, dtype)
    at = _targets(target)
    moved = [_tensor(_values(v), dtype, shift) for v in (x, weight)]
    out = tuple(_tensor(np.ones(v.shape), dtype, shift) for v in (x, weight))
    loss, lse = F.linear_cross_entropy_forward(x, weight, at)
    again, lse_again = F.linear_cross_entropy_forward(*moved, at)
    assert np.array_equal(loss.bits(), again.bits()) and np.array_equal(lse.bits(), lse_again.bits())
    dx, dw = F.linear_cross_entropy_backward(1.0, x, weight, at, lse)
    assert F.linear_cross_entropy_backward(1.0, *moved, at, lse, out=out) == out
    assert np.array_equal(dx.bits(), out[0].bits()) and np.array_equal(dw.bits(), out[1].bits())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 40, 150])
def test_rows_that_are_not_counted_take_no_part(rows, dtype):
    """Whatever an ignored row holds, results are those of the batch without it."""
    rng = _rng(4, rows)
    x, weight, target = _problem(rng, rows, 130, 48, dtype)
    target = rng.integers(0, 130, rows)
    there = np.sort(rng.permutation(2 * rows)[:rows])
    wide, wide_target = np.full((2 * rows, 48), np.nan), np.full(2 * rows, 7)
    wide[::3] = np.inf
    wide[there], wide_target[there] = _values(x), np.where(target == 7, 8, target)
    target = wide_target[there]
    padded = _tensor(wide, dtype)
    loss, lse = F.linear_cross_entropy_forward(x, weight, _targets(target))
    again, lse_again = F.linear_cross_entropy_forward(padded, weight, _targets(wide_target), ignore_index=7)
    assert abs(float(loss.numpy()) - float(again.numpy())) <= 1e-6 * abs(float(loss.numpy()))
    dx, dw = F.linear_cross_entropy_backward(2.0, x, weight, _targets(target), lse)
    dx_again, dw_again = F.linear_cross_entropy_backward(2.0, padded, weight, _targets(wide_target), lse_again,
                                                         ignore_index=7)
    rest = np.setdiff1d(np.arange(2 * rows), there)
    assert not np.any(lse_again.numpy()[rest]) and not np.any(_values(dx_again)[rest])
    _check_forward(again, None, _values(x), _values(weight), target, dtype)
    _check_backward(nt.Tensor(dx_again.numpy()[there]), dw_again, 2.0, _values(x), _values(weight), target,
                    lse_again.numpy()[there].astype(np.float64), dtype)


@pytest.mark.parametrize("rows", [1, 3, 70])
def test_no_row_counts(rows):
    x, weight, _ = _problem(_rng(5, rows), rows, 50, 24, "bfloat16")
    at = _targets(np.full(rows, -100))
    for reduction in ("mean", "sum", "none"):
        loss, lse = F.linear_cross_entropy_forward(x, weight, at, reduction=reduction)
        assert not np.any(loss.numpy()) and not np.any(lse.numpy())
        grad = 1.0 if reduction != "none" else nt.Tensor(np.ones(rows, np.float32), device=DEV)
        out = _tensor(np.ones(x.shape), "bfloat16"), _tensor(np.ones(weight.shape), "bfloat16")
        dx, dw = F.linear_cross_entropy_backward(grad, x, weight, at, lse, reduction=reduction, out=out)
        assert not np.any(dx.numpy()) and not np.any(dw.numpy())


def test_no_rows():
    x, weight = nt.Tensor(np.zeros((0, 8), np.float32), device=DEV), _tensor(np.ones((5, 8)), "float32")
    at = _targets(np.zeros(0))
    loss, lse = F.linear_cross_entropy_forward(x, weight, at)
    assert float(loss.numpy()) == 0.0 and lse.shape == (0,)
    assert F.linear_cross_entropy(x, weight, at, reduction="none").shape == (0,)
    out = (nt.Tensor(np.zeros((0, 8), np.float32), device=DEV), _tensor(np.ones((5, 8)), "float32"))
    F.linear_cross_entropy_backward(1.0, x, weight, at, lse, out=out)
    assert not np.any(out[1].numpy())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("wrong", [-1, 200, 2 ** 31 + 5, -2 ** 40])
def test_targets_that_are_no_class(wrong, rows, dtype):
    x, weight, target = _problem(_rng(6, rows), rows, 200, 56, dtype)
    target = np.where(target < 0, 3, target)
    target[1] = wrong
    loss, lse = F.linear_cross_entropy_forward(x, weight, _targets(target), reduction="none")
    _check_forward(loss, lse, _values(x), _values(weight), target, dtype, reduction="none")
    assert np.isnan(F.linear_cross_entropy(x, weight, _targets(target)).numpy())
    dx, dw = F.linear_cross_entropy_backward(1.0, x, weight, _targets(target), lse)
    assert np.array_equal(np.isnan(dx.numpy()).all(axis=1), np.arange(rows) == 1)
    assert np.isnan(dw.numpy()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 40])
def test_far_logits(rows, dtype):
    """Logits of hundreds, all far below zero or far above it, and ones that dwarf the others."""
    rng = _rng(7, rows)
    weight = _tensor(rng.standard_normal((333, 16)) + 3.0, dtype)
    x = _tensor(rng.standard_normal((rows, 16)) + np.linspace(-8, 8, rows)[:, None], dtype)
    target = rng.integers(0, 333, rows)
    loss, lse = F.linear_cross_entropy_forward(x, weight, _targets(target), reduction="none")
    _check_forward(loss, lse, _values(x), _values(weight), target, dtype, reduction="none")
    dx, dw = F.linear_cross_entropy_backward(1.0, x, weight, _targets(target), lse)
    _check_backward(dx, dw, 1.0, _values(x), _values(weight), target, _values(lse), dtype)


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(value, rows):
    """They reach their own row alone, where all that the row gives is NaN."""
    for dtype in DTYPES:
        x, weight, target = _problem(_rng(8, rows), rows, 150, 24, dtype)
        target = np.where(target < 0, 3, target)
        values = _values(x)
        values[1, 5] = value
        loss, lse = F.linear_cross_entropy_forward(_tensor(values, dtype), weight, _targets(target), reduction="none")
        assert np.array_equal(np.isnan(loss.numpy()), np.arange(rows) == 1)
        dx, _ = F.linear_cross_entropy_backward(1.0, _tensor(values, dtype), weight, _targets(target), lse)
        assert np.array_equal(np.isnan(dx.numpy()).all(axis=1), np.arange(rows) == 1)


@pytest.mark.parametrize("grad", [1.0, 65536.0, 2.0 ** -20, 0.0, -3.0])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_loss_scales(grad, dtype):
    """Float16's small gradients are what the formulas say, rounded once at the end."""
    x, weight, target = _problem(_rng(9), 90, 700, 64, dtype)
    at = _targets(target)
    _, lse = F.linear_cross_entropy_forward(x, weight, at)
    for given in (grad, nt.Tensor(np.float32(grad), device=DEV)):
        dx, dw = F.linear_cross_entropy_backward(given, x, weight, at, lse)
        _check_backward(dx, dw, grad, _values(x), _values(weight), target, _values(lse), dtype)


def test_leading_shapes_and_given_results():
    x, weight, target = _problem(_rng(10), 60, 90, 40, "bfloat16")
    at = _targets(target)
    loss, lse = F.linear_cross_entropy_forward(x, weight, at, reduction="none")
    dx, dw = F.linear_cross_entropy_backward(loss, x, weight, at, lse, reduction="none")
    folded = nt.Tensor._from_storage(x._data.narrow(0, 2400, (3, 20, 40)))
    at_folded = _targets(target.reshape(3, 20))
    out = tuple(nt.Tensor(np.zeros((3, 20), np.float32), device=DEV) for _ in range(2))
    made = F.linear_cross_entropy_forward(folded, weight, at_folded, reduction="none", out=out)
    assert made == out and made[0].shape == (3, 20)
    assert np.array_equal(loss.numpy(), out[0].numpy().reshape(-1)) and out[0]._version == 1
    dx2, dw2 = F.linear_cross_entropy_backward(out[0], folded, weight, at_folded, out[1], reduction="none")
    assert dx2.shape == (3, 20, 40)
    assert np.array_equal(dx.numpy(), dx2.numpy().reshape(60, 40)) and np.array_equal(dw.bits(), dw2.bits())
    single = nt.Tensor._from_storage(x._data.narrow(0, 40, (40,)))
    loss1 = F.linear_cross_entropy(single, weight, _targets(int(abs(target[0]) % 90)), reduction="none")
    assert loss1.shape == ()


@pytest.mark.parametrize("dtype", DTYPES)
def test_results_repeat(dtype):
    x, weight, target = _problem(_rng(11), 700, 900, 128, dtype)
    at = _targets(target)
    first = F.linear_cross_entropy_forward(x, weight, at)
    grads = F.linear_cross_entropy_backward(1.0, x, weight, at, first[1])
    for _ in range(3):
        again = F.linear_cross_entropy_forward(x, weight, at)
        assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(first, again))
        again = F.linear_cross_entropy_backward(1.0, x, weight, at, again[1])
        assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype, rows, classes, width", [("bfloat16", 16000, 20011, 64), ("float16", 5000, 70000, 40),
                                                         ("float32", 3000, 33000, 24)])
def test_pieces_of_the_vocabulary(dtype, rows, classes, width):
    """More than one piece, against PyTorch in 64 bits: as a whole, with independent roundings (see _check_backward)."""
    generator = torch.Generator(device="cuda").manual_seed(12)
    kind = getattr(torch, dtype)
    weight = (torch.randn(classes, width, generator=generator, device="cuda") * 0.3).to(kind)
    x = torch.randn(rows, width, generator=generator, device="cuda").to(kind)
    target = torch.randint(0, classes, (rows,), generator=generator, device="cuda")
    target[::7] = -100
    wrap = nt.Tensor._from_storage
    loss, lse = F.linear_cross_entropy_forward(wrap(x), wrap(weight), wrap(target))
    there = target != -100
    total, dw = 0.0, torch.zeros(classes, width, dtype=torch.float64, device="cuda")
    dx = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    squares = torch.zeros_like(dw)
    kept = torch.from_numpy(lse.numpy()).cuda()
    for first in range(0, rows, 1000):
        part = slice(first, first + 1000)
        z = torch.mm(x[part].double(), weight.double().t())
        expected = torch.logsumexp(z, dim=1)
        assert (kept[part] - expected)[there[part]].abs().max() < 1e-5
        index = target[part].clamp(min=0)
        total += ((expected - z.gather(1, index[:, None])[:, 0]) * there[part]).sum().item()
        dz = torch.exp(z - kept[part].double()[:, None])
        dz[torch.arange(len(index), device="cuda"), index] -= 1.0
        dz *= (there[part] / there.sum())[:, None]
        dx[part] = torch.mm(dz, weight.double())
        dw += torch.mm(dz.t().contiguous(), x[part].double())
        squares += torch.mm(dz.square().t().contiguous(), x[part].double().square())
        del z, dz
    assert abs(float(loss.numpy()) - total / there.sum().item()) < 1e-5
    got_dx, got_dw = F.linear_cross_entropy_backward(1.0, wrap(x), wrap(weight), wrap(target), lse)
    u = HALF_ULP[dtype]
    # Independent errors of dz (u of each, or float32's sums and exponentials, some 2**-20) and the final rounding.
    share = u if dtype != "float32" else 2.0 ** -20
    for got, exact, by in ((got_dw, dw, squares), (got_dx, dx, None)):
        got = torch.from_numpy(got.numpy()).cuda().double()
        terms = by.sum().sqrt() if by is not None else 2.0 * exact.norm() + 1e-30
        assert (got - exact).norm() <= 1.2 * share * (terms + exact.norm())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, classes, width", [(2500, 90, 24), (1500, 700, 72), (4000, 5, 8), (3000, 300, 100)])
def test_many_rows_of_few_classes(rows, classes, width, dtype):
    """The weight's gradient is a few tiles of a long sum, which is split."""
    x, weight, target = _problem(_rng(16, rows, classes), rows, classes, width, dtype)
    at = _targets(target)
    loss, lse = F.linear_cross_entropy_forward(x, weight, at)
    _check_forward(loss, lse, _values(x), _values(weight), target, dtype)
    dx, dw = F.linear_cross_entropy_backward(1.0, x, weight, at, lse)
    _check_backward(dx, dw, 1.0, _values(x), _values(weight), target, _values(lse), dtype)
    again = F.linear_cross_entropy_backward(1.0, x, weight, at, lse)
    assert np.array_equal(dx.bits(), again[0].bits()) and np.array_equal(dw.bits(), again[1].bits())


def test_streams():
    """Calls of two streams at once: each is what it is alone."""
    problems = [_problem(_rng(13, k), 300 + 50 * k, 2000, 256, "bfloat16") for k in range(2)]
    expected = []
    for x, weight, target in problems:
        loss, lse = F.linear_cross_entropy_forward(x, weight, _targets(target))
        expected.append([loss, lse, *F.linear_cross_entropy_backward(1.0, x, weight, _targets(target), lse)])
    at = [_targets(target) for _, _, target in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    for _ in range(4):
        made = [None, None]
        for k, (x, weight, _) in enumerate(problems):
            with torch.cuda.stream(streams[k]):
                loss, lse = F.linear_cross_entropy_forward(x, weight, at[k])
                made[k] = [loss, lse, *F.linear_cross_entropy_backward(1.0, x, weight, at[k], lse)]
        torch.cuda.synchronize()
        for k in range(2):
            assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(expected[k], made[k]))


def test_a_capture_is_refused():
    x, weight, target = _problem(_rng(14), 8, 40, 16, "float32")
    at = _targets(target)
    loss, lse = F.linear_cross_entropy_forward(x, weight, at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    out = nt.Tensor(np.zeros((8, 16), np.float32), device=DEV)
    with torch.cuda.graph(graph):
        F.layer_norm(x, 16, out=out)
        with pytest.raises(RuntimeError, match="capture"):
            F.linear_cross_entropy_forward(x, weight, at, out=(loss, lse))
        with pytest.raises(RuntimeError, match="capture"):
            F.linear_cross_entropy_backward(1.0, x, weight, at, lse, out=(out, weight))
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.bits(), F.layer_norm(x, 16).bits())


def test_gradients_reach_the_optimizer():
    """A tied-head training step as a program makes it: loss, gradients, accumulation, clip and AdamW."""
    rng = _rng(15)
    weight = nt.Parameter((rng.standard_normal((120, 32)) * 0.2).astype(np.float32), dtype="bfloat16", device=DEV)
    optimizer = nt.optim.AdamW([weight], lr=1e-2, master_weights=True)
    x, target = _tensor(rng.standard_normal((64, 32)), "bfloat16"), _targets(rng.integers(0, 120, 64))
    before = weight.numpy().copy()
    loss, lse = F.linear_cross_entropy_forward(x, weight, target)
    _, grad = F.linear_cross_entropy_backward(1.0, x, weight, target, lse)
    expected = _values(grad)
    nt.accumulate_grads([weight], [grad])
    assert np.array_equal(_values(weight.grad), expected)
    nt.optim.clip_grad_norm_([weight], 1.0)
    optimizer.step()
    assert np.any(weight.numpy() != before)
    with nt.no_grad(), pytest.raises(ValueError, match="overlap"):
        F.linear_cross_entropy_backward(1.0, x, weight, target, lse, out=(None, weight))
