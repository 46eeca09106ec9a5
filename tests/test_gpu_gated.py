"""The edge after a block that is normalized on both sides, on the device
against the 64-bit oracle, elementwise.

Bounds.  e = 2**-24, u the half ulp of a result's dtype.  Every operation
before a result's rounding is float32, and a float32 sum whose longest chain of
additions has length k is off by at most k e sum|terms| (higher orders are
below the slack of k).  A row's chains are at most `_chain(width)`: a lane's
share, then lanes and waves; a column's at most `_column_chain(rows)`: a lane's
rows, then lanes, workgroups and their slices.  Errors carry through the
formulas as written at each bound; a vector's gradient may be formed from the
sums of dt i and dt and the gate or weight afterwards, which changes no sum of
magnitudes."""

from __future__ import annotations

import gc

import numpy as np
import pytest
import torch

import namitorch_amd as nt
from namitorch_amd import functional as F
from oracle import gated as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E = 2.0 ** -24
HALF_ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}
PAIRS = [("float32", "float32"), ("float16", "float16"), ("float16", "float32"), ("bfloat16", "bfloat16"),
         ("bfloat16", "float32")]
GATES = ["none", "shared", "run", "row"]
# (runs, rows of a run, width): around the groups of eight, the lanes of a row and the widest rows in registers.
SHAPES = [(1, 1, 1), (1, 1, 8), (5, 1, 3), (2, 3, 9), (2, 2, 64), (1, 3, 100), (3, 11, 96), (1, 257, 40), (3, 3, 511),
          (1, 3, 1001), (4, 300, 24), (2, 1, 2050), (1, 2, 4096), (3, 1, 4104), (1, 3, 8192), (2, 1, 8191), (1, 2, 8200),
          (1, 3, 16384), (2, 1, 20003), (70, 9, 33), (600, 2, 16)]


def _chain(count):
    return count / 64 + 80


def _column_chain(rows):
    return rows / 64 + 400


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


def _values(tensor, shape=None):
    if tensor is None:
        return None
    made = tensor.numpy().astype(np.float64)
    return made if shape is None else made.reshape(shape)


class _Edge:
    """Inputs of one edge, as Tensors and as 64-bit rows."""

    def __init__(self, rng, runs, run, width, dtype, weight, gate="shared", gate_dtype=None, bias=True, shift=0):
        lead, rows = (runs, run), runs * run
        self.lead, self.rows, self.width, self.dtype = lead, rows, width, dtype
        vector = lambda scale, middle: _tensor(middle + scale * rng.standard_normal(width), weight, shift)  # noqa: E731
        self.u, self.w = vector(0.3, 1.0), vector(0.3, 1.0)
        self.k, self.b = (vector(0.2, 0.0), vector(0.2, 0.0)) if bias else (None, None)
        shape = {"none": None, "shared": (width,), "run": (runs, 1, width), "row": (*lead, width)}[gate]
        self.gate = None
        if shape is not None:
            self.gate = _tensor(0.5 + 0.4 * rng.standard_normal(shape), gate_dtype or dtype, shift)
        self.x = _tensor(0.5 * rng.standard_normal((*lead, width)) + 0.1, dtype, shift)
        self.residual = _tensor(rng.standard_normal((*lead, width)) + 0.5 * rng.standard_normal(width), dtype, shift)
        self.dy, self.dtotal = (_tensor(rng.standard_normal((*lead, width)), dtype, shift) for _ in range(2))
        self.vectors = (self.u, self.k, self.gate, self.w, self.b)

    def flat(self, tensor):
        return _values(tensor, (-1, self.width))

    def wide(self):
        return oracle._wide(self.flat(self.gate), self.rows)


def _near(got, expected, allowed, dtype, what):
    got = got.numpy().astype(np.float64).reshape(expected.shape)
    assert np.array_equal(np.isnan(got), np.isnan(expected)), what
    fine = np.isfinite(expected)
    bound = np.broadcast_to(HALF_ULP[dtype] * (np.abs(expected) + allowed) + TINY[dtype] + allowed, expected.shape)
    off = np.abs(got - expected)
    assert np.all(off[fine] <= bound[fine]), (what, (off - bound)[fine].max(), off[fine].max())


def _norm_errors(t, t_error, w, b, eps, rms):
    """Bounds of y, mean and rstd of rows that the device has with errors up to `t_error`."""
    k = _chain(t.shape[1])
    _, m, r = oracle.norm(t, w, b, eps, rms)
    mean_error = np.zeros(len(t)) if rms else k * E * np.abs(t).mean(axis=1) + t_error.mean(axis=1) + E * np.abs(m)
    centred = np.abs(t - m[:, None])
    centred_error = t_error + mean_error[:, None] + E * (centred + t_error + mean_error[:, None])
    # var: squares of values off by centred_error, a sum, a product; rstd: half of var's relative error.
    var = np.square(centred).mean(axis=1)
    var_error = (2 * centred * centred_error + centred_error ** 2).mean(axis=1) + (k + 3) * E * var
    rstd_error = r * (0.5 * var_error * r * r * 1.5 + 4 * E)
    scale = np.abs(w) if w is not None else 1.0
    h = centred * r[:, None]
    h_error = centred_error * r[:, None] + (centred + centred_error) * rstd_error[:, None] + E * h
    size = scale * (h + h_error) + (np.abs(b) if b is not None else 0.0)
    return scale * h_error + 2 * E * size, mean_error, rstd_error, size


def _check_forward(edge, made, scale=1.0, eps=1e-5, rms=False):
    y, total, *stats = made
    x, r = edge.flat(edge.x), edge.flat(edge.residual)
    u, k, w, b = (_values(v) for v in (edge.u, edge.k, edge.w, edge.b))
    gate = edge.flat(edge.gate) if edge.gate is not None else None
    want = oracle.forward(x, r, u, k, gate, w, b, scale, eps, rms)
    n_error, inner_mean_error, inner_rstd_error, n_size = _norm_errors(x, np.zeros(x.shape), u, k, eps, rms)
    wide = np.abs(edge.wide())
    # The gate may be multiplied into weight and bias first, the scaled residual rounds once, the sum once.
    total_error = wide * n_error + 4 * E * (wide * n_size + np.abs(scale * r))
    y_error, mean_error, rstd_error, _ = _norm_errors(want[1], total_error, w, b, eps, rms)
    _near(y, want[0], y_error, edge.dtype, "output")
    _near(total, want[1], total_error, edge.dtype, "total")
    if stats:
        names = ("inner_mean", "inner_rstd", "mean", "rstd")
        errors = (inner_mean_error, inner_rstd_error, mean_error, rstd_error)
        for name, stat, value, error in zip(names, stats, want[2:], errors):
            if rms and "mean" in name:
                assert stat is None
            else:
                assert stat.shape == edge.lead and stat.dtype is nt.float32
                _near(stat, value, error, "float32", name)


def _check_backward(edge, made, total, stats, dtotal, scale=1.0):
    rms = stats[0] is None
    x, t, dy = edge.flat(edge.x), edge.flat(total), edge.flat(edge.dy)
    dt_in = edge.flat(dtotal) if dtotal is not None else None
    u, k, w = (_values(v) for v in (edge.u, edge.k, edge.w))
    gate = edge.flat(edge.gate) if edge.gate is not None else None
    zero = np.zeros(edge.rows)
    im, ir, m, r = (zero if s is None else s.numpy().astype(np.float64).reshape(-1) for s in stats)
    *want, dt = oracle.backward(dy, dt_in, x, t, im, ir, m, r, u, k, gate, w, scale, rms)

    chain, columns = _chain(edge.width) + 3, _column_chain(edge.rows)

    def back(dy, dy_error, x, mean, rstd, weight):
        """(bound of the norm's input gradient, |normalized x|, its error)."""
        h = np.abs((x - mean[:, None]) * rstd[:, None])
        h_error = 2 * E * h
        g = np.abs(dy * weight)
        g_error = dy_error * np.abs(weight) + E * (g + dy_error * np.abs(weight))
        along = (g * h).mean(axis=1, keepdims=True)
        along_error = (chain + 4) * E * along + (g_error * (h + h_error) + g * h_error).mean(axis=1, keepdims=True)
        level = np.zeros_like(along) if rms else g.mean(axis=1, keepdims=True)
        level_error = np.zeros_like(along) if rms else chain * E * level + g_error.mean(axis=1, keepdims=True)
        inside = g_error + level_error + (h + h_error) * along_error + h_error * along
        return rstd[:, None] * (inside + 5 * E * (g + g_error + level + h * along)), h, h_error

    none = np.zeros(dy.shape)
    w1, u1 = (np.ones(edge.width) if v is None else v for v in (w, u))
    dt_error, h, h_error = back(dy, none, t, m, r, w1)
    dt_error = dt_error + E * (np.abs(dt) + dt_error) * 2
    wide = np.abs(edge.wide())
    dn, dn_error = np.abs(dt) * wide, dt_error * wide + 2 * E * (np.abs(dt) + dt_error) * wide
    dx_error, i, i_error = back(dt * edge.wide(), dn_error, x, im, ir, u1)
    n = i * np.abs(u1) + (0.0 if k is None else np.abs(k))
    n_error = (i_error + 2 * E * i) * np.abs(u1) + 2 * E * n

    def summed(value, error, axis=0):
        return error.sum(axis=axis) + (columns + 8) * E * (value + error).sum(axis=axis)

    errors = [dx_error, abs(scale) * dt_error + 2 * E * np.abs(scale * dt),
              summed(dn * i, dn_error * (i + i_error) + dn * i_error), summed(dn, dn_error), None,
              summed(np.abs(dy) * h, np.abs(dy) * h_error), summed(np.abs(dy), none)]
    if gate is not None:
        by_gate, by_gate_error = np.abs(dt) * n, dt_error * (n + n_error) + np.abs(dt) * n_error
        split = lambda v: v.reshape(len(gate), -1, edge.width)  # noqa: E731
        errors[4] = summed(split(by_gate), split(by_gate_error), axis=1)
    names = ("input", "residual", "inner_weight", "inner_bias", "gate", "weight", "bias")
    for name, got, value, error, given in zip(names, made, want, errors, (edge.x, edge.x, *edge.vectors)):
        if given is None:
            assert got is None
            continue
        assert (got.shape, got.dtype) == (given.shape, given.dtype), name
        _near(got, value, error, given.dtype.name, "grad_" + name)


def _run_forward(edge, scale=1.0, norm="layer", **more):
    return F.norm_gate_add_norm_forward(edge.x, edge.residual, edge.width, edge.u, edge.k, edge.gate, edge.w, edge.b,
                                        scale, norm=norm, **more)


def _run_backward(edge, made, dtotal, scale=1.0, **more):
    _, total, *stats = made
    return F.norm_gate_add_norm_backward(edge.dy, dtotal, edge.x, total, *stats, edge.u, edge.k, edge.gate, edge.w,
                                         edge.b, scale, **more)


@pytest.mark.parametrize("dtype, weight", PAIRS)
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("runs, run, width", SHAPES)
def test_both_passes(runs, run, width, norm, dtype, weight):
    place = SHAPES.index((runs, run, width)) + PAIRS.index((dtype, weight)) + (norm == "rms")
    gate = GATES[place % 4]
    rng = _rng(1, runs, run, width, place)
    edge = _Edge(rng, runs, run, width, dtype, weight, gate, ["float32", dtype][place % 2], bias=place % 3 != 0)
    scale = [1.0, 0.5, -1.25][place % 3]
    made = _run_forward(edge, scale, norm)
    _check_forward(edge, made, scale, rms=norm == "rms")
    alone = F.norm_gate_add_norm(edge.x, edge.residual, (width,), edge.u, edge.k, edge.gate, edge.w, edge.b, scale,
                                 norm=norm)
    assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(alone, made))
    for dtotal in (edge.dtotal, None):
        _check_backward(edge, _run_backward(edge, made, dtotal, scale), made[1], made[2:], dtotal, scale)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("runs, run, width", [(2, 5, 72), (3, 40, 200), (2, 2, 1001), (1, 9, 8208)])
def test_gates(runs, run, width, gate, dtype):
    """Every gate at sizes of each kernel, without the vectors that may be absent."""
    for norm in ("layer", "rms"):
        edge = _Edge(_rng(2, runs, run, width), runs, run, width, dtype, dtype, gate, bias=norm == "layer")
        if norm == "rms":
            edge.u = edge.w = None
            edge.vectors = (None, None, edge.gate, None, None)
        made = _run_forward(edge, 1.0, norm)
        _check_forward(edge, made, rms=norm == "rms")
        _check_backward(edge, _run_backward(edge, made, edge.dtotal), made[1], made[2:], edge.dtotal)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("gate", ["shared", "run", "row"])
@pytest.mark.parametrize("runs, run, width", [(4, 700, 64), (2, 1500, 24), (1, 4099, 16), (3, 777, 136)])
def test_many_rows(runs, run, width, gate, dtype):
    edge = _Edge(_rng(3, runs, run, width), runs, run, width, dtype, "float32", gate)
    made = _run_forward(edge)
    _check_forward(edge, made)
    _check_backward(edge, _run_backward(edge, made, edge.dtotal), made[1], made[2:], edge.dtotal)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("gate", ["shared", "run", "row"])
@pytest.mark.parametrize("width, shift", [(64, 1), (96, 3), (65, 1), (1024, 4), (8192, 1), (7, 1)])
def test_unaligned_arrays(width, shift, gate, dtype):
    """The same values from and to arrays that start anywhere."""
    plain, moved = (_Edge(_rng(4, width), 2, 6, width, dtype, dtype, gate, shift=s) for s in (0, shift))
    made = _run_forward(plain)
    shapes = [v.shape for v in made]
    out = tuple(_tensor(np.ones(s), v.dtype.name, shift) for s, v in zip(shapes, made))
    assert _run_forward(moved, out=out) == out
    assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(made, out))
    grads = _run_backward(plain, made, plain.dtotal)
    out2 = tuple(_tensor(np.ones(v.shape), v.dtype.name, shift) for v in grads)
    assert _run_backward(moved, out, moved.dtotal, out=out2) == out2
    for got in (grads, out2):
        _check_backward(plain, got, made[1], made[2:], plain.dtotal)


def test_shapes_of_gates():
    """A gate's row is that of its leading dimensions, in any shape that says so."""
    edge = _Edge(_rng(5), 6, 4, 40, "float32", "float32", "run")
    expected = _run_forward(edge)[0].bits().reshape(-1)
    x, residual = (nt.Tensor(_values(v).reshape(2, 3, 4, 40).astype(np.float32), device=DEV)
                   for v in (edge.x, edge.residual))
    gate = nt.Tensor(_values(edge.gate).reshape(2, 3, 1, 40).astype(np.float32), device=DEV)
    made = F.norm_gate_add_norm(x, residual, 40, edge.u, edge.k, gate, edge.w, edge.b)[0]
    assert np.array_equal(made.bits().reshape(-1), expected)
    both = F.norm_gate_add_norm(x, residual, (4, 40), None, None, nt.Tensor(np.ones((2, 1, 4, 40), np.float32), device=DEV))
    assert np.array_equal(both[0].bits(), F.norm_gate_add_norm(x, residual, (4, 40))[0].bits())


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("width", [128, 9000])
def test_a_closed_gate(width, dtype):
    """A gate of zero leaves the residual stream as it is (to the bit), and its scale alone where that is not one."""
    edge = _Edge(_rng(6), 1, 20, width, dtype, dtype, "none")
    edge.gate = _tensor(np.zeros(width), dtype)
    for scale in (1.0, 2.0):
        made = _run_forward(edge, scale)
        assert np.array_equal(made[1].numpy(), scale * edge.residual.numpy())
        _check_forward(edge, made, scale)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("width", [64, 1000, 9000])
def test_rows_that_are_not_finite(width, norm):
    """They reach their own row; the rows beside it are what they were."""
    edge = _Edge(_rng(7, width), 1, 9, width, "float32", "float32")
    y, total, *_ = _run_forward(edge, norm=norm)
    values = edge.x.numpy().copy()
    values[0, 3, width // 2], values[0, 5, 0] = np.nan, np.inf
    edge.x = _tensor(values, "float32")
    got_y, got_total, *_ = _run_forward(edge, norm=norm)
    rest = [k for k in range(9) if k not in (3, 5)]
    assert np.isnan(got_y.numpy()[0, [3, 5]]).all()
    for a, b in ((y, got_y), (total, got_total)):
        assert np.array_equal(a.numpy()[0, rest], b.numpy()[0, rest])


@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_constant_rows(norm):
    """No deviation at all: the norm is its bias."""
    x = _tensor(np.full((4, 96), 3.0), "float32")
    k = _tensor(np.linspace(-1, 1, 96), "float32")
    y, total = F.norm_gate_add_norm(x, x, 96, None, k, norm="layer")
    assert np.allclose(total.numpy(), 3.0 + k.numpy(), rtol=0, atol=1e-5)
    zeros = _tensor(np.zeros((4, 96)), "float32")
    y, total = F.norm_gate_add_norm(zeros, zeros, 96, norm=norm)
    assert not np.any(y.numpy()) and not np.any(total.numpy())


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_no_rows(lead):
    make = lambda shape, value=0.0: nt.Tensor(np.full(shape, value, np.float32), device=DEV)  # noqa: E731
    x, vector = make((*lead, 16)), make(16, 1.0)
    made = F.norm_gate_add_norm_forward(x, x, 16, vector, vector, vector, vector, vector)
    assert made[0].shape == x.shape and made[5].shape == lead
    out = (make((*lead, 16)), make((*lead, 16)), *(make(16, 1.0) for _ in range(5)))
    F.norm_gate_add_norm_backward(x, None, x, x, *made[2:], vector, vector, vector, vector, vector, out=out)
    assert not any(np.any(v.numpy()) for v in out[2:])


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("runs, run, width", [(3, 700, 200), (2, 3, 8192), (40, 33, 64)])
def test_results_repeat(runs, run, width, gate):
    edge = _Edge(_rng(8, runs), runs, run, width, "bfloat16", "float32", gate)
    made = _run_forward(edge)
    grads = _run_backward(edge, made, edge.dtotal)
    for _ in range(3):
        again = _run_forward(edge)
        assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(made, again))
        again = _run_backward(edge, made, edge.dtotal)
        assert all(a is b is None or np.array_equal(a.bits(), b.bits()) for a, b in zip(grads, again))


def test_captured_forward_calls():
    """With every result given, a forward call is replayed; what needs workspace or allocates is refused."""
    edge = _Edge(_rng(9), 2, 3, 96, "bfloat16", "float32", "run")
    made = _run_forward(edge)
    out = tuple(_tensor(np.zeros(v.shape), v.dtype.name) for v in made)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    gc.disable()                                         # no finalizer may run HIP calls mid-capture
    try:
        with torch.cuda.graph(graph):
            _run_forward(edge, out=out)
            with pytest.raises(RuntimeError, match="capture"):
                _run_forward(edge)
            with pytest.raises(RuntimeError, match="capture"):
                _run_backward(edge, made, None)
    finally:
        gc.enable()
    for k in range(3):
        values = _rng(10, k).standard_normal(edge.x.shape).astype(np.float32)
        edge.x.copy_(nt.Tensor(values, dtype="bfloat16", device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(out, _run_forward(edge)))


def test_streams():
    """Calls of two streams at once: each is what it is alone."""
    edges = [_Edge(_rng(11, k), 2, 400, 256, "bfloat16", "float32", "run") for k in range(2)]
    expected = []
    for edge in edges:
        made = _run_forward(edge)
        expected.append((*made, *_run_backward(edge, made, edge.dtotal)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in edges]
    for _ in range(4):
        got = []
        for edge, stream in zip(edges, streams):
            with torch.cuda.stream(stream):
                made = _run_forward(edge)
                got.append((*made, *_run_backward(edge, made, edge.dtotal)))
        torch.cuda.synchronize()
        for want, have in zip(expected, got):
            assert all(np.array_equal(a.bits(), b.bits()) for a, b in zip(want, have))


@pytest.mark.parametrize("dtype, gate", [("bfloat16", "run"), ("float32", "row"), ("float16", "shared")])
@pytest.mark.parametrize("runs, run, width", [(2, 1400, 1536), (2, 900, 2560), (2, 300, 5120)])
def test_rows_of_odd_numbers_of_waves(runs, run, width, gate, dtype):
    """More rows than workgroups hold at a time, of three, five and ten waves each."""
    edge = _Edge(_rng(19, runs, run, width), runs, run, width, dtype, "float32", gate)
    made = _run_forward(edge)
    _check_forward(edge, made)
    _check_backward(edge, _run_backward(edge, made, edge.dtotal), made[1], made[2:], edge.dtotal)
