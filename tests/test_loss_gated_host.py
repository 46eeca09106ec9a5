"""The linear cross entropy and the edge after a block without a GPU: the
64-bit oracles' gradients against differences, and what the entry points
refuse before any device is asked."""

from __future__ import annotations

import numpy as np
import pytest

import namitorch_amd as nt
from namitorch_amd import _native, functional as F
from oracle import gated, loss

STEP = 2.0 ** -13       # central differences: off by step^2 times a third derivative and 2^-52 over the step, below 1e-6


def _slope(f, array, index):
    kept = array[index]
    array[index] = kept + STEP
    above = f()
    array[index] = kept - STEP
    below = f()
    array[index] = kept
    return (above - below) / (2 * STEP)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_gradient_against_differences(reduction):
    rng = np.random.Generator(np.random.PCG64(5))
    x, weight = rng.standard_normal((5, 4)), rng.standard_normal((7, 4))
    target = np.array([3, -100, 0, 6, 3])
    grad = rng.standard_normal(5) if reduction == "none" else 1.7

    def value():
        return float(np.sum(np.asarray(grad) * loss.forward(x, weight, target, reduction=reduction)[0]))

    _, lse = loss.forward(x, weight, target, reduction=reduction)
    dx, dw, _ = loss.backward(grad, x, weight, target, lse, reduction=reduction)
    for array, grads in ((x, dx), (weight, dw)):
        for index in np.ndindex(array.shape):
            assert abs(_slope(value, array, index) - grads[index]) < 1e-6
    assert not dx[1].any()


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("gate_rows", [0, 1, 2, 6])
def test_edge_gradient_against_differences(gate_rows, rms):
    rng = np.random.Generator(np.random.PCG64(6 + gate_rows))
    x, r, dy, dt = (rng.standard_normal((6, 5)) for _ in range(4))
    u, k, w, b = (rng.standard_normal(5) for _ in range(4))
    gate = rng.standard_normal((gate_rows, 5)) if gate_rows else None

    def value():
        y, total, *_ = gated.forward(x, r, u, k, gate, w, b, 0.75, 1e-3, rms)
        return float((y * dy).sum() + (total * dt).sum())

    _, total, *stats = gated.forward(x, r, u, k, gate, w, b, 0.75, 1e-3, rms)
    dx, dr, du, dk, dgate, dw, db, _ = gated.backward(dy, dt, x, total, *stats, u, k, gate, w, 0.75, rms)
    for array, grads in ((x, dx), (r, dr), (u, du), (k, dk), (gate, dgate), (w, dw), (b, db)):
        if array is None:
            continue
        for index in np.ndindex(array.shape):
            assert abs(_slope(value, array, index) - grads[index]) < 1e-6


# ---- refusals: device Tensors that own no memory, which nothing may read or write ----------------------
@pytest.fixture
def launches(monkeypatch):
    """The library's launches, recorded instead of made."""
    from types import SimpleNamespace

    from namitorch_amd.backends import _backends, _graph_capture

    made = []
    monkeypatch.setitem(_backends, nt.Device("cuda:0"), SimpleNamespace(adamw=object()))
    monkeypatch.setattr(_graph_capture, "capturing", lambda: False)
    monkeypatch.setattr(F, "current_stream", lambda device: 0)

    class Library:
        def __getattr__(self, name):
            return lambda *args: made.append((name, args)) or 0

    monkeypatch.setattr(_native, "load", Library)
    return made


def _tensor(shape, dtype=nt.float32):
    return nt.Tensor._from_storage(nt.DeviceArray._make(None, 1 << 20, shape, dtype, nt.Device("cuda:0")))


def _int(shape, dtype="int64"):
    return _tensor(shape, nt.dtype.normalize_dtype(dtype))


def test_loss_refusals(launches):
    x, w, t = _tensor((2, 3, 8)), _tensor((50, 8)), _int((2, 3))
    lse, each = _tensor((2, 3)), _tensor((2, 3))
    out = dict(out=(_tensor(()), lse))
    good = lambda **more: F.linear_cross_entropy_forward(x, w, t, **{**out, **more})  # noqa: E731
    good()
    F.linear_cross_entropy_backward(2.0, x, w, t, lse, out=(_tensor((2, 3, 8)), _tensor((50, 8))))
    assert [name for name, _ in launches] == ["nt_linear_cross_entropy", "nt_linear_cross_entropy_backward"]
    launches.clear()
    back = lambda g=1.0, a=x, b=w, c=t, d=lse, **more: F.linear_cross_entropy_backward(  # noqa: E731
        g, a, b, c, d, **{"out": (_tensor((2, 3, 8)), _tensor((50, 8))), **more})
    refused = [
        (TypeError, "input must be a NamiTorch Tensor", lambda: F.linear_cross_entropy(np.zeros((3, 8)), w, t)),
        (TypeError, "float16, bfloat16 or float32", lambda: F.linear_cross_entropy(_tensor((2, 3, 8), nt.float64), w, t)),
        (TypeError, "weight must be a NamiTorch Tensor", lambda: F.linear_cross_entropy(x, None, t)),
        (TypeError, "weight has dtype", lambda: F.linear_cross_entropy(x, _tensor((50, 8), nt.float16), t)),
        (ValueError, "weight has shape", lambda: F.linear_cross_entropy(x, _tensor((50, 9)), t)),
        (ValueError, "weight has shape", lambda: F.linear_cross_entropy(x, _tensor((0, 8)), t)),
        (ValueError, "weight has shape", lambda: F.linear_cross_entropy(_tensor((2, 3, 0)), _tensor((50, 0)), t)),
        (ValueError, "at least one dimension", lambda: F.linear_cross_entropy(_tensor(()), w, t)),
        (TypeError, "target must be int64 or int32", lambda: F.linear_cross_entropy(x, w, _tensor((2, 3)))),
        (TypeError, "target must be int64 or int32", lambda: F.linear_cross_entropy(x, w, _int((2, 3), "int16"))),
        (TypeError, "target must be a NamiTorch Tensor", lambda: F.linear_cross_entropy(x, w, [1, 2])),
        (ValueError, "target has shape", lambda: F.linear_cross_entropy(x, w, _int((6,)))),
        (ValueError, "reduction must be", lambda: good(reduction="median")),
        (ValueError, "reduction must be", lambda: good(reduction=None)),
        (TypeError, "ignore_index must be an integer", lambda: good(ignore_index=1.0)),
        (TypeError, "ignore_index must be an integer", lambda: good(ignore_index=True)),
        (ValueError, "ignore_index must be in", lambda: good(ignore_index=1 << 63)),
        (TypeError, "out must be a tuple of 2", lambda: good(out=lse)),
        (ValueError, "out: loss has shape", lambda: good(out=(each, lse))),
        (TypeError, "out: lse has dtype", lambda: good(out=(_tensor(()), _tensor((2, 3), nt.float16)))),
        (TypeError, "grad_loss must be", lambda: back("1")),
        (TypeError, "grad_loss must be", lambda: back(True)),
        (TypeError, "as each row has a loss", lambda: back(1.0, reduction="none")),
        (ValueError, "grad_loss has shape", lambda: back(each)),
        (ValueError, "grad_loss has shape", lambda: back(_tensor(()), reduction="none")),
        (TypeError, "grad_loss must be float32", lambda: back(_tensor((), nt.float16))),
        (ValueError, "lse has shape", lambda: back(d=_tensor((6,)))),
        (TypeError, "lse must be float32", lambda: back(d=_tensor((2, 3), nt.bfloat16))),
        (ValueError, "out: grad_weight has shape", lambda: back(out=(_tensor((2, 3, 8)), _tensor((8, 50))))),
    ]
    for error, message, call in refused:
        with pytest.raises(error, match=message):
            call()
    assert not launches


def test_edge_refusals(launches):
    x, vector, stat = _tensor((2, 3, 8)), _tensor((8,)), _tensor((2, 3))
    same = lambda: _tensor((2, 3, 8))  # noqa: E731
    good = lambda a=x, r=x, shape=8, out=None, **more: F.norm_gate_add_norm(  # noqa: E731
        a, r, shape, out=out or (same(), same()), **more)
    for gate in (None, vector, _tensor((2, 1, 8)), _tensor((1, 1, 8)), _tensor((2, 3, 8))):
        good(gate=gate)
        assert launches[-1][1][8] == (0 if gate is None else gate.numel() // 8)
    good(a=_tensor((2, 3, 8), nt.float16), r=_tensor((2, 3, 8), nt.float16), gate=vector,
         out=(_tensor((2, 3, 8), nt.float16), _tensor((2, 3, 8), nt.float16)))
    back = lambda stats=(stat,) * 4, **more: F.norm_gate_add_norm_backward(  # noqa: E731
        x, None, x, x, *stats, **{"out": (same(), same()) + (None,) * 5, **more})
    back()
    back(stats=(None, stat, None, stat))
    launches.clear()
    refused = [
        (ValueError, "residual has shape", lambda: good(r=_tensor((3, 8)))),
        (TypeError, "residual has dtype", lambda: good(r=_tensor((2, 3, 8), nt.float16))),
        (ValueError, "normalized_shape", lambda: good(shape=(3, 9))),
        (ValueError, "inner_weight has shape", lambda: good(inner_weight=_tensor((9,)))),
        (TypeError, "weights and biases must have one dtype", lambda: F.norm_gate_add_norm(
            _tensor((2, 8), nt.float16), _tensor((2, 8), nt.float16), 8, vector, _tensor((8,), nt.float16))),
        (TypeError, "bias must be float32 or float32", lambda: good(bias=_tensor((8,), nt.float16))),
        (TypeError, "gate must be a NamiTorch Tensor", lambda: good(gate=0.5)),
        (TypeError, "gate must be", lambda: good(gate=_tensor((8,), nt.float16))),
        (ValueError, "gate has shape", lambda: good(gate=_tensor((9,)))),
        (ValueError, "gate has shape", lambda: good(gate=_tensor((1, 3, 8)))),
        (ValueError, "gate has shape", lambda: good(gate=_tensor((3, 8)))),
        (ValueError, "gate has shape", lambda: good(gate=_tensor((2, 2, 8)))),
        (ValueError, "gate has shape", lambda: good(gate=_tensor(()))),
        (TypeError, "residual_scale must be a real", lambda: good(residual_scale="1")),
        (TypeError, "residual_scale must be a real", lambda: good(residual_scale=True)),
        (ValueError, "residual_scale must be finite", lambda: good(residual_scale=float("nan"))),
        (ValueError, "residual_scale must be finite", lambda: good(residual_scale=1e39)),
        (ValueError, "eps must be", lambda: good(eps=-1.0)),
        (ValueError, "norm must be", lambda: good(norm="batch")),
        (ValueError, "norm must be", lambda: good(norm=0)),
        (ValueError, "root mean square norms have none", lambda: F.norm_gate_add_norm_forward(
            x, x, 8, norm="rms", out=(same(), same(), stat, stat, None, stat))),
        (ValueError, "given together", lambda: back(stats=(None, stat, stat, stat))),
        (TypeError, "rstd must be a NamiTorch Tensor", lambda: back(stats=(stat, stat, stat, None))),
        (TypeError, "inner_rstd must be a NamiTorch Tensor", lambda: back(stats=(stat, None, stat, stat))),
        (ValueError, "rstd has shape", lambda: back(stats=(stat, stat, stat, _tensor((3,))))),
        (ValueError, "inner_mean has shape", lambda: back(stats=(_tensor((2,)), stat, stat, stat))),
        (ValueError, "the edge has no such parameter", lambda: back(out=(same(), same(), vector, None, None, None, None))),
        (TypeError, "out must be a tuple of 7", lambda: back(out=(None, None))),
    ]
    for error, message, call in refused:
        with pytest.raises(error, match=message):
            call()
    assert not launches


def test_captures_are_refused_before_a_launch(launches, monkeypatch):
    from namitorch_amd.backends import _graph_capture

    monkeypatch.setattr(_graph_capture, "capturing", lambda: True)
    x, w, t, lse = _tensor((3, 8)), _tensor((50, 8)), _int((3,)), _tensor((3,))
    calls = (lambda: F.linear_cross_entropy(x, w, t, out=_tensor(())),
             lambda: F.linear_cross_entropy_backward(1.0, x, w, t, lse, out=(_tensor((3, 8)), _tensor((50, 8)))),
             lambda: F.norm_gate_add_norm(x, x, 8), lambda: F.norm_gate_add_norm(x, x, 8, out=(_tensor((3, 8)), None)),
             lambda: F.norm_gate_add_norm_backward(x, None, x, x, lse, lse, lse, lse))
    for call in calls:
        with pytest.raises(RuntimeError, match="capture"):
            call()
    assert not launches
    F.norm_gate_add_norm(x, x, 8, out=(_tensor((3, 8)), _tensor((3, 8))))
    F.norm_gate_add_norm_forward(x, x, 8, norm="rms", out=(_tensor((3, 8)), _tensor((3, 8)), None, lse, None, _tensor((3,))))
    assert [name for name, _ in launches] == ["nt_norm_gate_add_norm"] * 2


# ---- the C ABI's own checks, which come before any device call ------------------------------------------
def _loss_arguments(**changed):
    arguments = dict(device=0, x=4096, weight=8192, dtype=_native.NT_F32, target=16384, target_size=8, ignore=-100,
                     reduction=1, loss=20480, lse=24576, rows=2, classes=5, width=8, stream=None)
    assert not set(changed) - set(arguments)
    return tuple({**arguments, **changed}.values())


@pytest.mark.parametrize("changed, status, message", [
    (dict(dtype=_native.NT_F64), _native.NT_ERR_TYPE, "float32, float16 or bfloat16"),
    (dict(target_size=2), _native.NT_ERR_TYPE, "int32 or int64"),
    (dict(reduction=3), _native.NT_ERR_VALUE, "reduction"),
    (dict(width=0), _native.NT_ERR_VALUE, "width"),
    (dict(width=(1 << 21) + 1), _native.NT_ERR_VALUE, "width"),
    (dict(classes=0), _native.NT_ERR_VALUE, "classes"),
    (dict(classes=1 << 30), _native.NT_ERR_VALUE, "classes"),
    (dict(rows=1 << 24), _native.NT_ERR_VALUE, "rows"),
    (dict(x=None), _native.NT_ERR_VALUE, "NULL"),
    (dict(loss=None), _native.NT_ERR_VALUE, "NULL"),
    (dict(target=16388), _native.NT_ERR_VALUE, "aligned"),
    (dict(x=4098), _native.NT_ERR_VALUE, "aligned"),
    (dict(lse=20480), _native.NT_ERR_VALUE, "overlaps"),
    (dict(loss=4160 - 4), _native.NT_ERR_VALUE, "overlaps"),
])
def test_c_refusals_of_the_loss(changed, status, message):
    library = _native.load()
    assert library.nt_linear_cross_entropy(*_loss_arguments(**changed)) == status
    assert message in library.nt_last_error().decode()


def _edge_arguments(**changed):
    arguments = dict(device=0, x=4096, residual=8192, dtype=_native.NT_F16, inner_weight=None, inner_bias=None,
                     gate=12288, gate_dtype=_native.NT_F32, gate_rows=2, weight=None, bias=None,
                     weight_dtype=_native.NT_F16, scale=1.0, eps=1e-5, rms=0, total=16384, y=20480, inner_mean=24576,
                     inner_rstd=28672, mean=32768, rstd=36864, rows=4, width=8, stream=None)
    assert not set(changed) - set(arguments)
    return tuple({**arguments, **changed}.values())


@pytest.mark.parametrize("changed, status, message", [
    (dict(dtype=_native.NT_F64), _native.NT_ERR_TYPE, "float32, float16 or bfloat16"),
    (dict(weight=4000, weight_dtype=_native.NT_BF16), _native.NT_ERR_TYPE, "weights"),
    (dict(gate_dtype=_native.NT_BF16), _native.NT_ERR_TYPE, "gate"),
    (dict(gate_rows=3), _native.NT_ERR_VALUE, "divide"),
    (dict(gate_rows=0), _native.NT_ERR_VALUE, "divide"),
    (dict(width=0), _native.NT_ERR_VALUE, "width"),
    (dict(width=(1 << 24) + 1), _native.NT_ERR_VALUE, "width"),
    (dict(rows=1 << 31), _native.NT_ERR_VALUE, "rows"),
    (dict(residual=None), _native.NT_ERR_VALUE, "NULL"),
    (dict(gate=12290), _native.NT_ERR_VALUE, "aligned"),
    (dict(total=4096), _native.NT_ERR_VALUE, "overlaps"),
    (dict(y=12288 + 60), _native.NT_ERR_VALUE, "overlaps"),
    (dict(mean=None), _native.NT_ERR_VALUE, "together"),
    (dict(rms=1), _native.NT_ERR_VALUE, "together"),
    (dict(rstd=None), _native.NT_ERR_VALUE, "together"),
])
def test_c_refusals_of_the_edge(changed, status, message):
    library = _native.load()
    assert library.nt_norm_gate_add_norm(*_edge_arguments(**changed)) == status
    assert message in library.nt_last_error().decode()
