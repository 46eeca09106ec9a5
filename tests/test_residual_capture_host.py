"""Layer norm and dropout in a stream capture, without a GPU: with capture
reported as active, a gradient whose accumulation or unscaling is still
deferred is refused as an input and as a result.  Its write would be recorded
into the graph and marked as done, though nothing has run: the gradient would
lack it until a replay, and every further replay would apply it again."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

import namitorch_amd as nt
from namitorch_amd import functional as F
from namitorch_amd.backends import _backends, _graph_capture
from namitorch_amd.tensor import GradTransform

WRITES = ("pending", "incoming")


@pytest.fixture
def queued(monkeypatch):
    """Operations that reach the device while it is being captured."""
    made = []
    backend = SimpleNamespace(
        adamw=object(), accumulate_tensors=lambda stored, incoming, assign: made.append("accumulate"),
        apply_grad_transform=lambda tensors, transform: made.append("transform"))
    monkeypatch.setitem(_backends, nt.Device("cuda:0"), backend)
    monkeypatch.setattr(_graph_capture, "capturing", lambda: True)
    return made


def _tensor(shape, dtype=nt.float32):
    """A device Tensor that owns no memory: nothing here may read or write it."""
    return nt.Tensor._from_storage(nt.DeviceArray._make(None, 1 << 20, shape, dtype, nt.Device("cuda:0")))


def _deferred(shape, kind):
    tensor = _tensor(shape)
    if kind == "pending":
        tensor._pending = GradTransform(scale=2.0)
    else:
        tensor._incoming = (_tensor(shape), 0)
    return tensor


def _calls(value, rows, columns):
    """Every place of a Tensor shaped like the activations, the weight and the statistics."""
    x, w, s, out = _tensor((4, 8)), _tensor((8,)), _tensor((4,)), _tensor((4, 8))
    return {
        "norm input": lambda: F.layer_norm(value, 8, w, w, out=out),
        "norm weight": lambda: F.layer_norm(x, 8, columns, w, out=out),
        "norm bias": lambda: F.layer_norm(x, 8, w, columns, out=out),
        "norm output": lambda: F.layer_norm(x, 8, w, w, out=value),
        "norm mean": lambda: F.layer_norm_forward(x, 8, w, w, out=(out, rows, s)),
        "backward gradient": lambda: F.layer_norm_backward(value, x, s, s, w, w),
        "backward mean": lambda: F.layer_norm_backward(x, x, rows, s, w, w),
        "backward grad_weight": lambda: F.layer_norm_backward(x, x, s, s, w, w, out=(out, columns, w)),
        "dropout input": lambda: F.dropout(value, 0.5, seed=1, out=out),
        "dropout input, none dropped": lambda: F.dropout(value, 0.0, seed=1, out=out),
        "dropout output": lambda: F.dropout(x, 0.0, seed=1, out=value),
        "edge residual": lambda: F.dropout_add_layer_norm(x, value, 8, w, w, out=(out, x)),
        "edge total": lambda: F.dropout_add_layer_norm(x, x, 8, w, w, out=(out, value)),
        "edge backward grad_total": lambda: F.dropout_add_layer_norm_backward(x, value, x, s, s, w, w),
    }


@pytest.mark.parametrize("kind", WRITES)
@pytest.mark.parametrize("place", list(_calls(None, None, None)))
def test_deferred_gradients_are_refused_in_a_capture(queued, place, kind):
    value, rows, columns = (_deferred(shape, kind) for shape in ((4, 8), (4,), (8,)))
    markers = [(t._pending, t._incoming, t._version_counter.value) for t in (value, rows, columns)]
    with pytest.raises(RuntimeError, match="capture"):
        _calls(value, rows, columns)[place]()
    assert queued == []
    assert markers == [(t._pending, t._incoming, t._version_counter.value) for t in (value, rows, columns)]


@pytest.mark.parametrize("kind", WRITES)
def test_outside_a_capture_they_are_written_back(queued, monkeypatch, kind):
    monkeypatch.setattr(_graph_capture, "capturing", lambda: False)
    value = _deferred((4, 8), kind)
    assert F.dropout(value, 0.0, seed=1) is value
    assert queued == ["transform" if kind == "pending" else "accumulate"]
    assert value._pending is None and value._incoming is None
