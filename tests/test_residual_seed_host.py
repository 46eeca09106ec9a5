"""An edge that drops elements names its seed (without a GPU: the call is
refused before anything is launched).  With a default, every edge of every
step would drop the same elements and nothing would say so."""

from __future__ import annotations

import re
from types import SimpleNamespace

import pytest

import namitorch_amd as nt
from namitorch_amd import _native, functional as F
from namitorch_amd.backends import _backends, _graph_capture

NEEDED = "^" + re.escape("seed is needed where elements are dropped (p > 0 in training).") + "$"


@pytest.fixture
def launched(monkeypatch):
    """(entry, drop threshold, seed) of each launch, none of which runs."""
    made = []

    class Library:
        def __getattr__(self, name):
            def entry(*arguments):
                made.append((name, *arguments[8 if name.endswith("norm") else 9:][:2]))
                return 0
            return entry

    monkeypatch.setitem(_backends, nt.Device("cuda:0"), SimpleNamespace())
    monkeypatch.setattr(_native, "load", Library)
    monkeypatch.setattr(_graph_capture, "capturing", lambda: False)
    with nt.runtime.stream((0, 0)):
        yield made


def _tensor(shape):
    return nt.Tensor._from_storage(nt.DeviceArray._make(None, 1 << 20, shape, nt.float32, nt.Device("cuda:0")))


def _calls(rows, **arguments):
    x, s = _tensor((rows, 8)), _tensor((rows,))
    return (lambda: F.dropout_add_layer_norm(x, x, 8, out=(x, x), **arguments),
            lambda: F.dropout_add_layer_norm_forward(x, x, 8, out=(x, x, s, s), **arguments),
            lambda: F.dropout_add_layer_norm_backward(x, x, x, s, s, out=(x, x, None, None), **arguments))


@pytest.mark.parametrize("arguments", [{"p": 0.1}, {"p": 0.1, "offset": 3}, {"p": 1.0}, {"p": 0.1, "seed": None}])
def test_a_mask_needs_a_seed(launched, arguments):
    for call in _calls(4, **arguments):
        with pytest.raises(TypeError, match=NEEDED):
            call()
    assert launched == []


@pytest.mark.parametrize("rows, arguments, threshold, seed", [
    (4, {"p": 0.1, "seed": 7}, 6554, 7), (4, {"p": 0.1, "seed": 0}, 6554, 0), (4, {}, 0, 0), (4, {"p": 0.0}, 0, 0),
    (4, {"p": 0.1, "training": False}, 0, 0), (0, {"p": 0.1}, 6554, 0)])
def test_calls_that_draw_nothing_need_none(launched, rows, arguments, threshold, seed):
    for call in _calls(rows, **arguments):
        call()
    assert [entry[1:] for entry in launched] == [(threshold, seed)] * 3
