"""What the linear cross entropy and the gated edge refuse, and in whose name, without a GPU."""

from __future__ import annotations

import numpy as np
import pytest

import namitorch_amd as nt
from namitorch_amd import functional as F
from test_loss_gated_host import _int, _tensor, launches  # noqa: F401 - a fixture


@pytest.mark.parametrize("value", [1e39, -1e300, 2.0 ** 128, np.float64(4e38), 10 ** 39])
def test_a_loss_gradient_that_float32_does_not_hold(launches, value):  # noqa: F811
    """Passed on it would be infinite, and with it gradients that may be finite."""
    x, w, t, lse = _tensor((3, 8)), _tensor((50, 8)), _int((3,)), _tensor((3,))
    with pytest.raises(ValueError, match="grad_loss must be within float32's range"):
        F.linear_cross_entropy_backward(value, x, w, t, lse, out=(_tensor((3, 8)), _tensor((50, 8))))
    assert not launches


@pytest.mark.parametrize("value", [3.4028234663852886e38, float("inf"), -float("inf"), 0.0, 2, np.float32(1.5)])
def test_loss_gradients_that_it_holds(launches, value):  # noqa: F811
    """Infinities among them: a scaler skips such a step."""
    x, w, t, lse = _tensor((3, 8)), _tensor((50, 8)), _int((3,)), _tensor((3,))
    F.linear_cross_entropy_backward(value, x, w, t, lse, out=(_tensor((3, 8)), _tensor((50, 8))))
    (name, arguments), = launches
    assert name == "nt_linear_cross_entropy_backward" and arguments[2] == float(value)


def test_the_edge_is_refused_in_its_own_name(launches, monkeypatch):  # noqa: F811
    from namitorch_amd.backends import _graph_capture

    host, device, stat = nt.Tensor(np.ones((3, 8), np.float32)), _tensor((3, 8)), _tensor((3,))
    for call in (lambda: F.norm_gate_add_norm(host, host, 8),
                 lambda: F.norm_gate_add_norm_backward(host, None, host, host, stat, stat, stat, stat)):
        with pytest.raises(RuntimeError, match="^The gated edge runs only on HIP devices"):
            call()
    monkeypatch.setattr(_graph_capture, "capturing", lambda: True)
    for call in (lambda: F.norm_gate_add_norm(device, device, 8), lambda: F.norm_gate_add_norm_forward(device, device, 8),
                 lambda: F.norm_gate_add_norm_backward(device, None, device, device, stat, stat, stat, stat)):
        with pytest.raises(RuntimeError, match="^The gated edge.* capture"):
            call()
    assert not launches
