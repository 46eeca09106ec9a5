"""A gradient whose accumulation or unscaling is still deferred, handed to
layer norm or dropout inside a real stream capture: the call raises, the
graph holds none of it, and the gradient reads as ever afterwards, however
often the graph is replayed."""

from __future__ import annotations

import gc

import numpy as np
import pytest
import torch

import namitorch_amd as nt
from namitorch_amd import functional as F

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _deferred(kind, rng):
    """(a parameter whose gradient has a deferred write, the values that the gradient reads as)."""
    parameter = nt.Parameter(rng.standard_normal((8, 64)).astype(np.float32), device=DEV)
    first, second = (rng.standard_normal((8, 64)).astype(np.float32) for _ in range(2))
    nt.accumulate_grads([parameter], [nt.Tensor(first, device=DEV)])
    if kind == "incoming":
        nt.accumulate_grads([parameter], [nt.Tensor(second, device=DEV)], defer=True)
        assert parameter.grad._incoming is not None
        return parameter, first + second
    scaler = nt.GradScaler(init_scale=256.0)
    scaler.scale(nt.Tensor(np.float32(1.0), device=DEV))
    assert scaler.unscale_(nt.optim.AdamW([parameter], lr=1e-3))
    assert parameter.grad._pending is not None
    return parameter, first / np.float32(256.0)


@pytest.mark.parametrize("kind", ["incoming", "pending"])
def test_deferred_gradient_in_a_capture(kind):
    rng = np.random.Generator(np.random.PCG64(31))
    parameter, expected = _deferred(kind, rng)
    gradient, version = parameter.grad, parameter.grad._version
    x = nt.Tensor(rng.standard_normal((8, 64)).astype(np.float32), device=DEV)
    out = nt.Tensor(np.zeros((8, 64), np.float32), device=DEV)
    y, mean, rstd = F.layer_norm_forward(x, 64)
    calls = (lambda: F.layer_norm(gradient, 64, out=out), lambda: F.layer_norm(x, 64, out=gradient),
             lambda: F.dropout(gradient, 0.0, seed=1, out=out), lambda: F.dropout(gradient, 0.5, seed=1, out=out),
             lambda: F.dropout_add_layer_norm(x, gradient, 64, out=(out, y)),
             lambda: F.layer_norm_backward(gradient, x, mean, rstd))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    gc.disable()                                         # no finalizer may run HIP calls mid-capture
    try:
        with torch.cuda.graph(graph):
            F.layer_norm(x, 64, out=out)
            for call in calls:
                with pytest.raises(RuntimeError, match="capture"):
                    call()
    finally:
        gc.enable()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    assert gradient._version == version
    assert np.array_equal(gradient.numpy(), expected)
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(gradient.numpy(), expected)
    assert np.array_equal(out.bits(), F.layer_norm(x, 64).bits())
    assert np.array_equal(F.dropout(gradient, 0.0, seed=1).numpy(), expected)
