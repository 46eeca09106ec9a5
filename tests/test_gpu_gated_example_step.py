"""One training step of examples/gated_lm.py: each parameter moves against its own gradient, as AdamW's first step says."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_gpu_gated_example as base

pytestmark = pytest.mark.gpu

gated_lm, nt = base.gated_lm, base.gated_lm.nt
LR, EPS = 3e-3, 1e-8


def test_a_step_moves_each_parameter_against_its_gradient():
    """After one step the corrected moments are g and g**2, so the step is lr g / (|g| + eps) with g clipped: off by some
    2**-14 of lr (1 - 0.999 of float32 numbers alone is off by 2**-14 of itself, of which the root takes half) and by
    two roundings of the value.  Where g is zero nothing moves."""
    nt.runtime.set_stream_provider(lambda device: torch.cuda.current_stream(device).cuda_stream)
    model = gated_lm.GatedModel(70, 48, 96, 2, 3, dtype=torch.float32)
    optimizer = nt.optim.AdamW(model.parameters, lr=LR, weight_decay=0.0, eps=EPS)
    generator = torch.Generator(device="cuda").manual_seed(5)
    tokens, target = (torch.randint(0, 70, (4, 11), generator=generator, device="cuda") for _ in range(2))
    target[:, 8:] = gated_lm.IGNORED
    _, gradients = model.gradients(tokens, torch.tensor([0, 2, 0, 1], device="cuda"), target)
    before = [value.double().cpu().numpy() for value in model.values]
    grads = [np.array(g.numpy(), dtype=np.float64) for g in gradients]
    nt.accumulate_grads(model.parameters, gradients)
    nt.amp.fused_step(optimizer, None, max_norm=1.0)
    torch.cuda.synchronize()
    norm = np.sqrt(sum(np.square(g).sum() for g in grads))
    assert len(grads) == len(model.values)
    for was, value, grad in zip(before, model.values, grads):
        now, clipped = value.double().cpu().numpy(), grad * min(1.0, 1.0 / norm)
        moved = LR * clipped / (np.abs(clipped) + EPS)
        assert np.any(grad != 0.0)
        assert np.all(np.abs(now - (was - moved)) <= LR * 2.0 ** -12 + 2.0 ** -23 * np.abs(was))
        assert np.array_equal(now[grad == 0.0], was[grad == 0.0])
