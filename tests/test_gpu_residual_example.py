"""The operators run together as a training program uses them: the example's
gradients against PyTorch's float64 autograd with the oracle's masks, and its
training loop."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import residual

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


def test_gradients_of_the_network():
    """Relative error of each gradient: float32 products of up to 200 terms and norms in a chain of ten operations,
    (200 + 10 * 100) * 2**-24 = 7e-5 in the worst case."""
    import residual_mlp
    model = residual_mlp.ResidualMLP(40, 200, 2, 5, p=0.2, seed=3)
    generator = torch.Generator(device="cuda").manual_seed(4)
    for weight, bias in model.norms:                     # away from ones and zeros
        weight.add_(0.2 * torch.randn(weight.shape, generator=generator, device="cuda"))
        bias.add_(0.2 * torch.randn(bias.shape, generator=generator, device="cuda"))
    x = torch.randn(33, 40, generator=generator, device="cuda")
    target = torch.randn(33, 5, generator=generator, device="cuda")
    loss, gradients = model.gradients(x, target)
    gradients = [g.numpy().astype(np.float64) for g in gradients]

    leaves = [v.double().cpu().requires_grad_() for v in model.values]
    mask = [torch.from_numpy(residual.mask((33, 40), 0.2, 3, k)) for k in range(3)]
    norm = lambda t, k: torch.nn.functional.layer_norm(t, (40,), leaves[4 + 2 * k], leaves[5 + 2 * k], 1e-5)  # noqa: E731
    stream = x.double().cpu() * mask[0]
    for k in range(2):
        branch = torch.relu(norm(stream, k) @ leaves[2 * k]) @ leaves[2 * k + 1]
        stream = stream + branch * mask[1 + k]
    expected = (norm(stream, 2) @ leaves[-1] - target.double().cpu()).square().mean()
    expected.backward()
    assert abs(loss.item() - expected.item()) <= 7e-5 * expected.item()
    for got, leaf in zip(gradients, leaves):
        want = leaf.grad.numpy()
        assert np.linalg.norm(got - want) <= 7e-5 * np.linalg.norm(want)


def test_training_lowers_the_loss():
    import residual_mlp
    losses, served, _ = residual_mlp.train(steps=150)
    assert np.isfinite(losses).all()
    assert np.mean(losses[-10:]) < 0.5 * np.mean(losses[:10])
    assert served < np.mean(losses[:10])
