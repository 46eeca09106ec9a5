"""The gated model of examples/gated_lm.py: its gradients against PyTorch's
own derivative of the same model in 64 bits, its scores against its training
path's loss, and a short training run."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

import gated_lm  # noqa: E402

pytestmark = pytest.mark.gpu


def _reference(model, tokens, tags, target):
    """(loss, gradients) by PyTorch in 64 bits, from the model's definition."""
    values = [v.detach().double().requires_grad_() for v in model.values]
    blocks = model.blocks
    embedding, products = values[0], values[1:1 + 2 * blocks]
    norms, gates, head = values[1 + 2 * blocks:2 + 4 * blocks], values[2 + 4 * blocks:2 + 5 * blocks], values[-1]

    def norm(x, weight):
        return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-5) * weight

    stream = embedding[tokens]
    y = norm(stream, norms[0])
    for k in range(blocks):
        branch = torch.relu(y @ products[2 * k]) @ products[2 * k + 1]
        stream = model.scale * stream + gates[k][tags][:, None] * norm(branch, norms[2 * k + 1])
        y = norm(stream, norms[2 * k + 2])
    logits = (y @ head.t()).reshape(-1, head.shape[0])
    loss = torch.nn.functional.cross_entropy(logits, target.reshape(-1), ignore_index=gated_lm.IGNORED)
    return loss.item(), torch.autograd.grad(loss, values)


def test_gradients():
    """In float32 every difference is a chain of a few dozen float32 operations and products of up to 96 terms (each
    2**-24 relative to the sum of magnitudes): some 2**-15 of a gradient's norm bounds them with room."""
    gated_lm.nt.runtime.set_stream_provider(lambda device: torch.cuda.current_stream(device).cuda_stream)
    model = gated_lm.GatedModel(70, 48, 96, 2, 3, dtype=torch.float32)
    generator = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(0, 70, (4, 11), generator=generator, device="cuda")
    tags = torch.tensor([0, 2, 0, 1], device="cuda")
    target = torch.randint(0, 70, (4, 11), generator=generator, device="cuda")
    target[:, 8:] = gated_lm.IGNORED
    loss, gradients = model.gradients(tokens, tags, target)
    expected, reference = _reference(model, tokens, tags, target)
    assert abs(float(loss.numpy()) - expected) <= 2.0 ** -15 * abs(expected)
    assert len(gradients) == len(reference)
    for got, exact in zip(gradients, reference):
        got = torch.from_numpy(got.numpy()).cuda().double()
        assert got.shape == exact.shape
        assert (got - exact).norm() <= 2.0 ** -15 * exact.norm()


def test_scores_are_the_training_path_s_loss():
    """A sequence scored row by row is the mean of what a batch of it gives: the same float32 operations in other
    orders, products of 64 terms and a sum over 300 classes, so within some 2**-15."""
    model = gated_lm.GatedModel(300, 64, 96, 2, 3, dtype=torch.float32)
    generator = torch.Generator(device="cuda").manual_seed(4)
    tokens, target = (torch.randint(0, 300, (6,), generator=generator, device="cuda") for _ in range(2))
    loss, _ = model.gradients(tokens[None], torch.tensor([2], device="cuda"), target[None])
    served = model.score(tokens, 2, target)
    assert abs(served.mean().item() - float(loss.numpy())) <= 2.0 ** -15 * float(loss.numpy())


def test_it_trains():
    losses, served, _ = gated_lm.train(steps=12)
    assert len(losses) == 12 and len(served) == 5
    assert np.all(np.isfinite(losses)) and np.all(np.isfinite(served))
