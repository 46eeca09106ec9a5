"""A small residual network trained and served with the package's operators.

The residual path is the package's (``namitorch_amd.functional``): dropout of
the input, a layer norm, then one edge per block (dropout of the block's
branch, added to the stream, and the next norm) with their backward passes.
PyTorch does the matrix products on the same device memory.  Gradients go to
``accumulate_grads``, the step is ``amp.fused_step`` with a clip, and
``answer`` runs single rows through the same weights without dropout.

Run: ``python examples/residual_mlp.py`` (an MI355X and PyTorch)."""

from __future__ import annotations

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import namitorch_amd as nt
from namitorch_amd import functional as F


def shared(value: torch.Tensor) -> nt.Tensor:
    """The same memory as a Tensor of the package."""
    return nt.Tensor._from_storage(value)


class ResidualMLP:
    """``blocks`` of ``relu(norm(x) A) B`` on a stream ``width`` wide, then a norm and a linear head."""

    def __init__(self, width: int, hidden: int, blocks: int, outputs: int, p: float = 0.1, seed: int = 1):
        generator = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, columns):
            return torch.randn(rows, columns, generator=generator, device="cuda") * rows ** -0.5

        self.width, self.p, self.seed, self.calls = width, p, seed, 0
        self.products = [(matrix(width, hidden), matrix(hidden, width) * 0.5) for _ in range(blocks)]
        self.norms = [(torch.ones(width, device="cuda"), torch.zeros(width, device="cuda")) for _ in range(blocks + 1)]
        self.head = matrix(width, outputs)
        self.values = [v for pair in self.products for v in pair] + [v for pair in self.norms for v in pair] + [self.head]
        self.parameters = [nt.Parameter._from_storage(v, True) for v in self.values]
        first = 2 * blocks
        self.affine = [tuple(self.parameters[first + 2 * k:first + 2 * k + 2]) for k in range(blocks + 1)]

    def _edge(self, k: int, branch: torch.Tensor, stream: torch.Tensor, offset: int):
        """The edge after block k: (norm of the new stream, new stream, mean, rstd), in new PyTorch memory."""
        made = [torch.empty_like(stream), torch.empty_like(stream)] + [stream.new_empty(stream.shape[0]) for _ in "mr"]
        F.dropout_add_layer_norm_forward(shared(branch), shared(stream), self.width, *self.affine[k + 1], self.p,
                                         seed=self.seed, offset=offset, out=tuple(map(shared, made)))
        return made

    def gradients(self, x: torch.Tensor, target: torch.Tensor):
        """(loss, gradients in the order of ``parameters``) of the mean squared error of one batch.  Every dropout of
        the run has an offset of its own."""
        blocks, offset = len(self.products), self.calls * (len(self.products) + 1)
        self.calls += 1
        stream = torch.empty_like(x)
        F.dropout(shared(x), self.p, seed=self.seed, offset=offset, out=shared(stream))
        y, mean, rstd = torch.empty_like(x), x.new_empty(x.shape[0]), x.new_empty(x.shape[0])
        F.layer_norm_forward(shared(stream), self.width, *self.affine[0], out=tuple(map(shared, (y, mean, rstd))))
        kept = [(y, stream, mean, rstd)]
        inner = []
        for k, (a, b) in enumerate(self.products):
            inner.append(torch.relu(torch.mm(kept[-1][0], a)))
            kept.append(self._edge(k, torch.mm(inner[-1], b), kept[-1][1], offset + 1 + k))
        error = torch.mm(kept[-1][0], self.head) - target
        loss = error.square().mean()

        d_out = error * (2.0 / error.numel())
        head = torch.mm(kept[-1][0].t(), d_out)
        dy, d_stream = torch.mm(d_out, self.head.t()), None
        products, norms = [None] * blocks, [None] * (blocks + 1)
        for k in reversed(range(blocks)):
            _, total, mean, rstd = kept[k + 1]
            d_branch, d_total = torch.empty_like(dy), torch.empty_like(dy)
            grads = F.dropout_add_layer_norm_backward(
                shared(dy), None if d_stream is None else shared(d_stream), shared(total), shared(mean), shared(rstd),
                *self.affine[k + 1], self.p, seed=self.seed, offset=offset + 1 + k,
                out=(shared(d_branch), shared(d_total), None, None))
            norms[k + 1], d_stream = grads[2:], d_total
            a, b = self.products[k]
            d_inner = torch.mm(d_branch, b.t()).mul_(inner[k] > 0)
            products[k] = (torch.mm(kept[k][0].t(), d_inner), torch.mm(inner[k].t(), d_branch))
            dy = torch.mm(d_inner, a.t())
        # The input is data: its gradient (the first norm's, plus d_stream, through dropout) is not needed.
        _, stream, mean, rstd = kept[0]
        norms[0] = F.layer_norm_backward(shared(dy), shared(stream), shared(mean), shared(rstd), *self.affine[0])[1:]
        flat = [shared(g) for pair in products for g in pair] + [g for pair in norms for g in pair] + [shared(head)]
        return loss, flat

    def answer(self, x: torch.Tensor) -> torch.Tensor:
        """The network's output for a few rows: no dropout, no statistics."""
        stream = shared(x)
        y = torch.empty_like(x)
        F.layer_norm(stream, self.width, *self.affine[0], out=shared(y))
        for k, (a, b) in enumerate(self.products):
            branch = torch.mm(torch.relu(torch.mm(y, a)), b)
            y, total = torch.empty_like(x), torch.empty_like(x)
            F.dropout_add_layer_norm(shared(branch), stream, self.width, *self.affine[k + 1], self.p, training=False,
                                     out=(shared(y), shared(total)))
            stream = shared(total)
        return torch.mm(y, self.head)


def train(steps: int = 200, rows: int = 512, width: int = 96, hidden: int = 200, blocks: int = 3):
    """Losses of fitting a fixed random function of the input."""
    nt.runtime.set_stream_provider(lambda device: torch.cuda.current_stream(device).cuda_stream)
    model = ResidualMLP(width, hidden, blocks, 8)
    optimizer = nt.optim.AdamW(model.parameters, lr=2e-3, weight_decay=0.01)
    generator = torch.Generator(device="cuda").manual_seed(7)
    teacher = torch.randn(width, 8, generator=generator, device="cuda") * width ** -0.5
    losses = []
    for _ in range(steps):
        x = torch.randn(rows, width, generator=generator, device="cuda")
        loss, gradients = model.gradients(x, torch.tanh(torch.mm(x, teacher)))
        nt.accumulate_grads(model.parameters, gradients)
        nt.amp.fused_step(optimizer, None, max_norm=1.0)
        optimizer.zero_grad()
        losses.append(loss)
    x = torch.randn(3, width, generator=generator, device="cuda")
    served = (model.answer(x) - torch.tanh(torch.mm(x, teacher))).square().mean()
    return torch.stack(losses).tolist(), served.item(), model


if __name__ == "__main__":
    history, served, _ = train()
    print(f"loss {history[0]:.4f} -> {history[-1]:.4f}; three rows served with error {served:.4f}")
