"""A small language model of gated blocks, trained and scored with the package's operators.

The model is a stream of token embeddings, then blocks that are normalized on
both sides: each block's output meets its norm, a gate for each sequence, the
residual stream and the next block's norm in one call
(``norm_gate_add_norm``); the head's loss never holds its logits
(``linear_cross_entropy``).  PyTorch does the blocks' own products and the
embedding's lookup on the same device memory.  Gradients go to
``accumulate_grads``, the step is ``amp.fused_step`` with a clip, and
``score`` gives the loss of a sequence's next token as it is served, a row at
a time.

Run: ``python examples/gated_lm.py`` (an MI355X and PyTorch)."""

from __future__ import annotations

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import namitorch_amd as nt
from namitorch_amd import functional as F

IGNORED = -100


def shared(value: torch.Tensor) -> nt.Tensor:
    """The same memory as a Tensor of the package."""
    return nt.Tensor._from_storage(value)


class GatedModel:
    """``blocks`` of ``relu(y A) B`` between root mean square norms, each with a gate made from the sequence's tag."""

    def __init__(self, classes: int, width: int, hidden: int, blocks: int, tags: int, dtype=torch.bfloat16, seed=1):
        generator = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, columns, scale=1.0):
            return (torch.randn(rows, columns, generator=generator, device="cuda") * (scale * columns ** -0.5)).to(dtype)

        self.width, self.blocks, self.scale = width, blocks, 0.9
        self.embedding = matrix(classes, width, width ** 0.5)
        self.products = [(matrix(width, hidden), matrix(hidden, width)) for _ in range(blocks)]
        self.norms = [torch.ones(width, device="cuda", dtype=dtype) for _ in range(2 * blocks + 1)]
        self.gates = [(0.5 + 0.1 * torch.randn(tags, width, generator=generator, device="cuda")).to(dtype)
                      for _ in range(blocks)]
        self.head = matrix(classes, width)
        self.values = [self.embedding, *(m for pair in self.products for m in pair), *self.norms, *self.gates, self.head]
        self.parameters = [nt.Parameter._from_storage(v, True) for v in self.values]

    def _edge(self, k: int, branch, stream, gate):
        """Norm of block k's output, gate, stream and the next norm: what the backward call reads, in new memory."""
        lead = stream.shape[:-1]
        made = [torch.empty_like(stream), torch.empty_like(stream)] + [
            None if n % 2 == 0 else torch.empty(lead, device="cuda") for n in range(4)]
        F.norm_gate_add_norm_forward(shared(branch), shared(stream), self.width, shared(self.norms[2 * k + 1]), None,
                                     shared(gate), shared(self.norms[2 * k + 2]), None, self.scale, norm="rms",
                                     out=tuple(None if m is None else shared(m) for m in made))
        return made

    def _first(self, x):
        """The first block's input: the root mean square norm of the embeddings."""
        x = x.float()
        return (x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-5) * self.norms[0].float())

    def gradients(self, tokens, tags, target):
        """(loss, gradients in the order of ``parameters``): ``tokens`` and ``target`` are sequences of rows, ``tags``
        one number for each sequence; targets that are ``IGNORED`` do not count."""
        stream = self.embedding[tokens]
        with torch.enable_grad():                       # PyTorch's own derivative of the first norm
            leaf, weight = stream.detach().requires_grad_(), self.norms[0].detach().requires_grad_()
            x = leaf.float()
            y_first = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + 1e-5) * weight.float()
        y = y_first.detach().to(stream.dtype)
        kept, inner = [(y, stream)], []
        for k, (a, b) in enumerate(self.products):
            inner.append(torch.relu(kept[-1][0] @ a))
            branch = inner[-1] @ b
            kept.append((*self._edge(k, branch, kept[-1][1], self.gates[k][tags][:, None].contiguous()), branch))
        at = [shared(kept[-1][0]), self.parameters[-1], shared(target)]
        loss, lse = F.linear_cross_entropy_forward(*at, ignore_index=IGNORED)
        dy, d_head = torch.empty_like(y), torch.empty_like(self.head)
        F.linear_cross_entropy_backward(1.0, *at, lse, ignore_index=IGNORED, out=(shared(dy), shared(d_head)))

        d_stream = None
        products, norms = [None] * self.blocks, [None] * (2 * self.blocks + 1)
        gates = [torch.zeros_like(gate) for gate in self.gates]
        for k in reversed(range(self.blocks)):
            _, total, _, inner_rstd, _, rstd, branch = kept[k + 1]
            gate = self.gates[k][tags][:, None].contiguous()
            d_branch, d_before, d_gate = torch.empty_like(dy), torch.empty_like(dy), torch.empty_like(gate)
            d_inner_norm, d_norm = (torch.empty_like(self.norms[0]) for _ in range(2))
            F.norm_gate_add_norm_backward(
                shared(dy), None if d_stream is None else shared(d_stream), shared(branch), shared(total), None,
                shared(inner_rstd), None, shared(rstd), shared(self.norms[2 * k + 1]), None, shared(gate),
                shared(self.norms[2 * k + 2]), None, self.scale,
                out=(shared(d_branch), shared(d_before), shared(d_inner_norm), None, shared(d_gate), shared(d_norm), None))
            norms[2 * k + 1], norms[2 * k + 2], d_stream = d_inner_norm, d_norm, d_before
            gates[k].index_add_(0, tags, d_gate[:, 0])
            a, b = self.products[k]
            flat = lambda v: v.reshape(-1, v.shape[-1])  # noqa: E731
            d_inner = (d_branch @ b.t()) * (inner[k] > 0)
            products[k] = (flat(kept[k][0]).t() @ flat(d_inner), flat(inner[k]).t() @ flat(d_branch))
            dy = d_inner @ a.t()
        d_leaf, norms[0] = torch.autograd.grad(y_first, (leaf, weight), dy.float())
        d_embedding = torch.zeros_like(self.embedding, dtype=torch.float32)
        d_embedding.index_add_(0, tokens.reshape(-1), (d_leaf + d_stream).reshape(-1, self.width).float())
        grads = [d_embedding.to(self.embedding.dtype), *(g for pair in products for g in pair), *norms, *gates, d_head]
        return loss, [shared(g.contiguous()) for g in grads]

    def score(self, tokens, tag, target) -> torch.Tensor:
        """The loss of each next token of one sequence, a row at a time, as a server has them."""
        made = []
        for token, following in zip(tokens, target):
            stream = self.embedding[token][None]
            y = self._first(stream).to(stream.dtype)
            for k, (a, b) in enumerate(self.products):
                branch, out = torch.relu(y @ a) @ b, (torch.empty_like(stream), torch.empty_like(stream))
                F.norm_gate_add_norm(shared(branch), shared(stream), self.width, shared(self.norms[2 * k + 1]), None,
                                     shared(self.gates[k][tag]), shared(self.norms[2 * k + 2]), None, self.scale,
                                     norm="rms", out=tuple(map(shared, out)))
                y, stream = out
            loss = torch.empty(1, device="cuda")
            F.linear_cross_entropy(shared(y), self.parameters[-1], shared(following[None]), reduction="none",
                                   out=shared(loss))
            made.append(loss)
        return torch.cat(made)


def train(steps: int = 60, classes: int = 500, width: int = 128, hidden: int = 256, blocks: int = 2, tags: int = 3):
    """Losses of learning a random successor of each token, another for each tag."""
    nt.runtime.set_stream_provider(lambda device: torch.cuda.current_stream(device).cuda_stream)
    model = GatedModel(classes, width, hidden, blocks, tags)
    optimizer = nt.optim.AdamW(model.parameters, lr=3e-3, weight_decay=0.01, master_weights=True)
    generator = torch.Generator(device="cuda").manual_seed(7)
    successor = torch.randint(0, classes, (tags, classes), generator=generator, device="cuda")
    losses = []
    for _ in range(steps):
        tokens = torch.randint(0, classes, (16, 48), generator=generator, device="cuda")
        tag = torch.randint(0, tags, (16,), generator=generator, device="cuda")
        target = torch.gather(successor[tag], 1, tokens)
        target[:, 40:] = IGNORED                        # padding
        loss, gradients = model.gradients(tokens, tag, target)
        nt.accumulate_grads(model.parameters, gradients)
        nt.amp.fused_step(optimizer, None, max_norm=1.0)
        optimizer.zero_grad()
        losses.append(loss)
    tokens = torch.randint(0, classes, (5,), generator=generator, device="cuda")
    served = model.score(tokens, 1, successor[1][tokens])
    return [float(loss.numpy()) for loss in losses], served.tolist(), model


if __name__ == "__main__":
    history, served, _ = train()
    print(f"loss {history[0]:.4f} -> {history[-1]:.4f}; next tokens scored {', '.join(f'{s:.3f}' for s in served)}")
