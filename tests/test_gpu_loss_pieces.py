"""The linear cross entropy over several pieces of the vocabulary, against PyTorch's 64-bit products on the device.

A piece is as much as keeps the logits' gradient, or packed weights, within a set number of bytes, or a launch within
its work-items; test_loss_rules_host.py asserts that the sizes here have the pieces that stand beside them.

Bounds, element by element, e = 2**-24 and u the half ulp of the dtype (float32's three parts hold a value to
2**-24).  A sum of k products, in any order and over any pieces, is off by 2 k e of the sum of their magnitudes (the
matrix cores may truncate each step), of float32's six products a pair by 12 k e and the 2**-23 that is left out.
exp(z - lse) is off by the logit's error and the roundings of its argument, 4 e (|z| + |lse|), and 4 e of its own; dz by
u more, in float16 by half the smallest subnormal too, 2**-25, after a scale of 2**14 or more.  Results are multiplied
by a rounded factor, 3 e, and rounded once, off by TINY where they are subnormal."""

from __future__ import annotations

import pytest
import torch

import namitorch_amd as nt
from namitorch_amd import functional as F

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF_ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}

# dtype, rows, classes, width, pieces of the forward pass and of the backward one.
PIECES = [
    ("bfloat16", 16000, 70011, 64, 1, 3),       # weights read in place, whose last lines do not fill a step
    ("float16", 16000, 40011, 40, 1, 2),        # packed weights
    ("float32", 8192, 50257, 24, 1, 3),         # three planes of everything
    ("bfloat16", 70000, 9000, 40, 1, 2),        # the weight's gradient is split along the rows in each piece
    ("bfloat16", 4200001, 300, 8, 1, 2),        # pieces of the fewest classes, split likewise
    ("float32", 6, 1500001, 128, 2, 2),         # packed weights in both passes, few rows
    ("float16", 7, 9000003, 40, 2, 2),
    ("float32", 300, 400001, 520, 2, 2),        # the same, larger tiles
]
# The forward pass alone, in pieces for its launches' sake.
MANY_ROWS = ("bfloat16", 4200001, 33001, 64, 2)


def _off(k, dtype):
    return 2 * k * E if dtype != "float32" else 12 * k * E + 2.0 ** -23


def _problem(dtype, rows, classes, width):
    generator = torch.Generator(device="cuda").manual_seed(classes)
    kind = getattr(torch, dtype)
    weight = (torch.randn(classes, width, generator=generator, device="cuda") * (2.0 / width ** 0.5)).to(kind)
    target = torch.randint(0, classes, (rows,), generator=generator, device="cuda")
    x = torch.randn(rows, width, generator=generator, device="cuda")
    x = (x + 2.0 * torch.rand(rows, 1, generator=generator, device="cuda") * weight[target].float()).to(kind)
    target[::7] = -100
    target[3], target[5] = 0, classes - 1
    return x, weight, target


def _lse_bound(z_off, expected, classes):
    return z_off.amax(dim=1) + (classes / 1024 + 200) * E + 4 * E * expected.abs()


def _check(got, exact, bound, dtype):
    bound = bound + (HALF_ULP[dtype] + 3 * E) * (exact.abs() + bound) + TINY[dtype]
    wrong = (got.double() - exact).abs() > bound
    assert not wrong.any(), (int(wrong.sum()), wrong.nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype, rows, classes, width, forward, backward", PIECES)
def test_pieces(dtype, rows, classes, width, forward, backward):
    x, weight, target = _problem(dtype, rows, classes, width)
    wrap, at = nt.Tensor._from_storage, (nt.Tensor._from_storage(v) for v in (x, weight, target))
    at = tuple(at)
    loss, lse = torch.full((), -1.0, device="cuda"), torch.full((rows,), -1.0, device="cuda")
    F.linear_cross_entropy_forward(*at, out=(wrap(loss), wrap(lse)))
    got_dx, got_dw = torch.full_like(x, 7.0), torch.full_like(weight, 7.0)
    F.linear_cross_entropy_backward(1.0, *at, wrap(lse), out=(wrap(got_dx), wrap(got_dw)))

    there = target != -100
    count, u = int(there.sum()), HALF_ULP[dtype]
    wd = weight.double()
    w_size = wd.abs()
    dw, dw_off, dw_size = (torch.zeros_like(wd) for _ in range(3))
    total = total_off = 0.0
    each = max(1, min(rows, (1 << 26) // classes))
    for first in range(0, rows, each):
        part = slice(first, first + each)
        here, kept = there[part], lse[part].double()
        xd = x[part].double() * here[:, None]
        z = torch.mm(xd, wd.t().contiguous())
        z_off = torch.mm(xd.abs(), w_size.t().contiguous()) * _off(width, dtype)
        expected = torch.logsumexp(z, dim=1)
        lse_off = _lse_bound(z_off, expected, classes)
        assert torch.all((kept - expected).abs()[here] <= lse_off[here])
        assert torch.all(kept[~here] == 0.0)
        place = target[part].clamp(min=0)[:, None]
        losses = (expected - z.gather(1, place)[:, 0])[here]
        total += losses.sum().item()
        total_off += (lse_off[here] + z_off.gather(1, place)[here, 0] + 2 * E * losses.abs()).sum().item()

        dz = torch.exp(z - kept[:, None])
        dz_off = 1.01 * dz * (z_off + 4 * E * (z.abs() + kept.abs()[:, None] + 1.0))
        del z, z_off
        dz.scatter_add_(1, place, torch.full_like(place, -1, dtype=torch.float64))
        dz_off = (1 + u) * dz_off + u * dz.abs() + (2.0 ** -39 if dtype == "float16" else 0.0)
        dz, dz_off = dz * here[:, None], dz_off * here[:, None]
        dz_size = dz.abs() + dz_off
        bound = torch.mm(dz_off, w_size) + torch.mm(dz_size, w_size) * _off(classes, dtype)
        _check(got_dx[part], torch.mm(dz, wd) / count, bound / count, dtype)
        dw += torch.mm(dz.t().contiguous(), xd)
        dw_off += torch.mm(dz_off.t().contiguous(), xd.abs())
        dw_size += torch.mm(dz_size.t().contiguous(), xd.abs())
    assert abs(loss.item() - total / count) <= (total_off + 2 * E * total) / count
    _check(got_dw, dw / count, (dw_off + dw_size * _off(rows, dtype)) / count, dtype)
    assert not torch.any(got_dx[~there])


def test_pieces_of_many_rows():
    """Some of them, the first and the last among them, against 64 bits."""
    dtype, rows, classes, width, _ = MANY_ROWS
    x, weight, target = _problem(dtype, rows, classes, width)
    wrap = nt.Tensor._from_storage
    each, lse = (torch.full((rows,), -1.0, device="cuda") for _ in range(2))
    F.linear_cross_entropy_forward(wrap(x), wrap(weight), wrap(target), reduction="none", out=(wrap(each), wrap(lse)))
    some = torch.cat([torch.arange(1000), torch.arange(1000, rows - 1000, 4099), torch.arange(rows - 1000, rows)]).cuda()
    there, place = (target[some] != -100), target[some].clamp(min=0)[:, None]
    xd, wd = x[some].double(), weight.double()
    z = torch.mm(xd, wd.t().contiguous())
    z_off = torch.mm(xd.abs(), wd.abs().t().contiguous()) * _off(width, dtype)
    expected = torch.logsumexp(z, dim=1)
    lse_off = _lse_bound(z_off, expected, classes)
    losses = expected - z.gather(1, place)[:, 0]
    losses_off = lse_off + z_off.gather(1, place)[:, 0] + 2 * E * losses.abs()
    assert torch.all((lse[some].double() - expected).abs()[there] <= lse_off[there])
    assert torch.all((each[some].double() - losses).abs()[there] <= losses_off[there])
    assert not torch.any(lse[target == -100]) and not torch.any(each[target == -100])
