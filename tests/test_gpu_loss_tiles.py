"""The linear cross entropy at sizes of each choice of tiles, against PyTorch's 64-bit products on the device.

Bounds, element by element, e = 2**-24 and u the half ulp of the dtype (float32's three parts hold a value to
2**-24).  A sum of k products is off by 2 k e of the sum of their magnitudes (the matrix cores may truncate each
step), of float32's six products a pair by 12 k e and the 2**-23 that is left out.  exp(z - lse) is off by the
logit's error and the roundings of its argument, 4 e (|z| + |lse|), and 4 e of its own; dz by u more, in float16
by half the smallest subnormal too, 2**-25, after a scale of 2**14 or more.  Results are multiplied by a rounded
factor, 3 e, and rounded once, off by TINY where they are subnormal."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import namitorch_amd as nt
from namitorch_amd import functional as F

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF_ULP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def _off(k, dtype):
    return 2 * k * E if dtype != "float32" else 12 * k * E + 2.0 ** -23


def _get(tensor):
    values = tensor.numpy()
    return torch.from_numpy(np.ascontiguousarray(values.astype(np.float64))).cuda()


def _product(a, b):
    return torch.mm(a, b.contiguous())


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows, classes, width", [
    (129, 50304, 520),      # tall logits, gradients of 128 x 128
    (256, 33001, 1024),     # the same, with weights read in place whose last lines do not fill a step
    (200, 17000, 72),       # the same, little of it
    (200, 10007, 1001),     # small logits for want of tiles
    (300, 3000, 520),       # 128 x 128
    (777, 10007, 1001),     # large logits, gradients of 128 x 128
    (1040, 32100, 1000),    # large ones
])
def test_tiles(rows, classes, width, dtype):
    generator = torch.Generator(device="cuda").manual_seed(rows)
    kind = getattr(torch, dtype)
    weight = (torch.randn(classes, width, generator=generator, device="cuda") * (2.0 / width ** 0.5)).to(kind)
    target = torch.randint(0, classes, (rows,), generator=generator, device="cuda")
    x = torch.randn(rows, width, generator=generator, device="cuda")
    x = (x + 2.0 * torch.rand(rows, 1, generator=generator, device="cuda") * weight[target].float()).to(kind)
    target[::7] = -100
    wrap = nt.Tensor._from_storage
    loss, lse = F.linear_cross_entropy_forward(wrap(x), wrap(weight), wrap(target))
    got_dx, got_dw = F.linear_cross_entropy_backward(1.0, wrap(x), wrap(weight), wrap(target), lse)

    there = target != -100
    count, u = int(there.sum()), HALF_ULP[dtype]
    xd, wd = x.double() * there[:, None], weight.double()
    z = _product(xd, wd.t())
    z_off = _product(xd.abs(), wd.abs().t()) * _off(width, dtype)
    expected = torch.logsumexp(z, dim=1)
    kept = _get(lse)
    lse_off = z_off.amax(dim=1) + (classes / 1024 + 200) * E + 4 * E * expected.abs()
    assert torch.all((kept - expected).abs()[there] <= lse_off[there])
    assert torch.all(kept[~there] == 0.0)
    at = target.clamp(min=0)[:, None]
    each = (expected - z.gather(1, at)[:, 0])[there]
    each_off = lse_off[there] + z_off.gather(1, at)[there, 0] + 2 * E * each.abs()
    assert abs(float(loss.numpy()) - each.sum().item() / count) <= (each_off.sum().item() + 2 * E * each.sum().item()) / count

    dz = torch.exp(z - kept[:, None])
    dz_off = 1.01 * dz * (z_off + 4 * E * (z.abs() + kept.abs()[:, None] + 1.0))
    del z, z_off
    dz.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float64))
    dz_off = (1 + u) * dz_off + u * dz.abs() + (2.0 ** -39 if dtype == "float16" else 0.0)
    dz, dz_off = dz * there[:, None], dz_off * there[:, None]
    for got, exact, off, size, depth in (
            (got_dx, _product(dz, wd), _product(dz_off, wd.abs()), _product(dz.abs() + dz_off, wd.abs()), classes),
            (got_dw, _product(dz.t(), xd), _product(dz_off.t(), xd.abs()), _product((dz.abs() + dz_off).t(), xd.abs()),
             rows)):
        exact, bound = exact / count, (off + size * _off(depth, dtype)) / count
        bound = bound + (u + 3 * E) * (exact.abs() + bound) + TINY[dtype]
        wrong = (_get(got) - exact).abs() > bound
        assert not wrong.any(), (int(wrong.sum()), wrong.nonzero()[:4].tolist())


def test_two_threads():
    """Calls of two threads, on streams of their own and on one, give what each gives alone."""
    generator = torch.Generator(device="cuda").manual_seed(3)
    wrap = nt.Tensor._from_storage

    def made(rows, classes, width):
        weight = torch.randn(classes, width, generator=generator, device="cuda") * 0.1
        x = torch.randn(rows, width, generator=generator, device="cuda")
        target = torch.randint(0, classes, (rows,), generator=generator, device="cuda")
        return wrap(x), wrap(weight), wrap(target)

    def call(problem):
        loss, lse = F.linear_cross_entropy_forward(*problem)
        return (loss, lse, *F.linear_cross_entropy_backward(1.0, *problem, lse))

    problems = [made(300, 1500, 72), made(70, 4000, 128)]
    alone = [[np.array(t.numpy()) for t in call(problem)] for problem in problems]
    torch.cuda.synchronize()
    for shared in (True, False):
        found = [None, None]

        def work(k, stream):
            with torch.cuda.stream(stream):
                results = [call(problems[k]) for _ in range(20)]
                stream.synchronize()
                found[k] = [[np.array(t.numpy()) for t in result] for result in results]

        one = torch.cuda.Stream()
        threads = [threading.Thread(target=work, args=(k, one if shared else torch.cuda.Stream())) for k in range(2)]
        for thread in threads:
            thread.start()
        for thread in threads:
            thread.join()
        for k in range(2):
            assert found[k] is not None
            for result in found[k]:
                assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(result, alone[k]))
