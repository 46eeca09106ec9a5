"""What a training or serving program asks of the residual path's operators, as measurable cases.

A transformer's residual stream meets three operators between its matrix products: dropout, the addition, and layer
norm, with their gradients.  The cases call them as ``namitorch_amd.functional`` offers them:

* ``norm``: layer norm of rows; ``norm_grad``: its backward pass, with the gradients of weight and bias;
* ``drop``: dropout (its backward pass is the same call on the gradient);
* ``edge``: dropout of a branch, added to the residual stream, and the layer norm of the sum; ``edge_grad``: its
  backward pass.

The dropout mask is never stored.  Element ``i`` of the flattened tensor is dropped where the 16-bit number
``u(seed, offset, i)`` is below ``T = round(65536 p)``; kept elements are multiplied by ``65536 / (65536 - T)``.
``u`` is half ``i % 2`` of word ``i % 8 // 2`` of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
numbers: as easy as 1, 2, 3", 2011) with the 64-bit counter words ``i // 8`` and ``offset`` and the key ``seed``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
_EPS = 1e-5
# Activations of the largest listed case (bytes of one such tensor): what a drawn one may have at most.
_LARGEST = 16384 * 4096 * 2


def listed():
    return [
        # Serving, one sequence: the final norm of one new token of GPT-2 124M.  Launch and host cost.
        {"name": "norm_token", "kind": "norm", "rows": 1, "width": 768, "dtype": "float16", "weight": "float16",
         "stats": False},
        # Training GPT-2 124M: 8 sequences of 1024, bfloat16 activations, float32 weights.
        {"name": "norm_gpt2", "kind": "norm", "rows": 8192, "width": 768, "dtype": "bfloat16", "weight": "float32"},
        # Float32 with sizes that fit nothing: packed sequences of odd length, an odd model width.
        {"name": "norm_odd", "kind": "norm", "rows": 5003, "width": 1001, "dtype": "float32", "weight": "float32"},
        # The backward pass of GPT-2 124M's norms, weights in the activations' type.
        {"name": "norm_grad_gpt2", "kind": "norm_grad", "rows": 8192, "width": 768, "dtype": "bfloat16",
         "weight": "bfloat16"},
        # Few rows, each long: the column sums have little to run over, the rows much.
        {"name": "norm_grad_wide", "kind": "norm_grad", "rows": 129, "width": 8192, "dtype": "float16",
         "weight": "float32"},
        # GPT 1.3B in float32 (2048 wide, 4 sequences of 2048).
        {"name": "norm_grad_1p3b", "kind": "norm_grad", "rows": 8192, "width": 2048, "dtype": "float32",
         "weight": "float32"},
        # Dropout of a short batch's embeddings.
        {"name": "drop_small", "kind": "drop", "rows": 33, "width": 768, "dtype": "float32", "p": 0.1},
        # Dropout inside GPT 1.3B's feed-forward layer (8192 wide).
        {"name": "drop_ffn", "kind": "drop", "rows": 8192, "width": 8192, "dtype": "bfloat16", "p": 0.1},
        # Serving a batch of 64 sequences, one token each: residual addition and norm, no dropout.
        {"name": "edge_tokens", "kind": "edge", "rows": 64, "width": 2048, "dtype": "bfloat16", "weight": "bfloat16",
         "p": 0.0, "stats": False},
        # The edge between two blocks of GPT-2 124M in training.
        {"name": "edge_gpt2", "kind": "edge", "rows": 8192, "width": 768, "dtype": "bfloat16", "weight": "float32",
         "p": 0.1},
        # Its backward pass.
        {"name": "edge_grad_gpt2", "kind": "edge_grad", "rows": 8192, "width": 768, "dtype": "bfloat16",
         "weight": "float32", "p": 0.1},
        # The largest: 16384 tokens of a 4096-wide model, float16.
        {"name": "edge_grad_4096", "kind": "edge_grad", "rows": 16384, "width": 4096, "dtype": "float16",
         "weight": "float32", "p": 0.1},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "drop", "edge", "edge_grad"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    width = _spread(rng, 8, 16384)
    rows = _spread(rng, 1, max(1, min(65536, _LARGEST // (width * _SIZE[dtype]))))
    case = {"kind": kind, "rows": rows, "width": width, "dtype": dtype}
    if kind != "drop":
        case["weight"] = rng.choice([dtype, "float32"])
        case["bias"] = rng.random() < 0.8
    if kind not in ("norm", "norm_grad"):
        case["p"] = rng.choice([0.1, 0.1, 0.2, 0.5]) if kind == "drop" else rng.choice([0.0, 0.1, 0.1, 0.35])
    if kind in ("norm", "edge"):
        case["stats"] = rng.random() < 0.7
    return case


# ---- inputs -----------------------------------------------------------------------------------------
def _normal(generator, shape, dtype, scale=1.0, shift=None):
    values = torch.randn(shape, generator=generator, device="cuda").mul_(scale)
    if shift is not None:
        values.add_(shift)
    return values.to(_TORCH[dtype])


def _inputs(case, seed):
    """Activations with an offset and a few strong columns, as residual streams have them; weights near one."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    shape, dtype, kind = (case["rows"], case["width"]), case["dtype"], case["kind"]
    given = {}
    if kind != "drop":
        given["weight"] = _normal(generator, (case["width"],), case["weight"], 0.2, 1.0)
        given["bias"] = _normal(generator, (case["width"],), case["weight"], 0.1) if case.get("bias", True) else None
        strong = 0.2 * torch.randn(case["width"], generator=generator, device="cuda")
        strong[::97] *= 8.0
    if kind in ("norm", "drop"):
        given["input"] = _normal(generator, shape, dtype, 1.0, strong if kind == "norm" else None)
    elif kind == "edge":
        given["input"] = _normal(generator, shape, dtype, 0.5)
        given["residual"] = _normal(generator, shape, dtype, 1.0, strong)
    else:
        name = "input" if kind == "norm_grad" else "total"
        given[name] = _normal(generator, shape, dtype, 1.0, strong)
        # What the forward pass kept of each row.
        var, mean = torch.var_mean(given[name].double(), dim=1, correction=0)
        given["mean"], given["rstd"] = mean.float(), var.add_(_EPS).rsqrt_().float()
        given["grad_output"] = _normal(generator, shape, dtype, 0.05)
        if kind == "edge_grad":
            given["grad_total"] = _normal(generator, shape, dtype, 0.05)
    if "p" in case:
        given["seed"], given["offset"] = 0x9E3779B97F4A7C15 * (2 * seed + 1) % 2**64, 1000 + seed
    return given


def _outputs(case):
    """What one call writes, by name: (shape, dtype)."""
    shape, dtype, kind = (case["rows"], case["width"]), case["dtype"], case["kind"]
    stats = {"mean": (shape[:1], "float32"), "rstd": (shape[:1], "float32")} if case.get("stats", True) else {}
    if kind == "drop":
        return {"output": (shape, dtype)}
    if kind == "norm":
        return {"output": (shape, dtype), **stats}
    if kind == "edge":
        return {"output": (shape, dtype), "total": (shape, dtype), **stats}
    made = {"grad_input": (shape, dtype)}
    if kind == "edge_grad":
        made["grad_residual"] = (shape, dtype)
    made["grad_weight"] = (shape[1:], case["weight"])
    if case.get("bias", True):
        made["grad_bias"] = (shape[1:], case["weight"])
    return made


def prepare(case, seed):
    held = {"case": case, "given": _inputs(case, seed)}
    if own:
        # A program that shares the GPU with PyTorch: launches follow PyTorch's stream, the package's Tensors are
        # PyTorch's memory, and each step's results go to the same buffers.
        import namitorch_amd as nt
        nt.runtime.set_stream_provider(lambda device: torch.cuda.current_stream(device).cuda_stream)
        wrap = lambda value: nt.Tensor._from_storage(value) if isinstance(value, torch.Tensor) else value  # noqa: E731
        held["tensors"] = {name: wrap(value) for name, value in held["given"].items()}
        held["results"] = {name: torch.empty(shape, dtype=_TORCH[dtype], device="cuda")
                           for name, (shape, dtype) in _outputs(case).items()}
        names = {"norm_grad": ("grad_input", "grad_weight", "grad_bias"),
                 "edge_grad": ("grad_input", "grad_residual", "grad_weight", "grad_bias")}.get(case["kind"])
        made = {name: wrap(value) for name, value in held["results"].items()}
        held["out"] = tuple(map(made.get, names)) if names else tuple(made.values())
    return held


# ---- the calls ----------------------------------------------------------------------------------------
def _run_own(held):
    from namitorch_amd import functional as F
    case, t, out = held["case"], held["tensors"], held["out"]
    kind, shape = case["kind"], (case["width"],)
    if kind == "norm":
        if case.get("stats", True):
            F.layer_norm_forward(t["input"], shape, t["weight"], t["bias"], _EPS, out=out)
        else:
            F.layer_norm(t["input"], shape, t["weight"], t["bias"], _EPS, out=out[0])
    elif kind == "norm_grad":
        F.layer_norm_backward(t["grad_output"], t["input"], t["mean"], t["rstd"], t["weight"], t["bias"], out=out)
    elif kind == "drop":
        F.dropout(t["input"], case["p"], seed=t["seed"], offset=t["offset"], out=out[0])
    elif kind == "edge":
        call = F.dropout_add_layer_norm_forward if case.get("stats", True) else F.dropout_add_layer_norm
        call(t["input"], t["residual"], shape, t["weight"], t["bias"], case["p"], _EPS, seed=t["seed"],
             offset=t["offset"], out=out)
    else:
        F.dropout_add_layer_norm_backward(t["grad_output"], t["grad_total"], t["total"], t["mean"], t["rstd"],
                                          t["weight"], t["bias"], case["p"], seed=t["seed"], offset=t["offset"],
                                          out=out)
    return held["results"]


# ---- the plain forms ------------------------------------------------------------------------------------
_LOW = 0xFFFFFFFF


def _kept(count, p, seed, offset):
    """(truth value per element of the flat tensor, factor of the kept ones).  Products of 32-bit words wrap in
    64 bits, of which both halves are read."""
    threshold = round(65536 * p)
    group = torch.arange(-(-count // 8), device="cuda")
    a, b = group & _LOW, group >> 32
    c = torch.full_like(group, offset & _LOW)
    d = torch.full_like(group, offset >> 32 & _LOW)
    k, m = seed & _LOW, seed >> 32 & _LOW
    for _ in range(10):
        left, right = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = right >> 32 & _LOW ^ b ^ k, right & _LOW, left >> 32 & _LOW ^ d ^ m, left & _LOW
        k, m = k + 0x9E3779B9 & _LOW, m + 0xBB67AE85 & _LOW
    halves = torch.stack([half for word in (a, b, c, d) for half in (word & 0xFFFF, word >> 16)], dim=1)
    factor = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    return halves.view(-1)[:count] >= threshold, factor


def _dropped(x, p, seed, offset):
    if p == 0.0:
        return x
    kept, factor = _kept(x.numel(), p, seed, offset)
    return torch.where(kept.view(x.shape), x * factor, 0.0)


def _normed(x, weight, bias):
    mean = x.mean(dim=1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + _EPS)
    y = centred * rstd * weight.float()
    return (y if bias is None else y + bias.float()), mean.view(-1), rstd.view(-1)


def _normed_grad(grad, x, given):
    """Gradients of the norm by its input (32 bits), weight and bias."""
    weight, bias = given["weight"], given["bias"]
    hat = (x - given["mean"][:, None]) * given["rstd"][:, None]
    by = grad * weight.float()
    grad_x = (by - by.mean(dim=1, keepdim=True) - hat * (by * hat).mean(dim=1, keepdim=True)) * given["rstd"][:, None]
    made = {"grad_weight": (grad * hat).sum(dim=0).to(weight.dtype)}
    if bias is not None:
        made["grad_bias"] = grad.sum(dim=0).to(bias.dtype)
    return grad_x, made


def _run_plain(held):
    case, given = held["case"], held["given"]
    kind, dtype, stats = case["kind"], _TORCH[case["dtype"]], case.get("stats", True)
    if kind == "drop":
        return {"output": _dropped(given["input"].float(), case["p"], given["seed"], given["offset"]).to(dtype)}
    if kind in ("norm", "edge"):
        x = given["input"].float()
        if kind == "edge":
            x = _dropped(x, case["p"], given["seed"], given["offset"]) + given["residual"].float()
        y, mean, rstd = _normed(x, given["weight"], given["bias"])
        made = {"output": y.to(dtype)}
        if kind == "edge":
            made["total"] = x.to(dtype)
        return {**made, "mean": mean, "rstd": rstd} if stats else made
    grad = given["grad_output"].float()
    if kind == "norm_grad":
        grad_x, made = _normed_grad(grad, given["input"].float(), given)
        return {"grad_input": grad_x.to(dtype), **made}
    grad_x, made = _normed_grad(grad, given["total"].float(), given)
    grad_x = grad_x + given["grad_total"].float()
    grad_in = _dropped(grad_x, case["p"], given["seed"], given["offset"])
    return {"grad_input": grad_in.to(dtype), "grad_residual": grad_x.to(dtype), **made}


def run(held):
    return _run_own(held) if own else _run_plain(held)


# ---- the definition in 64 bits ------------------------------------------------------------------------------
def _mask64(count, p, seed, offset):
    """1 / (1 - T / 65536) for each kept element and 0 for each dropped one, with NumPy's unsigned words."""
    threshold = round(65536 * p)
    word = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    groups = -(-count // 8)
    state = np.empty((4, groups), dtype=np.uint64)
    state[0] = np.arange(groups, dtype=np.uint64)
    state[1] = state[0] >> shift
    state[0] &= word
    state[2], state[3] = offset % 2**32, offset // 2**32
    key = [seed % 2**32, seed // 2**32]
    for _ in range(10):
        first = state[0] * np.uint64(0xD2511F53)
        second = state[2] * np.uint64(0xCD9E8D57)
        state[0] = (second >> shift) ^ state[1] ^ np.uint64(key[0])
        state[2] = (first >> shift) ^ state[3] ^ np.uint64(key[1])
        state[1] = second & word
        state[3] = first & word
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    numbers = np.ascontiguousarray(state.T.astype("<u4")).view("<u2").reshape(-1)[:count]
    made = torch.from_numpy(numbers.astype(np.int32)).cuda() >= threshold
    return made.double() * (1.0 / (1.0 - threshold / 65536.0) if threshold < 65536 else 0.0)


def exact(case, seed):
    if case["rows"] * case["width"] > 70_000_000:
        return None
    given = {name: value.double() if isinstance(value, torch.Tensor) else value
             for name, value in _inputs(case, seed).items()}
    kind = case["kind"]
    mask = 1.0
    if case.get("p"):
        mask = _mask64(case["rows"] * case["width"], case["p"], given["seed"], given["offset"])
        mask = mask.view(case["rows"], case["width"])
    if kind == "drop":
        return {"output": given["input"] * mask}
    weight = given["weight"]
    if kind in ("norm", "edge"):
        x = given["input"] if kind == "norm" else given["input"] * mask + given["residual"]
        variance, mean = torch.var_mean(x, dim=1, correction=0)
        deviation = torch.sqrt(variance + _EPS)
        y = (x - mean.unsqueeze(1)) / deviation.unsqueeze(1) * weight
        if given["bias"] is not None:
            y = y + given["bias"]
        made = {"output": y, "mean": mean, "rstd": 1.0 / deviation, "total": x if kind == "edge" else None}
        return {name: made[name] for name in _outputs(case)}
    # Of the two projections that the norm's Jacobian takes out, each as a vector product per row.
    rows, rstd = given["input" if kind == "norm_grad" else "total"], given["rstd"].unsqueeze(1)
    hat = (rows - given["mean"].unsqueeze(1)) * rstd
    dy = given["grad_output"]
    made = {"grad_weight": torch.sum(dy * hat, 0), "grad_bias": torch.sum(dy, 0)}
    by = dy * weight
    along, level = torch.sum(by * hat, 1, keepdim=True), torch.sum(by, 1, keepdim=True)
    made["grad_input"] = rstd * (by - (level + hat * along) / case["width"])
    if kind == "edge_grad":
        made["grad_residual"] = made["grad_input"] + given["grad_total"]
        made["grad_input"] = made["grad_residual"] * mask
    return {name: made[name] for name in _outputs(case)}


# ---- what one pass cannot do without ----------------------------------------------------------------------
def work(case):
    n, rows, width = case["rows"] * case["width"], case["rows"], case["width"]
    size, kind = _SIZE[case["dtype"]], case["kind"]
    random = 10 * n if case.get("p") else 0             # integer operations of the generator, eight elements a call
    if kind == "drop":
        return {"bytes": 2 * size * n, "flops": random + n}
    vectors = (2 if case.get("bias", True) else 1) * width * _SIZE[case["weight"]]
    stats = 8 * rows if case.get("stats", True) else 0
    if kind in ("norm", "edge"):
        return {"bytes": (2 if kind == "norm" else 4) * size * n + vectors + stats, "flops": 8 * n + random}
    read = width * _SIZE[case["weight"]]
    return {"bytes": (3 if kind == "norm_grad" else 5) * size * n + vectors + read + stats, "flops": 14 * n + random}
