"""The ends of a block and the end of a model, as measurable cases.

Four calls of ``namitorch_amd.functional``, each on the path that carries a model's values and gradients between its
matrix products and its optimizer:

* ``loss``: softmax cross entropy of ``input @ weight.T`` over a large vocabulary, whose logits are never kept, and
  ``loss_grad``: its backward pass, the gradients of both factors;
* ``gated``: the edge after a block that is normalized on both sides, ``total = s residual + gate norm(branch)`` and
  the norm of ``total`` for the next block, and ``gated_grad``: its backward pass.

With ``z = x W^T`` (rows ``i``, classes ``v``), target ``t_i`` and ``c`` rows that are not ignored:
``lse_i = log sum_v exp z_iv``, ``loss_i = lse_i - z_i,t_i``, both zero in ignored rows, of which the mean (over
``c``), the sum or each is returned; ``dz_iv = g_i (exp(z_iv - lse_i) - [v = t_i])`` with ``g_i = grad_loss / c`` (or
the sum's or the row's own) and zero in ignored rows; ``dx = dz W``, ``dW = dz^T x``.

With ``N(x; w, b) = (x - mean) rstd w + b`` (``rms``: no mean): ``total = s r + a N(x; u, k)``, ``y = N(total; w, b)``
and, given ``dy`` and what ``total`` gets from elsewhere, the gradients of ``x``, ``r``, ``u``, ``k``, ``a``, ``w``
and ``b``.  The gate ``a`` has one row for all tokens, one for each sequence, or one for each token.
"""

from __future__ import annotations

import math

import torch

own = False

_TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
_EPS = 1e-5
_IGNORED = -100
_SHARE_IGNORED = 0.1
_MOST_WORK = 6 * 8192 * 32000 * 4096        # operations of the largest listed loss
_MOST_LOGITS = 8192 * 50257                 # what the plain form holds at a time
_MOST_WEIGHT = 32000 * 4096
_MOST_ROWS = 16384 * 4096                   # elements of the largest listed edge


def listed():
    return [
        # Scoring one token with GPT-2 124M: the head is read once, the rest is launch and host cost.
        {"name": "loss_token", "kind": "loss", "rows": 1, "classes": 50257, "width": 768, "dtype": "float16",
         "reduction": "none"},
        # Training GPT-2 124M: 8 sequences of 1024, a tenth of the tokens is padding.
        {"name": "loss_gpt2", "kind": "loss", "rows": 8192, "classes": 50257, "width": 768, "dtype": "bfloat16",
         "reduction": "mean"},
        # Float32 with sizes that fit nothing.
        {"name": "loss_odd", "kind": "loss", "rows": 777, "classes": 10007, "width": 1001, "dtype": "float32",
         "reduction": "mean"},
        # A short batch with a weight for each token, the head of GPT 1.3B in float16 under a loss scale.
        {"name": "loss_grad_short", "kind": "loss_grad", "rows": 129, "classes": 50304, "width": 2048,
         "dtype": "float16", "reduction": "none"},
        # The backward pass in float32, sizes that fit nothing.
        {"name": "loss_grad_odd", "kind": "loss_grad", "rows": 777, "classes": 10007, "width": 1001,
         "dtype": "float32", "reduction": "mean"},
        # The backward pass of GPT-2 124M.
        {"name": "loss_grad_gpt2", "kind": "loss_grad", "rows": 8192, "classes": 50257, "width": 768,
         "dtype": "bfloat16", "reduction": "mean"},
        # The largest: the untied head of the Llama-7B layout, 8192 tokens.
        {"name": "loss_grad_7b", "kind": "loss_grad", "rows": 8192, "classes": 32000, "width": 4096,
         "dtype": "bfloat16", "reduction": "mean"},
        # Serving one token of a 4096-wide model with root mean square norms.
        {"name": "gated_token", "kind": "gated", "rows": 1, "sequences": 1, "width": 4096, "dtype": "float16",
         "weight": "float16", "norm": "rms", "gate": "shared", "bias": False, "scale": 1.0, "stats": False},
        # Training: 8 sequences of 1024 of a 768-wide model, a gate for each sequence.
        {"name": "gated_768", "kind": "gated", "rows": 8192, "sequences": 8, "width": 768, "dtype": "bfloat16",
         "weight": "float32", "norm": "layer", "gate": "sequence", "bias": True, "scale": 1.0},
        # Its backward pass.
        {"name": "gated_grad_768", "kind": "gated_grad", "rows": 8192, "sequences": 8, "width": 768,
         "dtype": "bfloat16", "weight": "float32", "norm": "layer", "gate": "sequence", "bias": True, "scale": 1.0},
        # Float32, odd sizes, a gate that the model computes for each token.
        {"name": "gated_grad_odd", "kind": "gated_grad", "rows": 5003, "sequences": 1, "width": 1001,
         "dtype": "float32", "weight": "float32", "norm": "layer", "gate": "token", "bias": True, "scale": 0.5},
        # 16384 tokens of a 4096-wide model: root mean square norms, a learned gate of each channel.
        {"name": "gated_grad_4096", "kind": "gated_grad", "rows": 16384, "sequences": 8, "width": 4096,
         "dtype": "bfloat16", "weight": "bfloat16", "norm": "rms", "gate": "shared", "bias": False, "scale": 1.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["loss", "loss_grad", "gated", "gated_grad"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind in ("loss", "loss_grad"):
        while True:
            rows, classes, width = _spread(rng, 1, 16384), _spread(rng, 256, 131072), _spread(rng, 32, 8192)
            if rng.random() < 0.5:
                width = max(8, width // 64 * 64)
            if (6 * rows * classes * width <= _MOST_WORK and rows * classes <= _MOST_LOGITS
                    and classes * width <= _MOST_WEIGHT):
                return {"kind": kind, "rows": rows, "classes": classes, "width": width, "dtype": dtype,
                        "reduction": rng.choice(["mean", "mean", "sum", "none"])}
    width = _spread(rng, 8, 16384)
    rows = _spread(rng, 1, max(1, min(65536, 2 * _MOST_ROWS // (width * _SIZE[dtype]))))
    sequences = rng.choice([1, 2, 4, 7, 16])
    if sequences > rows:
        sequences = 1
    case = {"kind": kind, "rows": rows // sequences * sequences, "sequences": sequences, "width": width,
            "dtype": dtype, "weight": rng.choice([dtype, "float32"]), "norm": rng.choice(["layer", "rms"]),
            "gate": rng.choice(["shared", "sequence", "token", "none"]), "bias": rng.random() < 0.6,
            "scale": rng.choice([1.0, 1.0, 0.5, 1.25])}
    if kind == "gated":
        case["stats"] = rng.random() < 0.7
    return case


# ---- inputs -----------------------------------------------------------------------------------------
def _normal(generator, shape, dtype, scale=1.0, shift=None):
    values = torch.randn(shape, generator=generator, device="cuda").mul_(scale)
    if shift is not None:
        values += shift
    return values.to(_TORCH[dtype])


def _grad_loss(case):
    """The loss's own gradient, a number: one, or under float16 a loss scale."""
    return 4096.0 if case["dtype"] == "float16" else 1.0


def _loss_inputs(case, seed):
    """A model that has learnt something: frequent classes, logits a few units wide, the target's raised."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rows, classes, width = case["rows"], case["classes"], case["width"]
    dtype = _TORCH[case["dtype"]]
    uniform = torch.rand(rows, generator=generator, device="cuda", dtype=torch.float64)
    target = (torch.exp(uniform * math.log(classes + 1)) - 1).long().clamp_(0, classes - 1)
    weight = torch.randn(classes, width, generator=generator, device="cuda").mul_(2.0 * width ** -0.5)
    # The target's logit gains about 0 to 12.
    lift = 3.0 * torch.rand(rows, 1, generator=generator, device="cuda")
    x = torch.randn(rows, width, generator=generator, device="cuda").addcmul_(weight[target], lift)
    given = {"input": x.to(dtype), "weight": weight.to(dtype)}
    if rows > 1:
        target[torch.rand(rows, generator=generator, device="cuda") < _SHARE_IGNORED] = _IGNORED
    given["target"] = target
    if case["kind"] == "loss_grad":
        lse = torch.empty(rows, device="cuda", dtype=torch.float32)
        weight = given["weight"].float()
        for first in range(0, rows, 2048):              # what the forward pass kept
            logits = given["input"][first:first + 2048].float() @ weight.t()
            most = logits.amax(dim=1, keepdim=True)
            lse[first:first + 2048] = (logits - most).double().exp_().sum(dim=1).log_().add_(most[:, 0]).float()
        given["lse"] = lse
        if case["reduction"] == "none":
            given["grad_loss"] = torch.rand(rows, generator=generator, device="cuda") * (_grad_loss(case) / rows)
        else:
            given["grad_loss"] = _grad_loss(case)
    return given


def _gate_shape(case):
    rows, sequences, width = case["rows"], case["sequences"], case["width"]
    return {"shared": (width,), "sequence": (sequences, 1, width),
            "token": (sequences, rows // sequences, width)}[case["gate"]]


def _gated_inputs(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rows, width, dtype, weight = case["rows"], case["width"], case["dtype"], case["weight"]
    shape = (case["sequences"], rows // case["sequences"], width)
    given = {}
    for name in ("inner_weight", "weight"):
        given[name] = _normal(generator, (width,), weight, 0.2, 1.0)
    for name in ("inner_bias", "bias"):
        given[name] = _normal(generator, (width,), weight, 0.1) if case["bias"] else None
    given["gate"] = None if case["gate"] == "none" else _normal(generator, _gate_shape(case), dtype, 0.3, 0.5)
    # A residual stream has a few channels that stand out.
    strong = 0.2 * torch.randn(width, generator=generator, device="cuda")
    strong[::97] *= 8.0
    given["input"] = _normal(generator, shape, dtype, 0.5, 0.05)
    if case["kind"] == "gated":
        given["residual"] = _normal(generator, shape, dtype, 1.0, strong)
        return given
    given["total"] = _normal(generator, shape, dtype, 1.0, strong)
    for name, of in (("inner_", "input"), ("", "total")):      # what the forward pass kept of each row
        values = given[of].double()
        mean = values.mean(dim=2) if case["norm"] == "layer" else values.new_zeros(shape[:2])
        var = (values * values).mean(dim=2) - mean * mean
        given[name + "mean"] = mean.float() if case["norm"] == "layer" else None
        given[name + "rstd"] = (var + _EPS).rsqrt_().float()
    given["grad_output"] = _normal(generator, shape, dtype, 0.05)
    given["grad_total"] = _normal(generator, shape, dtype, 0.05)
    return given


def _inputs(case, seed):
    return _loss_inputs(case, seed) if case["kind"] in ("loss", "loss_grad") else _gated_inputs(case, seed)


def _outputs(case):
    """What one call writes, by name: (shape, dtype), or None for what it has not."""
    kind, dtype, rows, width = case["kind"], case["dtype"], case["rows"], case["width"]
    if kind == "loss":
        return {"loss": ((rows,) if case["reduction"] == "none" else (), "float32"), "lse": ((rows,), "float32")}
    if kind == "loss_grad":
        return {"grad_input": ((rows, width), dtype), "grad_weight": ((case["classes"], width), dtype)}
    lead = (case["sequences"], rows // case["sequences"])
    data, vector = ((*lead, width), dtype), ((width,), case["weight"])
    if kind == "gated":
        made = {"output": data, "total": data}
        if case.get("stats", True):
            stat, mean = (lead, "float32"), (lead, "float32") if case["norm"] == "layer" else None
            made.update(inner_mean=mean, inner_rstd=stat, mean=mean, rstd=stat)
        return made
    shift = vector if case["bias"] else None
    return {"grad_input": data, "grad_residual": data, "grad_inner_weight": vector, "grad_inner_bias": shift,
            "grad_gate": None if case["gate"] == "none" else (_gate_shape(case), dtype),
            "grad_weight": vector, "grad_bias": shift}


def prepare(case, seed):
    held = {"case": case, "given": _inputs(case, seed)}
    if own:
        # A program that shares the GPU with PyTorch: launches follow PyTorch's stream, the package's Tensors are
        # PyTorch's memory, and each step's results go to the same buffers.
        import namitorch_amd as nt
        nt.runtime.set_stream_provider(lambda device: torch.cuda.current_stream(device).cuda_stream)
        wrap = lambda value: nt.Tensor._from_storage(value) if isinstance(value, torch.Tensor) else value  # noqa: E731
        held["tensors"] = {name: wrap(value) for name, value in held["given"].items()}
        made = {name: None if what is None else torch.empty(what[0], dtype=_TORCH[what[1]], device="cuda")
                for name, what in _outputs(case).items()}
        held["results"] = {name: value for name, value in made.items() if value is not None}
        held["out"] = tuple(map(wrap, made.values()))
    return held


# ---- the calls ----------------------------------------------------------------------------------------
def _run_own(held):
    from namitorch_amd import functional as F
    case, t, out = held["case"], held["tensors"], held["out"]
    kind = case["kind"]
    if kind == "loss":
        F.linear_cross_entropy_forward(t["input"], t["weight"], t["target"], reduction=case["reduction"], out=out)
    elif kind == "loss_grad":
        F.linear_cross_entropy_backward(t["grad_loss"], t["input"], t["weight"], t["target"], t["lse"],
                                        reduction=case["reduction"], out=out)
    elif kind == "gated":
        call = F.norm_gate_add_norm_forward if case.get("stats", True) else F.norm_gate_add_norm
        call(t["input"], t["residual"], (case["width"],), t["inner_weight"], t["inner_bias"], t["gate"], t["weight"],
             t["bias"], case["scale"], _EPS, norm=case["norm"], out=out)
    else:
        F.norm_gate_add_norm_backward(t["grad_output"], t["grad_total"], t["input"], t["total"], t["inner_mean"],
                                      t["inner_rstd"], t["mean"], t["rstd"], t["inner_weight"], t["inner_bias"],
                                      t["gate"], t["weight"], t["bias"], case["scale"], out=out)
    return held["results"]


# ---- the plain forms ------------------------------------------------------------------------------------
def _plain_loss(case, given):
    target = given["target"]
    logits = given["input"].float() @ given["weight"].float().t()
    most = logits.amax(dim=1, keepdim=True)
    counted = target != _IGNORED
    picked = logits.gather(1, target.clamp(min=0)[:, None])[:, 0]
    lse = logits.sub_(most).exp_().sum(dim=1).log_() + most[:, 0]
    loss, lse = torch.where(counted, lse - picked, 0.0), torch.where(counted, lse, 0.0)
    if case["reduction"] != "none":
        loss = loss.double().sum()
        if case["reduction"] == "mean":
            loss = loss / counted.sum().clamp(min=1)
    return {"loss": loss.float(), "lse": lse}


def _plain_loss_grad(case, given):
    target, x, weight = given["target"], given["input"].float(), given["weight"].float()
    counted = target != _IGNORED
    scale = given["grad_loss"] * counted.float()
    if case["reduction"] == "mean":
        scale = scale / counted.sum().clamp(min=1)
    grad = (x @ weight.t()).sub_(given["lse"][:, None]).exp_()
    place = target.clamp(min=0)[:, None]
    grad.scatter_add_(1, place, torch.full_like(place, -1, dtype=torch.float32))
    grad *= scale[:, None]
    return {"grad_input": (grad @ weight).to(given["input"].dtype),
            "grad_weight": (grad.t() @ x).to(given["weight"].dtype)}


def _centred(x, norm):
    """(x - mean, mean), or (x, None) for root mean square norms."""
    if norm == "rms":
        return x, None
    mean = x.mean(dim=-1, keepdim=True)
    return x - mean, mean


def _plain_norm(x, weight, bias, norm):
    centred, mean = _centred(x, norm)
    rstd = torch.rsqrt((centred * centred).mean(dim=-1, keepdim=True) + _EPS)
    y = centred * rstd * weight.float()
    return y if bias is None else y + bias.float(), None if mean is None else mean[..., 0], rstd[..., 0]


def _plain_gated(case, given):
    dtype, norm = _TORCH[case["dtype"]], case["norm"]
    inner, inner_mean, inner_rstd = _plain_norm(given["input"].float(), given["inner_weight"], given["inner_bias"], norm)
    if given["gate"] is not None:
        inner = inner * given["gate"].float()
    total = given["residual"].float() * case["scale"] + inner
    y, mean, rstd = _plain_norm(total, given["weight"], given["bias"], norm)
    made = {"output": y.to(dtype), "total": total.to(dtype)}
    if case.get("stats", True):
        stats = {"inner_mean": inner_mean, "inner_rstd": inner_rstd, "mean": mean, "rstd": rstd}
        made.update((name, value) for name, value in stats.items() if value is not None)
    return made


def _plain_norm_grad(grad, x, mean, rstd, weight):
    """(gradient of the norm's input, normalized input)."""
    hat = (x if mean is None else x - mean[..., None]) * rstd[..., None]
    by = grad * weight.float()
    inner = by - hat * (by * hat).mean(dim=-1, keepdim=True)
    if mean is not None:
        inner = inner - by.mean(dim=-1, keepdim=True)
    return inner * rstd[..., None], hat


def _plain_gated_grad(case, given):
    dtype, vector, every = _TORCH[case["dtype"]], _TORCH[case["weight"]], (0, 1)
    grad = given["grad_output"].float()
    through, hat = _plain_norm_grad(grad, given["total"].float(), given["mean"], given["rstd"], given["weight"])
    made = {"grad_weight": (grad * hat).sum(dim=every).to(vector)}
    if case["bias"]:
        made["grad_bias"] = grad.sum(dim=every).to(vector)
    total = through + given["grad_total"].float()
    made["grad_residual"] = (total * case["scale"]).to(dtype)
    gated = total if given["gate"] is None else total * given["gate"].float()
    by_input, inner = _plain_norm_grad(gated, given["input"].float(), given["inner_mean"], given["inner_rstd"],
                                       given["inner_weight"])
    made["grad_input"] = by_input.to(dtype)
    made["grad_inner_weight"] = (gated * inner).sum(dim=every).to(vector)
    if case["bias"]:
        made["grad_inner_bias"] = gated.sum(dim=every).to(vector)
    if given["gate"] is not None:
        branch = inner * given["inner_weight"].float()
        if case["bias"]:
            branch = branch + given["inner_bias"].float()
        by_gate = total * branch
        if case["gate"] == "shared":
            by_gate = by_gate.sum(dim=every)
        elif case["gate"] == "sequence":
            by_gate = by_gate.sum(dim=1, keepdim=True)
        made["grad_gate"] = by_gate.to(dtype)
    return {name: made[name] for name, what in _outputs(case).items() if what is not None}


_PLAIN = {"loss": _plain_loss, "loss_grad": _plain_loss_grad, "gated": _plain_gated, "gated_grad": _plain_gated_grad}


def run(held):
    return _run_own(held) if own else _PLAIN[held["case"]["kind"]](held["case"], held["given"])


# ---- the definitions in 64 bits ------------------------------------------------------------------------------
def _exact_loss(case, given, rows_at_once=1024):
    x, weight, target = given["input"].double(), given["weight"].double(), given["target"]
    known = target >= 0
    index = torch.where(known, target, 0)
    backward = case["kind"] == "loss_grad"
    if backward:
        share = known.double() * given["grad_loss"]
        if case["reduction"] == "mean":
            share /= max(1, int(known.sum()))
        dx, dw = torch.empty_like(x), torch.zeros_like(weight)
    lse, own_logit = x.new_empty(x.shape[0]), x.new_empty(x.shape[0])
    for first in range(0, x.shape[0], rows_at_once):
        part = slice(first, first + rows_at_once)
        z = torch.mm(x[part], weight.t())
        if backward:
            z = torch.exp(z - given["lse"][part].double()[:, None])
            z[torch.arange(z.shape[0], device=z.device), index[part]] -= 1.0
            z *= share[part][:, None]
            dx[part] = torch.mm(z, weight)
            dw.addmm_(z.t(), x[part])
        else:
            lse[part] = torch.logsumexp(z, dim=1)
            own_logit[part] = z[torch.arange(z.shape[0], device=z.device), index[part]]
    if backward:
        return {"grad_input": dx, "grad_weight": dw}
    loss, lse = (lse - own_logit) * known.double(), lse * known.double()
    if case["reduction"] == "sum":
        loss = loss.sum()
    elif case["reduction"] == "mean":
        loss = loss.sum() / max(1, int(known.sum()))
    return {"loss": loss, "lse": lse}


def _exact_gated(case, given):
    layer = case["norm"] == "layer"
    x, r = given["input"].double(), given["residual"].double()

    def normal(v, scale, shift):
        mean = v.mean(-1) if layer else None
        away = v - mean.unsqueeze(-1) if layer else v
        rstd = 1.0 / torch.sqrt(away.square().mean(-1) + _EPS)
        y = away * rstd.unsqueeze(-1) * scale.double()
        return (y + shift.double() if shift is not None else y), mean, rstd

    branch, inner_mean, inner_rstd = normal(x, given["inner_weight"], given["inner_bias"])
    gate = 1.0 if given["gate"] is None else given["gate"].double()
    total = case["scale"] * r + gate * branch
    y, mean, rstd = normal(total, given["weight"], given["bias"])
    made = {"output": y, "total": total, "inner_mean": inner_mean, "inner_rstd": inner_rstd, "mean": mean,
            "rstd": rstd}
    return {name: made[name] for name, what in _outputs(case).items() if what is not None}


def _exact_gated_grad(case, given):
    """Sums of products, from the derivative of each step of the definition."""
    at = {name: value.double() if isinstance(value, torch.Tensor) else value for name, value in given.items()}
    width = case["width"]

    def back(dy, v, mean, rstd, scale):
        away = v if mean is None else v - mean.unsqueeze(-1)
        rstd = rstd.unsqueeze(-1)
        d_hat = dy * scale
        d_away = d_hat * rstd - away * rstd ** 3 * (d_hat * away).sum(-1, keepdim=True) / width
        if mean is not None:
            d_away = d_away - d_away.sum(-1, keepdim=True) / width
        return d_away, away * rstd

    d_total, hat = back(at["grad_output"], at["total"], at["mean"], at["rstd"], at["weight"])
    d_total = d_total + at["grad_total"]
    gate = 1.0 if at["gate"] is None else at["gate"]
    d_branch = d_total * gate
    d_input, inner = back(d_branch, at["input"], at["inner_mean"], at["inner_rstd"], at["inner_weight"])
    made = {"grad_input": d_input, "grad_residual": d_total * case["scale"],
            "grad_inner_weight": (d_branch * inner).sum((0, 1)), "grad_inner_bias": d_branch.sum((0, 1)),
            "grad_weight": (at["grad_output"] * hat).sum((0, 1)), "grad_bias": at["grad_output"].sum((0, 1))}
    if at["gate"] is not None:
        branch = inner * at["inner_weight"] + (0.0 if at["inner_bias"] is None else at["inner_bias"])
        made["grad_gate"] = (d_total * branch).sum_to_size(_gate_shape(case))
    return {name: made[name] for name, what in _outputs(case).items() if what is not None}


def exact(case, seed):
    given = _inputs(case, seed)
    if case["kind"] in ("loss", "loss_grad"):
        return _exact_loss(case, given)
    return _exact_gated(case, given) if case["kind"] == "gated" else _exact_gated_grad(case, given)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    kind, rows, width, size = case["kind"], case["rows"], case["width"], _SIZE[case["dtype"]]
    if kind in ("loss", "loss_grad"):
        factors = (rows + case["classes"]) * width * size
        counted = rows if rows == 1 else round(rows * (1 - _SHARE_IGNORED))
        product = 2 * counted * case["classes"] * width
        per_row = rows * (8 + 4)                        # target and lse
        if kind == "loss":
            return {"bytes": factors + per_row + 4 * (rows if case["reduction"] == "none" else 1), "flops": product}
        return {"bytes": 2 * factors + per_row + (4 * rows if case["reduction"] == "none" else 0), "flops": 3 * product}
    n = rows * width
    gate = {"none": 0, "shared": width, "sequence": case["sequences"] * width, "token": n}[case["gate"]] * size
    vectors = (4 if case["bias"] else 2) * width * _SIZE[case["weight"]]
    stats = (16 if case["norm"] == "layer" else 8) * rows
    if kind == "gated":
        return {"bytes": 4 * size * n + gate + vectors + (stats if case.get("stats", True) else 0), "flops": 16 * n}
    read = (3 if case["bias"] else 2) * width * _SIZE[case["weight"]]   # the last bias has no part in it
    return {"bytes": 6 * size * n + 2 * gate + vectors + read + stats, "flops": 32 * n}
