"""Operators between a transformer's matrix products, layer norm, dropout
and the edges of the residual path that join them, and the loss at its end.

The reference has layer norm, root mean square norm, dropout and cross entropy
in ``namitorch/nn`` (the norms over the kernels of
``backends/cuda/normalization.py:56-157``); root mean square norms are here
within the gated edge alone.  This package has no autograd, so each operator
comes as a forward call that returns what its backward call reads, and a
backward call that returns gradients to hand to ``accumulate_grads`` or to the
layer below:

* ``layer_norm`` / ``layer_norm_forward`` / ``layer_norm_backward``;
* ``dropout`` / ``dropout_backward``;
* ``dropout_add_layer_norm`` / ``..._forward`` / ``..._backward``:
  ``total = dropout(input) + residual`` and the layer norm of it, the edge
  between two sublayers, in one pass over the data;
* ``norm_gate_add_norm`` / ``..._forward`` / ``..._backward``: ``total =
  residual_scale * residual + gate * N(input)`` and the norm of it, the edge
  after a block that is normalized on both sides;
* ``linear_cross_entropy`` / ``..._forward`` / ``..._backward``: softmax cross
  entropy of ``input @ weight.T``, whose logits are never in memory.

Tensors are float16, bfloat16 or float32 on a HIP device; weight and bias
(and their gradients) have the activations' dtype or float32.  Statistics and
sums are float32, values are rounded once (the loss's backward call rounds
the logits' gradient to the operands' dtype too).  A row that holds an
infinity or NaN gives NaN outputs (but the gated edge's ``total`` of a root
mean square norm over an infinity NaN there alone: the norm is zero beside it).

No mask is stored.  Whether element ``i`` of the flattened tensor is dropped
depends on ``(seed, offset, i)`` alone (Philox4x32-10, 16 bits per element),
so the backward call, or a second forward one, takes the same numbers and
finds the same mask.  Programs keep one ``seed`` per run and give every call
of the run an ``offset`` of its own.  ``p`` is used as the nearest multiple
of 2**-16, in the factor of the kept elements too.  A dropped element is
zero, whatever it held.

``out`` takes Tensors to write instead of new ones: one Tensor, or a tuple in
the order of the results (``None`` entries are allocated).  They overlap
neither inputs nor one another; ``dropout`` may write its own input.  Launches
go to the calling thread's current stream.  In a stream capture the forward
calls of the norms and edges run when ``out`` names every result and nothing
is dropped (a replay would repeat the mask); the others raise, those of the
loss among them (they take workspace), and so does a call that is given a
gradient whose accumulation or unscaling is still deferred.
"""

from __future__ import annotations

import math
from numbers import Integral, Real

from . import _native
from .array import DeviceArray
from .backends import _backends, ensure_same_device, get_backend
from .backends._graph_capture import reject_during_capture
from .dtype import bfloat16, float16, float32, int32, int64
from .runtime import current_stream
from .tensor import Tensor, device_views

_DTYPES = frozenset((float16, bfloat16, float32))
_MAX_SEED = 1 << 64
# Of float32, in which the kernels add it: past the most rstd would be zero, and
# below the least a constant row, which is its bias, would be NaN.
_LEAST_EPS, _MOST_EPS = 2.0 ** -149, (2.0 - 2.0 ** -23) * 2.0 ** 127


# ---- arguments ----------------------------------------------------------------------------------
def _current(value: Tensor) -> Tensor:
    """`value` with its deferred accumulation and transform written back.  In
    a capture that write would be recorded instead of run, while the marker
    that asks for it is gone: refused, as every in-place write there."""
    if value._pending is not None or value._incoming is not None:
        reject_during_capture("In-place Tensor updates")
        value._materialize()
    return value


def _activation(value, name: str, like: Tensor | None = None, what: str = "Layer norm and dropout") -> int:
    """Address of an activation (or gradient) Tensor, of `like`'s shape, dtype and device."""
    if not isinstance(value, Tensor):
        raise TypeError(f"{name} must be a NamiTorch Tensor, got {type(value).__name__}.")
    if like is None:
        if value._device not in _backends or value._ptr is None:
            backend = get_backend(value)     # which also puts a device under the capture checks
            if value._ptr is None:
                backend._unsupported(what)
        if value._dtype not in _DTYPES:
            raise TypeError(f"{name} must be float16, bfloat16 or float32, got {value._dtype.name}.")
    else:
        if value._shape != like._shape:
            raise ValueError(f"{name} has shape {value._shape}; expected {like._shape}.")
        if value._dtype is not like._dtype:
            raise TypeError(f"{name} has dtype {value._dtype.name}; expected {like._dtype.name}.")
        if value._device is not like._device:
            ensure_same_device(like, value)
    return _current(value)._ptr


def _affine(value, name: str, shape: tuple, like: Tensor) -> int | None:
    """Address of weight or bias, or None when absent."""
    if value is None:
        return None
    if not isinstance(value, Tensor):
        raise TypeError(f"{name} must be a NamiTorch Tensor, got {type(value).__name__}.")
    if value._shape != shape:
        raise ValueError(f"{name} has shape {value._shape}; expected {shape}.")
    if value._dtype is not like._dtype and value._dtype is not float32:
        raise TypeError(f"{name} must be {like._dtype.name} or float32, got {value._dtype.name}.")
    if value._device is not like._device:
        ensure_same_device(like, value)
    return _current(value)._ptr


def _affine_pair(weight, bias, shape: tuple, like: Tensor) -> tuple:
    """(weight address, bias address, their dtype code)."""
    scale, shift = _affine(weight, "weight", shape, like), _affine(bias, "bias", shape, like)
    if weight is not None and bias is not None and weight._dtype is not bias._dtype:
        raise TypeError(f"weight and bias must have one dtype, got {weight._dtype.name} and {bias._dtype.name}.")
    present = weight if weight is not None else bias
    return scale, shift, (like if present is None else present)._dtype._code


def _statistic(value, name: str, shape: tuple, like: Tensor) -> int:
    if not isinstance(value, Tensor):
        raise TypeError(f"{name} must be a NamiTorch Tensor, got {type(value).__name__}.")
    if value._shape != shape:
        raise ValueError(f"{name} has shape {value._shape}; expected {shape}.")
    if value._dtype is not float32:
        raise TypeError(f"{name} must be float32, got {value._dtype.name}.")
    if value._device is not like._device:
        ensure_same_device(like, value)
    return _current(value)._ptr


def _normalized(value: Tensor, normalized_shape) -> tuple:
    """(leading shape, normalized shape, rows, width)."""
    shape = normalized_shape
    if type(shape) is not tuple:
        shape = (int(shape),) if isinstance(shape, Integral) else tuple(shape)
    lead = len(value._shape) - len(shape)
    if not shape or lead < 0 or value._shape[lead:] != shape:
        raise ValueError(f"normalized_shape {shape} must be the trailing dimensions of {value._shape}.")
    return _split(value, lead)


def _split(value: Tensor, lead: int) -> tuple:
    shape = value._shape[lead:]
    width = math.prod(shape)
    if width == 0:
        raise ValueError(f"Layer norm needs at least one element per row, got normalized shape {shape}.")
    return value._shape[:lead], shape, math.prod(value._shape[:lead]), width


def _epsilon(eps) -> float:
    if type(eps) is not float:
        if isinstance(eps, bool) or not isinstance(eps, Real):
            raise TypeError("eps must be a real number.")
        eps = float(eps)
    if eps != 0.0 and not _LEAST_EPS <= eps <= _MOST_EPS:
        raise ValueError(f"eps must be finite and nonnegative as a float32, got {eps}.")
    return eps


def _threshold(p) -> int:
    """Drop threshold of the 16-bit numbers: p rounded to a multiple of 2**-16."""
    if type(p) is not float:
        if isinstance(p, bool) or not isinstance(p, Real):
            raise TypeError("p must be a real number.")
        p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be between 0 and 1, got {p}.")
    return round(p * 65536)


def _counter(value, name: str) -> int:
    if type(value) is not int:
        if isinstance(value, bool) or not isinstance(value, Integral):
            raise TypeError(f"{name} must be an integer.")
        value = int(value)
    if not 0 <= value < _MAX_SEED:
        raise ValueError(f"{name} must be in [0, 2**64), got {value}.")
    return value


def _training_threshold(p, training) -> int:
    threshold = _threshold(p)
    if training is True:
        return threshold
    if training is not False:
        raise TypeError("training must be a Python bool.")
    return 0


def _edge_mask(x: Tensor, p, training, seed, offset) -> tuple:
    """(threshold, seed, offset) of an edge's dropout.  A call that draws
    numbers names its seed: with a common default every edge of every step
    would drop the same elements."""
    threshold = _training_threshold(p, training)
    if seed is None:
        if threshold and x._numel:
            reject_during_capture("Dropout")
            raise TypeError("seed is needed where elements are dropped (p > 0 in training).")
        seed = 0
    return threshold, _counter(seed, "seed"), _counter(offset, "offset")


# ---- results ------------------------------------------------------------------------------------
def _given(out, count: int) -> tuple:
    """The `out` argument as `count` entries."""
    if out is None:
        return (None,) * count
    if count == 1 and isinstance(out, Tensor):
        return (out,)
    if not isinstance(out, (tuple, list)) or len(out) != count:
        raise TypeError(f"out must be {'a Tensor' if count == 1 else f'a tuple of {count} Tensors'}.")
    return tuple(out)


def _result(given, name: str, shape: tuple, dtype, like: Tensor) -> Tensor:
    """The Tensor a call writes: `given`, checked, or a new one."""
    if given is None:
        return device_views(DeviceArray.empty(shape, dtype, like._device), (0,), (shape,))[0]
    if not isinstance(given, Tensor):
        raise TypeError(f"out: {name} must be a NamiTorch Tensor, got {type(given).__name__}.")
    if given._shape != shape:
        raise ValueError(f"out: {name} has shape {given._shape}; expected {shape}.")
    if given._dtype is not dtype:
        raise TypeError(f"out: {name} has dtype {given._dtype.name}; expected {dtype.name}.")
    if given._device is not like._device:
        ensure_same_device(like, given)
    given._check_inplace()
    if given._pending is not None or given._incoming is not None:
        # The launch replaces what is deferred; one that is only recorded does not yet.
        reject_during_capture("In-place Tensor updates")
    return given


def _launch(status: int, given: tuple) -> None:
    """Raise what the library refused; otherwise the in-place bookkeeping of
    the given Tensors that the launch overwrites."""
    if status:
        _native.check(status)
    for tensor in given:
        if tensor is not None:
            tensor._pending = tensor._incoming = tensor._known_item = None
            tensor._version_counter.increment()


# ---- layer norm -----------------------------------------------------------------------------------
def layer_norm(input, normalized_shape, weight=None, bias=None, eps=1e-5, *, out=None) -> Tensor:
    """Layer norm over the trailing dimensions ``normalized_shape``:
    ``(x - mean) / sqrt(var + eps) * weight + bias`` per row, with the biased
    variance.  The form for inference: no statistics are kept."""
    return _layer_norm(input, normalized_shape, weight, bias, eps, _given(out, 1), False)[0]


def layer_norm_forward(input, normalized_shape, weight=None, bias=None, eps=1e-5, *, out=None) -> tuple:
    """``(output, mean, rstd)``: :func:`layer_norm` and the float32 statistics
    of each row (of the leading shape) that :func:`layer_norm_backward` reads."""
    return _layer_norm(input, normalized_shape, weight, bias, eps, _given(out, 3), True)


def _layer_norm(x, normalized_shape, weight, bias, eps, given, stats: bool) -> tuple:
    source = _activation(x, "input")
    lead, shape, rows, width = _normalized(x, normalized_shape)
    scale, shift, code = _affine_pair(weight, bias, shape, x)
    eps = _epsilon(eps)
    if None in given:
        reject_during_capture("Layer norm without out")
    y = _result(given[0], "output", x._shape, x._dtype, x)
    mean = rstd = None
    if stats:
        mean = _result(given[1], "mean", lead, float32, x)
        rstd = _result(given[2], "rstd", lead, float32, x)
    device = x._device.index
    _launch(_native.load().nt_layer_norm(
        device, source, x._dtype._code, scale, shift, code, eps, y._ptr, mean._ptr if stats else None,
        rstd._ptr if stats else None, rows, width, current_stream(device)), given)
    return (y, mean, rstd)


def layer_norm_backward(grad_output, input, mean, rstd, weight=None, bias=None, *, out=None) -> tuple:
    """``(grad_input, grad_weight, grad_bias)`` of :func:`layer_norm_forward`
    at ``input`` with its ``mean`` and ``rstd``.  ``grad_weight`` and
    ``grad_bias`` have their parameter's shape and dtype, and are None where
    the parameter is None."""
    given = _given(out, 3)
    x = _activation(input, "input")
    dy = _activation(grad_output, "grad_output", input)
    _, shape, rows, width, mean_at, rstd_at = _kept(input, mean, rstd)
    scale, _, code = _affine_pair(weight, bias, shape, input)
    if None in given:
        reject_during_capture("Layer norm backward")
    dx = _result(given[0], "grad_input", input._shape, input._dtype, input)
    dw, db = _affine_results(given[1:], weight, bias, input)
    device = input._device.index
    _launch(_native.load().nt_layer_norm_backward(
        device, dy, x, input._dtype._code, mean_at, rstd_at, scale, code, dx._ptr, None if dw is None else dw._ptr,
        None if db is None else db._ptr, rows, width, current_stream(device)), given)
    return dx, dw, db


def _kept(x: Tensor, mean, rstd) -> tuple:
    """(leading shape, normalized shape, rows, width, mean address, rstd
    address): the statistics' shape says which dimensions were normalized."""
    if not isinstance(mean, Tensor):
        raise TypeError(f"mean must be a NamiTorch Tensor, got {type(mean).__name__}.")
    lead = len(mean._shape)
    if lead >= len(x._shape) or mean._shape != x._shape[:lead]:
        raise ValueError(f"mean has shape {mean._shape}, which is not the leading shape of {x._shape}.")
    return (*_split(x, lead), _statistic(mean, "mean", mean._shape, x), _statistic(rstd, "rstd", mean._shape, x))


def _affine_results(given, weight, bias, like: Tensor) -> tuple:
    made = []
    for parameter, name, out in ((weight, "grad_weight", given[0]), (bias, "grad_bias", given[1])):
        if parameter is None:
            if out is not None:
                raise ValueError(f"out: {name} was given, but the layer norm has no such parameter.")
            made.append(None)
        else:
            made.append(_result(out, name, parameter._shape, parameter._dtype, like))
    return tuple(made)


# ---- dropout --------------------------------------------------------------------------------------
def dropout(input, p=0.5, training=True, *, seed, offset=0, out=None) -> Tensor:
    """Each element zero with probability ``p``, otherwise divided by
    ``1 - p``.  With ``training=False`` or ``p`` rounding to zero the result
    is the input itself (or a copy of it in ``out``)."""
    return _dropout(input, p, training, seed, offset, out, "input")


def dropout_backward(grad_output, p=0.5, training=True, *, seed, offset=0, out=None) -> Tensor:
    """Gradient of :func:`dropout` with the same ``p``, ``seed`` and
    ``offset``: the same mask and factor applied to ``grad_output``."""
    return _dropout(grad_output, p, training, seed, offset, out, "grad_output")


def _dropout(x, p, training, seed, offset, out, name: str) -> Tensor:
    given, = outs = _given(out, 1)
    source = _activation(x, name)
    threshold = _training_threshold(p, training)
    seed, offset = _counter(seed, "seed"), _counter(offset, "offset")
    if given is None:
        if threshold == 0:
            return x
        reject_during_capture("Dropout")
    y = _result(given, "output", x._shape, x._dtype, x)
    device = x._device.index
    _launch(_native.load().nt_dropout(
        device, source, x._dtype._code, y._ptr, x._numel, threshold, seed, offset, current_stream(device)), outs)
    return y


# ---- the residual edge ------------------------------------------------------------------------------
def dropout_add_layer_norm(input, residual, normalized_shape, weight=None, bias=None, p=0.0, eps=1e-5,
                           training=True, *, seed=None, offset=0, out=None) -> tuple:
    """``(output, total)`` with ``total = dropout(input) + residual`` and
    ``output`` the layer norm of it.  The norm is taken before ``total`` is
    rounded to its dtype.  ``seed`` is needed where elements are dropped."""
    return _edge(input, residual, normalized_shape, weight, bias, p, eps, training, seed, offset, _given(out, 2),
                 False)[:2]


def dropout_add_layer_norm_forward(input, residual, normalized_shape, weight=None, bias=None, p=0.0, eps=1e-5,
                                   training=True, *, seed=None, offset=0, out=None) -> tuple:
    """``(output, total, mean, rstd)``: :func:`dropout_add_layer_norm` with
    the statistics that its backward call reads."""
    return _edge(input, residual, normalized_shape, weight, bias, p, eps, training, seed, offset, _given(out, 4), True)


def _edge(x, residual, normalized_shape, weight, bias, p, eps, training, seed, offset, given, stats: bool) -> tuple:
    source = _activation(x, "input")
    stream_in = _activation(residual, "residual", x)
    lead, shape, rows, width = _normalized(x, normalized_shape)
    scale, shift, code = _affine_pair(weight, bias, shape, x)
    eps = _epsilon(eps)
    threshold, seed, offset = _edge_mask(x, p, training, seed, offset)
    if None in given:
        reject_during_capture("Dropout" if threshold else "Layer norm without out")
    y = _result(given[0], "output", x._shape, x._dtype, x)
    total = _result(given[1], "total", x._shape, x._dtype, x)
    mean = rstd = None
    if stats:
        mean = _result(given[2], "mean", lead, float32, x)
        rstd = _result(given[3], "rstd", lead, float32, x)
    device = x._device.index
    _launch(_native.load().nt_dropout_add_layer_norm(
        device, source, stream_in, x._dtype._code, scale, shift, code, eps, threshold, seed, offset, total._ptr, y._ptr,
        mean._ptr if stats else None, rstd._ptr if stats else None, rows, width, current_stream(device)), given)
    return (y, total, mean, rstd)


def dropout_add_layer_norm_backward(grad_output, grad_total, total, mean, rstd, weight=None, bias=None, p=0.0,
                                    training=True, *, seed=None, offset=0, out=None) -> tuple:
    """``(grad_input, grad_residual, grad_weight, grad_bias)`` of
    :func:`dropout_add_layer_norm_forward`, from the gradients of its two
    results (``grad_total`` None: nothing else reads ``total``)."""
    given = _given(out, 4)
    t = _activation(total, "total")
    dy = _activation(grad_output, "grad_output", total)
    dt = None if grad_total is None else _activation(grad_total, "grad_total", total)
    _, shape, rows, width, mean_at, rstd_at = _kept(total, mean, rstd)
    scale, _, code = _affine_pair(weight, bias, shape, total)
    threshold, seed, offset = _edge_mask(total, p, training, seed, offset)
    if None in given:
        reject_during_capture("Layer norm backward")
    dx = _result(given[0], "grad_input", total._shape, total._dtype, total)
    dr = _result(given[1], "grad_residual", total._shape, total._dtype, total)
    dw, db = _affine_results(given[2:], weight, bias, total)
    device = total._device.index
    _launch(_native.load().nt_dropout_add_layer_norm_backward(
        device, dy, dt, t, total._dtype._code, mean_at, rstd_at, scale, code, threshold, seed, offset, dx._ptr, dr._ptr,
        None if dw is None else dw._ptr, None if db is None else db._ptr, rows, width, current_stream(device)), given)
    return dx, dr, dw, db


# ---- the edge after a block that is normalized on both sides --------------------------------------------
_NORMS = {"layer": 0, "rms": 1}


def norm_gate_add_norm(input, residual, normalized_shape, inner_weight=None, inner_bias=None, gate=None, weight=None,
                       bias=None, residual_scale=1.0, eps=1e-5, *, norm="layer", out=None) -> tuple:
    """``(output, total)`` with ``total = residual_scale * residual + gate *
    N(input)`` and ``output = N(total)``: the norm after a block, its gate, the
    residual stream and the norm before the next block, in one pass.

    ``N`` is layer norm over the trailing dimensions ``normalized_shape`` or,
    with ``norm="rms"``, the root mean square norm ``x / sqrt(mean(x**2) + eps)
    * weight + bias``; the first has ``inner_weight`` and ``inner_bias``, the
    second ``weight`` and ``bias`` (one dtype for all).  ``gate``, of the input's
    dtype or float32, has the normalized shape (one gate for all rows), or
    leading dimensions of the input before it, of which the last ones may be 1
    (one for each sequence of a batch, or for each row).  The second norm is
    taken before ``total`` is rounded to its dtype."""
    return _gated(input, residual, normalized_shape, inner_weight, inner_bias, gate, weight, bias, residual_scale, eps,
                  norm, _given(out, 2), False)[:2]


def norm_gate_add_norm_forward(input, residual, normalized_shape, inner_weight=None, inner_bias=None, gate=None,
                               weight=None, bias=None, residual_scale=1.0, eps=1e-5, *, norm="layer",
                               out=None) -> tuple:
    """``(output, total, inner_mean, inner_rstd, mean, rstd)``:
    :func:`norm_gate_add_norm` with the float32 statistics that its backward
    call reads.  With ``norm="rms"`` the means are None."""
    return _gated(input, residual, normalized_shape, inner_weight, inner_bias, gate, weight, bias, residual_scale, eps,
                  norm, _given(out, 6), True)


def _gated(x, residual, normalized_shape, inner_weight, inner_bias, gate, weight, bias, residual_scale, eps, norm, given,
           stats: bool) -> tuple:
    source = _activation(x, "input", None, "The gated edge")
    stream_in = _activation(residual, "residual", x)
    lead, shape, rows, width = _normalized(x, normalized_shape)
    vectors, code = _vectors((inner_weight, inner_bias, weight, bias), shape, x)
    gate_at, gate_code, gate_rows = _gate(gate, lead, shape, x)
    scale, eps, rms = _scale(residual_scale), _epsilon(eps), _norm_kind(norm)
    if stats and rms and (given[2] is not None or given[4] is not None):
        raise ValueError("out: a mean was given, but root mean square norms have none.")
    needed = given if not (stats and rms) else (given[0], given[1], given[3], given[5])
    if None in needed:
        reject_during_capture("The gated edge without out")
    y = _result(given[0], "output", x._shape, x._dtype, x)
    total = _result(given[1], "total", x._shape, x._dtype, x)
    kept, at = (None,) * 4, (None,) * 4
    if stats:
        kept = tuple(None if rms and place % 2 == 0 else _result(given[2 + place], name, lead, float32, x)
                     for place, name in enumerate(("inner_mean", "inner_rstd", "mean", "rstd")))
        at = tuple(None if k is None else k._ptr for k in kept)
    device = x._device.index
    _launch(_native.load().nt_norm_gate_add_norm(
        device, source, stream_in, x._dtype._code, vectors[0], vectors[1], gate_at, gate_code, gate_rows, vectors[2],
        vectors[3], code, scale, eps, rms, total._ptr, y._ptr, *at, rows, width, current_stream(device)), given)
    return (y, total, *kept)


def norm_gate_add_norm_backward(grad_output, grad_total, input, total, inner_mean, inner_rstd, mean, rstd,
                                inner_weight=None, inner_bias=None, gate=None, weight=None, bias=None,
                                residual_scale=1.0, *, out=None) -> tuple:
    """``(grad_input, grad_residual, grad_inner_weight, grad_inner_bias,
    grad_gate, grad_weight, grad_bias)`` of :func:`norm_gate_add_norm_forward`
    at ``input`` with its ``total`` and statistics (means None: root mean
    square norms), from the gradients of its two results (``grad_total`` None:
    nothing else reads ``total``).  A parameter's gradient has its shape and
    dtype, and is None where the parameter is None."""
    given = _given(out, 7)
    t = _activation(total, "total", None, "The gated edge")
    source = _activation(input, "input", total)
    dy = _activation(grad_output, "grad_output", total)
    dt = None if grad_total is None else _activation(grad_total, "grad_total", total)
    if (mean is None) != (inner_mean is None):
        raise ValueError("inner_mean and mean are given together, or both are None (root mean square norms).")
    if not isinstance(rstd, Tensor):
        raise TypeError(f"rstd must be a NamiTorch Tensor, got {type(rstd).__name__}.")
    lead = len(rstd._shape)
    if lead >= len(total._shape) or rstd._shape != total._shape[:lead]:
        raise ValueError(f"rstd has shape {rstd._shape}, which is not the leading shape of {total._shape}.")
    lead, shape, rows, width = _split(total, lead)
    stats = [None if value is None else _statistic(value, name, lead, total) for value, name in (
        (inner_mean, "inner_mean"), (inner_rstd, "inner_rstd"), (mean, "mean"), (rstd, "rstd"))]
    if stats[1] is None and inner_rstd is None:
        raise TypeError("inner_rstd must be a NamiTorch Tensor, got NoneType.")
    vectors, code = _vectors((inner_weight, inner_bias, weight, bias), shape, total)
    gate_at, gate_code, gate_rows = _gate(gate, lead, shape, total)
    scale = _scale(residual_scale)
    if None in given:
        reject_during_capture("The gated edge's backward call")
    dx = _result(given[0], "grad_input", total._shape, total._dtype, total)
    dr = _result(given[1], "grad_residual", total._shape, total._dtype, total)
    made = []
    for parameter, name, result in zip((inner_weight, inner_bias, gate, weight, bias),
                                       ("grad_inner_weight", "grad_inner_bias", "grad_gate", "grad_weight", "grad_bias"),
                                       given[2:]):
        if parameter is not None:
            made.append(_result(result, name, parameter._shape, parameter._dtype, total))
        elif result is None:
            made.append(None)
        else:
            raise ValueError(f"out: {name} was given, but the edge has no such parameter.")
    device = total._device.index
    _launch(_native.load().nt_norm_gate_add_norm_backward(
        device, dy, dt, source, t, total._dtype._code, *stats, vectors[0], vectors[1], gate_at, gate_code, gate_rows,
        vectors[2], code, scale, dx._ptr, dr._ptr, *(None if v is None else v._ptr for v in made), rows, width,
        current_stream(device)), given)
    return (dx, dr, *made)


def _vectors(values, shape: tuple, like: Tensor) -> tuple:
    """(addresses of the weights and biases, their dtype code)."""
    at, kind = [], None
    for value, name in zip(values, ("inner_weight", "inner_bias", "weight", "bias")):
        if value is None:
            at.append(None)
            continue
        at.append(_affine(value, name, shape, like))
        if kind is None:
            kind = value._dtype
        elif kind is not value._dtype:
            raise TypeError(f"weights and biases must have one dtype, got {kind.name} and {value._dtype.name}.")
    return at, (like._dtype if kind is None else kind)._code


def _gate(value, lead: tuple, shape: tuple, like: Tensor) -> tuple:
    """(address, dtype code, rows) of a gate; 0 rows where there is none."""
    if value is None:
        return None, like._dtype._code, 0
    if not isinstance(value, Tensor):
        raise TypeError(f"gate must be a NamiTorch Tensor, got {type(value).__name__}.")
    own = len(value._shape) - len(shape)
    before = value._shape[:own] if own >= 0 else None
    same = 0
    if before:
        while same < own and same < len(lead) and before[same] == lead[same]:
            same += 1
    if before is None or value._shape[own:] != shape or own not in (0, len(lead)) or any(n != 1 for n in before[same:]):
        raise ValueError(f"gate has shape {value._shape}; expected {shape}, or leading dimensions of {lead} before it, "
                         "the last of which may be 1.")
    if value._dtype is not like._dtype and value._dtype is not float32:
        raise TypeError(f"gate must be {like._dtype.name} or float32, got {value._dtype.name}.")
    if value._device is not like._device:
        ensure_same_device(like, value)
    return _current(value)._ptr, value._dtype._code, math.prod(before)


def _scale(value) -> float:
    if type(value) is not float:
        if isinstance(value, bool) or not isinstance(value, Real):
            raise TypeError("residual_scale must be a real number.")
        value = float(value)
    if not abs(value) <= _MOST_EPS:
        raise ValueError(f"residual_scale must be finite as a float32, got {value}.")
    return value


def _norm_kind(value) -> int:
    code = _NORMS.get(value) if isinstance(value, str) else None
    if code is None:
        raise ValueError(f"norm must be 'layer' or 'rms', got {value!r}.")
    return code


# ---- the loss -----------------------------------------------------------------------------------------
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(input, weight, target, *, ignore_index=-100, reduction="mean", out=None) -> Tensor:
    """Softmax cross entropy of the logits ``input @ weight.T`` against the
    class indices ``target``, without the logits ever being in memory.

    ``input``: ``(..., width)``; ``weight``: ``(classes, width)`` of the same
    dtype; ``target``: int64 or int32 of the leading shape.  Rows whose target
    is ``ignore_index`` are not counted: whatever their input holds, their
    loss is zero and they give no gradient.  ``reduction``: the ``"mean"`` over
    the counted rows (zero where there are none), their ``"sum"``, or
    ``"none"``, a loss for each row; float32 in every case.  A target that is
    no class makes its row's loss NaN, and the gradients."""
    return _linear_cross_entropy(input, weight, target, ignore_index, reduction, _given(out, 1), False)[0]


def linear_cross_entropy_forward(input, weight, target, *, ignore_index=-100, reduction="mean", out=None) -> tuple:
    """``(loss, lse)``: :func:`linear_cross_entropy` and the float32
    ``log(sum(exp(logits)))`` of each row (zero where it is not counted) that
    :func:`linear_cross_entropy_backward` reads."""
    return _linear_cross_entropy(input, weight, target, ignore_index, reduction, _given(out, 2), True)


def _linear_cross_entropy(x, weight, target, ignore_index, reduction, given, keep: bool) -> tuple:
    source = _activation(x, "input", None, "Linear cross entropy")
    head, classes, width = _head(weight, x)
    lead, at = x._shape[:-1], _targets(target, x)
    code, ignored = _reduction(reduction), _ignored(ignore_index)
    reject_during_capture("Linear cross entropy")
    loss = _result(given[0], "loss", lead if code == 0 else (), float32, x)
    lse = _result(given[1], "lse", lead, float32, x) if keep else None
    device = x._device.index
    _launch(_native.load().nt_linear_cross_entropy(
        device, source, head, x._dtype._code, at, target._dtype.itemsize, ignored, code, loss._ptr,
        lse._ptr if keep else None, math.prod(lead), classes, width, current_stream(device)), given)
    return loss, lse


def linear_cross_entropy_backward(grad_loss, input, weight, target, lse, *, ignore_index=-100, reduction="mean",
                                  out=None) -> tuple:
    """``(grad_input, grad_weight)`` of :func:`linear_cross_entropy_forward`
    with its ``lse`` and the same ``ignore_index`` and ``reduction``.  The
    logits' gradient is rounded to the operands' dtype on the way; float16's is
    scaled by one power of two for all rows, so that a row whose own gradient is
    2**-20 of the largest or less keeps few digits of its probabilities.
    ``grad_loss``, the gradient of the loss: a float32 Tensor of the loss's
    shape or, for a mean or sum, a number within float32's range (a loss scale;
    1 without one)."""
    given = _given(out, 2)
    x = _activation(input, "input", None, "Linear cross entropy")
    head, classes, width = _head(weight, input)
    lead, at = input._shape[:-1], _targets(target, input)
    code, ignored = _reduction(reduction), _ignored(ignore_index)
    kept = _statistic(lse, "lse", lead, input)
    value, grad = 0.0, None
    if isinstance(grad_loss, Tensor):
        grad = _statistic(grad_loss, "grad_loss", lead if code == 0 else (), input)
    elif isinstance(grad_loss, bool) or not isinstance(grad_loss, Real) or code == 0:
        raise TypeError("grad_loss must be a float32 Tensor of the loss's shape" +
                        (", as each row has a loss." if code == 0 else " or a real number."))
    else:
        value = float(grad_loss)
        if _MOST_EPS < abs(value) < math.inf:
            raise ValueError(f"grad_loss must be within float32's range, got {value}.")
    reject_during_capture("Linear cross entropy backward")
    dx = _result(given[0], "grad_input", input._shape, input._dtype, input)
    dw = _result(given[1], "grad_weight", weight._shape, weight._dtype, input)
    device = input._device.index
    _launch(_native.load().nt_linear_cross_entropy_backward(
        device, grad, value, x, head, input._dtype._code, at, target._dtype.itemsize, ignored, code, kept, dx._ptr,
        dw._ptr, math.prod(lead), classes, width, current_stream(device)), given)
    return dx, dw


def _head(weight, x: Tensor) -> tuple:
    """(address of the weight, classes, width)."""
    if not x._shape:
        raise ValueError("input must have at least one dimension.")
    if not isinstance(weight, Tensor):
        raise TypeError(f"weight must be a NamiTorch Tensor, got {type(weight).__name__}.")
    if len(weight._shape) != 2 or weight._shape[1] != x._shape[-1] or 0 in weight._shape:
        raise ValueError(f"weight has shape {weight._shape}; expected (classes, {x._shape[-1]}), neither of them zero.")
    if weight._dtype is not x._dtype:
        raise TypeError(f"weight has dtype {weight._dtype.name}; expected {x._dtype.name}.")
    if weight._device is not x._device:
        ensure_same_device(x, weight)
    return _current(weight)._ptr, *weight._shape


def _targets(target, x: Tensor) -> int:
    if not isinstance(target, Tensor):
        raise TypeError(f"target must be a NamiTorch Tensor, got {type(target).__name__}.")
    if target._dtype not in (int32, int64):
        raise TypeError(f"target must be int64 or int32, got {target._dtype.name}.")
    if target._shape != x._shape[:-1]:
        raise ValueError(f"target has shape {target._shape}; expected {x._shape[:-1]}.")
    if target._device is not x._device:
        ensure_same_device(x, target)
    return target._ptr


def _reduction(value) -> int:
    code = _REDUCTIONS.get(value) if isinstance(value, str) else None
    if code is None:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {value!r}.")
    return code


def _ignored(value) -> int:
    if isinstance(value, bool) or not isinstance(value, Integral):
        raise TypeError("ignore_index must be an integer.")
    if not -(1 << 63) <= value < 1 << 63:
        raise ValueError(f"ignore_index must be in [-2**63, 2**63), got {value}.")
    return int(value)


__all__ = ["layer_norm", "layer_norm_forward", "layer_norm_backward", "dropout", "dropout_backward",
           "dropout_add_layer_norm", "dropout_add_layer_norm_forward", "dropout_add_layer_norm_backward",
           "norm_gate_add_norm", "norm_gate_add_norm_forward", "norm_gate_add_norm_backward",
           "linear_cross_entropy", "linear_cross_entropy_forward", "linear_cross_entropy_backward"]
