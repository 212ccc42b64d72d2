"""Routing and low-rank adapters on tensors in HBM: what a model whose rows go to
clusters needs next to the clustering itself.

A router scores every row against the experts (for experts placed at the centres of a
``KMeans`` fit, a product with the centres) and ``route`` takes the best ones, with their
weights, counts and the balance loss that keeps all experts in use; ``adapt`` puts each
row through its expert, a low-rank adapter beside a projection that all rows share.  The
adapter of a row may as well be its request's, or its cluster's: ``HipKMeans.predict``
labels are valid ``ids``.

The tensors are PyTorch's (a ROCm build), on the device that the library was set up on.
The kernels run on the current stream like any torch operator: asynchronous, ordered
with the other work of that stream; a tensor made on another stream is the caller's to
wait for.  Rows may lie apart (``stride(0)``), their elements lie side by side.

``route`` and ``adapt`` record no autograd graph: their gradients are ``route_backward``
and ``adapt_backward``.  ``routed`` and ``adapted`` are the same operators inside
autograd.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _bridge

MAX_EXPERTS = 2048
MAX_TOP_K = 16
MAX_RANK = 128

_ADAPT, _ADAPT_BACKWARD, _ADAPT_IN_X = 0, 1, 2
_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class Routing(NamedTuple):
    """``route``'s results."""

    weights: torch.Tensor    # [n, k] float32
    experts: torch.Tensor    # [n, k] int32, -1: none
    counts: torch.Tensor     # [e] int32: rows that take each expert
    prob_sums: torch.Tensor  # [e] float32: its probabilities' sum over the rows
    rows: torch.Tensor       # [1] int32: rows that count
    loss: torch.Tensor       # [] float32


class AdaptGrads(NamedTuple):
    """``adapt_backward``'s results."""

    x: torch.Tensor
    down: torch.Tensor
    up: torch.Tensor
    gates: torch.Tensor | None


@functools.lru_cache(maxsize=1)
def _lib():
    """The bound library, checked once: set up, and on the HIP runtime that torch uses
    (a second one in the process would not know torch's memory and streams)."""
    _bridge._require()
    _bridge.require_torch_runtime()
    return _bridge._lib


@functools.lru_cache(maxsize=1)
def _device_index():
    return _lib().skmetal_hip_device()


def _fail(name):
    raise RuntimeError(f"{name} failed: {_bridge.last_error()}")


def _refuse(t, name, dtype, shape, device):
    """Says what is wrong with a tensor of another type, device or shape."""
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _rows(t, name, dtype, shape, device):
    """The row stride of the matrix `t`, whose rows' elements lie side by side."""
    if t.dtype != dtype or t.shape != shape or t.device != device:
        _refuse(t, name, dtype, shape, device)
    ld, one = t.stride()
    if one != 1 and shape[1] > 1:
        raise ValueError(f"{name}'s rows must have their elements side by side (stride(1) is {one})")
    return ld


def _vector(t, name, dtype, n, device):
    if t.dtype != dtype or t.shape != (n,) or t.device != device:
        _refuse(t, name, dtype, (n,), device)
    return t.stride(0)


def _dense(t, name, dtype, shape, device):
    if t.dtype != dtype or t.shape != shape or t.device != device:
        _refuse(t, name, dtype, shape, device)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _first(t, name):
    """The type code and device of the operator's first tensor."""
    code = _CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} is {t.dtype}, expected float32, bfloat16 or float16")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}, expected the GPU")
    if t.dim() != 2:
        raise ValueError(f"{name} has {t.dim()} dimensions, expected 2")
    device = t.device
    if device.index != _device_index():
        raise ValueError(f"{name} is on {device}, the library was set up on device {_device_index()}")
    return code, device


def _mask(mask, n, device):
    if mask is None:
        return None, 0
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"mask is {mask.dtype}, expected bool or uint8")
    return mask.data_ptr(), _vector(mask, "mask", mask.dtype, n, device)


def _workspace(size, device):
    if size == 0:
        return None, None
    w = torch.empty(size, dtype=torch.uint8, device=device)
    return w, w.data_ptr()


@functools.lru_cache(maxsize=4096)
def _route_workspace(n, e):
    return _lib().skmetal_hip_route_workspace(n, e)


@functools.lru_cache(maxsize=4096)
def _adapt_workspace(code, n, d, o, r, a, call):
    return _lib().skmetal_hip_adapt_workspace(code, n, d, o, r, a, call)


# the current stream's handle, without an object around it where torch offers that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device.index)


def _check_route(logits, top_k):
    code, device = _first(logits, "logits")
    n, e = logits.shape
    top_k = int(top_k)
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"logits has {e} experts, expected 1 to {MAX_EXPERTS}")
    if not 1 <= top_k <= min(e, MAX_TOP_K):
        raise ValueError(f"top_k={top_k} is not in [1, {min(e, MAX_TOP_K)}]")
    ld, one = logits.stride()
    if one != 1 and e > 1:
        raise ValueError(f"logits' rows must have their elements side by side (stride(1) is {one})")
    return code, device, n, e, top_k, ld


def _run_route(logits, top_k, mask, normalize, loss=None):
    """weights, experts and one tensor that holds counts, prob_sums, rows and, unless `loss` takes it, the loss."""
    code, device, n, e, k, ld = _check_route(logits, top_k)
    mask_ptr, mask_stride = _mask(mask, n, device)
    lib = _lib()
    weights = torch.empty((n, k), dtype=torch.float32, device=device)
    experts = torch.empty((n, k), dtype=torch.int32, device=device)
    whole = torch.empty(2 * e + 2, dtype=torch.int32, device=device)
    size = _route_workspace(n, e)
    ws, ws_ptr = _workspace(size, device)
    at = whole.data_ptr()
    if lib.skmetal_hip_route(code, logits.data_ptr(), ld, mask_ptr, mask_stride, n, e, k, 1 if normalize else 0, weights.data_ptr(), experts.data_ptr(),
                             at, at + 4 * e, at + 8 * e, at + 8 * e + 4 if loss is None else loss.data_ptr(), ws_ptr, size, _stream(device)):
        _fail("route")
    return weights, experts, whole


def _statistics(whole):
    """The parts of _run_route's last tensor."""
    e = whole.shape[0] // 2 - 1
    counts, sums, rows, loss = whole.split_with_sizes((e, e, 1, 1))
    return counts, sums.view(torch.float32), rows, loss


def route(logits, top_k, *, mask=None, normalize=False) -> Routing:
    """The `top_k` largest scores of every row of logits [n, e], equal ones by the lowest
    index, with their softmax probabilities as weights (over the row's e scores;
    `normalize` divides them by their sum over the chosen ones).  A score of -inf or NaN
    is excluded; a row that `mask` (bool [n]) leaves out, or whose scores are all
    excluded, takes no expert (-1, weight 0) and counts nowhere.  A score of +inf is the
    largest, and its row's weights are NaN like a softmax's, prob_sums and loss with them.

    ``loss`` = e / (top_k N^2) sum_j counts_j prob_sums_j over the N rows that count: 1
    where rows and probabilities are spread evenly, more where the same experts get
    both.  The same inputs give the same bits on every call."""
    weights, experts, whole = _run_route(logits, top_k, mask, normalize)
    e = logits.shape[1]
    counts, sums, rows, loss = whole.split_with_sizes((e, e, 1, 1))
    return Routing(weights, experts, counts, sums.view(torch.float32), rows, loss.view(torch.float32)[0])


def route_backward(logits, routing: Routing, *, grad_weights=None, grad_loss=None, mask=None, normalize=False):
    """The gradient of ``route``'s logits from those of its weights [n, top_k] and loss
    [] (float32 each; None: no gradient).  `routing`, `mask` and `normalize` are the
    forward call's; the counts have no gradient and are held constant.  For a loss over
    the rows of several processes, pass a routing whose counts and rows are their sums."""
    k = routing.experts.shape[1]
    code, device, n, e, k, ld = _check_route(logits, k)
    mask_ptr, mask_stride = _mask(mask, n, device)
    lib = _lib()
    w = _dense(routing.weights, "routing.weights", torch.float32, (n, k), device)
    x = _dense(routing.experts, "routing.experts", torch.int32, (n, k), device)
    c = _dense(routing.counts, "routing.counts", torch.int32, (e,), device)
    m = _dense(routing.rows, "routing.rows", torch.int32, (1,), device)
    dw = None if grad_weights is None else _dense(grad_weights, "grad_weights", torch.float32, (n, k), device)
    dl = None if grad_loss is None else _dense(grad_loss, "grad_loss", torch.float32, (), device)
    grad = torch.empty((n, e), dtype=logits.dtype, device=device)
    if lib.skmetal_hip_route_backward(code, logits.data_ptr(), ld, mask_ptr, mask_stride, n, e, k, 1 if normalize else 0, w, x, c, m, dw, dl,
                                      grad.data_ptr(), e, _stream(device)):
        _fail("route_backward")
    return grad


def _adapters(t, name, dtype, device):
    """The sizes and the adapter and rank strides of `t` [a, r, width]."""
    if t.dtype != dtype or t.device != device or t.dim() != 3:
        _refuse(t, name, dtype, ("adapters", "rank", "width"), device)
    sa, ld, one = t.stride()
    a, r, width = t.shape
    if one != 1 and width > 1:
        raise ValueError(f"{name}'s ranks must have their elements side by side (stride(2) is {one})")
    return a, r, width, sa, ld


def _check_adapt(x, first, down, up, ids, gates, scales):
    code, device = _first(x, first)
    n, width = x.shape
    ld, one = x.stride()
    if one != 1 and width > 1:
        raise ValueError(f"{first}'s rows must have their elements side by side (stride(1) is {one})")
    dtype = x.dtype
    a, r, d, down_sa, down_ld = _adapters(down, "down", dtype, device)
    a2, r2, o, up_sa, up_ld = _adapters(up, "up", dtype, device)
    if a2 != a or r2 != r:
        raise ValueError(f"down has shape {tuple(down.shape)} and up {tuple(up.shape)}: their adapters and ranks must agree")
    if not 1 <= r <= MAX_RANK:
        raise ValueError(f"a rank of {r} is not in [1, {MAX_RANK}]")
    ids_stride = _vector(ids, "ids", torch.int32, n, device)
    gate_ptr, gate_stride = (None, 0) if gates is None else (gates.data_ptr(), _vector(gates, "gates", torch.float32, n, device))
    scale_ptr = None if scales is None else _dense(scales, "scales", torch.float32, (a,), device)
    shared = (down.data_ptr(), down_sa, down_ld, up.data_ptr(), up_sa, up_ld, ids.data_ptr(), ids_stride, gate_ptr, gate_stride, scale_ptr)
    return code, device, n, d, o, r, a, width, ld, shared


def adapt(x, down, up, ids, *, base=None, gates=None, scales=None, out=None, return_low=False):
    """base + the low-rank adapter of every row of x [n, d]: with q = ids[i]

        out_i = base_i + gates_i scales_q up_q^T (down_q x_i)

    down [a, r, d] and up [a, r, o] (both by rank: up is the transpose of the usual
    up-projection), ids int32 [n] in any order, with any value outside [0, a) for a row
    without an adapter; base [n, o] is the shared projection's output (None: 0), gates
    [n] (a router's weights) and scales [a] are float32 (None: 1).  x, down, up, base
    and out have one type.  `out` may be base and may share memory with x (a residual
    stream in place: base=x, out=x); nothing else may share memory with it.  With `return_low` also returns down_q
    x_i, float32 [n, r], for ``adapt_backward``."""
    code, device, n, d, o, r, a, width, x_ld, shared = _check_adapt(x, "x", down, up, ids, gates, scales)
    if width != d:
        raise ValueError(f"x has {width} columns, down has {d}")
    dtype = x.dtype
    base_ptr, base_ld = (None, 0) if base is None else (base.data_ptr(), _rows(base, "base", dtype, (n, o), device))
    lib = _lib()
    x_ptr, call = x.data_ptr(), _ADAPT
    if out is None:
        out, out_ld = torch.empty((n, o), dtype=dtype, device=device), o
        out_ptr = out.data_ptr()
    else:
        out_ld = _rows(out, "out", dtype, (n, o), device)
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out requires a gradient, which this call does not record: use adapted, or torch.no_grad")
        torch.autograd.graph.increment_version(out)
        out_ptr, es = out.data_ptr(), dtype.itemsize
        if x_ptr < out_ptr + (n * out_ld + o) * es and out_ptr < x_ptr + (n * x_ld + d) * es:
            call = _ADAPT_IN_X  # or between x's rows, which the library finds out
    low = torch.empty((n, r), dtype=torch.float32, device=device) if return_low else None
    size = _adapt_workspace(code, n, d, o, r, a, call)
    ws, ws_ptr = _workspace(size, device)
    if lib.skmetal_hip_adapt(code, x_ptr, x_ld, *shared, base_ptr, base_ld, out_ptr, out_ld,
                             None if low is None else low.data_ptr(), n, d, o, r, a, ws_ptr, size, _stream(device)):
        _fail("adapt")
    return (out, low) if return_low else out


def adapt_backward(grad, x, down, up, ids, low, *, base=None, gates=None, scales=None) -> AdaptGrads:
    """The gradients of ``adapt`` from grad [n, o], that of its output; `low` is what the
    forward call returned.  The gradient of x is added to `base` [n, d] (the shared
    projection's part; None: 0); the gradient of the forward call's base is grad
    itself.  Those of down and up have their shapes and type, 0 for an adapter without
    rows; that of gates is None where there are none."""
    code, device, n, d, o, r, a, width, grad_ld, shared = _check_adapt(grad, "grad", down, up, ids, gates, scales)
    if width != o:
        raise ValueError(f"grad has {width} columns, up has {o}")
    dtype = grad.dtype
    x_ld = _rows(x, "x", dtype, (n, d), device)
    low_ptr = _dense(low, "low", torch.float32, (n, r), device)
    base_ptr, base_ld = (None, 0) if base is None else (base.data_ptr(), _rows(base, "base", dtype, (n, d), device))
    lib = _lib()
    grad_x = torch.empty((n, d), dtype=dtype, device=device)
    grad_down = torch.empty((a, r, d), dtype=dtype, device=device)
    grad_up = torch.empty((a, r, o), dtype=dtype, device=device)
    grad_gates = None if gates is None else torch.empty(n, dtype=torch.float32, device=device)
    size = _adapt_workspace(code, n, d, o, r, a, _ADAPT_BACKWARD)
    ws, ws_ptr = _workspace(size, device)
    if lib.skmetal_hip_adapt_backward(code, grad.data_ptr(), grad_ld, x.data_ptr(), x_ld, *shared, low_ptr, base_ptr, base_ld, grad_x.data_ptr(), d,
                                      grad_down.data_ptr(), grad_up.data_ptr(), None if grad_gates is None else grad_gates.data_ptr(), n, d, o, r, a,
                                      ws_ptr, size, _stream(device)):
        _fail("adapt_backward")
    return AdaptGrads(grad_x, grad_down, grad_up, grad_gates)


class _Routed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, mask, normalize):
        # the loss in memory of its own, the statistics whole and only cut apart outside: views that a
        # Function returns cannot be changed in place
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        weights, experts, whole = _run_route(logits, top_k, mask, normalize, loss)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(logits, mask, weights, experts, whole.clone())  # the caller may add up its own
        ctx.normalize = normalize
        ctx.mark_non_differentiable(experts, whole)
        ctx.set_materialize_grads(False)
        return weights, experts, whole, loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _experts, _whole, grad_loss):
        logits, mask, weights, experts, whole = ctx.saved_tensors
        counts, sums, rows, _ = _statistics(whole)
        grad = route_backward(logits, Routing(weights, experts, counts, sums, rows, None), grad_weights=None if grad_weights is None else grad_weights.contiguous(),
                              grad_loss=grad_loss, mask=mask, normalize=ctx.normalize)
        return grad, None, None, None


class _Adapted(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, down, up, ids, base, gates, scales):
        out, low = adapt(x, down, up, ids, base=base, gates=gates, scales=scales, return_low=True)
        ctx.save_for_backward(x, down, up, ids, low, gates, scales)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, down, up, ids, low, gates, scales = ctx.saved_tensors
        if grad.stride(1) != 1 and grad.shape[1] > 1:
            grad = grad.contiguous()
        g = adapt_backward(grad, x, down, up, ids, low, gates=gates, scales=scales)
        return g.x, g.down, g.up, None, grad if ctx.needs_input_grad[4] else None, g.gates, None


def routed(logits, top_k, *, mask=None, normalize=False) -> Routing:
    """``route`` inside autograd: weights and loss pass their gradients to logits.  loss,
    counts, prob_sums and rows may be changed in place (weighted, summed over processes);
    the gradient stays that of this call's own."""
    weights, experts, whole, loss = _Routed.apply(logits, top_k, mask, normalize)
    counts, sums, rows, _ = _statistics(whole)
    return Routing(weights, experts, counts, sums, rows, loss)


def adapted(x, down, up, ids, *, base=None, gates=None, scales=None):
    """``adapt`` inside autograd: gradients go to x, down, up, base and gates."""
    return _Adapted.apply(x, down, up, ids, base, gates, scales)
