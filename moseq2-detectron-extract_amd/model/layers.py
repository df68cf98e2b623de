"""Linear layers, grouped linear layers and layer norm of detection heads,
forward and backward, on gfx950 (include/mdx.h, csrc/linear.hip, csrc/norm.hip).

=======================  ========================================================
this module              what it computes
=======================  ========================================================
linear                   act(x W^T + b + r), float32 / float16 / bfloat16
linear_backward          its gradients: x, weight, bias, residual
grouped_linear           the same with one weight per group of ragged rows
grouped_linear_backward  its gradients
layer_norm               (x - mean) rstd gamma + beta over the last axis
layer_norm_backward      its gradients: x, gamma, beta
=======================  ========================================================

The reference takes these from torch.nn through Detectron2's heads
(FastRCNNConvFCHead, M/model/config.py:21-94).  All tensors live on one GPU
and work is enqueued on that GPU's current stream, without host
synchronisation, so the calls can be captured into a graph.  ``bias``,
``gamma`` / ``beta`` and their gradients are float32, everything else has the
input's dtype.  Leading axes are flattened; rows may be strided, other layouts
are copied first.  Gradients are explicit calls: tensors that require grad are
refused outside ``torch.no_grad()``, since no graph is recorded.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .._lib import call

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 3}
_MOST = 2 ** 31 - 1 - 2 ** 16  # rows, columns


class LinearGrads(NamedTuple):
    """Gradients of a linear layer; None where not asked for."""
    x: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]
    residual: Optional[torch.Tensor]


class LayerNormGrads(NamedTuple):
    """Gradients of a layer norm; None where not asked for."""
    x: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]


# ---------------------------------------------------------------------------
# plumbing
# ---------------------------------------------------------------------------
# A call on a few rows takes the GPU some 5 us, so what a call costs on the
# host counts: plain integers for pointers, the current stream's handle without
# a Stream object, and a device guard only where another device is current.
def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


class _on:
    """The device guard of a call: nothing where `device` is current."""

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _activation(name) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in ACTIVATIONS if a]} or None, not {name!r}")
    return ACTIVATIONS[name]


def _check(what: str, t: Optional[torch.Tensor], like: torch.Tensor, dtype=None, shape=None) -> None:
    """Type, place and shape of an operand (shapes before the device, so that
    wrong calls fail alike with and without a GPU)."""
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    dtype = like.dtype if dtype is None else dtype
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, not {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.layout != torch.strided:
        raise TypeError(f"{what} must be a dense tensor")
    if t.device != like.device:
        raise ValueError(f"{what} is on {t.device}, the input on {like.device}")


def _check_input(what: str, x: torch.Tensor, dims: int = 1) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    if x.layout != torch.strided:
        raise TypeError(f"{what} must be a dense tensor")
    if x.dim() < dims or x.shape[-1] < 1:
        raise ValueError(f"{what} must have {dims} or more axes, the last of at least 1 (got {tuple(x.shape)})")


def _check_run(x: torch.Tensor, *others) -> None:
    if torch.is_grad_enabled():
        for t in (x, *others):
            if t is not None and t.requires_grad:
                break
        else:
            t = None
    else:
        t = None
    if t is not None:
        raise ValueError("a tensor requires grad: call under torch.no_grad() and take the gradients with the "
                         "_backward function (no autograd graph is recorded)")
    if not x.is_cuda:
        raise ValueError("tensors must be on the GPU; there is no CPU fallback")


def _rows(t: torch.Tensor, copy: bool = True) -> Optional[torch.Tensor]:
    """t as (rows, width) with unit stride in a row and rows at a constant
    distance of at least the width; a copy where its layout allows no such
    view (None with copy=False)."""
    width = t.shape[-1]
    if t.is_contiguous():
        r = t if t.dim() == 2 else t.view(-1, width)
        if r.stride(0) == width:
            return r
    n = t.numel() // width
    if n == 0:
        return t.reshape(0, width)
    if width == 1 or t.stride(-1) == 1:
        # the axes that have more than one entry, outermost first
        lead = [(s, d) for s, d in zip(t.shape[:-1], t.stride()[:-1]) if s != 1]
        step = lead[-1][1] if lead else width
        if step >= width and all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])):
            return t.as_strided((n, width), (step, 1))
    return t.contiguous().view(n, width) if copy else None


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two (rows, width) views share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    ea, eb = a.element_size(), b.element_size()
    a0, b0 = a.data_ptr(), b.data_ptr()
    a1 = a0 + ((a.shape[0] - 1) * a.stride(0) + a.shape[1]) * ea
    b1 = b0 + ((b.shape[0] - 1) * b.stride(0) + b.shape[1]) * eb
    if a0 >= b1 or b0 >= a1:
        return False
    pitch = a.stride(0) * ea
    if pitch == b.stride(0) * eb:  # columns of one buffer lie beside each other
        at = (b0 - a0) % pitch
        return not (at >= a.shape[1] * ea and at + b.shape[1] * eb <= pitch)
    return True


def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()


def _output(out: torch.Tensor, reads, inplace=()) -> torch.Tensor:
    """The rows of the caller's `out`, which must not share memory with
    `reads`, nor in part with `inplace`."""
    rows = _rows(out, copy=False)
    if rows is None:
        raise ValueError("out must have rows of unit stride at a constant distance")
    for r in reads:
        if r is not None and _overlap(rows, r):
            raise ValueError("out shares memory with an input")
    for r in inplace:
        if r is not None and not _same(rows, r) and _overlap(rows, r):
            raise ValueError("out shares part of its memory with an input")
    return rows


def _ld(rows: Optional[torch.Tensor]) -> int:
    """Distance of the rows; a single row's is its width."""
    return 0 if rows is None else max(rows.stride(0), rows.shape[1])


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _limits(rows: int, *widths: int) -> None:
    if rows > _MOST or any(w > _MOST for w in widths):
        raise ValueError(f"at most {_MOST} rows and columns")


def _check_counts(counts, E: int, like: torch.Tensor) -> None:
    _check("counts", counts, like, torch.int32, (E,))
    if not counts.is_contiguous():
        raise ValueError("counts must be contiguous")


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
def linear(x, weight, bias=None, residual=None, activation=None, *, return_pre: bool = False, out=None):
    """act(x @ weight.T + bias + residual).

    x (..., K); weight (N, K); bias float32 (N,) or None; residual (..., N) or
    None; activation None / "none", "relu", "gelu", "gelu_tanh" or "silu".
    return_pre: also the activation's argument, in x's dtype, which
    linear_backward needs.  out: a tensor (..., N) to write, which may be the
    residual itself."""
    return _forward(x, None, weight, bias, residual, activation, return_pre, out)


def grouped_linear(x, counts, weight, bias=None, residual=None, activation=None, *, return_pre: bool = False,
                   out=None):
    """linear() of each group of rows with the group's own weight.

    x (T, K): the rows of group 0, then those of group 1, ...; counts int32
    (E,) on the GPU, the rows of each group (never read by the host; a
    negative count is 0, and what passes T is cut off); weight (E, N, K); bias
    float32 (E, N) or None; residual (T, N) or None.  Rows behind the last
    group: zeros in a new tensor, left as they were in `out`."""
    _check_input("x", x, 2)
    if x.dim() != 2:
        raise ValueError("x must be (T, K)")
    if counts is None:
        raise TypeError("counts must be a tensor")
    return _forward(x, counts, weight, bias, residual, activation, return_pre, out)


def _weight_shape(x, weight, grouped: bool):
    _check("weight", weight, x)
    if weight.dim() != (3 if grouped else 2) or weight.shape[-1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError(f"weight must be {'(E, N, K)' if grouped else '(N, K)'} with K = {x.shape[-1]} and no empty "
                         f"axis, not {tuple(weight.shape)}")
    if grouped and weight.shape[0] > 4096:
        raise ValueError("at most 4096 groups")
    return (weight.shape[0] if grouped else 0), weight.shape[-2], weight.shape[-1]


def _forward(x, counts, weight, bias, residual, activation, return_pre, out):
    _check_input("x", x)
    grouped = counts is not None
    E, N, K = _weight_shape(x, weight, grouped)
    act = _activation(activation)
    shape = (*x.shape[:-1], N)
    _check("bias", bias, x, torch.float32, (E, N) if grouped else (N,))
    _check("residual", residual, x, shape=shape)
    _check("out", out, x, shape=shape)
    if grouped:
        _check_counts(counts, E, x)
    _limits(x.numel() // K, N, K)
    _check_run(x, weight, bias, residual, out)
    with _on(x.device):
        xr = _rows(x)
        w = weight.contiguous() if grouped else _rows(weight)
        b = bias.contiguous() if bias is not None else None
        r = _rows(residual) if residual is not None else None
        fresh = out is None
        if fresh:
            out = x.new_empty(shape)
            o = out if len(shape) == 2 else out.view(-1, N)
        else:
            o = _output(out, (xr, w.view(-1, K), None if b is None else b.view(1, -1)), (r,))
        pre = x.new_empty(shape) if return_pre else None
        p = pre.view(-1, N) if return_pre else None
        M, dt = xr.shape[0], _DTYPES[x.dtype]
        if M:
            if grouped:
                # a new tensor's rows behind the last group are zeros; the
                # saved argument is always new
                if return_pre and not fresh:
                    pre.zero_()
                call("mdx_grouped_linear", _ptr(xr), _ld(xr), _ptr(w), _ptr(b), _ptr(r), _ld(r), _ptr(counts), E, M, N,
                     K, act, dt, _ptr(p), _ld(p), _ptr(o), _ld(o), int(fresh), _stream(x.device))
            else:
                nbytes = call("mdx_linear_workspace_bytes", M, N, K, dt)
                ws = _workspace(nbytes, x.device)
                call("mdx_linear", _ptr(xr), _ld(xr), _ptr(w), _ld(w), _ptr(b), _ptr(r), _ld(r), M, N, K, act, dt,
                     _ptr(p), _ld(p), _ptr(o), _ld(o), _ptr(ws), nbytes, _stream(x.device))
    return (out, pre) if return_pre else out


def linear_backward(grad, x, weight, pre=None, activation=None, *, need_x: bool = True, need_weight: bool = True,
                    need_bias: bool = False, need_residual: bool = False) -> LinearGrads:
    """Gradients of linear() for grad (..., N): with dz = grad * act'(pre),
    x = dz @ weight, weight = dz.T @ x, bias = dz's sum over the rows
    (float32), residual = dz (grad itself when there is no activation).  pre:
    what linear(..., return_pre=True) returned; not needed without an
    activation.  dz is rounded to x's dtype where it enters the products."""
    return _backward(grad, x, None, weight, pre, activation, need_x, need_weight, need_bias, need_residual)


def grouped_linear_backward(grad, x, counts, weight, pre=None, activation=None, *, need_x: bool = True,
                            need_weight: bool = True, need_bias: bool = False,
                            need_residual: bool = False) -> LinearGrads:
    """Gradients of grouped_linear() for grad (T, N).  weight (E, N, K) and
    bias (E, N) of a group without rows, and x and residual in the rows behind
    the last group, are zeros."""
    _check_input("x", x, 2)
    if x.dim() != 2:
        raise ValueError("x must be (T, K)")
    if counts is None:
        raise TypeError("counts must be a tensor")
    return _backward(grad, x, counts, weight, pre, activation, need_x, need_weight, need_bias, need_residual)


def _backward(grad, x, counts, weight, pre, activation, need_x, need_weight, need_bias, need_residual):
    _check_input("x", x)
    grouped = counts is not None
    E, N, K = _weight_shape(x, weight, grouped)
    act = _activation(activation)
    shape = (*x.shape[:-1], N)
    if grad is None:
        raise TypeError("grad must be a tensor")
    _check("grad", grad, x, shape=shape)
    _check("pre", pre, x, shape=shape)
    if act and pre is None:
        raise ValueError("an activation needs pre, from linear(..., return_pre=True)")
    if grouped:
        _check_counts(counts, E, x)
    _limits(x.numel() // K, N, K)
    _check_run(x, grad, weight, pre)
    dev = x.device
    with _on(dev):
        xr, gr = _rows(x), _rows(grad)
        w = weight.contiguous() if grouped else _rows(weight)
        z = _rows(pre) if act else None
        M, dt = xr.shape[0], _DTYPES[x.dtype]
        dx = x.new_empty(x.shape) if need_x else None
        dw = x.new_empty(weight.shape) if need_weight else None
        db = torch.empty((E, N) if grouped else (N,), dtype=torch.float32, device=dev) if need_bias else None
        # without an activation the residual's gradient is grad, but for the
        # rows that no group holds
        own = need_residual and (act or grouped)
        dr = x.new_empty(shape) if own else None
        flags = (int(need_x), int(need_weight), int(need_bias), int(own))
        if need_x or need_weight or need_bias or own:
            dxr, drr = (None if t is None else t.view(-1, t.shape[-1]) for t in (dx, dr))
            if grouped:
                nbytes = call("mdx_grouped_linear_backward_workspace_bytes", E, M, N, K, act, dt, *flags)
                ws = _workspace(nbytes, dev)
                call("mdx_grouped_linear_backward", _ptr(gr), _ld(gr), _ptr(xr), _ld(xr), _ptr(w), _ptr(z), _ld(z),
                     _ptr(counts), E, M, N, K, act, dt, _ptr(dxr), K, _ptr(dw), _ptr(db), _ptr(drr), N, 1, _ptr(ws),
                     nbytes, _stream(x.device))
            else:
                nbytes = call("mdx_linear_backward_workspace_bytes", M, N, K, act, dt, *flags)
                ws = _workspace(nbytes, dev)
                call("mdx_linear_backward", _ptr(gr), _ld(gr), _ptr(xr), _ld(xr), _ptr(w), _ld(w), _ptr(z), _ld(z), M,
                     N, K, act, dt, _ptr(dxr), K, _ptr(dw), K, _ptr(db), _ptr(drr), N, _ptr(ws), nbytes, _stream(x.device))
    return LinearGrads(dx, dw, db, (dr if own else grad) if need_residual else None)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, *, return_stats: bool = False, out=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (biased
    variance); weight / bias float32 (D,) or None.  return_stats: also mean and
    rstd = 1 / sqrt(var + eps), float32 (...), which layer_norm_backward
    needs.  out: a tensor like x to write, which may be x itself."""
    _check_input("x", x)
    D = x.shape[-1]
    _check("weight", weight, x, torch.float32, (D,))
    _check("bias", bias, x, torch.float32, (D,))
    _check("out", out, x, shape=x.shape)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    _limits(0, D)
    _check_run(x, weight, bias, out)
    with _on(x.device):
        xr = _rows(x)
        w, b = (None if t is None else t.contiguous() for t in (weight, bias))
        if out is None:
            out = x.new_empty(x.shape)
            o = out if x.dim() == 2 else out.view(-1, D)
        else:
            o = _output(out, [None if t is None else t.view(1, -1) for t in (w, b)], (xr,))
        mean, rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if return_stats else None
                      for _ in range(2))
        if xr.shape[0]:
            call("mdx_layer_norm", _ptr(xr), _ld(xr), _ptr(w), _ptr(b), xr.shape[0], D, float(eps), _DTYPES[x.dtype],
                 _ptr(o), _ld(o), _ptr(mean), _ptr(rstd), _stream(x.device))
    return (out, mean, rstd) if return_stats else out


def layer_norm_backward(grad, x, mean, rstd, weight=None, *, need_x: bool = True, need_weight: bool = True,
                        need_bias: bool = True) -> LayerNormGrads:
    """Gradients of layer_norm() for grad like x: x in its dtype, weight and
    bias (sums over the rows) in float32.  mean / rstd: float32 (...), what
    layer_norm(..., return_stats=True) returned."""
    _check_input("x", x)
    D = x.shape[-1]
    if grad is None or mean is None or rstd is None:
        raise TypeError("grad, mean and rstd must be tensors")
    _check("grad", grad, x, shape=x.shape)
    _check("mean", mean, x, torch.float32, x.shape[:-1])
    _check("rstd", rstd, x, torch.float32, x.shape[:-1])
    _check("weight", weight, x, torch.float32, (D,))
    _limits(0, D)
    _check_run(x, grad, mean, rstd, weight)
    dev = x.device
    with _on(dev):
        xr, gr = _rows(x), _rows(grad)
        m, r = mean.contiguous(), rstd.contiguous()
        w = weight.contiguous() if weight is not None else None
        n, dt = xr.shape[0], _DTYPES[x.dtype]
        dx = x.new_empty(x.shape) if need_x else None
        dw, db = (torch.empty(D, dtype=torch.float32, device=dev) if need else None
                  for need in (need_weight, need_bias))
        if need_x or need_weight or need_bias:
            nbytes = call("mdx_layer_norm_backward_workspace_bytes", n, D, dt) if need_weight or need_bias else 0
            ws = _workspace(nbytes, dev)
            call("mdx_layer_norm_backward", _ptr(gr), _ld(gr), _ptr(xr), _ld(xr), _ptr(m), _ptr(r), _ptr(w), n, D, dt,
                 _ptr(dx.view(-1, D) if need_x else None), D, _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(x.device))
    return LayerNormGrads(dx, dw, db)
