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
refused outside ``torch.no_grad()``, since no graph is recorded; so are tensors
with a forward-mode tangent, and calls under a tracer.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

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
# host counts: plain integers for pointers, no views where a pointer and a
# distance of rows are enough, the current stream's handle without a Stream
# object, and a device guard only where another device is current (a call of
# linear on 4 rows: 12.2 us with the general forms of these, 9.8 without, of
# which the launch is 4.4).
_Tensor, _strided = torch.Tensor, torch.strided
_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice
_tracing = torch._C._get_tracing_state
_mode, _PROXY = torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY


def _activation(name) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {[a for a in ACTIVATIONS if a]} or None, not {name!r}")
    return ACTIVATIONS[name]


def _check(what: str, t: Optional[torch.Tensor], like: torch.Tensor, dtype=None, shape=None) -> None:
    """Type, place and shape of an operand (shapes before the device, so that
    wrong calls fail alike with and without a GPU)."""
    if t is None:
        return
    if not isinstance(t, _Tensor):
        raise TypeError(f"{what} must be a tensor")
    if dtype is None:
        dtype = like.dtype
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, not {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.layout is not _strided:
        raise TypeError(f"{what} must be a dense tensor")
    if t.get_device() != like.get_device():
        raise ValueError(f"{what} is on {t.device}, the input on {like.device}")


def _check_input(what: str, x: torch.Tensor, dims: int = 1) -> None:
    if not isinstance(x, _Tensor):
        raise TypeError(f"{what} must be a tensor")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {x.dtype}")
    if x.layout is not _strided:
        raise TypeError(f"{what} must be a dense tensor")
    if x.dim() < dims or x.shape[-1] < 1:
        raise ValueError(f"{what} must have {dims} or more axes, the last of at least 1 (got {tuple(x.shape)})")


def _check_run(x: torch.Tensor, *others) -> None:
    """Refuses what would be lost without a word: derivatives in either mode,
    and a call that a tracer records as the allocation of its outputs."""
    if torch.is_grad_enabled():
        for t in (x, *others):
            if t is not None and t.requires_grad:
                raise ValueError("a tensor requires grad: call under torch.no_grad() and take the gradients with the "
                                 "_backward function (no autograd graph is recorded)")
    if forward_ad._current_level >= 0:
        for t in (x, *others):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("a tensor carries a tangent: there is no forward-mode derivative")
    if _tracing() is not None or _mode(_PROXY) is not None:
        raise RuntimeError("the call cannot be traced: capture it into a CUDA graph instead")
    if not x.is_cuda:
        raise ValueError("tensors must be on the GPU; there is no CPU fallback")


def _elsewhere(x: torch.Tensor) -> bool:
    """Whether x's device is not the current one."""
    return x.get_device() != _current()


def _rows(t: torch.Tensor, copy: bool = True) -> Optional[torch.Tensor]:
    """t as (rows, width) with unit stride in a row and rows at a constant
    distance of at least the width; a copy where its layout allows no such
    view (None with copy=False)."""
    width = t.shape[-1]
    if t.is_neg():  # of a conjugate's imaginary part: the memory holds -t
        if not copy:
            return None
        t = t.resolve_neg()
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


def _laid(t: Optional[torch.Tensor]):
    """t (or a copy, see _rows) and the distance of its rows."""
    if t is None:
        return None, 0
    width = t.shape[-1]
    if t.is_contiguous() and not t.is_neg():
        return t, width
    r = _rows(t)
    return r, max(r.stride(0), width)


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t, or a contiguous copy of what it stands for."""
    if t is None or t.is_contiguous() and not t.is_neg():
        return t
    return t.resolve_neg().contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, x: torch.Tensor) -> Optional[torch.Tensor]:
    return x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _limits(rows: int, *widths: int) -> None:
    if max(rows, *widths) > _MOST:
        raise ValueError(f"at most {_MOST} rows and columns")


def _norm_limits(rows: int, D: int) -> None:
    _limits(0, D)
    if D > 16384 and rows >= 2 ** 22:
        raise ValueError(f"at most {2 ** 22 - 1} rows of more than 16384 elements")


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
    if bias is not None:
        _check("bias", bias, x, torch.float32, (E, N) if grouped else (N,))
    if residual is not None:
        _check("residual", residual, x, shape=shape)
    if out is not None:
        _check("out", out, x, shape=shape)
    if grouped:
        _check_counts(counts, E, x)
    M = x.numel() // K
    _limits(M, N, K)
    _check_run(x, weight, bias, residual, out)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return _forward(x, counts, weight, bias, residual, activation, return_pre, out)
    xr, ldx = _laid(x)
    w, ldw = (_dense(weight), K) if grouped else _laid(weight)
    b = _dense(bias)
    r, ldr = _laid(residual)
    fresh = out is None
    if fresh:
        o = out = x.new_empty(shape)
        ldo = N
    else:
        o = _output(out, (_rows(xr), w.view(-1, K) if grouped else _rows(w), None if b is None else b.view(1, -1)),
                    () if r is None else (_rows(r),))
        ldo = max(o.stride(0), N)
    pre = x.new_empty(shape) if return_pre else None
    if M:
        dt, stream = _DTYPES[x.dtype], _stream(x.get_device())
        if grouped:
            # a new tensor's rows behind the last group are zeros; the saved
            # argument is always new
            if return_pre and not fresh:
                pre.zero_()
            call("mdx_grouped_linear", xr.data_ptr(), ldx, w.data_ptr(), _ptr(b), _ptr(r), ldr, counts.data_ptr(), E, M,
                 N, K, act, dt, _ptr(pre), N, o.data_ptr(), ldo, int(fresh), stream)
        else:
            nbytes = call("mdx_linear_workspace_bytes", M, N, K, dt)
            ws = _workspace(nbytes, x)
            call("mdx_linear", xr.data_ptr(), ldx, w.data_ptr(), ldw, _ptr(b), _ptr(r), ldr, M, N, K, act, dt, _ptr(pre),
                 N, o.data_ptr(), ldo, _ptr(ws), nbytes, stream)
    return (out, pre) if return_pre else out


def linear_backward(grad, x, weight, pre=None, activation=None, *, need_x: bool = True, need_weight: bool = True,
                    need_bias: bool = False, need_residual: bool = False) -> LinearGrads:
    """Gradients of linear() for grad (..., N): with dz = grad * act'(pre),
    x = dz @ weight, weight = dz.T @ x, bias = dz's sum over the rows
    (float32), residual = dz (grad itself when there is no activation).  pre:
    what linear(..., return_pre=True) returned; not needed without an
    activation.  dz is rounded to x's dtype where it enters the products (in
    float16 infinite beyond 65504 and zero below 3e-8, as between separate
    float16 layers: scale the loss); float32 operands keep all of it."""
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
    if pre is not None:
        _check("pre", pre, x, shape=shape)
    elif act:
        raise ValueError("an activation needs pre, from linear(..., return_pre=True)")
    if grouped:
        _check_counts(counts, E, x)
    M = x.numel() // K
    _limits(M, N, K)
    _check_run(x, grad, weight, pre)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return _backward(grad, x, counts, weight, pre, activation, need_x, need_weight, need_bias, need_residual)
    dx = x.new_empty(x.shape) if need_x else None
    dw = x.new_empty(weight.shape) if need_weight else None
    db = x.new_empty((E, N) if grouped else (N,), dtype=torch.float32) if need_bias else None
    # without an activation the residual's gradient is grad, but for the rows
    # that no group holds
    own = need_residual and (act or grouped)
    dr = x.new_empty(shape) if own else None
    if need_x or need_weight or need_bias or own:
        xr, ldx = _laid(x)
        gr, ldg = _laid(grad)
        w, ldw = (_dense(weight), K) if grouped else _laid(weight)
        z, ldz = _laid(pre) if act else (None, 0)
        dt, stream = _DTYPES[x.dtype], _stream(x.get_device())
        flags = (bool(need_x), bool(need_weight), bool(need_bias), bool(own))
        if grouped:
            nbytes = call("mdx_grouped_linear_backward_workspace_bytes", E, M, N, K, act, dt, *flags)
            ws = _workspace(nbytes, x)
            call("mdx_grouped_linear_backward", gr.data_ptr(), ldg, xr.data_ptr(), ldx, w.data_ptr(), _ptr(z), ldz,
                 counts.data_ptr(), E, M, N, K, act, dt, _ptr(dx), K, _ptr(dw), _ptr(db), _ptr(dr), N, 1, _ptr(ws),
                 nbytes, stream)
        else:
            nbytes = call("mdx_linear_backward_workspace_bytes", M, N, K, act, dt, *flags)
            ws = _workspace(nbytes, x)
            call("mdx_linear_backward", gr.data_ptr(), ldg, xr.data_ptr(), ldx, w.data_ptr(), ldw, _ptr(z), ldz, M, N, K,
                 act, dt, _ptr(dx), K, _ptr(dw), K, _ptr(db), _ptr(dr), N, _ptr(ws), nbytes, stream)
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
    _norm_limits(x.numel() // D, D)
    _check_run(x, weight, bias, out)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return layer_norm(x, weight, bias, eps, return_stats=return_stats, out=out)
    xr, ldx = _laid(x)
    w = _dense(weight)
    b = _dense(bias)
    if out is None:
        o = out = x.new_empty(x.shape)
        ldo = D
    else:
        o = _output(out, [None if t is None else t.view(1, -1) for t in (w, b)], (_rows(xr),))
        ldo = max(o.stride(0), D)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32) if return_stats else None
    rstd = x.new_empty(x.shape[:-1], dtype=torch.float32) if return_stats else None
    rows = x.numel() // D
    if rows:
        call("mdx_layer_norm", xr.data_ptr(), ldx, _ptr(w), _ptr(b), rows, D, float(eps), _DTYPES[x.dtype], o.data_ptr(), ldo,
             _ptr(mean), _ptr(rstd), _stream(x.get_device()))
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
    _norm_limits(x.numel() // D, D)
    _check_run(x, grad, mean, rstd, weight)
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return layer_norm_backward(grad, x, mean, rstd, weight, need_x=need_x, need_weight=need_weight,
                                       need_bias=need_bias)
    dx = x.new_empty(x.shape) if need_x else None
    dw = x.new_empty(D, dtype=torch.float32) if need_weight else None
    db = x.new_empty(D, dtype=torch.float32) if need_bias else None
    if need_x or need_weight or need_bias:
        xr, ldx = _laid(x)
        gr, ldg = _laid(grad)
        m, r = _dense(mean), _dense(rstd)
        w = _dense(weight)
        rows, dt = x.numel() // D, _DTYPES[x.dtype]
        nbytes = call("mdx_layer_norm_backward_workspace_bytes", rows, D, dt) if need_weight or need_bias else 0
        ws = _workspace(nbytes, x)
        call("mdx_layer_norm_backward", gr.data_ptr(), ldg, xr.data_ptr(), ldx, m.data_ptr(), r.data_ptr(), _ptr(w), rows,
             D, dt, _ptr(dx), D, _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(x.get_device()))
    return LayerNormGrads(dx, dw, db)
