"""Gated feed-forward block and its gradients: the other half of a model's layers, beside its mixers."""
from __future__ import annotations

import torch

from .. import _lib


def _rows(t, width):
    """Rows of ``width`` contiguous values at one distance, a view where there is one, and that distance."""
    if t.is_contiguous():
        return t, width
    t = _lib.rows2d(t, width)
    return t, _lib.row_stride(t)


def _prepare(x, w_gate, w_up, w_down, activation):
    if not (isinstance(x, torch.Tensor) and isinstance(w_gate, torch.Tensor) and isinstance(w_up, torch.Tensor) and
            isinstance(w_down, torch.Tensor)):
        raise TypeError("x, w_gate, w_up and w_down must be torch.Tensors")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (no CPU path)")
    dtype, dev = x.dtype, x.device
    if w_gate.dtype is not dtype or w_up.dtype is not dtype or w_down.dtype is not dtype:
        raise TypeError(f"w_gate ({w_gate.dtype}), w_up ({w_up.dtype}), w_down ({w_down.dtype}) and x ({dtype}) must have the "
                        "same dtype")
    if not dev == w_gate.device == w_up.device == w_down.device:
        raise ValueError("the weights must be on x's device")
    act = _lib.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(_lib.ACTIVATIONS)}")
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape:
        raise ValueError("w_gate and w_up must be (hidden, dim)")
    hidden, dim = w_gate.shape
    if w_down.dim() != 2 or w_down.shape[1] != hidden:
        raise ValueError(f"w_down must be (dim_out, {hidden})")
    out = w_down.shape[0]
    if hidden == 0 or dim == 0 or out == 0:
        raise ValueError("the weights must not be empty")
    if x.dim() < 1 or x.shape[-1] != dim:
        raise ValueError(f"x {tuple(x.shape)} must end in the weights' {dim} columns")
    (xr, xs), (g, gs), (u, us), (d, ds) = _rows(x, dim), _rows(w_gate, dim), _rows(w_up, dim), _rows(w_down, hidden)
    p = _lib.GatedFfParams(xr.numel() // dim, dim, hidden, out, xs, gs, us, ds, _lib.dtype_code(x), act,
                           xr.data_ptr(), g.data_ptr(), u.data_ptr(), d.data_ptr(), None)
    return p, (xr, g, u, d)   # (copies have to live until the call)


def gated_feed_forward(x, w_gate, w_up, w_down, *, activation: str = "silu", check_status: bool = False):
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``.

    x (..., dim), w_gate and w_up (hidden, dim) and w_down (dim_out, hidden) of one dtype, float32 or
    bfloat16; the weights may be row slices of a larger one.  ``activation`` is "silu", "gelu", "gelu_tanh" or "relu".
    Returns (..., dim_out) in x's dtype: products summed in float32, the hidden values rounded once to x's
    dtype (float32: not below its own accuracy; bfloat16, up to 4 tokens: kept in float32), the result once.  A
    value that is not finite makes its row's results so where the formula has them so; in float32 of more than 24
    tokens (and in its gradients) an infinity, or a hidden value above 3.396e38, gives NaN where the formula keeps an infinity or
    drops it.  ``check_status`` waits for the call and raises
    ``SsdError`` if a bounded wait inside a kernel gave up.  The result carries no autograd history:
    ``gated_feed_forward_grad`` gives the gradients.
    """
    p, rows = _prepare(x, w_gate, w_up, w_down, activation)
    y = torch.empty_like(x) if p.dim_out == p.dim and x.is_contiguous() else x.new_empty((*x.shape[:-1], p.dim_out))
    if p.tokens == 0:
        return y
    p.y = y.data_ptr()
    lib = _lib.load()
    with _lib.on_device(x.device):
        ws = y.new_empty(lib.ssd_gated_ff_workspace_bytes(p), dtype=torch.uint8)
        _lib.check(lib.ssd_gated_ff(p, ws.data_ptr(), ws.numel(), _lib.stream_of(y)))
        if check_status:
            _lib.check_device_status(ws)
    return y


def gated_feed_forward_grad(x, w_gate, w_up, w_down, grad_out, *, activation: str = "silu", weight_grad_dtype=None,
                            need_input_grad: bool = True, need_weight_grad: bool = True, check_status: bool = False):
    """Gradients of ``gated_feed_forward``: ``(grad_x, grad_w_gate, grad_w_up, grad_w_down)``.

    grad_out (..., dim_out) in x's dtype is the gradient that reaches the result; the hidden values are
    computed again from x.  grad_x has x's dtype, the weights' gradients ``weight_grad_dtype`` (default x's; float32
    for an accumulation over micro-batches).  Gradients that are not needed are None and cost nothing (frozen
    weights, or frozen layers below).  Equal calls give equal bits.
    """
    p, rows = _prepare(x, w_gate, w_up, w_down, activation)
    out_shape = (*x.shape[:-1], w_down.shape[0])
    if not isinstance(grad_out, torch.Tensor) or tuple(grad_out.shape) != out_shape or grad_out.device != x.device:
        raise ValueError(f"grad_out must be a {out_shape} tensor on x's device")
    if grad_out.dtype != x.dtype:
        raise TypeError(f"grad_out ({grad_out.dtype}) and x ({x.dtype}) must have the same dtype")
    wd = x.dtype if weight_grad_dtype is None else weight_grad_dtype
    if wd not in (torch.float32, torch.bfloat16):
        raise ValueError("weight_grad_dtype must be torch.float32 or torch.bfloat16")
    new = torch.zeros if p.tokens == 0 else torch.empty
    dev = x.device
    gx = new(x.shape, dtype=x.dtype, device=dev) if need_input_grad else None
    gw = [new(w.shape, dtype=wd, device=dev) if need_weight_grad else None for w in (w_gate, w_up, w_down)]
    if p.tokens == 0 or not (need_input_grad or need_weight_grad):
        return gx, *gw
    dy, dys = _rows(grad_out, p.dim_out)
    g = _lib.GatedFfGrads(dys, dy.data_ptr(), _lib.ptr(gx), *(_lib.ptr(t) for t in gw), wd is torch.bfloat16, 0)
    lib = _lib.load()
    with _lib.on_device(dev):
        ws = torch.empty(lib.ssd_gated_ff_grad_workspace_bytes(p, g), dtype=torch.uint8, device=dev)
        _lib.check(lib.ssd_gated_ff_grad(p, g, ws.data_ptr(), ws.numel(), _lib.stream_of(x)))
        if check_status:
            _lib.check_device_status(ws)
    return gx, *gw
