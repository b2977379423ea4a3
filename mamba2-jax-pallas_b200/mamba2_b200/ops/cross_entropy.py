"""Output projection and softmax cross entropy in one operator, with its gradients: the last
step of a language model.  The logits of a batch are never held as a whole."""
from __future__ import annotations

import torch

from .. import _lib


def _call(hidden, weight, targets, ignore_index, reduction, grad_loss, want_lse, want_hidden, want_weight,
          weight_grad_dtype, check_status):
    if reduction not in _lib.REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    y = _lib.index_list(targets, "targets")
    for t, name in ((hidden, "hidden"), (weight, "weight")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (no CPU path)")
    if weight.dim() != 2:
        raise ValueError("weight must be (vocab, dim)")
    vocab, dim = weight.shape
    if hidden.dim() < 1 or hidden.shape[-1] != dim:
        raise ValueError(f"hidden {tuple(hidden.shape)} must end in weight's {dim} columns")
    if tuple(hidden.shape[:-1]) != tuple(targets.shape):
        raise ValueError(f"targets {tuple(targets.shape)} must have hidden's shape without its last axis")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden ({hidden.dtype}) and weight ({weight.dtype}) must have the same dtype")
    if not hidden.device == weight.device == y.device:
        raise ValueError("hidden, weight and targets must be on one device")
    if vocab == 0 or dim == 0:
        raise ValueError("weight must not be empty")
    dtype = _lib.dtype_code(weight)
    wd = weight.dtype if weight_grad_dtype is None else weight_grad_dtype
    if wd not in (torch.float32, torch.bfloat16):
        raise ValueError("weight_grad_dtype must be torch.float32 or torch.bfloat16")
    x, w = _lib.rows2d(hidden, dim), _lib.rows2d(weight, dim)
    n, dev = y.numel(), x.device
    g = None
    if grad_loss is not None:
        want = tuple(targets.shape) if reduction == "none" else ()
        if not isinstance(grad_loss, torch.Tensor) or tuple(grad_loss.shape) != want or grad_loss.device != dev:
            raise ValueError(f"grad_loss must be a {want} tensor on hidden's device")
        g = _lib.dev(grad_loss, "grad_loss", torch.float32)
    new = x.new_zeros if n == 0 else x.new_empty
    loss = new(targets.shape if reduction == "none" else (), dtype=torch.float32)
    lse = new(targets.shape, dtype=torch.float32) if want_lse else None
    gx = new(hidden.shape) if want_hidden else None
    gw = new((vocab, dim), dtype=wd) if want_weight else None
    if n == 0:
        return loss, lse, gx, gw
    p = _lib.LinearCeParams(n, vocab, dim, _lib.row_stride(x), _lib.row_stride(w), int(ignore_index), dtype,
                            y.dtype is torch.int64, _lib.REDUCTIONS[reduction], wd is torch.bfloat16, x.data_ptr(),
                            w.data_ptr(), y.data_ptr(), _lib.ptr(g), loss.data_ptr(), _lib.ptr(lse), _lib.ptr(gx),
                            _lib.ptr(gw))
    lib = _lib.load()
    with _lib.on_device(dev):
        ws = x.new_empty(lib.ssd_linear_cross_entropy_workspace_bytes(p), dtype=torch.uint8)
        _lib.check(lib.ssd_linear_cross_entropy(p, ws.data_ptr(), ws.numel(), _lib.stream_of(x)))
        if check_status:
            _lib.check_device_status(ws)
    return loss, lse, gx, gw


def linear_cross_entropy(hidden, weight, targets, *, ignore_index: int = -100, reduction: str = "mean",
                         return_lse: bool = False, check_status: bool = False):
    """Cross entropy of ``softmax(hidden @ weight.T)`` against ``targets``.

    hidden (..., dim) and weight (vocab, dim) of one dtype, float32 or bfloat16; targets (...)
    int32 or int64.  Returns float32: a scalar, or with ``reduction="none"`` one loss per token;
    with ``return_lse`` also the log of each row's sum of exponentials (0 where ignored).  A target equal to
    ``ignore_index`` has loss 0 and does not count in the mean (a mean over no tokens is 0); any
    other target outside [0, vocab) has loss NaN.  ``check_status`` waits for the call and
    raises ``SsdError`` if a bounded wait inside a kernel gave up.  The result carries no autograd
    history, also where an input requires a gradient: ``linear_cross_entropy_grad`` gives both.
    """
    loss, lse, _, _ = _call(hidden, weight, targets, ignore_index, reduction, None, return_lse, False, False, None,
                            check_status)
    return (loss, lse) if return_lse else loss


def linear_cross_entropy_grad(hidden, weight, targets, *, ignore_index: int = -100, reduction: str = "mean",
                              grad_loss=None, weight_grad_dtype=None, need_hidden_grad: bool = True,
                              need_weight_grad: bool = True, check_status: bool = False):
    """``linear_cross_entropy`` and its gradients: ``(loss, grad_hidden, grad_weight)``.

    ``grad_loss`` is the gradient that reaches the loss: a float32 scalar tensor (a loss scale),
    or one value per token with ``reduction="none"``; default ones.  grad_hidden has hidden's
    dtype, grad_weight ``weight_grad_dtype`` (default weight's; float32 for an accumulation over
    micro-batches).  A gradient that is not needed is None and costs nothing (a frozen head, or
    frozen layers below).
    """
    loss, _, gx, gw = _call(hidden, weight, targets, ignore_index, reduction, grad_loss, False, need_hidden_grad,
                            need_weight_grad, weight_grad_dtype, check_status)
    return loss, gx, gw
