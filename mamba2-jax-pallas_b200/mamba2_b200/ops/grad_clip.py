"""Global gradient norm over many tensors, and clipping by it."""
from __future__ import annotations

from array import array

import torch

from .. import _lib

_DTYPE = {torch.float32: _lib.SSD_DTYPE_F32, torch.bfloat16: _lib.SSD_DTYPE_BF16}


def _checked(ts, name):
    ts = list(ts)
    for t in ts:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a list of torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be CUDA tensors (no CPU path)")
        if t.dtype not in _DTYPE:
            raise TypeError(f"unsupported dtype {t.dtype} (float32 or bfloat16)")
        if t.device != ts[0].device:
            raise ValueError(f"{name} must be on one device")
    return ts


def _run(grads, outs, max_norm, eps, scale):
    dev = grads[0].device
    norm = torch.empty((), device=dev, dtype=torch.float32)
    # ssd_grad_tensor_t: two addresses, the size, two 32-bit dtypes
    rec = array("q")
    for g, o in zip(grads, outs):
        rec.extend((g.data_ptr(), o.data_ptr(), g.numel(), _DTYPE[g.dtype] | _DTYPE[o.dtype] << 32))
    lib = _lib.load()
    addr = rec.buffer_info()[0]
    with torch.cuda.device(dev):
        n = lib.ssd_clip_grad_norm_workspace_bytes(addr, len(grads))
        ws = torch.empty(max(n, 8), device=dev, dtype=torch.uint8)
        _lib.check(lib.ssd_clip_grad_norm(addr, len(grads), float(max_norm), float(eps), int(scale), norm.data_ptr(),
                                          ws.data_ptr(), ws.numel(), _lib.stream_of(norm)))
    return norm


def grad_norm(grads):
    """2-norm over all tensors of ``grads`` (float32 or bfloat16, any mix and shapes): a float32
    scalar tensor.  Squares are summed in float64."""
    ts = [g.contiguous() for g in _checked(grads, "grads")]
    if not ts:
        raise ValueError("grads must not be empty")
    return _run(ts, ts, 0.0, 0.0, False)


def clip_grad_norm(grads, max_norm: float, *, eps: float = 1e-6, out=None, inplace: bool = False):
    """Scale gradients so that their global 2-norm is at most ``max_norm``.

    Returns ``(clipped, norm)``: ``grads`` times ``min(1, max_norm / (norm + eps))`` and the norm
    before clipping (a float32 scalar tensor on the device; nothing waits for it).  By default
    the clipped gradients are new tensors; ``inplace=True`` scales ``grads`` themselves, ``out``
    gives tensors of the same shapes to write to, float32 or bfloat16 (bfloat16 gradients into
    the float32 buffers of an optimizer).  A NaN norm makes every gradient NaN.
    """
    ts = _checked(grads, "grads")
    if not ts:
        raise ValueError("grads must not be empty")
    if not float(max_norm) >= 0.0 or not float(eps) >= 0.0:
        raise ValueError("max_norm and eps must be non-negative")
    if inplace:
        if out is not None:
            raise ValueError("give either out or inplace=True")
        for g in ts:
            if not g.is_contiguous():
                raise ValueError("inplace=True needs contiguous gradients")
        outs = ts
    else:
        ts = [g.contiguous() for g in ts]
        if out is None:
            outs = [torch.empty_like(g) for g in ts]
        else:
            outs = _checked(out, "out")
            if len(outs) != len(ts):
                raise ValueError(f"out has {len(outs)} tensors, grads {len(ts)}")
            for g, o in zip(ts, outs):
                if o.shape != g.shape or not o.is_contiguous():
                    raise ValueError("out must hold contiguous tensors of grads' shapes")
                if o.device != g.device:
                    raise ValueError("out and grads must be on one device")
    return outs, _run(ts, outs, max_norm, eps, True)
