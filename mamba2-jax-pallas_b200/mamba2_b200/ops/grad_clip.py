"""Global gradient norm over many tensors, and clipping by it."""
from __future__ import annotations

import math
import operator
from array import array

import torch

from .. import _lib

_DTYPE = {torch.float32: _lib.SSD_DTYPE_F32, torch.bfloat16: _lib.SSD_DTYPE_BF16}
_T = torch.Tensor
_dtype, _shape = operator.attrgetter("dtype"), operator.attrgetter("shape")


# A model has hundreds of tensors, and the kernels take a few microseconds where they are
# small: what is asked of each tensor goes through map() over the method itself.
def _checked(ts, name):
    """(list of tensors, the set of their dtypes, their device index), or an error."""
    ts = list(ts)
    if not ts:
        raise ValueError(f"{name} must not be empty")
    try:
        devices = set(map(_T.get_device, ts))
    except TypeError:
        raise TypeError(f"{name} must be a list of torch.Tensor") from None
    if -1 in devices:
        raise ValueError(f"{name} must be CUDA tensors (no CPU path)")
    if len(devices) != 1:
        raise ValueError(f"{name} must be on one device")
    dtypes = set(map(_dtype, ts))
    for d in dtypes:
        if d not in _DTYPE:
            raise TypeError(f"unsupported dtype {d} (float32 or bfloat16)")
    return ts, dtypes, devices.pop()


def _contiguous(ts):
    return ts if all(map(_T.is_contiguous, ts)) else [t.contiguous() for t in ts]


def _sizes(ts):
    return array("q", map(_T.numel, ts))


def _same_order(out, grads):
    """Every tensor of out has its gradient's shape, or is a flat piece of as many elements."""
    a, b = list(map(_shape, out)), list(map(_shape, grads))
    return a == b or all(x == y or (len(x) == 1 and x[0] == math.prod(y)) for x, y in zip(a, b))


def _run(grads, dtypes, outs, out_dtypes, sizes, max_norm, eps, scale):
    dev = grads[0].device
    norm = torch.empty((), device=dev, dtype=torch.float32)
    # ssd_grad_tensor_t: two addresses, the size, two 32-bit dtypes
    n = len(grads)
    rec = array("q", bytes(32 * n))
    rec[0::4] = array("q", map(_T.data_ptr, grads))
    rec[1::4] = rec[0::4] if outs is grads else array("q", map(_T.data_ptr, outs))
    rec[2::4] = sizes
    pairs = {(g, o): _DTYPE[g] | _DTYPE[o] << 32 for g in dtypes for o in out_dtypes}
    if len(pairs) == 1:
        rec[3::4] = array("q", pairs.values()) * n
    else:
        rec[3::4] = array("q", map(pairs.__getitem__, zip(map(_dtype, grads), map(_dtype, outs))))
    lib = _lib.load()
    addr = rec.buffer_info()[0]
    with _lib.on_device(dev):
        size = lib.ssd_clip_grad_norm_workspace_bytes(addr, n)
        ws = torch.empty(max(size, 8), device=dev, dtype=torch.uint8)
        _lib.check(lib.ssd_clip_grad_norm(addr, n, float(max_norm), float(eps), int(scale), norm.data_ptr(),
                                          ws.data_ptr(), ws.numel(), _lib.stream_of(norm)))
    return norm


def grad_norm(grads):
    """2-norm over all tensors of ``grads`` (float32 or bfloat16, any mix and shapes): a float32
    scalar tensor.  Squares are added in float32 by fours and those in float64: off by at most
    2.5 * 2^-24 of itself."""
    ts, dtypes, _ = _checked(grads, "grads")
    ts = _contiguous(ts)
    return _run(ts, dtypes, ts, dtypes, _sizes(ts), 0.0, 0.0, False)


def clip_grad_norm(grads, max_norm: float, *, eps: float = 1e-6, out=None, inplace: bool = False):
    """Scale gradients so that their global 2-norm is at most ``max_norm``.

    Returns ``(clipped, norm)``: ``grads`` times ``min(1, max_norm / (norm + eps))`` and the norm
    before clipping (a float32 scalar tensor on the device; nothing waits for it).  By default
    the clipped gradients are new tensors; ``inplace=True`` scales ``grads`` themselves, ``out``
    gives contiguous tensors of the same shapes (or flat pieces of as many elements) to write to,
    float32 or bfloat16 (bfloat16 gradients into the float32 buffers of an optimizer), none of which
    may overlap another or a gradient that is not its own.  A NaN norm makes every gradient NaN.
    Autograd does not see the writes (tensors' version counters stay).
    """
    ts, dtypes, device = _checked(grads, "grads")
    if not float(max_norm) >= 0.0 or not float(eps) >= 0.0:
        raise ValueError("max_norm and eps must be non-negative")
    sizes = _sizes(ts)
    if inplace:
        if out is not None:
            raise ValueError("give either out or inplace=True")
        if not all(map(_T.is_contiguous, ts)):
            raise ValueError("inplace=True needs contiguous gradients")
        outs, out_dtypes = ts, dtypes
    else:
        ts = _contiguous(ts)
        if out is None:
            outs, out_dtypes = [torch.empty_like(g) for g in ts], dtypes
        else:
            outs, out_dtypes, out_device = _checked(out, "out") if len(out) else ([], set(), device)
            if len(outs) != len(ts):
                raise ValueError(f"out has {len(outs)} tensors, grads {len(ts)}")
            if not _same_order(outs, ts) or not all(map(_T.is_contiguous, outs)):
                raise ValueError("out must hold contiguous tensors of grads' shapes, or flat pieces of their sizes")
            if out_device != device:
                raise ValueError("out and grads must be on one device")
    return outs, _run(ts, dtypes, outs, out_dtypes, sizes, max_norm, eps, True)
