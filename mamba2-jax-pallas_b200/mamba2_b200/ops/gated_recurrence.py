"""A gated linear recurrence per channel, its gradient and its single-token step: a sequence mixer that
trains, beside the SSD scan (``mamba_chunk_scan_combined_fwd``) and its step (``selective_state_update``)."""
from __future__ import annotations

import torch

from .. import _lib

_TILE = 32   # SSD_GATED_RECURRENCE_CHECKPOINT
_F32 = torch.float32


def _channels_last(t):
    """A view whose channels are contiguous, else a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _inputs(x, decay_gate, input_gate, decay, scale, dims):
    if not (isinstance(x, torch.Tensor) and isinstance(decay_gate, torch.Tensor) and
            isinstance(input_gate, torch.Tensor) and isinstance(decay, torch.Tensor)):
        raise TypeError("x, decay_gate, input_gate and decay must be torch.Tensors")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (no CPU path)")
    shape, dtype, dev = x.shape, x.dtype, x.device
    if len(shape) != dims or shape[-1] == 0:
        raise ValueError(f"x must be {'(batch, seqlen, dim)' if dims == 3 else '(batch, dim)'}, with channels")
    if decay_gate.shape != shape or input_gate.shape != shape:
        raise ValueError(f"decay_gate {tuple(decay_gate.shape)} and input_gate {tuple(input_gate.shape)} must have x's "
                         f"shape {tuple(shape)}")
    if decay_gate.dtype is not dtype or input_gate.dtype is not dtype:
        raise TypeError(f"decay_gate ({decay_gate.dtype}), input_gate ({input_gate.dtype}) and x ({dtype}) must have the "
                        "same dtype")
    if decay.shape != shape[-1:]:
        raise ValueError("decay must be (dim,)")
    if not dev == decay_gate.device == input_gate.device == decay.device:
        raise ValueError("decay_gate, input_gate and decay must be on x's device")
    if not 0 <= scale <= 3.4e38:
        raise ValueError("scale must be finite and not negative")
    if decay.dtype is not _F32 or not decay.is_contiguous():
        decay = decay.to(_F32).contiguous()
    return _lib.dtype_code(x), _channels_last(x), _channels_last(decay_gate), _channels_last(input_gate), decay


def _like(x):
    """A new contiguous tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _state(t, name, x):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.shape != (x.shape[0], x.shape[-1]):
        raise ValueError(f"{name} must be a (batch, dim) tensor on x's device")
    return t if t.dtype is _F32 and t.is_contiguous() else t.to(_F32).contiguous()


def _ids(seq_idx, x):
    if seq_idx is None:
        return None
    ids = _lib.index_list(seq_idx, "seq_idx")
    if ids.shape != x.shape[:2] or ids.device != x.device:
        raise ValueError("seq_idx must be (batch, seqlen) on x's device")
    if ids.dtype is torch.int32 or not ids.numel():
        return ids.to(torch.int32)
    # only where neighbours differ counts, and wider ids need not fit 32 bits
    seq = ids.new_zeros(ids.shape, dtype=torch.int32)
    torch.cumsum(ids[:, 1:] != ids[:, :-1], 1, dtype=torch.int32, out=seq[:, 1:])
    return seq


def _checkpoint_shape(x):
    return (x.shape[0], -(-x.shape[1] // _TILE), x.shape[2])


def _params(code, x, decay_gate, input_gate, decay, scale, *optional):
    ptrs = [None if t is None else t.data_ptr() for t in optional]
    return _lib.GatedRecurrenceParams(*x.shape, *x.stride()[:2], *decay_gate.stride()[:2], *input_gate.stride()[:2], code,
                                      scale, x.data_ptr(), decay_gate.data_ptr(), input_gate.data_ptr(), decay.data_ptr(),
                                      *ptrs)


def gated_recurrence(x, decay_gate, input_gate, decay, *, scale: float = 8.0, initial_state=None, seq_idx=None,
                     return_final_state: bool = False, return_checkpoints: bool = False, check_status: bool = False):
    """``h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t`` along the sequence, per channel, with
    ``a_t = exp(-scale softplus(decay) sigmoid(decay_gate_t))``.

    x, decay_gate and input_gate (batch, seqlen, dim) of one dtype, float32 or bfloat16, at any
    strides with contiguous channels (others are copied); decay (dim,); initial_state (batch, dim) or
    None for zeros; seq_idx (batch, seqlen) int32 or int64: a packed sequence starts where the id
    differs from the token before, and takes nothing of what came before (initial_state belongs to the first).
    Returns h (batch, seqlen, dim) in x's dtype, computed in float32 and rounded once; with
    ``return_final_state`` also the float32 state after the last token (batch, dim); with
    ``return_checkpoints`` also the float32 states that ``gated_recurrence_grad`` starts from,
    (batch, ceil(seqlen / 32), dim), which saves it a pass over the inputs.  A value that is
    not finite makes its channel so up to the next sequence.  ``check_status`` waits for the call and raises
    ``SsdError`` if a bounded wait inside a kernel gave up (unchecked, the channels concerned are NaN).  The
    results carry no autograd history.
    """
    code, xs, r, i, lam = _inputs(x, decay_gate, input_gate, decay, scale, 3)
    h0, ids = _state(initial_state, "initial_state", x), _ids(seq_idx, x)
    b, L, d = x.shape
    y = _like(xs)
    final = xs.new_empty((b, d), dtype=_F32) if return_final_state else None
    points = xs.new_empty(_checkpoint_shape(x), dtype=_F32) if return_checkpoints else None
    if b and L:
        status = xs.new_zeros(64, dtype=torch.int32) if check_status else None
        p = _params(code, xs, r, i, lam, scale, h0, ids, y, final, points, status)
        with _lib.on_device(x.device):
            _lib.check(_lib.load().ssd_gated_recurrence(p, _lib.stream_of(y)))
            if check_status:
                _lib.check_device_status(status)
    elif final is not None:
        final.zero_() if h0 is None else final.copy_(h0)
    if not (return_final_state or return_checkpoints):
        return y
    return (y,) + ((final,) if return_final_state else ()) + ((points,) if return_checkpoints else ())


def gated_recurrence_grad(x, decay_gate, input_gate, decay, grad_out, *, scale: float = 8.0, initial_state=None,
                          seq_idx=None, grad_final_state=None, checkpoints=None, check_status: bool = False):
    """Gradients of ``gated_recurrence``: ``(grad_x, grad_decay_gate, grad_input_gate, grad_decay,
    grad_initial_state)``.

    grad_out (batch, seqlen, dim) in x's dtype is the gradient that reaches h, grad_final_state
    (batch, dim) that of the final state (None for none).  The other arguments are those of the
    forward call; ``checkpoints`` what it returned with ``return_checkpoints`` (None: computed again, by one
    more pass over x and the gates).  The first three results have x's dtype, rounded once from float32;
    grad_decay (dim,) is float32, summed in a fixed order, so that equal calls give equal bits;
    grad_initial_state (batch, dim) is float32, or None where initial_state is.
    """
    code, xs, r, i, lam = _inputs(x, decay_gate, input_gate, decay, scale, 3)
    h0, ids = _state(initial_state, "initial_state", x), _ids(seq_idx, x)
    gf = _state(grad_final_state, "grad_final_state", x)
    if not isinstance(grad_out, torch.Tensor) or grad_out.shape != x.shape or grad_out.device != x.device:
        raise ValueError(f"grad_out must be a {tuple(x.shape)} tensor on x's device")
    if grad_out.dtype != x.dtype:
        raise TypeError(f"grad_out ({grad_out.dtype}) and x ({x.dtype}) must have the same dtype")
    if checkpoints is not None and (not isinstance(checkpoints, torch.Tensor) or checkpoints.dtype != _F32 or
                                    tuple(checkpoints.shape) != _checkpoint_shape(x) or checkpoints.device != x.device):
        raise ValueError(f"checkpoints must be the float32 {_checkpoint_shape(x)} tensor that gated_recurrence returned")
    g = _channels_last(grad_out)
    b, L, d = x.shape
    gx, gr, gi = _like(xs), _like(xs), _like(xs)
    gd = xs.new_empty(d, dtype=_F32)
    gh = xs.new_empty((b, d), dtype=_F32) if h0 is not None else None
    if not (b and L):
        gd.zero_()
        if gh is not None:
            gh.zero_() if gf is None else gh.copy_(gf)
        return gx, gr, gi, gd, gh
    points = None if checkpoints is None else checkpoints.contiguous()
    status = xs.new_zeros(64, dtype=torch.int32) if check_status else None
    p = _params(code, xs, r, i, lam, scale, h0, ids, None, None, points, status)
    q = _lib.GatedRecurrenceGrads(g.stride(0), g.stride(1), g.data_ptr(), _lib.ptr(gf), gx.data_ptr(), gr.data_ptr(),
                                  gi.data_ptr(), gd.data_ptr(), _lib.ptr(gh))
    lib = _lib.load()
    with _lib.on_device(x.device):
        ws = xs.new_empty(lib.ssd_gated_recurrence_grad_workspace_bytes(p), dtype=torch.uint8)
        _lib.check(lib.ssd_gated_recurrence_grad(p, q, ws.data_ptr(), ws.numel(), _lib.stream_of(gx)))
        if check_status:
            _lib.check_device_status(status)
    return gx, gr, gi, gd, gh


def gated_recurrence_update(state, x, decay_gate, input_gate, decay, *, scale: float = 8.0, inplace: bool = False):
    """One token of ``gated_recurrence``.  Returns ``(new_state, h)``.

    state (batch, dim) float32; x, decay_gate and input_gate (batch, dim); h has x's dtype.  The given state
    stays as it is; with ``inplace=True`` it is updated itself (it must be contiguous) and returned.
    """
    if not isinstance(state, torch.Tensor) or state.dtype != _F32:
        raise TypeError("state must be a float32 tensor")
    code, xs, r, i, lam = _inputs(x, decay_gate, input_gate, decay, scale, 2)
    if state.shape != x.shape or state.device != x.device:
        raise ValueError("state must be (batch, dim) on x's device")
    b, d = x.shape
    old = state
    if not state.is_contiguous():
        if inplace:
            raise ValueError("inplace=True needs a contiguous state")
        old = state.contiguous()
    new = state if inplace else torch.empty_like(old)
    y = _like(xs)
    if b:
        p = _lib.GatedRecurrenceUpdateParams(b, d, xs.stride(0), r.stride(0), i.stride(0), code, scale, xs.data_ptr(),
                                             r.data_ptr(), i.data_ptr(), lam.data_ptr(), old.data_ptr(), new.data_ptr(),
                                             y.data_ptr())
        with _lib.on_device(x.device):
            _lib.check(_lib.load().ssd_gated_recurrence_update(p, _lib.stream_of(y)))
    return new, y
