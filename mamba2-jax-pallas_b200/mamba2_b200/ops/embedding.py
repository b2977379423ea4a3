"""Token embedding and its gradient: the first step of a language model around the mixer layers."""
from __future__ import annotations

import torch

from .. import _lib

_DTYPES = (torch.float32, torch.bfloat16)


def _pad(padding_idx, vocab: int) -> int:
    if padding_idx is None:
        return -1
    padding_idx = int(padding_idx)
    if not 0 <= padding_idx < vocab:
        raise ValueError(f"padding_idx {padding_idx} is outside [0, {vocab})")
    return padding_idx


def embedding(tokens, weight, scale: float = 1.0, *, padding_idx=None, out_dtype=None):
    """``scale * weight[tokens]``, computed in float32 and rounded once.

    tokens (...) int32 or int64; weight (vocab, dim) float32 or bfloat16.  Returns (..., dim)
    in ``out_dtype`` (default: weight's dtype).  A token outside [0, vocab) or equal to
    ``padding_idx`` gives a zero row, whatever the table holds there (torch.nn.functional.embedding
    returns the row and stops only its gradient).  The result carries no autograd history, also
    where weight requires a gradient: ``embedding_grad`` gives it.
    """
    ids = _lib.index_list(tokens, "tokens")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be a (vocab, dim) tensor")
    if not weight.is_cuda:
        raise ValueError("weight must be a CUDA tensor (no CPU path)")
    dev = weight.device
    if ids.device != dev:
        raise ValueError("tokens and weight must be on one device")
    vocab, dim = weight.shape
    if vocab == 0 or dim == 0:
        raise ValueError("weight must not be empty")
    w_code = _lib.dtype_code(weight)
    if out_dtype is None:
        out_dtype = weight.dtype
    elif out_dtype not in _DTYPES:
        raise ValueError("out_dtype must be torch.float32 or torch.bfloat16")
    w = _lib.rows2d(weight, dim)
    pad = -1 if padding_idx is None else _pad(padding_idx, vocab)
    out = weight.new_empty((*ids.shape, dim), dtype=out_dtype)
    n = ids.numel()
    if n == 0:
        return out
    p = _lib.EmbeddingParams(n, vocab, dim, _lib.row_stride(w), pad, ids.dtype is torch.int64, w_code,
                             _lib.dtype_code(out), scale, ids.data_ptr(), w.data_ptr(), out.data_ptr())
    with _lib.on_device(dev):
        _lib.check(_lib.load().ssd_embedding(p, _lib.stream_of(out)))
    return out


def embedding_grad(tokens, grad_out, num_embeddings: int, scale: float = 1.0, *, padding_idx=None, out_dtype=None,
                   accumulate_into=None):
    """Gradient of ``embedding`` with respect to its weight: (num_embeddings, dim), dense.

    tokens (...) int32 or int64 and grad_out (..., dim) float32 or bfloat16.  Row v is
    ``scale`` times the sum of grad_out over the tokens equal to v, summed in float32 by sorted
    tokens (the same bits in every run) and rounded once to ``out_dtype`` (default: grad_out's
    dtype).  With ``accumulate_into`` (a float32 or bfloat16 (num_embeddings, dim) tensor, rows
    contiguous) the sums are added to that tensor, only the named rows are touched, and it is
    returned: the tied output projection's gradient, or that of an earlier micro-batch.  Autograd
    does not see that write.
    """
    ids = _lib.index_list(tokens, "tokens")
    vocab = int(num_embeddings)
    if vocab <= 0:
        raise ValueError("num_embeddings must be positive")
    if not isinstance(grad_out, torch.Tensor) or not grad_out.is_cuda:
        raise ValueError("grad_out must be a CUDA tensor (no CPU path)")
    shape = grad_out.shape
    if len(shape) < 1 or shape[:-1] != tokens.shape:
        raise ValueError(f"grad_out {tuple(shape)} must be tokens' shape {tuple(tokens.shape)} and one axis more")
    dev = grad_out.device
    if ids.device != dev:
        raise ValueError("tokens and grad_out must be on one device")
    dim = shape[-1]
    if dim == 0:
        raise ValueError("grad_out must not have an empty last axis")
    g_code = _lib.dtype_code(grad_out)
    g = _lib.rows2d(grad_out, dim)
    if accumulate_into is not None:
        out = accumulate_into
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError("out_dtype is accumulate_into's dtype")
        if not out.is_cuda or out.device != dev:
            raise ValueError("accumulate_into must be on grad_out's device")
        if tuple(out.shape) != (vocab, dim) or (dim > 1 and out.stride(1) != 1) or (vocab > 1 and out.stride(0) < dim):
            raise ValueError(f"accumulate_into must be ({vocab}, {dim}) with contiguous rows")
        out_stride = _lib.row_stride(out)
    else:
        out_dtype = grad_out.dtype if out_dtype is None else out_dtype
        if out_dtype not in _DTYPES:
            raise ValueError("out_dtype must be torch.float32 or torch.bfloat16")
        out = g.new_empty((vocab, dim), dtype=out_dtype)
        out_stride = dim
    pad = -1 if padding_idx is None else _pad(padding_idx, vocab)
    n = ids.numel()
    p = _lib.EmbeddingGradParams(n, vocab, dim, _lib.row_stride(g), out_stride, pad, ids.dtype is torch.int64, g_code,
                                 _lib.dtype_code(out), accumulate_into is not None, scale, ids.data_ptr(), g.data_ptr(),
                                 out.data_ptr())
    if accumulate_into is not None and n == 0:
        return out
    lib = _lib.load()
    size = lib.ssd_embedding_grad_workspace_bytes(p)
    ws = g.new_empty(max(size, 1), dtype=torch.uint8)
    with _lib.on_device(dev):
        _lib.check(lib.ssd_embedding_grad(p, ws.data_ptr(), size, _lib.stream_of(out)))
    return out
