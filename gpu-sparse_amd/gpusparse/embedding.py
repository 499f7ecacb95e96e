"""The encoder's first layer: rows of the vocabulary by token id, and their gradient.

The matrix is the one that the vocabulary head multiplies with (:mod:`gpusparse.vocab`), where both are tied: autograd adds
their gradients.  It may be in 8 bits for serving (:class:`gpusparse.Int8Rows`).  Work is queued on the current stream of
the weight's device.  What autograd records is a node in C++ (csrc/gs_autograd.cpp).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._tensors import _beyond_reverse_mode, _check_sizes, _on
from .int8 import Int8Rows, _gpu, _refuse_gradient

C = _lib.C
MAX_SCALE = torch.finfo(torch.float32).max
FEW_TOKENS = 1024  # whose gradient takes no workspace


def _lookup8(ids, weight, scale: float):
    vocab, dim = weight.values.shape
    dev = weight.values.device
    out = weight.values.new_empty((*ids.shape, dim), dtype=weight.dtype)
    row, value = weight.values.stride()
    a = _lib.GsLookup(ids.data_ptr(), weight.values.data_ptr(), weight.scales.data_ptr(), row, value, ids.numel(), -1, ids.element_size(),
                      _lib.GS_H_I8, _lib.HTYPE_OF_DTYPE[weight.dtype], vocab, dim, scale)
    with _on(dev):
        _lib.check(_lib.lib().gs_embed_tokens(C.byref(a), out.data_ptr(), _lib.stream_ptr(dev)), "gs_embed_tokens")
    return out


class _Embed(torch.autograd.Function):
    """For what knows functions of Python alone: a trace, which records this one, and dual tensors and functional transforms, which
    refuse it."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        ctx.save_for_backward(ids)
        ctx.call = ids.shape, ids.dtype, weight.device, weight.shape[0], scale, padding
        return _lib.autograd().embed_tokens(ids, weight, scale, padding)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        shape, dtype, dev, vocab, scale, padding = ctx.call
        if (ids.shape, ids.dtype, ids.device) != (shape, dtype, dev):  # hooks on saved tensors may move them, no more
            raise RuntimeError(f"the saved ids came back as {ids.dtype} {tuple(ids.shape)} on {ids.device}")
        return None, _lib.autograd().embed_tokens_grad(ids.contiguous(), grad, vocab, scale, padding), None, None


def embed_tokens(ids, weight, *, scale: float = 1.0, padding_idx: int | None = None):
    """``scale * weight[ids]``: [..., dim] of weight's type from ids [...] (int64 or int32) and weight [vocab, dim].

    An id outside [0, vocab) is padding: zeros, and no gradient.  padding_idx: an id of the vocabulary whose row is looked up
    but gets no gradient.  weight: float32, float16 or bfloat16 with any strides, or :class:`gpusparse.Int8Rows`, whose rows come
    out in its ``dtype`` and which has no gradient.  The gradient (first derivatives, in reverse mode) is summed in 32 bits over
    the tokens sorted by id: the same call gives the same bits.  Up to 2**28 tokens, 32768 values and 2**20 rows."""
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int64, torch.int32):
        raise ValueError("ids must be an int64 or int32 tensor")
    q8 = isinstance(weight, Int8Rows)
    if not q8:
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
            raise ValueError("weight must be a tensor [vocab, dim] or Int8Rows")
        if weight.dtype not in _lib.HTYPE_OF_DTYPE:
            raise ValueError(f"weight must be float32, float16 or bfloat16, got {weight.dtype}")
    scale = float(scale)
    if not abs(scale) <= MAX_SCALE:
        raise ValueError(f"scale must be finite in float32, got {scale}")
    vocab, dim = weight.shape
    padding = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None and not 0 <= padding < vocab:
        raise ValueError(f"padding_idx must be in [0, {vocab}), got {padding_idx}")
    _check_sizes(ids.numel(), dim, vocab)
    if not ids.is_cuda or weight.device != ids.device:
        _gpu(weight, "weight", ids=ids)
    ids = ids.contiguous()
    if q8:
        _refuse_gradient()
        return _lookup8(ids, weight, scale)
    if _beyond_reverse_mode():
        return _Embed.apply(ids, weight, scale, padding)
    return _lib.autograd().embed_tokens(ids, weight, scale, padding)
