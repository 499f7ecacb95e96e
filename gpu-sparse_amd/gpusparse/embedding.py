"""The encoder's first layer: rows of the vocabulary by token id, and their gradient.

The matrix is the one that the vocabulary head multiplies with (:mod:`gpusparse.vocab`), where both are tied: autograd adds
their gradients.  It may be in 8 bits for serving (:class:`gpusparse.Int8Rows`).  Work is queued on the current stream of
the weight's device.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._tensors import _bytes, _check_sizes, _differentiable, _on
from .int8 import Int8Rows, _gpu, _refuse_gradient

C = _lib.C
MAX_SCALE = torch.finfo(torch.float32).max
FEW_TOKENS = 1024  # whose gradient takes no workspace


def _lookup(ids, weight, scale: float, padding: int):
    """The rows, and the C struct of the call."""
    if isinstance(weight, Int8Rows):
        table, scales, wtype = weight.values, weight.scales.data_ptr(), _lib.GS_H_I8
    else:
        table, scales, wtype = weight, None, _lib.HTYPE_OF_DTYPE[weight.dtype]
    vocab, dim = table.shape
    dev = table.device
    out = table.new_empty((*ids.shape, dim), dtype=weight.dtype)
    row, value = table.stride()
    a = _lib.GsLookup(ids.data_ptr(), table.data_ptr(), scales, row, value, ids.numel(), padding, ids.element_size(), wtype,
                      _lib.HTYPE_OF_DTYPE[weight.dtype], vocab, dim, scale)
    with _on(dev):
        _lib.check(_lib.lib().gs_embed_tokens(C.byref(a), out.data_ptr(), _lib.stream_ptr(dev)), "gs_embed_tokens")
    return out, a


def _gradient(ctx, grad):
    ids, = ctx.saved_tensors
    a, dev = ctx.lookup, ctx.dev
    if (ids.data_ptr(), ids.shape, ids.stride(), ids.dtype) != ctx.at:  # hooks on saved tensors may move them, no more
        if (ids.shape, ids.dtype, ids.device) != (ctx.at[1], ctx.at[3], dev):
            raise RuntimeError(f"the saved ids came back as {ids.dtype} {tuple(ids.shape)} on {ids.device}")
        ids = ids.contiguous()
        a = _lib.GsLookup.from_buffer_copy(a)
        a.ids_d = ids.data_ptr()
    row = a.dim
    if not grad.is_contiguous():
        grad = grad.reshape(-1, a.dim)
        if grad.stride(1) != 1:
            grad = grad.contiguous()
        row = grad.stride(0)
    dw = grad.new_empty((a.vocab, a.dim))
    ws = _bytes(ctx.grad_bytes, dev) if ctx.grad_bytes else None
    with _on(dev):
        _lib.check(_lib.lib().gs_embed_tokens_grad(C.byref(a), grad.data_ptr(), row, dw.data_ptr(), _lib.ptr(ws), ctx.grad_bytes,
                                                   _lib.stream_ptr(dev)), "gs_embed_tokens_grad")
    return None, dw, None, None


_gradient_once = once_differentiable(_gradient)


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        out, ctx.lookup = _lookup(ids, weight, scale, padding)
        ctx.grad_bytes = 0
        if ids.numel() > FEW_TOKENS:
            need = C.c_size_t()
            _lib.check(_lib.lib().gs_embed_tokens_grad_workspace(C.byref(ctx.lookup), C.byref(need)), "gs_embed_tokens_grad_workspace")
            ctx.grad_bytes = need.value
        ctx.save_for_backward(ids)
        ctx.at = (ids.data_ptr(), ids.shape, ids.stride(), ids.dtype)
        ctx.dev = out.device
        return out

    @staticmethod
    def backward(ctx, grad):
        # what refuses a second derivative has nothing to do where none can be asked for (4 us)
        return _gradient_once(ctx, grad) if torch.is_grad_enabled() else _gradient(ctx, grad)


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
    if padding_idx is not None and not 0 <= int(padding_idx) < weight.shape[0]:
        raise ValueError(f"padding_idx must be in [0, {weight.shape[0]}), got {padding_idx}")
    _check_sizes(ids.numel(), weight.shape[1], weight.shape[0])
    dev = ids.device
    if dev.type != "cuda" or weight.device != dev:
        _gpu(weight, "weight", ids=ids)
    padding = -1 if padding_idx is None else int(padding_idx)
    ids = ids.contiguous()
    if q8:
        _refuse_gradient()
    elif _differentiable(weight):
        return _Embed.apply(ids, weight, scale, padding)
    return _lookup(ids, weight, scale, padding)[0]
