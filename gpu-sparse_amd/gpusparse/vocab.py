"""The vocabulary head of a learned sparse encoder, and the losses it is trained with.

An index holds what such an encoder answers with: a non-negative weight per
vocabulary term and text.  Its last layer is one product, hidden states times the
vocabulary's rows, ``l = hidden @ weight.T + bias``; the operators here are that
product with what follows it, without the ``[tokens, vocab]`` logits in memory:

- :func:`term_weights`: ``log(1 + relu(max of l over a text's kept tokens))``, the
  rows an index is built from and the queries it is searched with;
- :func:`vocab_loss`: softmax cross entropy over the vocabulary;
- :func:`distill_loss`: distillation from a teacher's top logits.

All three work with autograd (first derivatives, in reverse mode).  Tensors are float32, float16 or
bfloat16, hidden states and weight of one type; sums and softmaxes are in 32 bits, and
gradients of 16-bit tensors are rounded to their type.  So are a loss's gradients of 16-bit
logits before the products that make the others of them; float32 tensors keep 32 bits
throughout, at about six times the products.  Hidden states and weight may
have any strides, up to 2**28 rows (of term weights, 65535 texts), 32768 values and 2**20
terms; a 16-bit weight whose rows are 16-byte aligned and a multiple
of 64 values wide is read where it is, others are laid out once per call.  Work is queued
on the current stream of the tensors' device; results are deterministic.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._tensors import _bytes, _check_sizes, _differentiable, _on, _same_device
from .int8 import Int8Rows, _check_bias, _gpu, _refuse_gradient

C = _lib.C
REDUCTIONS = {"none": _lib.GS_REDUCE_NONE, "mean": _lib.GS_REDUCE_MEAN, "sum": _lib.GS_REDUCE_SUM}
MAX_TOP = 1024  # most teacher logits per row
SAVED_ALIGN = 256  # of what a loss saves for its gradient


def _check_head_sizes(hidden, weight):
    lead = hidden.shape[:-1]
    _check_sizes(max(lead.numel(), *lead) if lead else 1, weight.shape[1], weight.shape[0])  # a side may be long and another 0


def _check_head(hidden, weight, bias, dims: str) -> torch.device:
    for name, t in (("hidden", hidden), ("weight", weight)) + ((("bias", bias),) if bias is not None else ()):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype not in _lib.HTYPE_OF_DTYPE:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if weight.dim() != 2:
        raise ValueError(f"weight must be [vocab, dim], got {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype:
        raise ValueError(f"hidden ({hidden.dtype}) and weight ({weight.dtype}) must be of one type")
    if hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden must be {dims} with dim {weight.shape[1]}, got {tuple(hidden.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    _check_head_sizes(hidden, weight)
    dev = hidden.device
    if dev.type != "cuda":
        dev = _lib.require_gpu(dev)
    _same_device(dev, weight=weight, bias=bias)
    return dev


def _head(hidden, weight, bias) -> _lib.GsVocabHead:
    """The C struct of hidden [texts, length, dim] or [rows, dim], weight [vocab, dim] and a contiguous bias."""
    s, n = hidden.stride(), hidden.shape
    if len(n) == 2:
        s, n = (0, *s), (1, *n)
    return _lib.GsVocabHead(hidden.data_ptr(), s[0], s[1], s[2], weight.data_ptr(), weight.stride(0), weight.stride(1),
                            _lib.ptr(bias), _lib.HTYPE_OF_DTYPE[hidden.dtype],
                            _lib.GS_H_F32 if bias is None else _lib.HTYPE_OF_DTYPE[bias.dtype], n[0], n[1], n[2],
                            weight.shape[0])


def _upstream(grad: torch.Tensor) -> torch.Tensor:
    return grad if grad.dtype == torch.float32 and grad.is_contiguous() else grad.to(torch.float32).contiguous()


def _grads(ctx, hidden_shape, weight, dev):
    """Empty gradients of the inputs that need one (hidden, weight, bias)."""
    needs, vocab = ctx.needs_input_grad, weight.shape[0]
    return (torch.empty(hidden_shape, dtype=weight.dtype, device=dev) if needs[0] else None,
            torch.empty(weight.shape, dtype=weight.dtype, device=dev) if needs[1] else None,
            torch.empty(vocab, dtype=ctx.bias_dtype, device=dev) if needs[2] else None)


def _save(ctx, bias, *tensors):
    ctx.save_for_backward(*tensors)
    ctx.at = [(t.data_ptr(), t.shape, t.stride(), t.dtype) for t in tensors]
    ctx.dev = tensors[0].device
    ctx.bias_dtype = None if bias is None else bias.dtype


def _unpack(ctx):
    """The saved tensors, and whether they are where they were.  Hooks on them (offloading, packing) may bring them back at
    other addresses and in other strides, which what reads them has to bear, but not as tensors of another kind, whose memory
    the kernels would misread."""
    saved = ctx.saved_tensors
    if [(t.data_ptr(), t.shape, t.stride(), t.dtype) for t in saved] == ctx.at:
        return saved, True
    for t, (_, shape, _, dtype) in zip(saved, ctx.at):
        if (t.shape, t.dtype, t.device) != (shape, dtype, ctx.dev):
            raise RuntimeError(f"a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}, not as "
                               f"{dtype} {tuple(shape)} on {ctx.dev}")
    return saved, False


def _weights(hidden, weight, bias, mask, want_tokens: bool):
    """Weights, tokens or None, the call's head struct, and the bytes that a gradient's workspace takes."""
    dev = hidden.device
    texts, vocab = hidden.shape[0], weight.shape[0]
    weights = torch.empty((texts, vocab), dtype=torch.float32, device=dev)
    tokens = torch.empty((texts, vocab), dtype=torch.int32, device=dev) if want_tokens else None
    L, head = _lib.lib(), _head(hidden, weight, bias)
    need, grad_need = C.c_size_t(), C.c_size_t()
    with _on(dev):
        _lib.check(L.gs_term_weights_workspace(C.byref(head), want_tokens, C.byref(need), C.byref(grad_need)),
                   "gs_term_weights_workspace")
        ws = _bytes(need.value, dev)
        _lib.check(L.gs_term_weights(C.byref(head), _lib.ptr(mask), weights.data_ptr(), _lib.ptr(tokens), ws.data_ptr(),
                                     need.value, _lib.stream_ptr(dev)), "gs_term_weights")
    return weights, tokens, head, grad_need.value


class _TermWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, mask):
        weights, tokens, ctx.head, ctx.grad_bytes = _weights(hidden, weight, bias, mask, True)
        _save(ctx, bias, hidden, weight, weights, tokens)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(tokens)
        return weights, tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return None, None, None, None
        (hidden, weight, weights, tokens), still = _unpack(ctx)
        head = ctx.head
        if not still:
            weights, tokens = weights.contiguous(), tokens.contiguous()
            head = _moved(head, weight)
            head.hidden_d = hidden.data_ptr()
            head.hidden_text_stride, head.hidden_row_stride, head.hidden_dim_stride = hidden.stride()
        dev = ctx.dev
        dh, dw, db = _grads(ctx, hidden.shape, weight, dev)
        L, grad = _lib.lib(), _upstream(grad)
        with _on(dev):
            ws = _bytes(ctx.grad_bytes, dev)
            _lib.check(L.gs_term_weights_grad(C.byref(head), grad.data_ptr(), weights.data_ptr(), tokens.data_ptr(),
                                              _lib.ptr(dh), _lib.ptr(dw), _lib.ptr(db), ws.data_ptr(), ws.numel(),
                                              _lib.stream_ptr(dev)), "gs_term_weights_grad")
        return dh, dw, db, None


def _weights8(hidden, weight, bias, mask):
    dev = hidden.device
    weights = torch.empty((hidden.shape[0], weight.shape[0]), dtype=torch.float32, device=dev)
    L, head, need = _lib.lib(), _head(hidden, weight.values, bias), C.c_size_t()
    with _on(dev):
        _lib.check(L.gs_term_weights8_workspace(C.byref(head), C.byref(need)), "gs_term_weights8_workspace")
        ws = _bytes(need.value, dev) if need.value else None
        _lib.check(L.gs_term_weights8(C.byref(head), weight.scales.data_ptr(), _lib.ptr(mask), weights.data_ptr(), _lib.ptr(ws),
                                      need.value, _lib.stream_ptr(dev)), "gs_term_weights8")
    return weights


def _check_head8(hidden, weight, bias) -> torch.device:
    if hidden.dtype not in _lib.HTYPE_OF_DTYPE:
        raise ValueError(f"hidden must be float32, float16 or bfloat16, got {hidden.dtype}")
    if hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden must be [texts, length, dim] with dim {weight.shape[1]}, got {tuple(hidden.shape)}")
    _check_bias(bias, weight.shape[0])
    _check_head_sizes(hidden, weight)
    dev = hidden.device
    if dev.type != "cuda" or weight.values.device != dev or (bias is not None and bias.device != dev):
        dev = _gpu(hidden, "hidden", weight=weight, bias=bias)
    return dev


def term_weights(hidden, weight, bias=None, *, mask=None, return_tokens: bool = False):
    """Term weights of texts from an encoder's hidden states: float32 [texts, vocab],
    ``log(1 + relu(max over the text's kept tokens of hidden @ weight.T + bias))``.

    hidden: [texts, length, dim].  weight: [vocab, dim], or :class:`gpusparse.Int8Rows` of it: then the kept hidden states
    are taken in 8 bits as well, and there is neither a gradient nor return_tokens.  bias: [vocab] or None.
    mask: [texts, length], nonzero for the tokens that count (None: all do); the hidden
    states of the others are never read, and a text without any has weights 0.
    return_tokens: also the int32 [texts, vocab] lowest token that reaches the maximum
    (compared before the bias is added; -1 where the weight is 0), through which the gradient
    flows.  A NaN is the maximum of its text: the weight is NaN, and the gradient where it flows."""
    if not isinstance(hidden, torch.Tensor) or hidden.dim() != 3:
        raise ValueError("hidden must be [texts, length, dim]")
    q8 = isinstance(weight, Int8Rows)
    if q8 and return_tokens:
        raise ValueError("return_tokens goes with the gradient, which a vocabulary in 8 bits does not have")
    dev = _check_head8(hidden, weight, bias) if q8 else _check_head(hidden, weight, bias, "[texts, length, dim]")
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or tuple(mask.shape) != tuple(hidden.shape[:2]):
            raise ValueError(f"mask must be a tensor of shape {tuple(hidden.shape[:2])}")
        _same_device(dev, mask=mask)
        if mask.dtype not in (torch.bool, torch.uint8):
            mask = mask != 0
        mask = mask.contiguous()
    bias = None if bias is None else bias.contiguous()
    if q8:
        _refuse_gradient(hidden, bias)
        return _weights8(hidden, weight, bias, mask)
    if _differentiable(hidden, weight, bias):
        weights, tokens = _TermWeights.apply(hidden, weight, bias, mask)
    else:
        weights, tokens, _, _ = _weights(hidden, weight, bias, mask, bool(return_tokens))
    return (weights, tokens) if return_tokens else weights


def _losses(hidden, weight, bias, ids, logits, ignore_index, temperature, reduction):
    """The loss, what a gradient reads of the call (head and targets structs, saved bytes) and the bytes its workspace takes."""
    dev = hidden.device
    head = _head(hidden, weight, bias)
    if logits is None:
        targets = _lib.GsVocabTargets(_lib.ptr(ids), ignore_index, None, None, _lib.GS_H_F32, 0, 1.0)
    else:
        targets = _lib.GsVocabTargets(None, 0, _lib.ptr(ids), logits.data_ptr(), _lib.HTYPE_OF_DTYPE[logits.dtype],
                                      logits.shape[1], temperature)
    shape = (hidden.shape[0],) if reduction == _lib.GS_REDUCE_NONE else ()
    loss = torch.empty(shape, dtype=torch.float32, device=dev)
    L = _lib.lib()
    need, scratch, grad_need = C.c_size_t(), C.c_size_t(), C.c_size_t()
    with _on(dev):
        _lib.check(L.gs_vocab_loss_workspace(C.byref(head), C.byref(targets), C.byref(need), C.byref(scratch),
                                             C.byref(grad_need)), "gs_vocab_loss_workspace")
        saved, ws = _bytes(need.value, dev), _bytes(scratch.value, dev)
        _lib.check(L.gs_vocab_loss(C.byref(head), C.byref(targets), reduction, loss.data_ptr(), saved.data_ptr(),
                                   need.value, ws.data_ptr(), scratch.value, _lib.stream_ptr(dev)), "gs_vocab_loss")
    return loss, head, targets, saved, grad_need.value


def _moved(head, weight):
    """The head with its weight where it is now."""
    head = _lib.GsVocabHead.from_buffer_copy(head)
    head.weight_d, head.weight_row_stride, head.weight_dim_stride = weight.data_ptr(), weight.stride(0), weight.stride(1)
    return head


def _as_loss_read_it(head, weight, targets, saved_bytes):
    """The head and the weight, moved, as a gradient can read it: where it is, or from the copy among the saved bytes; where the
    loss made no copy and the weight came back in another layout, a contiguous one, as it was then."""
    need, other = C.c_size_t(), C.c_size_t()
    head = _moved(head, weight)
    with _on(weight.device):
        _lib.check(_lib.lib().gs_vocab_loss_workspace(C.byref(head), C.byref(targets), C.byref(need), C.byref(other),
                                                      C.byref(other)), "gs_vocab_loss_workspace")
    if need.value > saved_bytes:
        weight = weight.clone(memory_format=torch.contiguous_format)
        head = _moved(head, weight)
    return head, weight


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, ids, logits, ignore_index, temperature, reduction):
        loss, ctx.head, ctx.targets, saved, ctx.grad_bytes = _losses(hidden, weight, bias, ids, logits, ignore_index,
                                                                     temperature, reduction)
        # not the hidden states, nor the targets: what backward reads of them is among the saved bytes
        _save(ctx, bias, weight, saved)
        ctx.hidden_shape = hidden.shape
        ctx.reduction = reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (weight, saved), still = _unpack(ctx)
        head = ctx.head
        if not still:
            if saved.data_ptr() % SAVED_ALIGN or not saved.is_contiguous():
                saved = saved.clone(memory_format=torch.contiguous_format)
            head, weight = _as_loss_read_it(head, weight, ctx.targets, saved.numel())
        dev = ctx.dev
        dh, dw, db = _grads(ctx, ctx.hidden_shape, weight, dev)
        L, grad = _lib.lib(), _upstream(grad)
        with _on(dev):
            ws = _bytes(ctx.grad_bytes, dev)
            _lib.check(L.gs_vocab_loss_grad(C.byref(head), C.byref(ctx.targets), ctx.reduction, grad.data_ptr(),
                                            saved.data_ptr(), saved.numel(), _lib.ptr(dh), _lib.ptr(dw), _lib.ptr(db),
                                            ws.data_ptr(), ws.numel(), _lib.stream_ptr(dev)), "gs_vocab_loss_grad")
        return dh, dw, db, None, None, None, None, None


def _loss(hidden, weight, bias, ids, logits, ignore_index, temperature, reduction):
    lead = hidden.shape[:-1]
    bias = None if bias is None else bias.contiguous()
    rows = hidden if len(lead) == 1 else hidden.reshape(lead.numel(), hidden.shape[-1])  # a view is one more gradient
    args = (rows, weight, bias, ids, logits, ignore_index, temperature, REDUCTIONS[reduction])
    out = _VocabLoss.apply(*args) if _differentiable(hidden, weight, bias) else _losses(*args)[0]
    return out.reshape(lead) if reduction == "none" and len(lead) != 1 else out


def _check_rows(hidden, reduction):
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    if not isinstance(hidden, torch.Tensor) or hidden.dim() < 1:
        raise ValueError("hidden must be [..., dim]")


def _ids(t, shape, what, dev):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what} must be an int64 or int32 tensor")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(t.shape)}")
    _same_device(dev, **{what: t})
    return t.to(torch.int64).contiguous()


def vocab_loss(hidden, weight, targets, bias=None, *, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of ``hidden @ weight.T + bias`` over the vocabulary, without the logits.

    hidden: [..., dim]; targets: [...] int64 or int32 term ids.  A row whose target is
    ignore_index or outside the vocabulary is left out: its loss and gradient are 0, it does
    not count in the mean, and its hidden state is never read.  reduction: "mean" over the rows
    that count (0 when none does), "sum", or "none" (a loss per row).  float32."""
    _check_rows(hidden, reduction)
    dev = _check_head(hidden, weight, bias, "[..., dim]")
    ids = _ids(targets, hidden.shape[:-1], "targets", dev)
    return _loss(hidden, weight, bias, ids, None, int(ignore_index), 1.0, reduction)


def distill_loss(hidden, weight, teacher_ids, teacher_logits, bias=None, *, temperature: float = 1.0,
                 reduction: str = "mean"):
    """Distillation from a teacher's top logits: ``temperature**2 * sum_k q_k (log q_k - log p[id_k])``
    with ``q = softmax(teacher_logits / temperature)`` over a row's ids and
    ``p = softmax(l / temperature)`` over the whole vocabulary, l = hidden @ weight.T + bias
    never in memory.

    hidden: [..., dim]; teacher_ids: [..., top] int64 or int32, teacher_logits: [..., top]
    (float32, float16 or bfloat16), top <= 1024.  Ids outside the vocabulary (padding) are
    skipped, equal ids add up; a row without any other id is left out as in :func:`vocab_loss`.
    The teacher gets no gradient."""
    _check_rows(hidden, reduction)
    dev = _check_head(hidden, weight, bias, "[..., dim]")
    if not isinstance(teacher_logits, torch.Tensor) or teacher_logits.dtype not in _lib.HTYPE_OF_DTYPE:
        raise ValueError("teacher_logits must be a float32, float16 or bfloat16 tensor")
    if teacher_logits.dim() != hidden.dim() or teacher_logits.shape[:-1] != hidden.shape[:-1]:
        raise ValueError(f"teacher_logits must be {tuple(hidden.shape[:-1])} + (top,), got {tuple(teacher_logits.shape)}")
    top = teacher_logits.shape[-1]
    if not 1 <= top <= MAX_TOP:
        raise ValueError(f"{top} teacher logits per row: 1 to {MAX_TOP} are supported")
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    ids = _ids(teacher_ids, teacher_logits.shape, "teacher_ids", dev)
    _same_device(dev, teacher_logits=teacher_logits)
    logits = teacher_logits.detach().reshape(ids.numel() // top, top).contiguous()
    return _loss(hidden, weight, bias, ids.reshape(ids.numel() // top, top), logits, 0, float(temperature), reduction)
