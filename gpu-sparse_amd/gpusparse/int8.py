"""Rows in 8 bits, and products with them: weights as a serving encoder keeps them.

A row is kept as whole numbers of -127 .. 127 and one float32 scale: ``values = nearest(127 * x / max|x|)`` (ties to even),
``scale = max|x| / 127``, :class:`Int8Rows`.  What multiplies with such rows takes each token's hidden state in 8 bits as
well, within the call: sums are exact whole numbers, and the two scales and a bias come in at the end, in 32 bits.

- :func:`quantize_rows`: a weight's rows in 8 bits;
- :func:`int8_linear`: a linear layer with such a weight;
- :func:`gpusparse.term_weights` and :func:`gpusparse.embed_tokens` take a vocabulary in 8 bits.

A row with an infinity or a NaN has scale NaN, and what is made from it is NaN; a row whose largest magnitude is below
2**-94 counts as zeros.  There is no gradient: calls that autograd would record are refused.  Work is queued on the
current stream of the tensors' device.
"""
from __future__ import annotations

import torch

from . import _lib
from ._tensors import _bytes, _check_sizes, _differentiable, _on, _same_device

C = _lib.C
PAD = 128  # bytes that 8-bit rows are padded to
MAX_STRIDE = 1 << 20  # rows lie nearer than this, in bytes


def _padded(rows: int, dim: int, device) -> torch.Tensor:
    """Memory for 8-bit rows, zeros."""
    return torch.zeros((rows, -(-dim // PAD) * PAD), dtype=torch.int8, device=device)


def _in_place(values: torch.Tensor) -> bool:
    """Whether 8-bit rows can be read where they are: each starts 16-byte aligned, may be read up to its padding's end, and
    lies as near to the next as the kernels' offsets reach."""
    rows, dim = values.shape
    width = -(-dim // PAD) * PAD
    if values.stride(1) != 1 or values.stride(0) % PAD or not width <= values.stride(0) < MAX_STRIDE or values.data_ptr() % 16:
        return False
    return values.storage_offset() + (rows - 1) * values.stride(0) + width <= values.untyped_storage().nbytes()


class Int8Rows:
    """A matrix [rows, dim] in 8 bits: ``values`` int8 [rows, dim], ``scales`` float32 [rows], and ``dtype``, the type it
    came from, which lookups give back.  Scales may have either sign; a gradient that they ask for is left out.  Values
    that are not laid out as the kernels read them (rows padded to 128 bytes, less than 2**20 bytes apart) are copied once, here."""

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        if not isinstance(values, torch.Tensor) or values.dtype != torch.int8 or values.dim() != 2:
            raise ValueError("values must be an int8 tensor [rows, dim]")
        if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or tuple(scales.shape) != (values.shape[0],):
            raise ValueError(f"scales must be float32 [{values.shape[0]}]")
        if dtype not in _lib.HTYPE_OF_DTYPE:
            raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        if values.shape[1] < 1:
            raise ValueError("values must have at least one column")
        _same_device(values.device, "values", scales=scales)
        if not _in_place(values):
            padded = _padded(*values.shape, values.device)[:, : values.shape[1]]
            padded.copy_(values)
            values = padded
        self.values, self.scales, self.dtype = values, scales.detach().contiguous(), dtype

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def to(self, device) -> "Int8Rows":
        return Int8Rows(self.values.to(device), self.scales.to(device), self.dtype)

    def dequantize(self) -> torch.Tensor:
        """The values that the rows stand for, of ``dtype``."""
        return (self.values.float() * self.scales[:, None]).to(self.dtype)

    def __repr__(self) -> str:
        return f"Int8Rows({tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def _refuse_gradient(*inputs):
    if _differentiable(*inputs):
        raise ValueError("8-bit rows have no gradient, and calls with them no trace: call under torch.no_grad(), or with "
                         "detached tensors")


def _gpu(t, name: str, **others) -> torch.device:
    """The GPU that a call runs on, which is t's; refuses tensors that are elsewhere."""
    dev = t.device
    if dev.type != "cuda":
        dev = _lib.require_gpu(dev)
    _same_device(dev, name, **others)
    return dev


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """The rows of x [rows, dim] (float32, float16 or bfloat16, any strides) in 8 bits.  No gradient flows through it."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.dtype not in _lib.HTYPE_OF_DTYPE:
        raise ValueError("x must be a float32, float16 or bfloat16 tensor [rows, dim]")
    if x.shape[1] < 1:
        raise ValueError("x must have at least one column")
    _check_sizes(*x.shape)
    dev = _gpu(x, "x")
    x = x.detach()
    values = torch.empty((x.shape[0], -(-x.shape[1] // PAD) * PAD), dtype=torch.int8, device=dev)
    scales = torch.empty(x.shape[0], dtype=torch.float32, device=dev)
    with _on(dev):
        _lib.check(_lib.lib().gs_quantize_rows(x.data_ptr(), _lib.HTYPE_OF_DTYPE[x.dtype], x.shape[0], x.shape[1], x.stride(0),
                                               x.stride(1), values.data_ptr(), values.stride(0), scales.data_ptr(),
                                               _lib.stream_ptr(dev)), "gs_quantize_rows")
    return Int8Rows(values[:, : x.shape[1]], scales, x.dtype)


def _check_bias(bias, n: int):
    if bias is None:
        return
    if not isinstance(bias, torch.Tensor) or bias.dtype not in _lib.HTYPE_OF_DTYPE:
        raise ValueError("bias must be a float32, float16 or bfloat16 tensor")
    if tuple(bias.shape) != (n,):
        raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")


def int8_linear(x: torch.Tensor, weight: Int8Rows, bias=None, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` with a weight in 8 bits: [..., out] from x [..., dim] and weight [out, dim].

    x: float32, float16 or bfloat16, any strides; its rows are taken in 8 bits, each with a scale of its own.  bias: [out] or
    None.  dtype: of the result (None: x's), rounded once from 32 bits.  Up to 2**28 rows, 32768 values, 2**20 columns."""
    if not isinstance(weight, Int8Rows):
        raise ValueError(f"weight must be Int8Rows (see quantize_rows), got {type(weight).__name__}")
    if not isinstance(x, torch.Tensor) or x.dtype not in _lib.HTYPE_OF_DTYPE or x.dim() < 1:
        raise ValueError("x must be a float32, float16 or bfloat16 tensor [..., dim]")
    out, dim = weight.values.shape
    if x.shape[-1] != dim:
        raise ValueError(f"x must be [..., {dim}], got {tuple(x.shape)}")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _lib.HTYPE_OF_DTYPE:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    _check_bias(bias, out)
    _check_sizes(x.shape[:-1].numel(), dim, out)
    dev = x.device
    if dev.type != "cuda" or weight.values.device != dev or (bias is not None and bias.device != dev):
        dev = _gpu(x, "x", weight=weight, bias=bias)
    _refuse_gradient(x, bias)
    bias = None if bias is None else bias.contiguous()
    rows = x if x.dim() == 2 else x.reshape(-1, dim)
    y = x.new_empty((*x.shape[:-1], out), dtype=dtype)
    L = _lib.lib()
    a = _lib.GsLinear8(rows.data_ptr(), rows.stride(0), rows.stride(1), weight.values.data_ptr(), weight.values.stride(0),
                       weight.scales.data_ptr(), _lib.ptr(bias), y.data_ptr(), _lib.HTYPE_OF_DTYPE[x.dtype],
                       _lib.HTYPE_OF_DTYPE[dtype], _lib.GS_H_F32 if bias is None else _lib.HTYPE_OF_DTYPE[bias.dtype],
                       rows.shape[0], dim, out)
    need = C.c_size_t()
    with _on(dev):
        _lib.check(L.gs_int8_linear_workspace(C.byref(a), C.byref(need)), "gs_int8_linear_workspace")
        ws = _bytes(need.value, dev) if need.value else None
        _lib.check(L.gs_int8_linear(C.byref(a), _lib.ptr(ws), need.value, _lib.stream_ptr(dev)), "gs_int8_linear")
    return y
