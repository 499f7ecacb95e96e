"""What the encoder's operators check and ask of tensors."""
from __future__ import annotations

from contextlib import nullcontext

import torch
from torch.autograd import forward_ad


HERE = nullcontext()
MAX_ROWS, MAX_DIM, MAX_TERMS = 1 << 28, 1 << 15, 1 << 20


def _check_sizes(rows: int, dim: int, terms: int = 1):
    """The C entries' limits.  They are checked here as well since ctypes cuts a size that is beyond its field's 32 bits, so
    that those entries would see another, smaller one."""
    if rows > MAX_ROWS or dim > MAX_DIM or terms > MAX_TERMS:
        raise ValueError(f"{rows} rows, {dim} values, {terms} terms: at most {MAX_ROWS}, {MAX_DIM} and {MAX_TERMS} are supported")


def _same_device(dev, of="hidden", **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, {of} on {dev}")


def _on(dev):
    """The tensors' device as the current one; entering it costs more than asking whether it is."""
    return HERE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _bytes(n: int, dev) -> torch.Tensor:
    return torch.empty(int(n), dtype=torch.uint8, device=dev)


def _beyond_reverse_mode() -> bool:
    return (forward_ad._current_level >= 0 or torch._C._are_functorch_transforms_active()
            or torch._C._get_tracing_state() is not None)


def _differentiable(*inputs) -> bool:
    """Whether a call has to go through autograd: a gradient may be asked for, tensors may carry tangents or belong to a
    functional transform (both of which autograd refuses here), or a trace records it.  One that need not leaves autograd
    out (5 us of a query's 21)."""
    if torch.is_grad_enabled():
        for t in inputs:
            if t is not None and t.requires_grad:
                return True
    return _beyond_reverse_mode()
