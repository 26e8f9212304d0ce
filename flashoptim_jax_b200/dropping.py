"""Dropout from a counter-based generator, on the GPU.

Which elements stay is a function of (seed, offset, element number) that the kernels work out where they need it
(Philox4x32-10, see FoDropout in include/flashoptim_b200.h); no mask is stored, and the backward pass is the same
call on the gradient.  The reference leaves dropout to the model; it is here because the lookup of an embedding
table (embedding.py) and its gradient take it along in their own pass.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._dev import DTYPE_CODE, dtype_name, refuse_tangent, require_cuda, stream_ptr


def checked_dropout(p, seed, offset, device: torch.device) -> Tuple[float, int, int, Optional[torch.Tensor]]:
    """(p, seed, offset, device offset) in the ranges the library holds."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
    on_device = None
    if isinstance(offset, torch.Tensor):
        if offset.dtype not in (torch.int32, torch.int64) or offset.numel() != 1 or offset.device != device:
            raise ValueError(f"a tensor offset must be one int32 or int64 on {device}, got {tuple(offset.shape)} {dtype_name(offset.dtype)} on {offset.device}")
        on_device, offset = offset, 0
    return p, int(seed) % 2**64, int(offset) % 2**64, on_device


def fill_dropout(f: _lib.FoDropout, p: float, seed: int, offset: int, on_device: Optional[torch.Tensor]) -> None:
    f.p, f.seed, f.offset = p, seed, offset
    if on_device is not None:
        f.dev_offset, f.dev_offset_bits = on_device.data_ptr(), 8 * on_device.element_size()


def _run(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, seed: int, offset) -> torch.Tensor:
    p, seed, host_offset, on_device = checked_dropout(p, seed, offset, x.device)
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    f = _lib.FoDropout()
    fill_dropout(f, p, seed, host_offset, on_device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().fo_dropout(x.data_ptr(), 0 if residual is None else residual.data_ptr(), y.data_ptr(), DTYPE_CODE[x.dtype], x.numel(),
                                         ctypes.byref(f), stream_ptr(x.device)))
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        on_device = isinstance(offset, torch.Tensor)
        ctx.how = (p, seed, None if on_device else offset)
        ctx.save_for_backward(*([offset] if on_device else []))
        return _run(x, residual, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, seed, offset = ctx.how
        dx = _run(dy, None, p, seed, ctx.saved_tensors[0] if offset is None else offset) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, offset=0, *, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x with each element dropped (0, whatever it held) with probability `p` and the others multiplied by 1 / (1 - p); plus `residual`.

    `seed` and `offset` (whole numbers, taken modulo 2^64) and the element's place in row-major order decide what is dropped: give each layer
    a seed and each step an offset.  `offset` may be a one-element int32 or int64 CUDA tensor (the counter of a capturable
    optimizer's state, say), read when the kernel runs: a captured call then drops other elements at each replay.  Until the
    backward pass has run it must keep its value.  Differentiable in x and residual (once, in reverse mode); by hand, the gradient of x is
    `dropout(dy, p, seed, offset)` and that of the residual is dy."""
    y = _lib.host().dropout(x, p, seed, offset, residual)  # None: something to differentiate or convert first, or an error to report
    if y is not None:
        return y
    require_cuda(x, "x")
    refuse_tangent(x, "x")
    if x.dtype not in DTYPE_CODE:
        raise ValueError(f"dropout takes float32, bfloat16 or float16, got {dtype_name(x.dtype)}")
    if residual is not None:
        require_cuda(residual, "residual")
        refuse_tangent(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"residual of shape {tuple(residual.shape)}, {dtype_name(residual.dtype)}, on {residual.device} does not match "
                             f"x of shape {tuple(x.shape)}, {dtype_name(x.dtype)}, on {x.device}")
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        checked_dropout(p, seed, offset, x.device)
        return _Dropout.apply(x, residual, p, seed, offset)
    return _run(x, residual, p, seed, offset)
