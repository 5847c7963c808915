"""Dropout from a counter-based generator: the mask is a function of (seed,
counter, place) and is made again where it is needed, never stored.

The torch side of falcom_dropout (include/falcom_b200.h, which defines the
random bits); mx4.linear has the same dropout inside its rounding.  The
reference has none: its clients train with their framework's.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import abi
from . import mx4 as _mx4


def _run(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, seed: int, counter) -> torch.Tensor:
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    cols = x.shape[-1] if x.dim() else 1
    args = abi.DropoutArgsC(p, _mx4._seeded(seed, counter, x.device))
    _mx4._done(_mx4._library().falcom_dropout(
        x.data_ptr(), residual.data_ptr() if residual is not None else None, y.data_ptr(), _mx4._TYPES[x.dtype],
        x.numel() // cols if cols else 0, cols, ctypes.byref(args), _mx4._stream(x.device)), "falcom_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, counter):
        ctx.p, ctx.seed = p, seed
        # the counter as it is now, whatever it is when the gradient is asked for
        ctx.save_for_backward(counter.clone() if counter is not None else None)
        return _run(x.contiguous(), residual.contiguous() if residual is not None else None, p, seed, counter)

    @staticmethod
    def backward(ctx, dy):
        counter, = ctx.saved_tensors
        # through apply: the gradient of the gradient is the same operation again
        dx = _Dropout.apply(dy, None, ctx.p, ctx.seed, counter) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float = 0.5, seed: int = 0, counter: Optional[torch.Tensor] = None,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + (kept ? x / (1 - p) : 0), an element kept with probability
    1 - p (p to 16 bits).  Elements are numbered by row, a row being the last
    dimension.  A dropped element is 0 whatever x holds there, infinity and NaN
    included, and so is its gradient.  Give each step and place a seed of its
    own, or a counter (an int64 tensor on the device, read when the work runs)
    that is counted up."""
    _mx4._check(x, "x")
    if residual is not None:
        _mx4._check(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"residual is {residual.dtype} {tuple(residual.shape)} on {residual.device}, x {x.dtype} "
                             f"{tuple(x.shape)} on {x.device}")
    _mx4._drop(p, seed, counter, x.device)
    return _Dropout.apply(x, residual, float(p), int(seed), counter)
