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
    x = x.contiguous()
    if residual is not None:   # (as for x: a copy has to live until the call is made)
        residual = residual.contiguous()
    y = torch.empty_like(x)
    cols = x.shape[-1] if x.dim() else 1
    args = abi.DropoutArgsC(p, _mx4._seeded(seed, counter, x.device))
    _mx4._done(_mx4._library().falcom_dropout(
        x.data_ptr(), residual.data_ptr() if residual is not None else None, y.data_ptr(),
        _mx4._TYPES[x.dtype], x.numel() // cols if cols else 0, cols, ctypes.byref(args), _mx4._stream(x.device)),
        "falcom_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, counter):
        ctx.p, ctx.seed, ctx.counter = p, seed, None
        if counter is not None:   # as it is now, whatever it is when the gradient is asked for
            ctx.counter = counter.clone()
        return _run(x, residual, p, seed, counter)

    @staticmethod
    def backward(ctx, dy):
        need_x, need_residual = ctx.needs_input_grad[:2]
        dx = None
        if need_x:
            # through apply where a graph is wanted: the gradient of the gradient is the same operation again
            dx = (_Dropout.apply if torch.is_grad_enabled() else _run)(dy, None, ctx.p, ctx.seed, ctx.counter)
        return dx, dy if need_residual else None, None, None, None


def dropout(x: torch.Tensor, p: float = 0.5, seed: int = 0, counter: Optional[torch.Tensor] = None,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + (kept ? x / (1 - p) : 0), an element kept with probability
    1 - p (p to 16 bits).  Elements are numbered by row, a row being the last
    dimension.  A dropped element is 0 whatever x holds there, infinity and NaN
    included, and so is its gradient.  Give each step and place a seed of its
    own, or a counter (an int64 tensor on the device, read when the work runs)
    that is counted up.  Without a residual p = 0 returns x itself.  Where p is
    not 0 tangents of forward mode are refused (NotImplementedError)."""
    _mx4._check(x, "x")
    if residual is not None:
        _mx4._check(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise ValueError(f"residual is {residual.dtype} {tuple(residual.shape)} on {residual.device}, x {x.dtype} "
                             f"{tuple(x.shape)} on {x.device}")
    _mx4._check_p(p)
    if p == 0:   # the rest is torch's
        return x if residual is None else x + residual
    if not _mx4._differentiated(x, residual):
        return _run(x, residual, float(p), int(seed), counter)
    return _Dropout.apply(x, residual, float(p), int(seed), counter)
