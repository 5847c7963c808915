"""Microscaled 4-bit floating point on the GPU: models on their way to the
clients, and products with 4-bit factors on the tensor cores.

The torch side of falcom_mx4_* (include/falcom_b200.h, which defines the
format, the rounding and the random bits).  The reference has nothing of the
kind: its server sends models in 32 bits.  Vectors:

    sent = mx4.encode(weights, base=held)          # server: held follows what clients have
    mx4.decode(sent, out=mine, accumulate=True)    # client

(federated.Downlink is that pair with the server's copy.)  Matrices:

    w = mx4.quantize(weight)                       # once
    y = mx4.product(x, w, dtype=torch.bfloat16)    # x @ weight.t(), x rounded on the way
    y = mx4.linear(x, weight, p=0.1, seed=step)    # training: all three products in 4 bits

Calls queue work on the device's current stream and may be captured in a CUDA
graph.  Random rounding and dropout are functions of (seed, counter, place):
the same arguments give the same bits.  In a graph that is replayed a new seed
has to come from the device: `counter`, an int64 tensor that the caller counts
up, is read when the work runs.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import abi
from . import optim as _optim

_TYPES = {torch.float32: abi.TYPE_F32, torch.bfloat16: abi.TYPE_BF16, torch.float16: abi.TYPE_F16}
_bound = {}


def _library(path: Optional[str] = None) -> ctypes.CDLL:
    lib = _bound.get(path)
    if lib is None:
        lib = _optim._library(path)
        abi.bind_mx4(lib)
        _bound[path] = lib
    return lib


def _check(t, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is not a tensor")
    if t.dtype not in _TYPES:
        raise ValueError(f"{what} is {t.dtype}: float32, bfloat16 or float16 is wanted")
    if not t.is_cuda:
        raise ValueError(f"{what} is on {t.device}: a CUDA device is wanted")
    if t.layout != torch.strided or t.is_neg():
        raise ValueError(f"{what} does not hold its values as they are ({t.layout})")


def _check_type(dtype) -> None:
    if dtype not in _TYPES:
        raise ValueError(f"{dtype}: float32, bfloat16 or float16 is wanted")


def _same_device(device, **others) -> None:
    for what, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f"{what} is on {t.device}, the rest of the call on {device}")


def _stream(device: torch.device) -> int:
    return _optim._current_stream(device.index)


def _random(rounding: str, seed: int, counter: Optional[torch.Tensor], device) -> Optional[abi.RandomC]:
    if rounding not in ("nearest", "random"):
        raise ValueError(f"rounding is 'nearest' or 'random', got {rounding!r}")
    r = _seeded(seed, counter, device)
    return r if rounding == "random" else None


def _seeded(seed: int, counter: Optional[torch.Tensor], device) -> abi.RandomC:
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed must fit 64 bits, got {seed}")
    at = None
    if counter is not None:
        if not isinstance(counter, torch.Tensor) or counter.dtype != torch.int64 or counter.numel() != 1 \
                or counter.device != device:
            raise ValueError(f"counter must be one int64 on {device}")
        at = counter.data_ptr()
    return abi.RandomC(int(seed), at)


def _drop(p: float, seed: int, counter: Optional[torch.Tensor], device) -> Optional[abi.DropoutArgsC]:
    if not (p >= 0 and int(p * 65536 + 0.5) < 65536):
        raise ValueError(f"p must lie in [0, 1), got {p}")
    return abi.DropoutArgsC(float(p), _seeded(seed, counter, device)) if p > 0 else None


def _ref(c):
    return ctypes.byref(c) if c is not None else None


def _done(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed ({rc})")


def _scales_from(n: int) -> int:
    """Where a vector's scales begin in its buffer."""
    return -(-((n + 1) // 2) // 16) * 16


class Mx4Vector:
    """A vector in 4 bits: `buffer`, one run of bytes (to broadcast, to save),
    holds `codes` and, from the next multiple of 16 on, `scales`."""

    def __init__(self, n: int, buffer: torch.Tensor):
        self.n, self.buffer = n, buffer
        if buffer.dtype != torch.uint8 or buffer.dim() != 1 or buffer.numel() != self.size_of(n) \
                or not buffer.is_contiguous():
            raise ValueError(f"the buffer of {n} elements is {self.size_of(n)} contiguous bytes")
        self.codes = buffer[:(n + 1) // 2]
        self.scales = buffer[_scales_from(n):]

    @staticmethod
    def size_of(n: int) -> int:
        return _scales_from(n) + -(-n // abi.MX4_BLOCK)

    @staticmethod
    def empty(n: int, device) -> "Mx4Vector":
        """For a receiver: the buffer that a sent one is copied into.  (Zeroed:
        the bytes between codes and scales, up to 15, are nobody's.)"""
        return Mx4Vector(n, torch.zeros(Mx4Vector.size_of(n), dtype=torch.uint8, device=device))

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def decode(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return decode(self, dtype=dtype)


class Mx4Matrix:
    """A matrix [rows, cols] in 4 bits, rounded along its rows, in the layout
    of the tensor cores (include/falcom_b200.h)."""

    def __init__(self, rows: int, cols: int, codes: torch.Tensor, scales: torch.Tensor):
        self.rows, self.cols, self.codes, self.scales = rows, cols, codes, scales
        for what, t, size in (("codes", codes, self.sizes_of(rows, cols)[0]), ("scales", scales, self.sizes_of(rows, cols)[1])):
            if t.dtype != torch.uint8 or t.dim() != 1 or t.numel() != size or not t.is_contiguous() or t.device != codes.device:
                raise ValueError(f"the {what} of {rows} x {cols} are {size} contiguous bytes")
        self._c = abi.Mx4MatrixC(codes.data_ptr(), scales.data_ptr(), rows, cols)

    @staticmethod
    def sizes_of(rows: int, cols: int) -> Tuple[int, int]:
        """Bytes of codes and of scales."""
        panels = -(-cols // 256) if rows else 0
        return panels * -(-rows // 8) * 8 * 128, panels * -(-rows // 128) * 1024

    @staticmethod
    def empty(rows: int, cols: int, device) -> "Mx4Matrix":
        codes, scales = Mx4Matrix.sizes_of(rows, cols)
        both = torch.empty(codes + scales, dtype=torch.uint8, device=device)
        return Mx4Matrix(rows, cols, both[:codes], both[codes:])

    @property
    def shape(self) -> Tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        _check_type(dtype)
        out = torch.empty(self.rows, self.cols, dtype=dtype, device=self.device)
        _done(_library().falcom_mx4_dequantize(ctypes.byref(self._c), out.data_ptr(), _TYPES[dtype], self.cols,
                                               _stream(self.device)), "falcom_mx4_dequantize")
        return out


# ------------------------------------------------------------------ vectors

def encode(x: torch.Tensor, base: Optional[torch.Tensor] = None, rounding: str = "nearest", seed: int = 0,
           counter: Optional[torch.Tensor] = None) -> Mx4Vector:
    """x in 4 bits, as a vector in memory order.  With `base` (float32, what
    the receivers hold) the difference from it, and base then follows: it has
    what the difference reads back as added, so the next call's difference
    holds again what this one rounded away."""
    _check(x, "x")
    if not x.is_contiguous():
        raise ValueError(f"x must be contiguous, got strides {x.stride()}")
    if base is not None:
        _check(base, "base")
        if base.dtype != torch.float32 or base.numel() != x.numel() or not base.is_contiguous():
            raise ValueError(f"base must be {x.numel()} contiguous float32 values")
        _same_device(x.device, base=base)
    random = _random(rounding, seed, counter, x.device)
    n = x.numel()
    # not zeroed: the kernel writes all but the bytes between codes and scales
    sent = Mx4Vector(n, torch.empty(Mx4Vector.size_of(n), dtype=torch.uint8, device=x.device))
    at = sent.buffer.data_ptr()
    _done(_library().falcom_mx4_encode(x.data_ptr(), _TYPES[x.dtype], n, base.data_ptr() if base is not None else None,
                                       _ref(random), at, at + _scales_from(n), _stream(x.device)), "falcom_mx4_encode")
    if base is not None:
        torch.autograd.graph.increment_version(base)
    return sent


def decode(sent: Mx4Vector, out: Optional[torch.Tensor] = None, weight: float = 1.0, accumulate: bool = False,
           dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """weight times the values, into `out` (added to it with accumulate) or
    into a new vector of `dtype`."""
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs an out to add to")
        _check_type(dtype)
        out = torch.empty(sent.n, dtype=dtype, device=sent.device)
    _check(out, "out")
    if out.numel() != sent.n or not out.is_contiguous():
        raise ValueError(f"out must be {sent.n} contiguous values, got {tuple(out.shape)} with strides {out.stride()}")
    _same_device(out.device, sent=sent)
    at = sent.buffer.data_ptr()
    _done(_library().falcom_mx4_decode(at, at + _scales_from(sent.n), sent.n, weight, accumulate, out.data_ptr(),
                                       _TYPES[out.dtype], _stream(out.device)), "falcom_mx4_decode")
    torch.autograd.graph.increment_version(out)
    return out


# ----------------------------------------------------------------- matrices

def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as a matrix whose rows are runs of memory."""
    _check(x, what)
    if x.dim() < 1:
        raise ValueError(f"{what} has no dimensions")
    # (no reshape to -1: a last dimension of 0 leaves the rows undetermined)
    rows = 1
    for s in x.shape[:-1]:
        rows *= s
    x = x.detach().reshape(rows, x.shape[-1])
    if x.numel() and (x.stride(1) != 1 and x.shape[1] > 1 or x.stride(0) < x.shape[1] and rows > 1):
        x = x.contiguous()
    return x


def _quantize(x: torch.Tensor, along: str, random, drop) -> Tuple[Optional[Mx4Matrix], Optional[Mx4Matrix]]:
    rows, cols = x.shape
    by_rows = Mx4Matrix.empty(rows, cols, x.device) if along != "columns" else None
    by_cols = Mx4Matrix.empty(cols, rows, x.device) if along != "rows" else None
    _done(_library().falcom_mx4_quantize(x.data_ptr(), _TYPES[x.dtype], rows, cols, x.stride(0) if rows > 1 else cols,
                                         _ref(random), _ref(drop), _ref(by_rows._c) if by_rows else None,
                                         _ref(by_cols._c) if by_cols else None, _stream(x.device)),
          "falcom_mx4_quantize")
    return by_rows, by_cols


def quantize(x: torch.Tensor, along: str = "rows", rounding: str = "nearest", seed: int = 0,
             counter: Optional[torch.Tensor] = None) -> Union[Mx4Matrix, Tuple[Mx4Matrix, Mx4Matrix]]:
    """x (all but its last dimension are rows) in 4 bits: along its "rows";
    along its "columns", which gives the transposed matrix; or "both", from one
    read.  Products sum along the dimension that was rounded along."""
    if along not in ("rows", "columns", "both"):
        raise ValueError(f"along is 'rows', 'columns' or 'both', got {along!r}")
    x = _rows(x, "x")
    both = _quantize(x, along, _random(rounding, seed, counter, x.device), None)
    return both if along == "both" else both[0] or both[1]


def product(a: Union[torch.Tensor, Mx4Matrix], b: Mx4Matrix, dtype: torch.dtype = torch.bfloat16,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ b.t() in `dtype`, summed in float32.  A tensor `a` is rounded to the
    nearest 4-bit values on the way; its leading dimensions stay."""
    if not isinstance(b, Mx4Matrix):
        raise TypeError("b is not an Mx4Matrix: quantize it")
    lead = None
    if isinstance(a, torch.Tensor):
        lead = a.shape[:-1]
        x = _rows(a, "a")
        if x.shape[1] != b.cols:
            raise ValueError(f"a has {x.shape[1]} columns, b {b.cols}")
        _same_device(b.device, a=x)
        a = _quantize(x, "rows", None, None)[0]
    elif not isinstance(a, Mx4Matrix):
        raise TypeError("a is neither a tensor nor an Mx4Matrix")
    y = _product(a, b, dtype, None, out)
    return y if lead is None or out is not None else y.view(*lead, b.rows)


def _product(a: Mx4Matrix, b: Mx4Matrix, dtype: torch.dtype, drop, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if a.cols != b.cols:
        raise ValueError(f"a has {a.cols} columns, b {b.cols}")
    _same_device(b.device, a=a)
    if out is None:
        _check_type(dtype)
        out = torch.empty(a.rows, b.rows, dtype=dtype, device=b.device)
    else:
        _check(out, "out")
        if out.numel() != a.rows * b.rows or not out.is_contiguous():
            raise ValueError(f"out must be {a.rows} x {b.rows} contiguous values, got {tuple(out.shape)} with strides "
                             f"{out.stride()}")
        _same_device(b.device, out=out)
        torch.autograd.graph.increment_version(out)
    _done(_library().falcom_mx4_product(ctypes.byref(a._c), ctypes.byref(b._c), out.data_ptr(), _TYPES[out.dtype],
                                        b.rows, _ref(drop), _stream(b.device)), "falcom_mx4_product")
    return out


def errors() -> int:
    """Nonzero once a product on the current device gave up waiting for its own
    copies (never seen): what it left is then not to be used.  Waits for the
    device."""
    return _library().falcom_mx4_errors()


# ------------------------------------------------------------------- layers

class _Linear(torch.autograd.Function):
    """y = Q(D(x)) Q(w)^T, dx = D'(Q(dy) Q(w^T)^T), dw = Q(dy^T) Q(D(x)^T)^T:
    Q rounds along the summed dimension, the gradient at random, the rest to
    the nearest; D is dropout.  Rounding counts as the identity in the
    gradients.  What is kept for them is in 4 bits."""

    @staticmethod
    def forward(ctx, x, w, p, seed, counter):
        m = _rows(x, "x")
        drop = _drop(p, seed, counter, m.device)
        a, at = _quantize(m, "both" if ctx.needs_input_grad[1] else "rows", None, drop)
        b, bt = _quantize(_rows(w, "weight"), "both" if ctx.needs_input_grad[0] else "rows", None, None)
        ctx.p, ctx.seed, ctx.shapes, ctx.types = p, seed, (x.shape, w.shape), (x.dtype, w.dtype)
        # the counter as it is now, whatever it is when the gradients are asked for
        counter = counter.clone() if counter is not None else None
        ctx.save_for_backward(counter, *(t for m in (at, bt) for t in ((m.codes, m.scales) if m else (None, None))))
        return _product(a, b, x.dtype, None).view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        counter, a_codes, a_scales, b_codes, b_scales = ctx.saved_tensors
        (*lead, k), (n, _) = ctx.shapes
        g = _rows(dy, "the gradient")
        t = g.shape[0]
        need_x, need_w = ctx.needs_input_grad[:2]
        along = "both" if need_x and need_w else "rows" if need_x else "columns"
        by_rows, by_cols = _quantize(g, along, _seeded(ctx.seed, counter, g.device), None)
        dx = dw = None
        if need_x:
            dx = _product(by_rows, Mx4Matrix(k, n, b_codes, b_scales), ctx.types[0],
                          _drop(ctx.p, ctx.seed, counter, g.device)).view(*lead, k)
        if need_w:
            dw = _product(by_cols, Mx4Matrix(k, t, a_codes, a_scales), ctx.types[1], None)
        return dx, dw, None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, p: float = 0.0, seed: int = 0,
           counter: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dropout(x, p) @ weight.t() with both factors in 4 bits, in x's type; the
    gradients' products have their factors in 4 bits too (the incoming gradient
    rounded at random).  weight [n, k] may have another type than x [..., k].
    Give each step and layer a seed of its own, or a counter."""
    for t, what in ((x, "x"), (weight, "weight")):
        _check(t, what)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    _same_device(x.device, weight=weight)
    _drop(p, seed, counter, x.device)
    return _Linear.apply(x, weight, float(p), int(seed), counter)
