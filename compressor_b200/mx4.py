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
up, is read when the work runs.  As for any backward pass, torch can capture
linear's and dropout's only while no eager autograd graph of the same leaves is
alive (its nodes belong to another stream, and the capture ends with an
error).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as _forward_ad

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
    if t.layout is not torch.strided or t.is_neg():
        raise ValueError(f"{what} does not hold its values as they are ({t.layout})")


def _check_type(dtype) -> None:
    if dtype not in _TYPES:
        raise ValueError(f"{dtype}: float32, bfloat16 or float16 is wanted")


def _same_device(device, **others) -> None:
    for what, t in others.items():
        if t.device != device:
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


def _differentiated(x: torch.Tensor, other: Optional[torch.Tensor]) -> bool:
    """Whether autograd has to see a call: a gradient is wanted, or a tensor
    carries a tangent of forward mode (autograd then raises, for want of a
    rule).  Outside of a dual level there are none, and asking costs 1 us."""
    if torch.is_grad_enabled() and (x.requires_grad or (other is not None and other.requires_grad)):
        return True
    if getattr(_forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in (x, other))


def _check_p(p: float) -> None:
    if not (p >= 0 and int(p * 65536 + 0.5) < 65536):
        raise ValueError(f"p must lie in [0, 1) to 16 bits, got {p}")


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
    holds `codes` and, from the next multiple of 16 on, `scales`.  (The bytes
    between them, up to 15, are 0.)  `round` goes beside it: the number, an
    int64 tensor, of the federated.Downlink round that it was sent in, or None."""

    round: Optional[torch.Tensor] = None

    def __init__(self, n: int, buffer: torch.Tensor):
        if buffer.dtype != torch.uint8 or buffer.dim() != 1 or buffer.numel() != self.size_of(n) \
                or not buffer.is_contiguous():
            raise ValueError(f"the buffer of {n} elements is {self.size_of(n)} contiguous bytes")
        self.n, self.buffer = n, buffer

    @property
    def codes(self) -> torch.Tensor:
        return self.buffer[:(self.n + 1) // 2]

    @property
    def scales(self) -> torch.Tensor:
        return self.buffer[_scales_from(self.n):]

    @staticmethod
    def size_of(n: int) -> int:
        return _scales_from(n) + -(-n // abi.MX4_BLOCK)

    @staticmethod
    def empty(n: int, device) -> "Mx4Vector":
        """For a receiver: the buffer that a sent one is copied into (zeros until then)."""
        return Mx4Vector(n, torch.zeros(Mx4Vector.size_of(n), dtype=torch.uint8, device=device))

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def decode(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return decode(self, dtype=dtype)


class Mx4Matrix:
    """A matrix [rows, cols] in 4 bits, rounded along its rows, in the layout
    of the tensor cores (include/falcom_b200.h): `buffer`, one run of bytes,
    holds `codes` and `scales`.  (Padding in it is 0: products count on it.)"""

    def __init__(self, rows: int, cols: int, buffer: torch.Tensor):
        codes, scales = self.sizes_of(rows, cols)
        if buffer.dtype != torch.uint8 or buffer.dim() != 1 or buffer.numel() != codes + scales \
                or not buffer.is_contiguous():
            raise ValueError(f"the buffer of {rows} x {cols} is {codes + scales} contiguous bytes")
        self.rows, self.cols, self.buffer = rows, cols, buffer
        self._codes, self._c = codes, abi.Mx4MatrixC(None, None, rows, cols)

    @property
    def _ref(self):
        """For a call: the buffer as it lies now."""
        at = self.buffer.data_ptr()
        self._c.codes, self._c.scales = at, at + self._codes
        return ctypes.byref(self._c)

    @staticmethod
    def sizes_of(rows: int, cols: int) -> Tuple[int, int]:
        """Bytes of codes and of scales."""
        panels = -(-cols // 256) if rows else 0
        return panels * -(-rows // 8) * 8 * 128, panels * -(-rows // 128) * 1024

    @staticmethod
    def empty(rows: int, cols: int, device) -> "Mx4Matrix":
        """Room for a matrix (of a receiver, of a checkpoint)."""
        return Mx4Matrix(rows, cols, torch.empty(sum(Mx4Matrix.sizes_of(rows, cols)), dtype=torch.uint8, device=device))

    @property
    def codes(self) -> torch.Tensor:
        return self.buffer[:self._codes]

    @property
    def scales(self) -> torch.Tensor:
        return self.buffer[self._codes:]

    @property
    def shape(self) -> Tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        _check_type(dtype)
        out = torch.empty(self.rows, self.cols, dtype=dtype, device=self.device)
        _done(_library().falcom_mx4_dequantize(self._ref, out.data_ptr(), _TYPES[dtype], self.cols,
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
    sent = Mx4Vector(n, torch.empty(Mx4Vector.size_of(n), dtype=torch.uint8, device=x.device))   # written whole
    _done(_library().falcom_mx4_encode_vector(x.data_ptr(), _TYPES[x.dtype], n,
                                              base.data_ptr() if base is not None else None, _ref(random),
                                              sent.buffer.data_ptr(), _stream(x.device)), "falcom_mx4_encode_vector")
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
    """x as a matrix whose rows are runs of memory (for its address alone)."""
    _check(x, what)
    if x.dim() == 2 and x.is_contiguous():
        return x
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


def _quantize(x: torch.Tensor, along: str, random) -> Tuple[Optional[Mx4Matrix], Optional[Mx4Matrix]]:
    rows, cols = x.shape
    by_rows = Mx4Matrix.empty(rows, cols, x.device) if along != "columns" else None
    by_cols = Mx4Matrix.empty(cols, rows, x.device) if along != "rows" else None
    _done(_library().falcom_mx4_quantize(x.data_ptr(), _TYPES[x.dtype], rows, cols, x.stride(0) if rows > 1 else cols,
                                         _ref(random), None, by_rows._ref if by_rows else None,
                                         by_cols._ref if by_cols else None, _stream(x.device)), "falcom_mx4_quantize")
    return by_rows, by_cols


def quantize(x: torch.Tensor, along: str = "rows", rounding: str = "nearest", seed: int = 0,
             counter: Optional[torch.Tensor] = None) -> Union[Mx4Matrix, Tuple[Mx4Matrix, Mx4Matrix]]:
    """x (all but its last dimension are rows) in 4 bits: along its "rows";
    along its "columns", which gives the transposed matrix; or "both", from one
    read.  Products sum along the dimension that was rounded along.  (No
    gradients go through it, as none do through encode, decode and product.)"""
    if along not in ("rows", "columns", "both"):
        raise ValueError(f"along is 'rows', 'columns' or 'both', got {along!r}")
    x = _rows(x, "x")
    both = _quantize(x, along, _random(rounding, seed, counter, x.device))
    return both if along == "both" else both[0] or both[1]


def product(a: Union[torch.Tensor, Mx4Matrix], b: Mx4Matrix, dtype: torch.dtype = torch.bfloat16,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ b.t() in `dtype`, summed in float32.  A tensor `a` is rounded to the
    nearest 4-bit values on the way; its leading dimensions stay.  (For
    answering: no gradients go through it, as they do through linear.)"""
    if not isinstance(b, Mx4Matrix):
        raise TypeError("b is not an Mx4Matrix: quantize it")
    if isinstance(a, Mx4Matrix):
        return _product(a, b, dtype, out)
    x = _rows(a, "a")
    rows, cols = x.shape
    if cols != b.cols:
        raise ValueError(f"a has {cols} columns, b {b.cols}")
    device = b.device
    _same_device(device, a=x)
    y = _out(rows, b, dtype, out, a.shape[:-1])
    lib = _library()
    size = lib.falcom_mx4_work_bytes(rows, cols)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _done(lib.falcom_mx4_product_of(x.data_ptr(), _TYPES[x.dtype], rows, x.stride(0) if rows > 1 else cols, b._ref,
                                    y.data_ptr(), _TYPES[y.dtype], b.rows, work.data_ptr() if size else None,
                                    _stream(device)), "falcom_mx4_product_of")
    return y


def _out(rows: int, b: Mx4Matrix, dtype: torch.dtype, out: Optional[torch.Tensor], lead) -> torch.Tensor:
    if out is None:
        _check_type(dtype)
        return torch.empty(*lead, b.rows, dtype=dtype, device=b.device)
    _check(out, "out")
    if out.numel() != rows * b.rows or not out.is_contiguous():
        raise ValueError(f"out must be {rows} x {b.rows} contiguous values, got {tuple(out.shape)} with strides "
                         f"{out.stride()}")
    _same_device(b.device, out=out)
    torch.autograd.graph.increment_version(out)
    return out


def _product(a: Mx4Matrix, b: Mx4Matrix, dtype: torch.dtype, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if a.cols != b.cols:
        raise ValueError(f"a has {a.cols} columns, b {b.cols}")
    _same_device(b.device, a=a)
    out = _out(a.rows, b, dtype, out, (a.rows,))
    _done(_library().falcom_mx4_product(a._ref, b._ref, out.data_ptr(), _TYPES[out.dtype], b.rows, None,
                                        _stream(b.device)), "falcom_mx4_product")
    return out


def errors() -> int:
    """Nonzero when a product on the current device gave up waiting for its own
    copies since the last call that said so (never seen): results that may lack
    a part are NaN then.  Waits for the device."""
    return _library().falcom_mx4_errors()


# ------------------------------------------------------------------- layers

def _linear_forward(x, w, p, seed, counter, need_x, need_w):
    """y, the layer as the library has it, and what backward needs."""
    lib, device = _library(), x.device
    m, v = _rows(x, "x"), _rows(w, "weight")
    (rows, cols), outs = m.shape, v.shape[0]
    layer = abi.Mx4LinearC(rows, cols, outs, _TYPES[x.dtype], _TYPES[w.dtype], need_x, need_w, p,
                           _seeded(seed, counter, device))
    ref = ctypes.byref(layer)
    kept = torch.empty(lib.falcom_mx4_linear_kept_bytes(ref), dtype=torch.uint8, device=device)
    work = torch.empty(lib.falcom_mx4_linear_work_bytes(ref, 0), dtype=torch.uint8, device=device)
    y = torch.empty(*x.shape[:-1], outs, dtype=x.dtype, device=device)
    _done(lib.falcom_mx4_linear_forward(ref, m.data_ptr(), m.stride(0) if rows > 1 else cols, v.data_ptr(),
                                        v.stride(0) if outs > 1 else cols, y.data_ptr(), kept.data_ptr(),
                                        work.data_ptr(), _stream(device)), "falcom_mx4_linear_forward")
    return y, layer, kept


class _Linear(torch.autograd.Function):
    """falcom_mx4_linear_forward and _backward.  Rounding counts as the
    identity in the gradients; what is kept for them is in 4 bits."""

    @staticmethod
    def forward(ctx, x, w, p, seed, counter):
        y, ctx.layer, kept = _linear_forward(x, w, p, seed, counter, *ctx.needs_input_grad[:2])
        # the counter as it is now, whatever it is when the gradients are asked for
        ctx.save_for_backward(kept, counter.clone() if counter is not None else None)
        ctx.of = x.shape, x.dtype, w.shape, w.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib, device, layer = _library(), dy.device, ctx.layer
        kept, counter = ctx.saved_tensors
        x_shape, x_type, w_shape, w_type = ctx.of
        need_x, need_w = ctx.needs_input_grad[:2]
        g = _rows(dy, "the gradient")
        layer.random.counter = counter.data_ptr() if counter is not None else None
        ref = ctypes.byref(layer)
        work = torch.empty(lib.falcom_mx4_linear_work_bytes(ref, 1), dtype=torch.uint8, device=device)
        dx = torch.empty(x_shape, dtype=x_type, device=device) if need_x else None
        dw = torch.empty(w_shape, dtype=w_type, device=device) if need_w else None
        _done(lib.falcom_mx4_linear_backward(ref, g.data_ptr(), g.stride(0) if layer.rows > 1 else layer.outs,
                                             kept.data_ptr(), dx.data_ptr() if need_x else None,
                                             dw.data_ptr() if need_w else None, work.data_ptr(), _stream(device)),
              "falcom_mx4_linear_backward")
        return dx, dw, None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, p: float = 0.0, seed: int = 0,
           counter: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dropout(x, p) @ weight.t() with both factors in 4 bits, in x's type; the
    gradients' products have their factors in 4 bits too (the incoming gradient
    rounded at random).  weight [n, k] may have another type than x [..., k].
    Give each step and layer a seed of its own, or a counter.  Tangents of
    forward mode are refused (NotImplementedError)."""
    for t, what in ((x, "x"), (weight, "weight")):
        _check(t, what)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not go together")
    _same_device(x.device, weight=weight)
    _check_p(p)
    if not _differentiated(x, weight):
        return _linear_forward(x, weight, float(p), int(seed), counter, False, False)[0]
    return _Linear.apply(x, weight, float(p), int(seed), counter)
