"""Optimiser steps over many tensors on the GPU: gradient norm with clipping
coefficient (GradNorm) and AdamW with 32-bit or 8-bit states (AdamW).

The reference has no optimiser of its own: its server averages the decoded
updates and its clients train with their framework's.  These classes are the
torch side of falcom_norm_* and falcom_adamw_* (include/falcom_b200.h, which
defines every formula): one kernel launch for the whole list (a step: for
each pair of parameter and gradient type in it), results on the device,
nothing read back.  A server steps on the round's aggregate with
them (federated.ServerAdamW), a client on its local gradients:

    norm = GradNorm(grads)
    opt = AdamW(params, grads, lr=1e-3, weight_decay=0.01, state_bits=8)
    ...
    opt.step(clip=norm(max_norm=1.0))

Parameters and gradients are fixed lists of tensors: the addresses are read
once, so gradients are written in place from then on (zero_grad with
set_to_none=False; a step refuses parameters whose .grad was one of its
gradients and is so no longer).  Making an object waits for the device; it is
meant once per list.  Calls queue work on the device's current stream (the
steps of one AdamW have to be ordered: one stream, or events) and may be
captured in a CUDA graph; the hyperparameters are captured by value, the
step number, a clip coefficient and a learning rate given as a device tensor
are read when the graph runs.  Closing or dropping an object leaves what
graphs captured of it in place until they are gone.
"""
from __future__ import annotations

import ctypes
import math
import threading
from typing import Dict, List, Optional, Sequence, Union

import torch

from . import abi
from . import build as _build

_TYPES = {torch.float32: abi.TYPE_F32, torch.bfloat16: abi.TYPE_BF16, torch.float16: abi.TYPE_F16}
_libs: Dict[str, ctypes.CDLL] = {}
# (device index) -> cudaStream_t; the public route through a Stream object takes 2 us.  A torch without CUDA has none
# and no tensor that would get as far.
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _capturing(index: int) -> bool:
    """Whether the current stream of that device is being captured."""
    if torch.cuda.current_device() == index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def _library(path: Optional[str]) -> ctypes.CDLL:
    path = path or _build.OUT
    if path not in _libs:
        lib = ctypes.CDLL(path)
        abi.bind_optim(lib)
        _libs[path] = lib
    return _libs[path]


def _dense_strides(t: torch.Tensor) -> Optional[tuple]:
    """Strides of the dimensions longer than one if the tensor fills one run
    of memory without gaps or repeats (in any order of dimensions), else None."""
    dims = sorted((st, s) for s, st in zip(t.shape, t.stride()) if s > 1)
    run = 1
    for st, s in dims:
        if st != run:
            return None
        run *= s
    return tuple(st for s, st in zip(t.shape, t.stride()) if s > 1)


def _check_list(tensors: Sequence[torch.Tensor], what: str) -> List[torch.Tensor]:
    tensors = list(tensors)
    device = None
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} {i} is not a tensor")
        if t.dtype not in _TYPES:
            raise ValueError(f"{what} {i} is {t.dtype}: float32, bfloat16 or float16 is wanted")
        if not t.is_cuda:
            raise ValueError(f"{what} {i} is on {t.device}: a CUDA device is wanted")
        if t.layout != torch.strided or t.is_neg():
            raise ValueError(f"{what} {i} does not hold its values as they are ({t.layout}, negation pending: "
                             f"{t.layout == torch.strided and t.is_neg()})")
        device = t.device if device is None else device
        if t.device != device:
            raise ValueError(f"{what} {i} is on {t.device}, the first on {device}")
        if not t.is_contiguous() and t.numel() and _dense_strides(t) is None:
            raise ValueError(f"{what} {i} has gaps or repeats in memory (strides {t.stride()})")
    return tensors


def _device_of(tensors: Sequence[torch.Tensor]) -> torch.device:
    """Their device, with its index."""
    return tensors[0].device if tensors else torch.device("cuda", torch.cuda.current_device())


def _scalar_input(t: torch.Tensor, numel: int, device: torch.device, what: str) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device or t.numel() != numel \
            or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32 tensor of {numel} on {device}")
    return t.data_ptr()


def _ties(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor]) -> List[tuple]:
    """(index, parameter, its address, its gradient's) of the parameters that
    autograd writes the given gradients of."""
    return [(i, p, p.data_ptr(), g.data_ptr()) for i, (p, g) in enumerate(zip(params, grads))
            if p.requires_grad and (p.is_leaf or p.retains_grad) and p.numel() and p.grad is not None
            and p.grad.data_ptr() == g.data_ptr()]


def _check_ties(ties: List[tuple]) -> None:
    for i, p, p_at, g_at in ties:
        g = p.grad
        if g is None or g.data_ptr() != g_at:
            raise RuntimeError(f"the gradient of parameter {i} is no longer the tensor that this plan reads: keep it "
                               "with zero_grad(set_to_none=False), or make a new plan")
        if p.data_ptr() != p_at:
            raise RuntimeError(f"parameter {i} has moved since this plan was made: make a new one")


# (graphs, destroy, handle, memory) of dropped objects whose captured calls'
# graphs may still run
_kept: List[tuple] = []
_kept_lock = threading.RLock()   # a collector may come back here on the same thread


def _retire(graphs, destroy, handle: int, memory: tuple) -> None:
    """Destroys a plan, and lets go of the memory that its calls use, once no
    graph that captured them is left; looks after earlier ones too."""
    global _kept
    with _kept_lock:
        waiting, _kept = _kept + [(graphs, destroy, handle, memory)], []
        for item in waiting:
            if item[0](item[2]) > 0:
                _kept.append(item)
            else:
                item[1](item[2])


class GradNorm:
    """L2 norm over a list of tensors, and the coefficient that clips it.

    norm(max_norm, grad_scale) returns a new float32 tensor [norm,
    coefficient]: norm = |grad_scale| * sqrt(sum of squares), coefficient =
    min(1, max_norm / norm), NaN when the norm is not finite (in 64 bits: a
    norm above float32's range comes out as infinity beside its coefficient).
    Calls on different streams, and captured ones, do not share scratch
    memory."""

    def __init__(self, tensors: Sequence[torch.Tensor], lib_path: Optional[str] = None):
        self._h = None
        self.tensors = _check_list(tensors, "tensor")
        self._held = [t.detach() for t in self.tensors]   # the memory stays, whatever becomes of a tensor's data
        self.device = _device_of(self.tensors)
        self.lib = _library(lib_path)
        n = len(self.tensors)
        with torch.cuda.device(self.device):
            self._h = self.lib.falcom_norm_create(
                (ctypes.c_void_p * n)(*[t.data_ptr() for t in self.tensors]),
                (ctypes.c_size_t * n)(*[t.numel() for t in self.tensors]),
                (ctypes.c_int * n)(*[_TYPES[t.dtype] for t in self.tensors]), n)
        if not self._h:
            raise RuntimeError("falcom_norm_create failed")
        self._work_words = -(-self.lib.falcom_norm_work_bytes(self._h) // 8)
        self._pair = torch.empty(2, dtype=torch.float32, device=self.device)   # a result's shape
        self._work: Dict[int, torch.Tensor] = {}      # by stream
        self._captured: List[torch.Tensor] = []       # in use by graphs from then on
        # one each for the first captured calls, so that their graphs need not clear theirs
        self._spare = list(torch.zeros(8, self._work_words, dtype=torch.int64, device=self.device))
        torch.cuda.current_stream(self.device).synchronize()

    def __call__(self, max_norm: float = math.inf, grad_scale: float = 1.0) -> torch.Tensor:
        if not self._h:
            raise RuntimeError("GradNorm is closed")
        if not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        if not math.isfinite(grad_scale):
            raise ValueError(f"grad_scale must be finite, got {grad_scale}")
        stream = _current_stream(self.device.index)
        if _capturing(self.device.index):
            if self._spare:
                self._captured.append(self._spare.pop())
                work = self._captured[-1]
            else:   # of the graph's own memory, cleared by the graph
                work = torch.zeros(self._work_words, dtype=torch.int64, device=self.device)
        else:
            work = self._work.get(stream)
            if work is None:
                work = self._work[stream] = torch.zeros(self._work_words, dtype=torch.int64, device=self.device)
        out = torch.empty_like(self._pair)
        rc = self.lib.falcom_norm_run(self._h, grad_scale, max_norm, out.data_ptr(), work.data_ptr(), stream)
        if rc != 0:
            raise RuntimeError(f"falcom_norm_run failed ({rc})")
        return out

    def close(self) -> None:
        h, self._h = self._h, None
        if h:
            _retire(self.lib.falcom_norm_graphs, self.lib.falcom_norm_destroy, h,
                    (self._held, self._work, self._captured))

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class AdamW:
    """AdamW over a list of parameters and a list of gradients of the same
    shapes and memory order (types may differ from tensor to tensor).

    weight_decay: one value, or one per parameter.  state_bits 32 keeps both
    moments in float32; 8 keeps one byte each and two float32 scales per 256
    elements, rounded at random from `seed` (the same seed, state and step
    give the same bits).

    `state` holds the states as flat tensors, every parameter's from a
    multiple of 256 elements on (`offsets`): m, v, step (int64), and with 8
    bits m and v as float8_e4m3fn (v's code holds sqrt(v)) with m_scale and
    v_scale, one float32 per 256 elements."""

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], lr: float = 1e-3,
                 betas: Sequence[float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: Union[float, Sequence[float]] = 0.01, state_bits: int = 32, seed: int = 0,
                 lib_path: Optional[str] = None):
        self._h = None
        self.params = _check_list(params, "parameter")
        self.grads = _check_list(grads, "gradient")
        n = len(self.params)
        if len(self.grads) != n:
            raise ValueError(f"{n} parameters and {len(self.grads)} gradients")
        for i, (p, g) in enumerate(zip(self.params, self.grads)):
            both = p.is_contiguous() and g.is_contiguous()
            if p.shape != g.shape or (not both and p.numel() and _dense_strides(p) != _dense_strides(g)):
                raise ValueError(f"gradient {i} has shape {tuple(g.shape)} and strides {g.stride()}, its parameter "
                                 f"{tuple(p.shape)} and {p.stride()}")
        self.device = _device_of(self.params)
        if n and self.grads[0].device != self.device:
            raise ValueError(f"gradients are on {self.grads[0].device}, parameters on {self.device}")
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        decay = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
        if len(decay) != n or not all(math.isfinite(w) and w >= 0 for w in decay):
            raise ValueError("weight_decay is one value or one per parameter, none of them negative")
        if not 0 <= seed < 1 << 64:
            raise ValueError(f"seed must fit 64 bits, got {seed}")
        self.lr, (self.beta1, self.beta2), self.eps, self.seed = float(lr), betas, float(eps), int(seed)
        self._check_hyper(self.lr, 1.0)
        self.state_bits = state_bits
        self.lib = _library(lib_path)
        self._autograd = [p for p in self.params if p.requires_grad]
        self._tied = _ties(self.params, self.grads)
        self._held = [t.detach() for t in self.params + self.grads]   # the memory stays, whatever becomes of a tensor's data

        self.offsets, total = [], 0
        for p in self.params:
            self.offsets.append(total)
            total += -(-p.numel() // abi.ADAMW_BLOCK) * abi.ADAMW_BLOCK
        kind = torch.float32 if state_bits == 32 else torch.uint8
        state: Dict[str, torch.Tensor] = {k: torch.zeros(total, dtype=kind, device=self.device) for k in "mv"}
        if state_bits == 8:
            state = {k: t.view(torch.float8_e4m3fn) for k, t in state.items()}
            for k in ("m_scale", "v_scale"):
                state[k] = torch.zeros(total // abi.ADAMW_BLOCK, dtype=torch.float32, device=self.device)
        state["step"] = torch.zeros(1, dtype=torch.int64, device=self.device)
        self._state = state

        table = (abi.AdamWTensorC * n)()
        size = 4 if state_bits == 32 else 1
        base = {k: t.data_ptr() for k, t in state.items()}
        for c, p, g, o, w in zip(table, self.params, self.grads, self.offsets, decay):
            c.param, c.grad, c.n = p.data_ptr(), g.data_ptr(), p.numel()
            c.m, c.v = base["m"] + size * o, base["v"] + size * o
            if state_bits == 8:
                c.m_scale = base["m_scale"] + 4 * (o // abi.ADAMW_BLOCK)
                c.v_scale = base["v_scale"] + 4 * (o // abi.ADAMW_BLOCK)
            c.param_type, c.grad_type, c.weight_decay = _TYPES[p.dtype], _TYPES[g.dtype], w
        # steps may run on any stream from here on: the zeros are in place first
        torch.cuda.current_stream(self.device).synchronize()
        with torch.cuda.device(self.device):
            self._h = self.lib.falcom_adamw_create(table, n, state_bits, base["step"])
        if not self._h:
            raise RuntimeError("falcom_adamw_create failed")
        self._args = abi.AdamWArgsC()
        self._args_ref = ctypes.byref(self._args)
        self._given = None
        self._streams = set()

    @property
    def state(self) -> Dict[str, torch.Tensor]:
        """The states, to read, to save and to change in place; others' values
        come in with load_state (the plan goes on with these tensors whatever
        becomes of the dict)."""
        return dict(self._state)

    def _check_hyper(self, lr: float, grad_scale: float) -> None:
        if not (math.isfinite(lr) and lr >= 0):
            raise ValueError(f"lr must be finite and not negative, got {lr}")
        if not (0 <= self.beta1 < 1 and 0 <= self.beta2 < 1):
            raise ValueError(f"betas must lie in [0, 1), got {self.beta1}, {self.beta2}")
        if not 1.2e-38 <= self.eps < 3.4e38:
            raise ValueError(f"eps must be positive as a float32, got {self.eps}")
        if not abs(grad_scale) < 3.4e38:
            raise ValueError(f"grad_scale must be finite as a float32, got {grad_scale}")

    def step(self, lr: Union[None, float, torch.Tensor] = None, grad_scale: float = 1.0,
             clip: Optional[torch.Tensor] = None) -> None:
        """One step on the gradients as they are now, times grad_scale and, if
        `clip` (GradNorm's result) is given, its coefficient; a NaN
        coefficient skips the step.  lr: this call's learning rate instead of
        self.lr, a number or a float32 tensor of one element on the device."""
        if not self._h:
            raise RuntimeError("AdamW is closed")
        if self._tied:
            _check_ties(self._tied)
        a = self._args
        on_device = isinstance(lr, torch.Tensor)
        rate = self.lr if lr is None or on_device else float(lr)
        given = (rate, self.beta1, self.beta2, self.eps, grad_scale, self.seed)
        if given != self._given:
            self._check_hyper(rate, grad_scale)
            a.lr, a.beta1, a.beta2, a.eps, a.grad_scale, a.seed = given
            self._given = given
        a.lr_device = _scalar_input(lr, 1, self.device, "lr") if on_device else None
        a.clip = _scalar_input(clip, 2, self.device, "clip") if clip is not None else None
        stream = _current_stream(self.device.index)
        if stream not in self._streams and not _capturing(self.device.index):
            # the allocator may not reuse the states' memory under this stream's work
            for t in self._state.values():
                t.record_stream(torch.cuda.current_stream(self.device))
            self._streams.add(stream)
        rc = self.lib.falcom_adamw_step(self._h, self._args_ref, stream)
        if rc != 0:
            raise RuntimeError(f"falcom_adamw_step failed ({rc})")
        if self._autograd:
            # a graph that saved a parameter's old value must not use the new one
            torch.autograd.graph.increment_version(self._autograd)

    def load_state(self, state: Dict[str, torch.Tensor]) -> None:
        """Copies a `state` of the same layout into this one's (in place)."""
        if set(state) != set(self._state):
            raise ValueError(f"state has {sorted(state)}, wanted {sorted(self._state)}")
        for k, t in self._state.items():
            if state[k].shape != t.shape or state[k].dtype != t.dtype:
                raise ValueError(f"state {k} is {state[k].dtype} {tuple(state[k].shape)}, wanted {t.dtype} "
                                 f"{tuple(t.shape)}")
        for k, t in self._state.items():
            t.copy_(state[k])

    def moments(self) -> List[tuple]:
        """Both moments of every parameter, as new float32 tensors (m, v) in
        the parameter's shape and memory order."""
        flat = {"m": self._state["m"], "v": self._state["v"]}
        if self.state_bits == 8:
            flat = {k: (t.float().view(-1, abi.ADAMW_BLOCK) * self._state[k + "_scale"][:, None]).view(-1)
                    for k, t in flat.items()}
            flat["v"] = flat["v"].square()
        out = []
        for p, o in zip(self.params, self.offsets):
            out.append(tuple(flat[k][o:o + p.numel()].clone().as_strided(p.shape, p.stride()) for k in "mv"))
        return out

    def errors(self) -> int:
        """Nonzero once a step gave up waiting for its own memory copies (8-bit
        states; never seen): what it left is then not to be used.  Waits for
        all work of the device."""
        return self.lib.falcom_adamw_errors(self._h) if self._h else 0

    def close(self) -> None:
        h, self._h = self._h, None
        if h:
            _retire(self.lib.falcom_adamw_graphs, self.lib.falcom_adamw_destroy, h,
                    (self._held, self._state))

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
