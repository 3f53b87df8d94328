"""Argument checks and the launch shared by the operator wrappers.

A decode step calls several small operators, and a model calls them with the
same few signatures over and over.  A wrapper therefore keeps, per signature
(shapes, strides, types, devices and options of the arguments), the checked
argument struct without its pointers; a call with a known signature copies it
and sets the pointers."""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from .attention import status_word

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_status_ptrs = {}  # device index -> address of its status word (status_word keeps the tensor)


def _stream_of(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# (torch's own lookup without the Stream object around it, where there is one)
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream_of)


def status_ptr(index: int) -> int:
    ptr = _status_ptrs.get(index)
    if ptr is None:
        ptr = _status_ptrs[index] = status_word(torch.device("cuda", index)).data_ptr()
    return ptr


def sig(x: Optional[Tensor]):
    """What of a tensor the checks and the argument struct go by."""
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device())


class Plans(dict):
    """Checked argument structs by signature, at most a few hundred."""

    def keep(self, key, given, used, args) -> None:
        """Keeps ``args`` unless a tensor had to be copied for it."""
        if all(x is y for x, y in zip(given, used)):
            if len(self) >= 512:
                self.clear()
            self[key] = args


def copy(args):
    """A struct of one call's own."""
    return type(args).from_buffer_copy(args)


def tracked(*tensors: Optional[Tensor]) -> bool:
    """Whether autograd may want something of a call: an input that requires a
    gradient with the gradients on, or any call within a forward-mode level
    (its tensors may carry tangents whatever they require)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                return True
    return False


class _NoBackward(torch.autograd.Function):
    """A call whose results carry no gradient: a backward that reaches it
    raises, as forward-mode tangents do, where detached results would lose
    them silently."""

    @staticmethod
    def forward(ctx, what, run, *inputs):
        ctx.what = what
        return run()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what} has no backward: call it under torch.no_grad() or on detached tensors")


def no_backward(what: str, run, *inputs: Optional[Tensor]):
    """``run()`` (the results of a call on ``inputs``, some of them ``tracked``)
    with that mark."""
    return _NoBackward.apply(what, run, *inputs)


def dtype_code(x: Tensor, name: str) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {x.dtype} of {name}: bfloat16, float16 or float32")
    return code


def dense_d(x: Tensor) -> Tensor:
    return x if x.stride(-1) == 1 else x.contiguous()


def dense4(x: Tensor) -> Tuple[Tensor, "_lib.AiTensor4"]:
    """``x`` with its last dimension contiguous, and what the library is told of it."""
    b, h, t, d = x.stride()
    if d != 1:
        x = x.contiguous()
        b, h, t, _ = x.stride()
    return x, _lib.AiTensor4(x.data_ptr(), b, h, t)


def strides4(x: Tensor) -> "_lib.AiTensor4":
    return _lib.AiTensor4(None, *x.stride()[:3])


def on_device(name: str, x: Tensor, index: int) -> None:
    if x.get_device() != index:
        raise RuntimeError(f"{name} is on {x.device}, expected cuda:{index}")


def cuda_index(name: str, x: Tensor) -> int:
    if not x.is_cuda:
        raise RuntimeError(f"autoindexer_b200 operators run on CUDA tensors only ({name} is on {x.device})")
    return x.get_device()


def _typed(name: str, x: Tensor, dtype, shape: Tuple[int, ...], index: int) -> None:
    if x.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    if x.get_device() != index:
        on_device(name, x, index)


def ints(name: str, x: Tensor, shape: Tuple[int, ...], index: int) -> Tensor:
    """An int32 tensor of ``shape`` on the device with its last dimension contiguous."""
    _typed(name, x, torch.int32, shape, index)
    return x if x.stride(-1) == 1 else x.contiguous()


def floats(name: str, x: Tensor, shape: Tuple[int, ...], index: int) -> Tensor:
    """A contiguous float32 tensor of ``shape`` on the device."""
    _typed(name, x, torch.float32, shape, index)
    return x.contiguous()


def dense_positions(positions: Tensor) -> Tensor:
    return positions if positions.stride(-1) == 1 else positions.contiguous()


def positions_stride(positions: Tensor) -> int:
    """Elements from a batch row's ids to the next one's; 0: one row for all."""
    strides = positions.stride()
    return strides[0] if len(strides) == 2 and positions.size(0) > 1 else 0


def check_rope(a, rope, positions: Optional[Tensor], batch: int, seq_len: int, head_dim: int, index: int):
    """Sets what ``a`` says of the rotary table and the position ids; returns
    (cos, sin, positions) as the kernels read them, whose pointers
    ``point_rope`` sets."""
    if rope is None:
        if positions is not None:
            raise ValueError("positions without a rope table")
        return None, None, None
    if positions is None:
        raise ValueError("a rope table needs positions")
    cos, sin = rope
    n = cos.shape[0]
    shape = (n, head_dim // 2)
    cos, sin = floats("rope cos", cos, shape, index), floats("rope sin", sin, shape, index)
    if n == 0:
        raise ValueError("the rope table is empty")
    is_int64 = positions.dtype is torch.int64
    if not is_int64 and positions.dtype is not torch.int32:
        raise TypeError(f"positions must be int64 or int32, got {positions.dtype}")
    dims = positions.shape
    rows = 1 if len(dims) == 1 else dims[0] if dims else 0
    if len(dims) > 2 or rows not in (1, batch) or dims[-1] != seq_len:
        raise ValueError(f"positions must be ({seq_len},) or ({batch}, {seq_len}), got {tuple(dims)}")
    on_device("positions", positions, index)
    positions = dense_positions(positions)
    a.n_pos = n
    a.pos = _lib.AiPositions(None, positions_stride(positions), is_int64)
    return cos, sin, positions


def point_rope(a, cos: Optional[Tensor], sin: Optional[Tensor], positions: Optional[Tensor]) -> None:
    if cos is not None:
        a.rope_cos, a.rope_sin, a.pos.ptr = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()


def head_weight(name: str, w: Optional[Tensor], x: Tensor, index: int) -> Optional[Tensor]:
    """A norm weight ``(D,)`` of ``x``'s dtype or float32."""
    if w is None:
        return None
    if w.shape != x.shape[-1:]:
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(w.shape)}")
    if w.dtype is not x.dtype and w.dtype is not torch.float32:
        raise TypeError(f"{name} must be {x.dtype} or float32, got {w.dtype}")
    on_device(name, w, index)
    return w.contiguous()


def workspace(query, args, device: torch.device, what: str) -> Optional[Tensor]:
    """Allocates what the library asks for and sets it in ``args``."""
    n = ctypes.c_size_t(0)
    code = query(args, n)
    if code:
        _lib.check(code, what)
    if not n.value:
        return None
    ws = torch.empty(n.value, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), n.value
    return ws


def launch(fn, args, index: int, what: str) -> None:
    """Runs one library call on the device's current stream."""
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return launch(fn, args, index, what)
    code = fn(args, raw_stream(index))
    if code:
        _lib.check(code, what)
