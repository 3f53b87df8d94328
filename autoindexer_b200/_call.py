"""Argument checks and the launch shared by the operator wrappers."""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def dtype_code(x: Tensor, name: str) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {x.dtype} of {name}: bfloat16, float16 or float32")
    return code


def dense_d(x: Tensor) -> Tensor:
    return x if x.stride(-1) == 1 else x.contiguous()


def t4(x: Tensor) -> "_lib.AiTensor4":
    s = x.stride()
    return _lib.AiTensor4(x.data_ptr(), s[0], s[1], s[2])


def on_device(name: str, x: Tensor, device: torch.device) -> None:
    if x.device != device:
        raise RuntimeError(f"{name} is on {x.device}, expected {device}")


def cuda_device(name: str, x: Tensor) -> torch.device:
    if not x.is_cuda:
        raise RuntimeError(f"autoindexer_b200 operators run on CUDA tensors only ({name} is on {x.device})")
    return x.device


def ints(name: str, x: Tensor, shape: Tuple[int, ...], device: torch.device) -> Tensor:
    """An int32 tensor of ``shape`` on ``device`` with its last dimension contiguous."""
    if x.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {x.dtype}")
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    on_device(name, x, device)
    return x if x.stride(-1) == 1 else x.contiguous()


def floats(name: str, x: Tensor, shape: Tuple[int, ...], device: torch.device) -> Tensor:
    """A contiguous float32 tensor of ``shape`` on ``device``."""
    if x.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {x.dtype}")
    if tuple(x.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    on_device(name, x, device)
    return x.contiguous()


def fill_rope(a, rope, positions: Optional[Tensor], batch: int, seq_len: int, head_dim: int, device):
    """Sets the rotary table and the position ids of ``a``; returns the
    tensors to keep alive until the launch."""
    if rope is None:
        if positions is not None:
            raise ValueError("positions without a rope table")
        return None
    if positions is None:
        raise ValueError("a rope table needs positions")
    cos, sin = rope
    shape = (cos.shape[0], head_dim // 2)
    cos, sin = floats("rope cos", cos, shape, device), floats("rope sin", sin, shape, device)
    if shape[0] == 0:
        raise ValueError("the rope table is empty")
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"positions must be int64 or int32, got {positions.dtype}")
    rows = 1 if positions.dim() == 1 else positions.shape[0]
    if positions.dim() > 2 or positions.shape[-1] != seq_len or rows not in (1, batch):
        raise ValueError(f"positions must be ({seq_len},) or ({batch}, {seq_len}), got {tuple(positions.shape)}")
    on_device("positions", positions, device)
    if positions.stride(-1) != 1:
        positions = positions.contiguous()
    a.rope_cos, a.rope_sin, a.n_pos = cos.data_ptr(), sin.data_ptr(), shape[0]
    a.pos.ptr = positions.data_ptr()
    a.pos.stride_b = positions.stride(0) if rows > 1 else 0
    a.pos.is_int64 = positions.dtype == torch.int64
    return cos, sin, positions


def head_weight(name: str, w: Optional[Tensor], x: Tensor) -> Optional[Tensor]:
    """A norm weight ``(D,)`` of ``x``'s dtype or float32."""
    if w is None:
        return None
    if tuple(w.shape) != (x.shape[-1],):
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(w.shape)}")
    if w.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{name} must be {x.dtype} or float32, got {w.dtype}")
    on_device(name, w, x.device)
    return w.contiguous()


def workspace(query, args, device: torch.device, what: str) -> Optional[Tensor]:
    """Allocates what the library asks for and sets it in ``args``."""
    n = ctypes.c_size_t(0)
    _lib.check(query(ctypes.byref(args), ctypes.byref(n)), what)
    if not n.value:
        return None
    ws = torch.empty(n.value, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = ws.data_ptr(), n.value
    return ws


def launch(fn, args, device: torch.device, what: str) -> None:
    """Runs one library call on the device's current stream."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn(ctypes.byref(args), torch.cuda.current_stream(device).cuda_stream), what)
        return
    with torch.cuda.device(device):
        _lib.check(fn(ctypes.byref(args), torch.cuda.current_stream(device).cuda_stream), what)
