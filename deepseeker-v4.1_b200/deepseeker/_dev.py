"""Small helpers for passing torch tensors through the C ABI."""
from __future__ import annotations

import contextlib
import ctypes

import numpy as np
import torch
from torch.autograd import forward_ad


#: A clamp's limit is above this: what is not rounds to 0 in f32, which stands for no clamps.
LEAST_LIMIT = 2.0 ** -150


def stream_handle(device: torch.device | None = None) -> ctypes.c_void_p:
    """cudaStream_t of torch's current stream on `device`."""
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


_SAME = contextlib.nullcontext()


def on_device(device: torch.device):
    """Context in which `device` is the current one; nothing where it is already."""
    return _SAME if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def raw_stream(device: torch.device) -> int:
    """cudaStream_t of torch's current stream on `device` (a CUDA tensor's, so with an index) as an integer:
    what a call of a few microseconds can afford."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def rows_of(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """`t` (2-D) with rows that are contiguous runs, and their distance in elements; a copy where it has none."""
    rows, cols = t.shape
    ld, inner = t.stride()
    if inner == 1 or cols == 1:
        if rows <= 1:
            return t, cols
        if ld >= cols:
            return t, ld
    return t.contiguous(), cols


def new_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type (empty_like takes a third of empty's time and keeps strides)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def has_tangent(*ts) -> bool:
    """Whether one of `ts` carries a forward-mode derivative, which a result made through the C ABI would lose."""
    return forward_ad._current_level >= 0 and any(
        isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def require_cuda(t: torch.Tensor, name: str, dtype: torch.dtype | tuple | None = None) -> torch.Tensor:
    """Check that `t` is a CUDA tensor of the given dtype; return it contiguous."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dtype is not None:
        allowed = dtype if isinstance(dtype, tuple) else (dtype,)
        if t.dtype not in allowed:
            raise ValueError(f"{name} must have dtype {allowed}, got {t.dtype}")
    return t.contiguous()


def device_of(*ts: torch.Tensor) -> torch.device:
    for t in ts:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            return t.device
    return torch.device("cuda", torch.cuda.current_device())


def to_device(a, device: torch.device | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """numpy array / bytes / tensor -> contiguous CUDA tensor (host data is copied)."""
    if isinstance(a, (bytes, bytearray, memoryview)):
        a = np.frombuffer(a, dtype=np.uint8)
    if isinstance(a, np.ndarray):
        a = np.ascontiguousarray(a)
        if not a.flags.writeable:    # torch wants writable storage; the data is copied to the device anyway
            a = a.copy()
        t = torch.from_numpy(a)
    else:
        t = a
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    return t.to(device or torch.device("cuda"), non_blocking=False).contiguous()
