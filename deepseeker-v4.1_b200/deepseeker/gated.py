"""Dense gated feed-forward block with its backward pass (16-bit weights).

    y = (silu(min(x W1^T, L)) * clip(x W3^T, -L, L)) W2^T

the block that a layer's shared expert or a layer without routing evaluates
(the reference's ``shared_fn``, src/deepseeker/mlx_runner.py:776-781), for
prompts, single tokens and training.  ``gated_ffn`` takes part in autograd.
"""
from __future__ import annotations

import ctypes

import torch

from . import _abi
from ._dev import stream_handle

_DTYPES = {torch.bfloat16: _abi.DS_BF16, torch.float16: _abi.DS_F16}


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A 2-D tensor whose rows are contiguous runs, and their distance in elements."""
    rows, cols = t.shape
    if t.stride(1) == 1 or cols == 1:
        ld = t.stride(0) if rows > 1 else cols
        if ld >= cols:
            return t, ld
    return t.contiguous(), cols


def _check(x, w1, w3, w2, limit) -> tuple[int, int]:
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("x must be a bf16 or f16 CUDA tensor")
    if x.dim() < 1:
        raise ValueError("x must be [..., hidden]")
    for name, w in (("w1", w1), ("w3", w3), ("w2", w2)):
        if not isinstance(w, torch.Tensor) or w.device != x.device or w.dtype != x.dtype or w.dim() != 2:
            raise ValueError(f"{name} must be a 2-D {x.dtype} tensor on x's device")
    inter, hidden = w1.shape
    if x.shape[-1] != hidden or w3.shape != (inter, hidden) or w2.shape != (hidden, inter):
        raise ValueError("x [..., H], w1 [I, H], w3 [I, H], w2 [H, I] expected")
    if hidden < 1 or inter < 1:
        raise ValueError("hidden and inter must be at least 1")
    if limit is not None and not limit > 0:
        raise ValueError("limit must be positive, or None for no clamps")
    return hidden, inter


def _desc(x, w1, w3, w2, limit) -> tuple[_abi.DsGatedFfn, tuple]:
    """The call's descriptor, and the tensors that it points into."""
    (x, lx), (w1, l1), (w3, l3), (w2, l2) = _rows(x), _rows(w1), _rows(w3), _rows(w2)
    d = _abi.DsGatedFfn(x.shape[0], w1.shape[1], w1.shape[0], _DTYPES[x.dtype], limit or 0.0, x.data_ptr(),
                        w1.data_ptr(), w3.data_ptr(), w2.data_ptr(), lx, l1, l3, l2)
    return d, (x, w1, w3, w2)


def _workspace(size_fn: str, device, *args) -> torch.Tensor:
    n = ctypes.c_size_t(0)
    _abi.call(size_fn, *args, ctypes.byref(n))
    return torch.empty(n.value, dtype=torch.uint8, device=device)


def _forward(x, w1, w3, w2, limit, keep: bool):
    d, hold = _desc(x, w1, w3, w2, limit)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = pre = None
    if keep:
        cols = (w1.shape[0] + 7) // 8 * 8
        h = torch.empty(x.shape[0], cols, dtype=x.dtype, device=x.device)
        pre = torch.empty(2, x.shape[0], cols, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        ws = _workspace("ds_gated_ffn_workspace_size", x.device, ctypes.byref(d), int(keep))
        _abi.call("ds_gated_ffn", ctypes.byref(d), y.data_ptr(), h.data_ptr() if keep else None,
                  pre.data_ptr() if keep else None, ws.data_ptr(), ws.numel(), stream_handle(x.device))
    return y, h, pre


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w3, w2, limit):
        y, h, pre = _forward(x, w1, w3, w2, limit, True)
        ctx.save_for_backward(x, w1, w3, w2, h, pre)
        ctx.limit = limit
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w1, w3, w2, h, pre = ctx.saved_tensors
        d, hold = _desc(x, w1, w3, w2, ctx.limit)
        dy, ld = _rows(dy)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None
                 for t, need in zip((x, w1, w3, w2), ctx.needs_input_grad)]
        with torch.cuda.device(x.device):
            ws = _workspace("ds_gated_ffn_backward_workspace_size", x.device, ctypes.byref(d), dy.data_ptr(), ld)
            _abi.call("ds_gated_ffn_backward", ctypes.byref(d), h.data_ptr(), pre.data_ptr(), dy.data_ptr(), ld,
                      *(None if g is None else g.data_ptr() for g in grads), ws.data_ptr(), ws.numel(),
                      stream_handle(x.device))
        return (*grads, None)


def gated_ffn(x: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor,
              limit: float | None = None) -> torch.Tensor:
    """x [..., H], w1 and w3 [I, H], w2 [H, I], all bf16 or all f16 -> [..., H].

    ``limit``: the clamps of the gate (from above) and of the up projection
    (both sides), as in ``moe_layer``; None for none.  Differentiable in x and
    the weights: between the passes the block keeps h (16 bits) and both
    pre-activations (f32), 10 bytes per token and intermediate feature.  The
    gradient of a clamped value is 0.
    """
    hidden, _ = _check(x, w1, w3, w2, limit)
    rows = x.reshape(-1, hidden)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w1, w3, w2)):
        return _GatedFFN.apply(rows, w1, w3, w2, limit).view(x.shape)
    return _forward(rows, w1, w3, w2, limit, False)[0].view(x.shape)


def status(device: torch.device | None = None) -> int:
    """Error bits of the block's calls on `device` since the last query (2: a
    bounded device wait gave up; outputs are then undefined).  Waits for the stream."""
    err = torch.zeros(1, dtype=torch.int32)
    with torch.cuda.device(device):
        _abi.call("ds_gated_ffn_status", err.data_ptr(), stream_handle(device))
        torch.cuda.current_stream(device).synchronize()
    return int(err[0])
