"""Layer norm with its backward pass: what stands in front of a layer's router and blocks.

    y = (x - mean) / sqrt(var + eps) * weight + bias      over the last dimension

(the reference has an RMS norm only, src/deepseeker/mlx_forward.py:45).
``layer_norm`` takes part in autograd (reverse mode; operands with forward-mode
derivatives are refused).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _abi
from ._dev import has_tangent, new_like, on_device, raw_stream, rows_of

_DTYPES = {torch.float32: _abi.DS_F32, torch.bfloat16: _abi.DS_BF16, torch.float16: _abi.DS_F16}
_MOST = 1 << 20   # features
_MOST_EPS = 2.0 ** 127


def _check(x, weight, bias, eps) -> torch.dtype:
    """Checks the operands; the type of the parameters."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("x must be a f32, bf16 or f16 CUDA tensor")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MOST:
        raise ValueError("x must be [..., H] with H in [1, 2^20]")
    dev, dtype = x.get_device(), None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.get_device() != dev or t.shape != x.shape[-1:]:
            raise ValueError(f"{name} must be a tensor [H] on x's device")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise ValueError(f"{name} must be f32 or of x's type")
        if dtype is not None and t.dtype != dtype:
            raise ValueError("weight and bias must have one type")
        dtype = t.dtype
    if not 0 <= eps < _MOST_EPS:
        raise ValueError("eps must be a number >= 0 that f32 holds")
    if has_tangent(x, weight, bias):
        raise ValueError("layer_norm has no forward-mode derivatives: an operand is a dual tensor")
    return dtype or torch.float32


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device: int, rows: int, cols: int) -> int:
    """Workspace of a backward pass with parameters on `device`, the current one (sizes follow its SMs)."""
    n = ctypes.c_size_t(0)
    _abi.check(_abi.lib().ds_layer_norm_backward_workspace_size(rows, cols, ctypes.byref(n)),
               "ds_layer_norm_backward_workspace_size")
    return n.value


def _forward(x, weight, bias, eps, kind, keep: bool):
    """y, and what the backward pass reads beside its operands."""
    xr, ld = rows_of(x)
    weight, bias, dev = _dense(weight), _dense(bias), x.device
    y = new_like(x)
    stats = torch.empty((x.shape[0], 2), dtype=torch.float32, device=dev) if keep else None
    with on_device(dev):
        _abi.check(_abi.lib().ds_layer_norm(
            xr.data_ptr(), _DTYPES[x.dtype], x.shape[0], x.shape[1], ld, None if weight is None else weight.data_ptr(),
            None if bias is None else bias.data_ptr(), _DTYPES[kind], eps, y.data_ptr(),
            None if stats is None else stats.data_ptr(), raw_stream(dev)), "ds_layer_norm")
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, kind):
        y, stats = _forward(x, weight, bias, eps, kind, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.kind = kind
        return y

    @staticmethod
    def backward(ctx, dy):
        # a graph of the gradients (create_graph) is refused where it is used; plain passes skip that wrapper's cost
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _backward(ctx, dy):
    x, weight, stats = ctx.saved_tensors
    (rows, cols), dev = x.shape, x.device
    (xr, ld), (dr, ld_dy), weight = rows_of(x), rows_of(dy), _dense(weight)
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dx = new_like(x) if need_x else None
    dw, db = (torch.empty(cols, dtype=ctx.kind, device=dev) if need else None for need in (need_w, need_b))
    n, ws = 0, None
    with on_device(dev):
        if need_w or need_b:
            n = _workspace_bytes(dev.index, rows, cols)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _abi.check(_abi.lib().ds_layer_norm_backward(
            xr.data_ptr(), _DTYPES[x.dtype], rows, cols, ld, None if weight is None else weight.data_ptr(),
            _DTYPES[ctx.kind], stats.data_ptr(), dr.data_ptr(), ld_dy,
            *[None if t is None else t.data_ptr() for t in (dx, dw, db, ws)], n, raw_stream(dev)),
            "ds_layer_norm_backward")
    return dx, dw, db, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """x [..., H] f32, bf16 or f16 -> the same shape and type; weight and bias
    [H], f32 or of x's type (None: 1 and 0).  Differentiable in x, weight and
    bias; between the passes it keeps x and two f32 values per row.

    Statistics and sums are f32, each result is rounded once.  Squares of
    differences to the mean have to stay inside f32: magnitudes up to about
    1e19 / sqrt(H).
    """
    kind = _check(x, weight, bias, eps)
    rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(rows, weight, bias, eps, kind)
    else:
        y = _forward(rows, weight, bias, eps, kind, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)
