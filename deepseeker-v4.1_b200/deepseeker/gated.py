"""Dense gated feed-forward block with its backward pass (16-bit weights).

    y = (silu(min(x W1^T, L)) * clip(x W3^T, -L, L)) W2^T

the block that a layer's shared expert or a layer without routing evaluates
(the reference's ``shared_fn``, src/deepseeker/mlx_runner.py:776-781), for
prompts, single tokens and training.  ``gated_ffn`` takes part in autograd
(reverse mode; operands with forward-mode derivatives are refused).
"""
from __future__ import annotations

import ctypes

import torch

from . import _abi
from ._dev import LEAST_LIMIT, has_tangent, new_like, on_device, raw_stream, rows_of, stream_handle

_DTYPES = {torch.bfloat16: _abi.DS_BF16, torch.float16: _abi.DS_F16}
_MOST = 1 << 17   # hidden, inter


def _check(x, w1, w3, w2, limit) -> int:
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("x must be a bf16 or f16 CUDA tensor")
    dev, dtype = x.get_device(), x.dtype
    for name, w in (("w1", w1), ("w3", w3), ("w2", w2)):
        if not isinstance(w, torch.Tensor) or w.get_device() != dev or w.dtype != dtype or w.dim() != 2:
            raise ValueError(f"{name} must be a 2-D {dtype} tensor on x's device")
    inter, hidden = w1.shape
    if x.dim() < 1 or x.shape[-1] != hidden or w3.shape != (inter, hidden) or w2.shape != (hidden, inter):
        raise ValueError("x [..., H], w1 [I, H], w3 [I, H], w2 [H, I] expected")
    if not (1 <= hidden <= _MOST and 1 <= inter <= _MOST):   # before they become 32-bit fields
        raise ValueError("hidden and inter must be in [1, 2^17]")
    if limit is not None and not limit > LEAST_LIMIT:
        raise ValueError("limit must be positive in f32, or None for no clamps")
    if has_tangent(x, w1, w3, w2):
        raise ValueError("gated_ffn has no forward-mode derivatives: an operand is a dual tensor")
    return hidden


def _desc(x, w1, w3, w2, limit) -> tuple[_abi.DsGatedFfn, tuple]:
    """The call's descriptor, and the tensors that it points into."""
    inter, hidden = w1.shape
    if x.is_contiguous() and w1.is_contiguous() and w3.is_contiguous() and w2.is_contiguous():
        lx = l1 = l3 = hidden
        l2 = inter
    else:
        (x, lx), (w1, l1), (w3, l3), (w2, l2) = rows_of(x), rows_of(w1), rows_of(w3), rows_of(w2)
    d = _abi.DsGatedFfn(x.shape[0], hidden, inter, _DTYPES[x.dtype], limit or 0.0, x.data_ptr(), w1.data_ptr(),
                        w3.data_ptr(), w2.data_ptr(), lx, l1, l3, l2)
    return d, (x, w1, w3, w2)


def _pre_bytes(x, w1) -> int:
    """Bytes of g and u in f32, which lead the buffer kept for the backward pass; h follows."""
    return 8 * x.shape[0] * ((w1.shape[0] + 7) // 8 * 8)


def _forward(x, w1, w3, w2, limit, keep: bool):
    """y, and the buffer (pre-activations, h) that the backward pass reads."""
    d, hold = _desc(x, w1, w3, w2, limit)
    lib, ref, dev = _abi.lib(), ctypes.byref(d), x.device
    y = new_like(x)
    kept = h = pre = None
    with on_device(dev):
        if keep:
            n = _pre_bytes(x, w1)
            kept = torch.empty(n + n // 4, dtype=torch.uint8, device=dev)
            pre = kept.data_ptr()
            h = pre + n
        n = ctypes.c_size_t(0)
        _abi.check(lib.ds_gated_ffn_workspace_size(ref, keep, ctypes.byref(n)), "ds_gated_ffn_workspace_size")
        ws = torch.empty(n.value, dtype=torch.uint8, device=dev) if n.value else None
        _abi.check(lib.ds_gated_ffn(ref, y.data_ptr(), h, pre, None if ws is None else ws.data_ptr(), n.value,
                                    raw_stream(dev)), "ds_gated_ffn")
    return y, kept


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w3, w2, limit):
        y, kept = _forward(x, w1, w3, w2, limit, True)
        ctx.save_for_backward(x, w1, w3, w2, kept)
        ctx.limit = limit
        return y

    @staticmethod
    def backward(ctx, dy):
        # a graph of the gradients (create_graph) is refused where it is used; plain passes skip that wrapper's cost
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _backward(ctx, dy):
    x, w1, w3, w2, kept = ctx.saved_tensors
    d, hold = _desc(x, w1, w3, w2, ctx.limit)
    dy, ld = rows_of(dy)
    lib, ref, dev = _abi.lib(), ctypes.byref(d), x.device
    grads = [new_like(t) if need else None for t, need in zip((x, w1, w3, w2), ctx.needs_input_grad)]
    pre, n = kept.data_ptr(), ctypes.c_size_t(0)
    with on_device(dev):
        _abi.check(lib.ds_gated_ffn_backward_workspace_size(ref, dy.data_ptr(), ld, ctypes.byref(n)),
                   "ds_gated_ffn_backward_workspace_size")
        ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
        _abi.check(lib.ds_gated_ffn_backward(ref, pre + _pre_bytes(x, w1), pre, dy.data_ptr(), ld,
                                             *[None if g is None else g.data_ptr() for g in grads],
                                             ws.data_ptr(), n.value, raw_stream(dev)), "ds_gated_ffn_backward")
    return (*grads, None)


_backward_once = torch.autograd.function.once_differentiable(_backward)


def gated_ffn(x: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor,
              limit: float | None = None) -> torch.Tensor:
    """x [..., H], w1 and w3 [I, H], w2 [H, I], all bf16 or all f16 -> [..., H].

    ``limit``: the clamps of the gate (from above) and of the up projection
    (both sides), as in ``moe_layer``; None for none.  Differentiable in x and
    the weights: between the passes the block keeps h (16 bits) and both
    pre-activations (f32), 10 bytes per token and intermediate feature.  The
    gradient of a clamped value is 0, that of one that equals the limit (taken
    in f32) is not; the exact sums decide, not their f32 rounding.

    h and the gradients of both projections are operands of the next products
    and have their type.  In f16 one beyond 65,504 is infinite, and so is (or
    becomes NaN) what it enters: its row of y and dx, its column of a weight's
    gradient.  A ``limit`` up to 255 keeps h (at most limit^2) inside; without
    one, blocks whose h may grow that large belong in bf16.
    """
    hidden = _check(x, w1, w3, w2, limit)
    rows = x if x.dim() == 2 else x.reshape(-1, hidden)
    if torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w3.requires_grad or w2.requires_grad):
        y = _GatedFFN.apply(rows, w1, w3, w2, limit)
    else:
        y = _forward(rows, w1, w3, w2, limit, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


def status(device: torch.device | None = None) -> int:
    """Error bits of the block's calls on `device` since the last query (2: a
    bounded device wait gave up; outputs are then undefined).  Waits for the stream."""
    err = torch.zeros(1, dtype=torch.int32)
    with torch.cuda.device(device):
        _abi.check(_abi.lib().ds_gated_ffn_status(err.data_ptr(), stream_handle(device)), "ds_gated_ffn_status")
        torch.cuda.current_stream(device).synchronize()
    return int(err[0])
