"""Balance loss of a router and its counts per expert, with gradients: what the routers of ``deepseeker.moe`` are
trained with.

The reference only serves (its routers: src/deepseeker/mlx_forward.py:62-81),
so the loss follows the usual definition: for a sequence of n valid tokens with
k of E experts each, c_e the times that expert e was chosen and P_e its mean
share of the scores,

    loss = sum_e (c_e E / (k n)) P_e

which is 1 where choices or scores are even.  ``balance_loss`` takes part in
autograd (reverse mode; the counts are taken as given).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _abi
from ._dev import has_tangent, new_like, on_device, raw_stream, rows_of

_DTYPES = {torch.float32: _abi.DS_F32, torch.bfloat16: _abi.DS_BF16, torch.float16: _abi.DS_F16}
_KINDS = {"softmax": _abi.DS_ROUTE_SOFTMAX, "sqrtsoftplus": _abi.DS_ROUTE_SQRTSOFTPLUS}
_MOST_EXPERTS, _MOST_TOP_K = 1024, 32


def _check(logits, ids, kind, valid, offsets) -> None:
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in _DTYPES or logits.dim() != 2:
        raise ValueError("logits must be a f32, bf16 or f16 CUDA tensor [tokens, experts]")
    dev, tokens = logits.get_device(), logits.shape[0]
    if not isinstance(ids, torch.Tensor) or ids.get_device() != dev or ids.dtype != torch.int32 or ids.dim() != 2:
        raise ValueError("ids must be an int32 tensor [tokens, top_k] on the logits' device")
    if ids.shape[0] != tokens or not 1 <= ids.shape[1] <= _MOST_TOP_K or tokens * ids.shape[1] >= 1 << 31:
        raise ValueError(f"ids must be [tokens, top_k], top_k in [1, {_MOST_TOP_K}], fewer than 2^31 in all")
    if not 1 <= logits.shape[1] <= _MOST_EXPERTS:
        raise ValueError(f"experts must be in [1, {_MOST_EXPERTS}]")
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {sorted(_KINDS)}")
    if valid is not None and (not isinstance(valid, torch.Tensor) or valid.get_device() != dev
                              or valid.dtype != torch.bool or valid.shape != (tokens,)):
        raise ValueError("valid must be a bool tensor [tokens] on the logits' device")
    if offsets is not None and (not isinstance(offsets, torch.Tensor) or offsets.get_device() != dev
                                or offsets.dtype not in (torch.int32, torch.int64) or offsets.dim() != 1
                                or not 1 <= offsets.shape[0] <= (1 << 24) + 1):
        raise ValueError("offsets must be an int32 or int64 tensor [sequences + 1] on the logits' device")
    if has_tangent(logits):
        raise ValueError("balance_loss has no forward-mode derivatives: logits is a dual tensor")


def _desc(logits, ids, kind, valid, offsets) -> tuple[_abi.DsBalance, tuple]:
    """The call's descriptor, and the tensors that it points into."""
    logits, ld = rows_of(logits)
    ids = None if ids is None else ids.contiguous()
    valid = None if valid is None else valid.contiguous()
    offsets = None if offsets is None else offsets.contiguous()
    tokens, experts = logits.shape
    d = _abi.DsBalance(logits.data_ptr(), tokens, ld, _DTYPES[logits.dtype], experts,
                       1 if ids is None else ids.shape[1], kind, None if ids is None else ids.data_ptr(),
                       None if valid is None else valid.data_ptr(), None if offsets is None else offsets.data_ptr(),
                       offsets is not None and offsets.dtype == torch.int64,
                       1 if offsets is None else offsets.shape[0] - 1)
    return d, (logits, ids, valid, offsets)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device: int, tokens: int, experts: int, sequences: int) -> int:
    """Workspace of a call on `device`, the current one (sizes follow its SMs)."""
    d = _abi.DsBalance(256, tokens, experts, _abi.DS_F32, experts, 1, _abi.DS_ROUTE_SOFTMAX, 256, None, 256, 0, sequences)
    n = ctypes.c_size_t(0)
    _abi.check(_abi.lib().ds_balance_loss_workspace_size(ctypes.byref(d), ctypes.byref(n)), "ds_balance_loss_workspace_size")
    return n.value


def _forward(logits, ids, kind, valid, offsets):
    """loss, counts, and the coefficients that the backward pass reads."""
    d, hold = _desc(logits, ids, kind, valid, offsets)
    dev, sequences, experts = logits.device, d.sequences, d.experts
    lead = () if offsets is None else (sequences,)
    loss = torch.empty(lead, dtype=torch.float32, device=dev)
    counts = torch.empty((*lead, experts), dtype=torch.int32, device=dev)
    coef = torch.empty(sequences * experts, dtype=torch.float32, device=dev)
    with on_device(dev):
        n = _workspace_bytes(dev.index, d.tokens, experts, sequences)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)   # of its own: the coefficients outlive the call
        _abi.check(_abi.lib().ds_balance_loss(ctypes.byref(d), loss.data_ptr(), counts.data_ptr(), coef.data_ptr(),
                                              ws.data_ptr(), n, raw_stream(dev)), "ds_balance_loss")
    return loss, counts, coef


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, kind, valid, offsets):
        loss, counts, coef = _forward(logits, ids, kind, valid, offsets)
        ctx.save_for_backward(logits, valid, offsets, coef)
        ctx.kind = kind
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)   # of the counts, which have none
        return loss, counts

    @staticmethod
    def backward(ctx, dloss, _):
        if dloss is None:
            return None, None, None, None, None
        # a graph of the gradients (create_graph) is refused where it is used; plain passes skip that wrapper's cost
        return _backward_once(ctx, dloss) if torch.is_grad_enabled() else _backward(ctx, dloss)


def _backward(ctx, dloss):
    logits, valid, offsets, coef = ctx.saved_tensors
    d, hold = _desc(logits, None, ctx.kind, valid, offsets)
    dloss, dev = dloss.contiguous(), logits.device
    dlogits = new_like(logits)
    with on_device(dev):
        _abi.check(_abi.lib().ds_balance_loss_backward(ctypes.byref(d), coef.data_ptr(), dloss.data_ptr(),
                                                       dlogits.data_ptr(), raw_stream(dev)), "ds_balance_loss_backward")
    return dlogits, None, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def balance_loss(logits: torch.Tensor, ids: torch.Tensor, kind: str = "softmax", valid: torch.Tensor | None = None,
                 offsets: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, counts) of a router's logits [T, E] (f32, bf16, f16) and the
    experts that it chose, ids [T, k] int32 (``moe.route_softmax_topk``,
    ``moe.route_sqrtsoftplus``; -1, like any number outside [0, E), stands for
    no expert, and every entry counts, a repeated one too).

    kind: the scores whose shares are balanced, "softmax" or "sqrtsoftplus"
    (``sqrt(softplus(l))`` over its sum).  valid [T] bool: rows where it is
    False are not looked at.  offsets [S + 1] int32 or int64, ascending: rows
    offsets[s] .. offsets[s + 1] - 1 are sequence s, with a loss and counts of
    its own; other rows belong to none.  Without offsets all rows are one
    sequence.

    loss f32, 0-d or [S], is differentiable in the logits (rows that are not
    valid or in no sequence get 0); counts int32 [E] or [S, E].  A sequence
    without valid tokens has loss 0.  Sums are f32; scores below 2^-126 are 0
    (square roots of softplus from logits of -174.7 on), and a row of none but
    such has no shares and no gradient.
    """
    _check(logits, ids, kind, valid, offsets)
    kind = _KINDS[kind]
    if torch.is_grad_enabled() and logits.requires_grad:
        return _BalanceLoss.apply(logits, ids, kind, valid, offsets)
    return _forward(logits, ids, kind, valid, offsets)[:2]
