"""Gradients of the dense gated block (deepseeker.gated) where many
pre-activations lie close to the clamps' limit.

A clamp's derivative jumps at the limit, so an element whose g or |u| is taken
to be on the wrong side of it has a whole gradient where it should have none.
The definition decides by the exact sums: no allowance is made for elements
that f32 sums bring to the other side.

Tolerance, as without clamps: with v half the 16-bit type's unit roundoff
(2^-9 bf16, 2^-12 f16), every output is a sum of products a b with one factor
rounded once (0.85 v in the root mean square) and is rounded once itself, so
  |error|_2 <= v |output|_2 + 0.58 v (1 + 3 / sqrt(n)) |R|_2,  R^2 = sum a^2 b^2,
n the smaller of the number of outputs and of rounded factors, plus f16's
spacing at 0 (2^-24) per rounding.
"""
from __future__ import annotations

import pytest
import torch

from deepseeker import gated

pytestmark = pytest.mark.gpu
HALF_UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


def close_to(T, H, I, dtype, device, limit, peak=0, seed=0):
    """A block whose g and |u| are the limit give or take 2^-13 of it: a part of
    the contraction adds up to +-limit exactly (half of it ones times
    +-limit / n, a power of two), the rest to small normal values.  ``peak``: on
    the way there the sums rise to peak times the limit and come back.  Three
    rows have g = limit and |u| = limit exactly."""
    gen = torch.Generator(device=device).manual_seed(seed)
    n = lambda r, c: torch.randn(r, c, generator=gen, device=device)  # noqa: E731
    flat = 1 << ((H // 2).bit_length() - 1)            # a power of two, at most half of H
    x, w1, w3 = n(T, H), n(I, H), n(I, H)
    small = 2.0 ** -13 * limit * (H - flat) ** -0.5
    x[:, :flat] = 1.0
    sign = torch.where(torch.rand(I, 1, generator=gen, device=device) < 0.5, -1.0, 1.0)
    for w, s in ((w1, 1.0), (w3, sign)):
        w *= small
        w[:, :flat] = s * limit / flat
        if peak:                                       # + p, - p, and once the limit in between
            w[:, : flat // 2] = s * limit / flat * 2 * (peak + 1)
            w[:, flat // 2: flat] = -s * limit / flat * 2 * peak
    x[:3, flat:] = 0.0
    return (x.to(dtype), w1.to(dtype), w3.to(dtype), (n(H, I) * I ** -0.5).to(dtype)), n(T, H).to(dtype)


def reference(ins, dy, limit):
    """Outputs and gradients of the definition in 64 bits, and (|R|, n) of each."""
    x, w1, w3, w2, dy = (t.detach().double() for t in (*ins, dy))
    g, u = (x @ w1.T).requires_grad_(), (x @ w3.T).requires_grad_()
    gc, uc = g.clamp(max=limit), u.clamp(-limit, limit)
    h = gc * torch.sigmoid(gc) * uc
    dg, du = torch.autograd.grad(h, (g, u), dy @ w2)
    h = h.detach()
    s = lambda t: t.square()  # noqa: E731
    want = (h @ w2.T, dg @ w1 + du @ w3, dg.T @ x, du.T @ x, dy.T @ h)
    sums = (s(h) @ s(w2).T, s(dg) @ s(w1) + s(du) @ s(w3), s(dg).T @ s(x), s(du).T @ s(x), s(dy).T @ s(h))
    return want, [(float(r.sum().sqrt()), min(r.numel(), h.numel())) for r in sums]


def run(ins, dy, limit):
    a = [t.detach().requires_grad_() for t in ins]
    y = gated.gated_ffn(*a, limit=limit)
    return (y.detach(), *torch.autograd.grad(y, a, dy))


def check(ins, dy, limit):
    dtype, got = dy.dtype, run(ins, dy, limit)
    for name, a, b, (R, n) in zip(("y", "dx", "dw1", "dw3", "dw2"), got, *reference(ins, dy, limit)):
        v, err = HALF_UNIT[dtype], float((a.double() - b).norm())
        bound = v * float(b.norm()) + 0.58 * v * (1 + 3 / n ** 0.5) * R + 2.0 ** -23 * b.numel() ** 0.5
        assert err <= bound, f"{name}: {err} > {bound} (relative {err / float(b.norm()):.2e})"
    assert gated.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,I,limit,peak", [
    (5, 64, 40, 1.0, 0), (16, 4096, 264, 0.5, 0), (37, 512, 256, 2.0, 0), (100, 1000, 201, 1.0, 0), (128, 2048, 136, 1.0, 16),
    (129, 256, 264, 1.0, 0), (300, 1000, 203, 0.5, 0), (333, 4096, 72, 1.0, 0), (600, 2048, 520, 4.0, 16), (300, 16, 64, 1.0, 0)])
def test_values_close_to_the_limit(T, H, I, limit, peak, dtype, cuda):
    check(*close_to(T, H, I, dtype, cuda, limit, peak, seed=T + H), limit)


@pytest.mark.parametrize("T", [50, 200])
def test_strided_operands_close_to_the_limit(T, cuda):
    """Unaligned operands behind NaN: only the operands' own values decide."""
    ins, dy = close_to(T, 520, 72, torch.float16, cuda, 1.0, seed=T)
    want = run(ins, dy, 1.0)
    check(ins, dy, 1.0)
    for pad, off in ((8, 8), (5, 3), (4, 0)):
        views = []
        for t in (*ins, dy):
            big = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=cuda)
            big[:, off:off + t.shape[1]] = t
            views.append(big[:, off:off + t.shape[1]])
        assert all(torch.equal(a, b) for a, b in zip(run(views[:4], views[4], 1.0), want)), (pad, off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,I,limit", [(2048, 4096, 2048, 1.0), (3000, 1001, 1003, 1.5), (1500, 640, 4096, 1.5), (64, 2048, 4096, 1.5)])
def test_normal_values_reach_the_clamps(T, H, I, limit, dtype, cuda):
    """Pre-activations of unit variance: a few per ten million lie within the error of an f32 sum of the limit."""
    gen = torch.Generator(device=cuda).manual_seed(T)
    n = lambda r, c, s: (torch.randn(r, c, generator=gen, device=cuda) * s).to(dtype)  # noqa: E731
    check((n(T, H, 1.0), n(I, H, H ** -0.5), n(I, H, H ** -0.5), n(H, I, I ** -0.5)), n(T, H, 1.0), limit)


def test_wide_spread_values(cuda):
    """Rows of very different size, with single large values that cancel: the distance at which a sum may be
    on the wrong side goes by the operands, not by the limit."""
    for T in (40, 300):
        (x, w1, w3, w2), dy = close_to(T, 1024, 96, torch.bfloat16, cuda, 1.0, seed=T)
        x[:, -1], x[:, -2] = 2.0 ** 10, 2.0 ** 10       # + 256 at the end of every sum, and - 256
        w1[:, -1], w1[:, -2], w3[:, -1], w3[:, -2] = 0.25, -0.25, -0.25, 0.25
        check((x, w1, w3, w2), dy, 1.0)
