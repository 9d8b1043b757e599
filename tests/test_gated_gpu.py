"""Dense gated feed-forward block (deepseeker.gated): forward and gradients
against the formulas in 64 bits.

Tolerances.  Let v be half the 16-bit type's unit roundoff (2^-9 bf16, 2^-12
f16): rounding to nearest is off by at most 2 v of the value, and by 0.85 v in
the root mean square over values of all mantissas.  Every output is a sum of
products a b of which one factor a (h, dg or du) was rounded once, and is
rounded once itself: independent errors of 0.85 v |output| and 0.85 v R with
R^2 = sum_k a_k^2 b_k^2 (about the output's own square unless the sum
cancels).  Where R = |output| that is 1.2 v |output| together; asserted is
  |error|_2 <= v |output|_2 + 0.58 v (1 + 3 / sqrt(n)) |R|_2,
1.58 v there, the last factor for the spread of the 2-norm of n independent
errors (n: the smaller of the number of outputs and of rounded factors), plus
ATOL per value (f16's spacing at 0, 2^-24, once per rounding).  The f32
accumulation of a few thousand terms adds 1e-3 v.

A clamp's derivative jumps at the limit, so a g or |u| that the f32 sums bring
to the other side of it changes a whole gradient.  Each of K / 16 additions
loses at most 2^-22 of a partial sum about as large as the limit L: values
within (K / 16) 2^-22 L of the limit may go either way, and their whole
products are added to the bound (F below).
"""
from __future__ import annotations

import pytest
import torch

from deepseeker import gated

pytestmark = pytest.mark.gpu
HALF_UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
ATOL = 2.0 ** -24


def make(T, H, I, dtype, device, seed=0, scale=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda a, b, s: (torch.randn(a, b, generator=g, device=device) * s).to(dtype)  # noqa: E731
    return (r(T, H, scale), r(I, H, 1.5 * H ** -0.5), r(I, H, 1.5 * H ** -0.5), r(H, I, I ** -0.5)), r(T, H, 1.0)


def formula(x, w1, w3, w2, limit):
    """The block in float64; autograd gives the gradients of the definition."""
    g, u = x @ w1.T, x @ w3.T
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return (g * torch.sigmoid(g) * u) @ w2.T


def scales(x, w1, w3, w2, dy, limit):
    """(|R|_2, n, F) of y, dx, dw1, dw3, dw2: see the module's head."""
    x, w1, w3, w2, dy = (t.detach().double() for t in (x, w1, w3, w2, dy))
    g, u = (x @ w1.T).requires_grad_(), (x @ w3.T).requires_grad_()
    gc, uc = (g.clamp(max=limit), u.clamp(-limit, limit)) if limit else (g, u)
    h = gc * torch.sigmoid(gc) * uc
    dh = dy @ w2
    dg, du = torch.autograd.grad(h, (g, u), dh)
    s = lambda t: t.detach().square()  # noqa: E731
    sums = (s(h) @ s(w2).T, s(dg) @ s(w1) + s(du) @ s(w3), s(dg).T @ s(x), s(du).T @ s(x), s(dy).T @ s(h))
    flips = [0.0] * 5
    if limit:
        near = x.shape[1] / 16 * 2.0 ** -22 * limit
        p = torch.sigmoid(gc.detach())
        fg = (dh * uc.detach() * p * (1 + gc.detach() * (1 - p))) * ((g.detach() - limit).abs() <= near)
        fu = (dh * gc.detach() * p) * ((u.detach().abs() - limit).abs() <= near)
        flips[1:4] = [float((a).norm()) for a in (fg @ w1 + fu @ w3, fg.T @ x, fu.T @ x)]
    return [(float(r.sum().sqrt()), min(r.numel(), h.numel()), f) for r, f in zip(sums, flips)]


def check(got, want, dtype, scale, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    (R, n, F), u = scale, HALF_UNIT[dtype]
    err = float((got - want).norm())
    bound = u * float(want.norm()) + 0.58 * u * (1 + 3 / n ** 0.5) * R + F + 2 * ATOL * want.numel() ** 0.5
    assert err <= bound, f"{what}: {err} > {bound} (relative {err / max(float(want.norm()), 1e-30):.2e})"


def both(ins, dy, limit):
    a = [t.detach().requires_grad_() for t in ins]
    y = gated.gated_ffn(*a, limit=limit)
    grads = torch.autograd.grad(y, a, dy)
    b = [t.detach().double().requires_grad_() for t in ins]
    yw = formula(*b, limit)
    return (y.detach(), *grads), (yw.detach(), *torch.autograd.grad(yw, b, dy.double()))


SIZES = [(1, 64, 64), (1, 4096, 2048), (2, 128, 96), (15, 72, 200), (16, 256, 128), (17, 1000, 711), (33, 513, 40),
         (64, 640, 1280), (65, 8, 8), (127, 1, 1), (130, 64, 4096), (200, 4096, 72), (384, 1288, 1000), (640, 2048, 2048), (128, 384, 257), (129, 2048, 512), (255, 96, 1024), (257, 1024, 264),
         (300, 30, 2050), (1, 7, 3), (1000, 512, 520), (2049, 256, 328)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,I", SIZES)
def test_block_and_gradients(T, H, I, dtype, cuda):
    ins, dy = make(T, H, I, dtype, cuda, seed=T + H)
    for limit in (None, 1.0):
        got, want = both(ins, dy, limit)
        for name, a, b, s in zip(("y", "dx", "dw1", "dw3", "dw2"), got, want, scales(*ins, dy, limit)):
            check(a, b, dtype, s, f"{name} limit={limit}")
    assert gated.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,I", [(2048, 4096, 2048), (777, 2560, 1288), (3000, 1001, 1003), (5001, 640, 1000),
                                   (2500, 1024, 1003), (2500, 1003, 1024),
                                   (16384, 256, 264)])
def test_large(T, H, I, dtype, cuda):
    ins, dy = make(T, H, I, dtype, cuda, seed=5, scale=0.25 if dtype == torch.float16 else 1.0)
    for limit in (None, 1.0):
        got, want = both(ins, dy, limit)
        for name, a, b, s in zip(("y", "dx", "dw1", "dw3", "dw2"), got, want, scales(*ins, dy, limit)):
            check(a, b, dtype, s, f"{name} limit={limit}")
    assert gated.status() == 0


def test_forward_without_gradients_is_the_same(cuda):
    ins, _ = make(70, 200, 88, torch.bfloat16, cuda)
    with torch.no_grad():
        a = gated.gated_ffn(*ins, limit=2.0)
    b = gated.gated_ffn(*[t.requires_grad_() for t in ins], limit=2.0)
    assert torch.equal(a, b.detach())


def test_repeats_bit_for_bit(cuda):
    for T in (1, 40, 600):
        ins, dy = make(T, 520, 264, torch.bfloat16, cuda)
        first, _ = both(ins, dy, None)
        for _ in range(3):
            again, _ = both(ins, dy, None)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gradient_against_differences(cuda):
    """Directional derivatives of the 64-bit formula by central differences.

    L(p) = sum(y dy).  With step s along a unit-scale direction the central
    difference of the 64-bit formula is off by O(s^2) and 1e-16 / s: s = 1e-5
    leaves less than 1e-9 relative.  The kernel's gradients are off by at most
    2 v |grad| (above: 1.58 v and the factor's few per cent), so <grad, d> along
    a direction d is within 2 v |grad| |d| of it."""
    ins, dy = make(24, 96, 64, torch.float16, cuda, seed=3)
    got, _ = both(ins, dy, 1.0)
    base = [t.double() for t in ins]
    gen = torch.Generator(device=cuda).manual_seed(9)
    for i in range(4):
        v = torch.randn(base[i].shape, generator=gen, device=cuda, dtype=torch.float64)
        f = lambda s: (formula(*[b + s * v if j == i else b for j, b in enumerate(base)], 1.0) * dy.double()).sum()  # noqa: E731,B023
        diff = float((f(1e-5) - f(-1e-5)) / 2e-5)
        grad = got[1 + i].double()
        bound = 2 * HALF_UNIT[torch.float16] * float(grad.norm()) * float(v.norm())
        assert abs(float((grad * v).sum()) - diff) <= bound


def test_strides_offsets_and_leading_dimensions(cuda):
    T, H, I = 45, 136, 72
    ins, dy = make(T, H, I, torch.bfloat16, cuda)
    want = both(ins, dy, None)[0]

    def views(pad, off):
        out = []
        for t in (*ins, dy):
            big = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=cuda)
            big[:, off:off + t.shape[1]] = t
            out.append(big[:, off:off + t.shape[1]])
        return out

    for pad, off in ((8, 0), (8, 8), (5, 3), (1, 1), (16, 2)):
        *v, vdy = views(pad, off)
        assert all(torch.equal(a, b) for a, b in zip(both(v, vdy, None)[0], want)), (pad, off)
    col = [t.t().contiguous().t() for t in ins]                     # column-major operands
    assert all(torch.equal(a, b) for a, b in zip(both(col, dy.t().contiguous().t(), None)[0], want))
    x3 = ins[0].view(5, 9, H)
    assert torch.equal(gated.gated_ffn(x3, *ins[1:]).view(T, H), want[0])
    one = ins[0][:1].expand(T, H).requires_grad_()                   # a broadcast input
    y = gated.gated_ffn(one, *ins[1:])
    g, = torch.autograd.grad(y, one, dy)
    rep = ins[0][:1].repeat(T, 1).requires_grad_()
    y2 = gated.gated_ffn(rep, *ins[1:])
    assert torch.equal(y, y2) and torch.equal(g, torch.autograd.grad(y2, rep, dy)[0])
    assert torch.equal(gated.gated_ffn(ins[0][0], *ins[1:]), gated.gated_ffn(ins[0][:1], *ins[1:])[0])


def test_shared_and_frozen_weights(cuda):
    ins, dy = make(20, 64, 48, torch.bfloat16, cuda)
    x, w1, w3, w2 = ins
    full = both(ins, dy, None)[0]
    for keep in range(4):                                            # one gradient at a time
        a = [t.detach().requires_grad_(i == keep) for i, t in enumerate(ins)]
        g, = torch.autograd.grad(gated.gated_ffn(*a), a[keep], dy)
        assert torch.equal(g, full[1 + keep])
    w = w1.detach().requires_grad_()                                 # one matrix as gate and up: gradients add
    g, = torch.autograd.grad(gated.gated_ffn(x, w, w, w2), w, dy)
    b = w1.double().requires_grad_()
    gw, = torch.autograd.grad(formula(x.double(), b, b, w2.double(), None), b, dy.double())
    # two rounded gradients and their rounded sum
    assert float((g.double() - gw).norm()) <= 4 * HALF_UNIT[torch.bfloat16] * float(gw.norm())


def test_broadcast_gradient_and_accumulation(cuda):
    """A loss that sums y hands down an expanded gradient; a second backward pass adds to .grad."""
    ins, _ = make(33, 72, 40, torch.bfloat16, cuda)
    a = [t.detach().requires_grad_() for t in ins]
    want = both(ins, torch.ones(33, 72, dtype=torch.bfloat16, device=cuda), 2.0)[0]
    gated.gated_ffn(a[0].view(3, 11, 72), *a[1:], limit=2.0).sum().backward()
    assert all(torch.equal(t.grad, w) for t, w in zip(a, want[1:]))
    gated.gated_ffn(*a, limit=2.0).sum().backward()
    assert all(torch.equal(t.grad, w + w) for t, w in zip(a, want[1:]))


def test_second_derivatives_are_refused(cuda):
    ins, dy = make(6, 64, 32, torch.bfloat16, cuda)
    a = [t.detach().requires_grad_() for t in ins]
    want = both(ins, dy, None)[0]
    up = dy.detach().requires_grad_()
    grads = torch.autograd.grad(gated.gated_ffn(*a), a, up, create_graph=True)
    assert all(torch.equal(g, w) for g, w in zip(grads, want[1:]))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grads[0].sum(), up)


def test_no_tokens(cuda):
    ins, _ = make(3, 64, 32, torch.bfloat16, cuda)
    x = ins[0][:0].detach().requires_grad_()
    w = [t.detach().requires_grad_() for t in ins[1:]]
    y = gated.gated_ffn(x, *w)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, (x, *w), torch.empty_like(y))
    assert grads[0].shape == (0, 64) and all(float(g.abs().sum()) == 0 for g in grads[1:])


def test_non_finite_values_stay_in_their_row(cuda):
    ins, dy = make(40, 72, 56, torch.bfloat16, cuda)
    x = ins[0].clone()
    x[7, 3], x[9, 5] = float("nan"), float("inf")
    for limit in (None, 1.0):
        clean = gated.gated_ffn(*ins, limit=limit)
        y = gated.gated_ffn(x, *ins[1:], limit=limit)
        keep = [i for i in range(40) if i not in (7, 9)]
        assert torch.equal(y[keep], clean[keep])
        assert torch.isnan(y[7]).all()
        want = formula(x.double(), *[t.double() for t in ins[1:]], limit)
        assert torch.equal(torch.isnan(y[9]), torch.isnan(want[9]))
    big = gated.gated_ffn(ins[0] * 1e4, *ins[1:])                    # saturated gates stay finite
    assert torch.isfinite(big).all()


def test_another_stream(cuda):
    ins, dy = make(50, 128, 96, torch.bfloat16, cuda)
    want = both(ins, dy, None)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(ins, dy, None)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_in_a_graph(cuda):
    ins, _ = make(4, 256, 128, torch.bfloat16, cuda)
    want = gated.gated_ffn(*ins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gated.gated_ffn(*ins)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


def test_training_step_in_a_graph(cuda):
    for T in (20, 300):
        ins, dy = make(T, 256, 136, torch.bfloat16, cuda)
        want = both(ins, dy, 1.0)[0]
        a = [t.detach().requires_grad_() for t in ins]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                                # autograd runs once outside the capture
            torch.autograd.grad(gated.gated_ffn(*a, limit=1.0), a, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = gated.gated_ffn(*a, limit=1.0)
            out = [y.detach(), *torch.autograd.grad(y, a, dy)]
        for o in out:
            o.zero_()
        graph.replay()
        assert all(torch.equal(o, w) for o, w in zip(out, want))


def test_two_streams_at_once(cuda):
    cases = [make(T, 512, 264, torch.bfloat16, cuda, seed=T) for T in (7, 700)]
    want = [both(ins, dy, None)[0] for ins, dy in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(*cases[i], None)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in (0, 1) for g in got[i] for a, b in zip(g, want[i]))


def test_refusals(cuda):
    (x, w1, w3, w2), _ = make(4, 64, 32, torch.bfloat16, cuda)
    bad = [(x.float(), w1, w3, w2), (x.cpu(), w1, w3, w2), (x, w1.half(), w3, w2), (x, w1, w3[:31], w2),
           (x, w1, w3, w2.t()), (x[:, :63], w1, w3, w2), (x, w1[0], w3, w2), (x, w1.cpu(), w3, w2),
           (x, w1[:0], w3[:0], w2[:, :0])]
    for args in bad:
        with pytest.raises(ValueError):
            gated.gated_ffn(*args)
    for limit in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            gated.gated_ffn(x, w1, w3, w2, limit=limit)
