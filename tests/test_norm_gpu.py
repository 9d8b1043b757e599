"""Layer norm (deepseeker.norm) and its gradients against the formulas in 64 bits.

Tolerances, derived before the first run, u = 2^-24 the unit roundoff of f32.
A sum of n values in f32 is off by at most c u sum|v|, c its longest chain of
additions: 64 covers up to 32 values a thread, a tree over 1024 threads and the
roundings of the values themselves; beyond 32768 features a thread adds H / 1024.
With A = mean|x|, d = c u A r bounds the mean's error over the deviation, so

  xh     E = d + |xh| (c u + d^2 + 4 u)       (the variance takes d^2 from the mean's error)
  y      |w| E + 4 u (|xh w| + |b|) + v |y|   v: unit roundoff of the result's type
  dx     r (c u mean|g| + |m2| E + |xh| (c u mean|g xh| + mean(|g| E)) + 4 u (|g| + |m1| + |xh m2|))
         + |dx| (c u + d^2 + 4 u) + v |dx|
  dw     sum |dy| E + k u sum |dy xh| + v |dw|, db the same without E; k = rows / 8 + 64 covers the
         rows that one block adds, its warps, and the joined blocks
and in f16 half of its smallest number, 2^-25, more.
"""
from __future__ import annotations

import itertools

import pytest
import torch

from deepseeker import norm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return 2.0 ** -25 if dtype == F16 else 0.0


def data(rows, cols, dtype, device, seed=0, gap=0, shift=0.5):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, cols + gap, generator=g, device=device)
    x = (x + shift * torch.randn(1, cols + gap, generator=g, device=device)) * torch.exp(
        0.5 * torch.randn(rows, 1, generator=g, device=device))
    return x.to(dtype)[:, :cols]


def formula(x, w, b, eps, dy=None):
    """Results and bounds {name: (value, bound without the last rounding)} in 64 bits."""
    rows, cols = x.shape
    c = (64 + (cols / 1024 if cols > 8192 else 0)) * U
    x = x.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * r
    w = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    d = c * x.abs().mean(1, keepdim=True) * r
    rel = c + d * d + 4 * U
    e = d + xh.abs() * rel
    out = {"y": (xh * w + b, w.abs() * e + 4 * U * ((xh * w).abs() + b.abs()))}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - m1 - xh * m2)
    off = (c * g.abs().mean(1, keepdim=True) + m2.abs() * e
           + xh.abs() * (c * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e).mean(1, keepdim=True))
           + 4 * U * (g.abs() + m1.abs() + (xh * m2).abs()))
    k = (rows / 8 + 64) * U
    out["dx"] = (dx, r * off + dx.abs() * rel)
    out["dw"] = ((dy * xh).sum(0), (dy.abs() * e).sum(0) + k * (dy * xh).abs().sum(0))
    out["db"] = (dy.sum(0), k * dy.abs().sum(0))
    return out


def check(got, want, name):
    value, bound = want
    assert got.shape == value.shape
    bound = bound + unit(got.dtype) * (value.abs() + bound) + least(got.dtype)
    err = (got.double() - value).abs()
    if got.dtype == F16:
        # f16 ends at 65504 = 2^16 - 2^5: from 65520, half a step of 2^5 above, values round to infinity
        over = (value.abs() + bound >= 65520) & torch.isinf(got) & (got.sign() == value.sign())
        err = torch.where(over, torch.zeros_like(err), err)
    assert bool((err <= bound).all()), (name, float((err - bound).max()), float(err.max()))


def train(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = norm.layer_norm(*leaves, eps=eps)
    live = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, live, dy))
    return {"y": y.detach(), **{n: next(grads) for n, t in zip(("dx", "dw", "db"), leaves) if t is not None}}


SHAPES = [(1, 1), (2, 2), (1, 16), (3, 33), (9, 64), (17, 250), (5, 711), (8, 1024), (1, 1025), (300, 1000), (64, 2560),
          (7, 4096), (1100, 4095), (2, 8192), (3, 8193), (1, 16384), (2, 32768), (5, 32769), (20, 40000), (4099, 72),
          (70001, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_gradients(rows, cols, dtype, cuda):
    for kind in {dtype, F32}:
        x, dy = data(rows, cols, dtype, cuda, seed=rows), data(rows, cols, dtype, cuda, seed=cols + 7)
        w, b = (1 + 0.3 * data(1, cols, F32, cuda, seed=1)[0]).to(kind), data(1, cols, F32, cuda, seed=2)[0].to(kind)
        want = formula(x, w, b, 1e-5, dy)
        got = train(x, w, b, dy)
        for name, t in got.items():
            assert t.dtype == (kind if name in ("dw", "db") else dtype)
            check(t, want[name], name)
        assert torch.equal(norm.layer_norm(x, w, b), got["y"])
        again = train(x, w, b, dy)
        assert all(torch.equal(again[n], got[n]) for n in got)


@pytest.mark.parametrize("has_w,has_b", list(itertools.product((False, True), repeat=2)))
def test_parameters_left_out(has_w, has_b, cuda):
    x, dy = data(37, 512, BF16, cuda), data(37, 512, BF16, cuda, seed=5)
    w = 1 + data(1, 512, F32, cuda, seed=1)[0] if has_w else None
    b = data(1, 512, F32, cuda, seed=2)[0] if has_b else None
    want = formula(x, w, b, 1e-5, dy)
    for name, t in train(x, w, b, dy).items():
        check(t, want[name], name)


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 1), (1, 2), (0, 2)])
@pytest.mark.parametrize("cols", [96, 2048, 9000])
def test_some_gradients(which, cols, cuda):
    x, dy = data(21, cols, F32, cuda), data(21, cols, F32, cuda, seed=5)
    w, b = data(1, cols, F32, cuda, seed=1)[0], data(1, cols, F32, cuda, seed=2)[0]
    want = train(x, w, b, dy)
    leaves = [t.clone().requires_grad_(i in which) for i, t in enumerate((x, w, b))]
    grads = torch.autograd.grad(norm.layer_norm(*leaves), [leaves[i] for i in which], dy)
    for i, g in zip(which, grads):
        assert torch.equal(g, want[("dx", "dw", "db")[i]])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [40, 1000, 4096, 33000])
def test_strides_and_alignments(cols, dtype, cuda):
    x, dy = data(11, cols, dtype, cuda), data(11, cols, dtype, cuda, seed=5)
    w, b = data(1, cols, F32, cuda, seed=1)[0].to(dtype), data(1, cols, F32, cuda, seed=2)[0].to(dtype)
    want = formula(x, w, b, 1e-5, dy)

    def placed(t, pad, off):
        big = torch.full((t.shape[0], cols + pad), float("nan"), dtype=dtype, device=cuda)
        big[:, off:off + cols] = t
        return big[:, off:off + cols]

    for pad, off in ((8, 0), (8, 8), (10, 2), (1, 1), (3, 0)):
        for name, t in train(placed(x, pad, off), w, b, placed(dy, 16 - pad, 0)).items():
            check(t, want[name], name)
    odd = torch.zeros(2 * cols + 1, dtype=dtype, device=cuda)
    odd[1::2] = w
    for name, t in train(x.t().contiguous().t(), odd[1::2], b, dy.t().contiguous().t()).items():
        check(t, want[name], name)
    off_w = torch.cat([w[:1], w])[1:]                                   # contiguous, off the 16-byte grid
    for name, t in train(x, off_w, b, dy).items():
        check(t, want[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [1, 6, 1400])
@pytest.mark.parametrize("cols", [1, 7, 31, 32, 33, 127, 129, 256, 257, 511, 513, 640, 1023, 1024, 1025, 2047, 2050, 4094,
                                  4097, 8191, 8192])
def test_rows_anywhere(cols, rows, dtype, cuda):
    """Rows that begin and end between 16-byte boundaries, among values that are no numbers; several turns a block."""
    x, dy = data(rows, cols, dtype, cuda, seed=cols), data(rows, cols, dtype, cuda, seed=rows + 5)
    w, b = data(1, cols, F32, cuda, seed=1)[0], data(1, cols, F32, cuda, seed=2)[0]
    want = formula(x, w, b, 1e-5, dy)

    def placed(t, pad, off):
        big = torch.full((rows * (cols + pad) + 2 * off,), float("nan"), dtype=dtype, device=cuda)
        view = big[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        view.copy_(t)
        return view

    seen = []
    for pad, off in ((0, 1), (5, 0), (1, 3)):
        got = train(placed(x, pad, off), w, b, placed(dy, 3 - pad % 3, off + 2))
        for name, t in got.items():
            check(t, want[name], name)
        seen.append(got)
    # the order of a row's sums follows from its columns, but for rows that lie on 16 bytes (of the three, the single
    # one at the beginning of its buffer), which are summed in vectors
    if rows > 1 or cols * x.element_size() % 16:
        assert all(torch.equal(seen[0][n], seen[i][n]) for n in want for i in (1, 2))


def test_shapes(cuda):
    x = data(24, 80, BF16, cuda)
    w, b = data(1, 80, BF16, cuda, seed=1)[0], data(1, 80, BF16, cuda, seed=2)[0]
    y = norm.layer_norm(x, w, b)
    assert torch.equal(norm.layer_norm(x.view(2, 3, 4, 80), w, b), y.view(2, 3, 4, 80))
    assert torch.equal(norm.layer_norm(x[5], w, b), y[5])
    a = x.view(2, 12, 80).clone().requires_grad_()
    p = w.clone().requires_grad_()
    norm.layer_norm(a, p, b).sum().backward()                           # dy of stride 0
    want = train(x, w, b, torch.ones_like(x))
    assert torch.equal(a.grad.view(24, 80), want["dx"]) and torch.equal(p.grad, want["dw"])
    for rows in (0,):
        e = x[:rows].clone().requires_grad_()
        p = w.clone().requires_grad_()
        y = norm.layer_norm(e, p, b)
        dx, dw = torch.autograd.grad(y, (e, p), torch.zeros_like(y))
        assert y.shape == dx.shape == (0, 80) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_values(dtype, cuda):
    x = data(12, 600, dtype, cuda)
    x[1] = 3.0                                                          # no deviation: y = b
    x[2] = 0.0
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    x[5, 9] = -float("inf")
    x[6] = (x[6].float() + 200).to(dtype)                               # a mean far from 0
    x[7] = (x[7].float() * 1e-4).to(dtype)                              # deviations below sqrt(eps)
    w, b = data(1, 600, F32, cuda, seed=1)[0], data(1, 600, F32, cuda, seed=2)[0]
    y = norm.layer_norm(x, w, b)
    bad = torch.tensor([3, 4, 5], device=cuda)
    good = torch.tensor([0, 1, 2, 6, 7, 8, 9, 10, 11], device=cuda)
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[1:3], b.to(dtype).expand(2, 600))
    dy = data(12, 600, dtype, cuda, seed=9)
    want = formula(x[good], w, b, 1e-5, dy[good])
    check(y[good], want["y"], "y")
    got = train(x, w, b, dy)
    check(got["dx"][good], want["dx"], "dx")
    assert torch.isnan(got["dx"][bad]).all() and torch.isnan(got["dw"]).all()
    zero = train(x[good], w, b, torch.zeros_like(dy[good]))
    assert not any(zero[n].any() for n in ("dx", "dw", "db"))


def test_eps(cuda):
    x = data(5, 128, F32, cuda) * 1e-3
    for eps in (0.0, 1e-12, 1e-5, 10.0):
        check(norm.layer_norm(x, eps=eps), formula(x, None, None, eps)["y"], eps)


def test_against_differences(cuda):
    """Central differences of the 64-bit form at steps of 2^-10: off by its third derivative, below 1e-4 of the
    largest gradient here."""
    x, dy = data(3, 24, F32, cuda), data(3, 24, F32, cuda, seed=3)
    w, b = 1 + data(1, 24, F32, cuda, seed=1)[0], data(1, 24, F32, cuda, seed=2)[0]
    got = train(x, w, b, dy)

    def loss(*t):
        return (formula(*t, 1e-5)["y"][0] * dy.double()).sum()

    for i, name in enumerate(("dx", "dw", "db")):
        t = [v.double() for v in (x, w, b)]
        num = torch.zeros_like(t[i])
        for at in range(num.numel()):
            for sign in (1, -1):
                s = [v.clone() for v in t]
                s[i].view(-1)[at] += sign * 2.0 ** -10
                num.view(-1)[at] += sign * loss(*s) * 2.0 ** 9
        assert float((got[name].double() - num).abs().max()) <= 1e-3 * float(num.abs().max())


def test_streams_and_graph(cuda):
    x, dy = data(200, 1536, BF16, cuda), data(200, 1536, BF16, cuda, seed=3)
    w, b = data(1, 1536, F32, cuda, seed=1)[0], data(1, 1536, F32, cuda, seed=2)[0]
    want = train(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)

    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    held = dy.clone()
    with torch.cuda.stream(side):                                       # warm-up of the allocator
        torch.autograd.grad(norm.layer_norm(*leaves), leaves, held)
    torch.cuda.synchronize()
    from deepseeker import moe

    graph = torch.cuda.CUDAGraph()
    with moe.graph_capture(graph):
        y = norm.layer_norm(*leaves)
        grads = torch.autograd.grad(y, leaves, held)
    for seed in (3, 11):
        nx, nd = data(200, 1536, BF16, cuda, seed=seed), data(200, 1536, BF16, cuda, seed=seed + 1)
        with torch.no_grad():
            leaves[0].copy_(nx)
            held.copy_(nd)
        graph.replay()
        want = train(nx, w, b, nd)
        for t, n in zip((y, *grads), ("y", "dx", "dw", "db")):
            assert torch.equal(t, want[n])


def test_many_values(cuda):
    """Rows past 2^32 elements."""
    rows, cols = (1 << 20) + 3, 4096
    x = torch.empty(rows, cols, dtype=BF16, device=cuda)
    x.view(-1)[: 1 << 24].normal_()
    torch.cuda.synchronize()
    x[1 << 12:] = x[: 1 << 12].repeat(rows // (1 << 12), 1)[: rows - (1 << 12)]
    w = torch.ones(cols, dtype=F32, device=cuda, requires_grad=True)
    y = norm.layer_norm(x.requires_grad_(), w)
    at = torch.tensor([0, 4096, 1 << 19, rows - 2, rows - 1], device=cuda)
    xs = x.detach()[at]
    want = formula(xs, None, None, 1e-5, xs)
    check(y.detach()[at], want["y"], "y")
    dx, = torch.autograd.grad(y, x, x.detach())
    check(dx[at], want["dx"], "dx")


@pytest.mark.parametrize("cols", [96, 1000, 4096, 8200, 40000])
def test_a_row_does_not_depend_on_the_others(cols, cuda):
    x, dy = data(1500, cols, BF16, cuda), data(1500, cols, BF16, cuda, seed=3)
    w, b = data(1, cols, F32, cuda, seed=1)[0], data(1, cols, F32, cuda, seed=2)[0]
    whole = train(x, w, b, dy)
    for lo, hi in ((0, 1), (7, 9), (1490, 1500)):
        part = train(x[lo:hi], w, b, dy[lo:hi])
        assert torch.equal(part["y"], whole["y"][lo:hi]) and torch.equal(part["dx"], whole["dx"][lo:hi])


def test_calls_at_once(cuda):
    """Eager steps on three streams, then two captured steps replayed side by side."""
    cases = [(data(r, c, BF16, cuda, seed=r), data(1, c, F32, cuda, seed=1)[0], data(1, c, F32, cuda, seed=2)[0],
              data(r, c, BF16, cuda, seed=r + 1)) for r, c in ((900, 1024), (40, 711), (300, 4096))]
    want = [train(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(train(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(g[n], w[n]) for g, w in zip(got, want) for n in w)
    from deepseeker import moe

    held, graphs = [], []
    for x, w, b, dy in cases[:2]:
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with moe.graph_capture(graph):
            y = norm.layer_norm(*leaves)
            held.append((leaves, y, torch.autograd.grad(y, leaves, dy)))
        graphs.append(graph)
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, y, grads), w in zip(held, want):
            assert all(torch.equal(t, w[n]) for t, n in zip((y, *grads), ("y", "dx", "dw", "db")))


def test_refusals(cuda):
    x, w = data(4, 64, BF16, cuda), data(1, 64, F32, cuda)[0]
    for bad in ((x.double(),), (x.cpu(),), (x, w[:63]), (x, w.double()), (x, w.cpu()), (x, w.half()),
                (x, w, w.bfloat16()), (x[0, 0],), (x[:, :0],), ("x",)):
        with pytest.raises(ValueError):
            norm.layer_norm(*bad)
    for eps in (-1e-5, float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError):
            norm.layer_norm(x, eps=eps)
    a = x.float().requires_grad_()
    g, = torch.autograd.grad(norm.layer_norm(a, w).square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        for at in range(3):
            ops = [x.float(), w, w]
            ops[at] = torch.autograd.forward_ad.make_dual(ops[at], torch.ones_like(ops[at]))
            with pytest.raises(ValueError, match="forward-mode"):
                norm.layer_norm(*ops)
