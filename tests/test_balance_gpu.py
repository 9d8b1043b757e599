"""Balance loss (deepseeker.balance), its counts and its gradient against their definition in 64 bits.

Tolerances, derived before the first run, u = 2^-24.  A share p is off by a
factor 1 +- q: CUDA's expf, log1pf and sqrtf by a few units each (16 u with the
roundings around them), the row's sum by 64 u (32 values a lane at most, five
shuffles), and for softmax the rounding of l - max by |l - max| u.  Counts are
exact.  The sum over rows has chains of at most 64 + T / 256 additions, all of
one sign:
  loss   (max q + (64 + T / 256) u) loss
  dl     with d = sum p c (positive terms: off by (max q + 64 u) d), t = g p or
         g slope / Z:  |t| (q |c - d| + (max q + 64 u) d + 4 u (c + d)),
         what underflows in p below 2^-126, and the result's rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

from deepseeker import balance, moe

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def data(T, E, k, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    l = (torch.randn(T, E, generator=g, device=device) * 1.5 + torch.randn(1, E, generator=g, device=device)).to(dtype)
    ids = torch.randint(0, E, (T, k), generator=g, device=device, dtype=torch.int32)
    return l, ids


def definition(l, ids, kind, dloss, valid=None, offsets=None):
    """(loss, bound), counts, (dlogits, bound) in 64 bits, sequence by sequence."""
    T, E = l.shape
    k = ids.shape[1]
    ends = [0, T] if offsets is None else offsets.tolist()
    S = len(ends) - 1
    dl, bl = torch.zeros(T, E, dtype=torch.float64, device=l.device), torch.zeros(T, E, dtype=torch.float64, device=l.device)
    losses, bounds, counts = [], [], []
    for s in range(S):
        rows = torch.arange(ends[s], max(ends[s + 1], ends[s]), device=l.device)
        if valid is not None:
            rows = rows[valid[rows]]
        n = rows.numel()
        chosen = ids[rows].reshape(-1).long()
        c = torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
        counts.append(c.int())
        if n == 0:
            losses.append(torch.zeros((), dtype=torch.float64, device=l.device))
            bounds.append(losses[-1])
            continue
        x = l[rows].double()
        if kind == "softmax":
            off = (x.amax(1, keepdim=True) - x).nan_to_num(0.0, posinf=0.0)
            p = torch.softmax(x, 1).nan_to_num(0.0)            # a row of -inf has no shares
            slope = p
            q = (80 + off) * U
        else:
            sp = torch.logaddexp(x, torch.zeros_like(x))
            a = sp.sqrt()
            z = a.sum(1, keepdim=True)
            p = a / z
            slope = (torch.sigmoid(x) / (2 * a) / z).nan_to_num(0.0)
            q = torch.full_like(x, 80 * U)
        coef = c.double() * E / (k * n * n)
        loss = (p.sum(0) * coef).sum()
        losses.append(loss)
        bounds.append(loss * (q.max() + (64 + T / 256 + 4) * U))
        d = (p * coef).sum(1, keepdim=True)
        g = float(dloss.reshape(-1)[s])
        dl[rows] = g * slope * (coef - d)
        bl[rows] = abs(g) * slope * (q * (coef - d).abs() + (q.max() + 64 * U) * d + 4 * U * (coef + d)) \
            + abs(g) * 2.0 ** -120 * (coef + d)
    if offsets is None:
        return (losses[0], bounds[0]), counts[0], (dl, bl)
    stack = lambda t, *shape: torch.stack(t) if t else torch.zeros(0, *shape, device=l.device)  # noqa: E731
    return (stack(losses), stack(bounds)), stack(counts, E).int(), (dl, bl)


def close(got, value, bound):
    unit = torch.finfo(got.dtype).eps / 2
    bound = bound + unit * (value.abs() + bound) + (2.0 ** -25 if got.dtype == F16 else 2.0 ** -150)
    err = (got.double() - value).abs()
    assert got.shape == value.shape and bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


def run(l, ids, kind, dloss, **kw):
    leaf = l.detach().requires_grad_()
    loss, counts = balance.balance_loss(leaf, ids, kind=kind, **kw)
    dl, = torch.autograd.grad(loss, leaf, dloss)
    assert loss.dtype == F32 and counts.dtype == torch.int32 and dl.dtype == l.dtype and not counts.requires_grad
    return loss.detach(), counts, dl


def check(l, ids, kind, dloss, **kw):
    loss, counts, dl = run(l, ids, kind, dloss, **kw)
    want, n, grad = definition(l, ids, kind, dloss, **kw)
    assert counts.shape == n.shape and torch.equal(counts, n)
    close(loss, *want)
    close(dl, *grad)
    quiet = balance.balance_loss(l, ids, kind=kind, **kw)
    assert torch.equal(quiet[0], loss) and torch.equal(quiet[1], counts)
    again = run(l, ids, kind, dloss, **kw)
    assert all(torch.equal(a, b) for a, b in zip(again, (loss, counts, dl)))
    return loss, counts, dl


SHAPES = [(1, 1, 1), (1, 8, 2), (2, 3, 1), (7, 16, 2), (61, 16, 2), (300, 60, 4), (513, 64, 8), (1000, 7, 3), (129, 128, 8),
          (2049, 160, 6), (4097, 256, 8), (333, 257, 5), (777, 384, 6), (100, 512, 32), (70, 1024, 8), (65, 1023, 3),
          (70001, 12, 2), (20000, 100, 4)]


@pytest.mark.parametrize("kind", ["softmax", "sqrtsoftplus"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,E,k", SHAPES)
def test_one_sequence(T, E, k, dtype, kind, cuda):
    l, ids = data(T, E, k, dtype, cuda, seed=T + E)
    check(l, ids, kind, torch.tensor(0.7, device=cuda))


@pytest.mark.parametrize("kind", ["softmax", "sqrtsoftplus"])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("ends", [[0, 700], [0, 0, 1, 2, 2, 699, 700], [3, 300, 300, 650], [5, 5], [700, 700], [0],
                                  list(range(0, 701)), [0, 350] + [350] * 40 + [351, 700]])
def test_sequences(ends, wide, kind, cuda):
    l, ids = data(700, 40, 3, F32, cuda, seed=len(ends))
    off = torch.tensor(ends, dtype=torch.int64 if wide else torch.int32, device=cuda)
    g = torch.rand(len(ends) - 1, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)) - 0.3
    valid = torch.rand(700, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)) > 0.2
    check(l, ids, kind, g, offsets=off)
    masked = l.clone()
    masked[~valid] = float("nan")                                       # not looked at
    loss, counts, dl = run(masked, ids, kind, g, offsets=off, valid=valid)
    want, n, grad = definition(l, ids, kind, g, offsets=off, valid=valid)
    assert torch.equal(counts, n)
    close(loss, *want)
    close(dl, *grad)
    assert not dl[~valid].any() and not dl[: ends[0]].any() and not dl[ends[-1]:].any()


def test_sequences_are_alone(cuda):
    """A sequence's results are those of a call of its own, up to the order of its sums."""
    l, ids = data(5000, 256, 8, F32, cuda)
    off = torch.tensor([0, 1, 1234, 1234, 4000, 5000], dtype=torch.int32, device=cuda)
    loss, counts, dl = run(l, ids, "softmax", torch.ones(5, device=cuda), offsets=off)
    for s, (a, b) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        if a == b:
            assert float(loss[s]) == 0.0 and not counts[s].any()
            continue
        one = run(l[a:b], ids[a:b], "softmax", torch.tensor(1.0, device=cuda))
        assert torch.equal(one[1], counts[s]) and abs(float(one[0] - loss[s])) <= 200 * U * float(loss[s])
        want, _, grad = definition(l[a:b], ids[a:b], "softmax", torch.tensor(1.0))
        close(dl[a:b], *grad)


@pytest.mark.parametrize("kind", ["softmax", "sqrtsoftplus"])
def test_values(kind, cuda):
    l, ids = data(90, 48, 4, F32, cuda)
    l[3] = -math.inf                                                    # no expert left
    l[4, 5:] = -math.inf
    l[5] = 0.0
    l[6] = -300.0                                                       # roots that underflow one by one
    l[7, 0] = 300.0
    l[8] = torch.linspace(-120, 60, 48, device=cuda)
    ids[0] = -1
    ids[1] = torch.tensor([7, 7, 7, 7], device=cuda)                    # a repeated one counts every time
    ids[2] = torch.tensor([48, 1 << 30, -(1 << 31), 2], device=cuda)
    g = torch.tensor(-1.3, device=cuda)
    if kind == "softmax":
        check(l, ids, kind, g)
    else:
        # exp(-150) is 0 in f32: row 6 has no shares, where 64 bits still give it even ones
        keep = torch.tensor([i for i in range(90) if i not in (3, 6)], device=cuda)
        check(l[keep], ids[keep], kind, g)
        loss, counts, dl = run(l, ids, kind, g)
        assert torch.isfinite(loss) and torch.isfinite(dl).all() and not dl[3].any() and not dl[6].any()
    for bad in (math.nan, math.inf):
        x = l.clone()
        x[10, 3] = bad
        loss, counts, dl = run(x, ids, kind, g)
        assert torch.isnan(loss) and torch.isnan(dl[10]).any() and torch.isfinite(dl[11:]).all()
        assert torch.equal(counts, balance.balance_loss(l, ids, kind=kind)[1])


def test_even_routing_gives_one(cuda):
    l = torch.zeros(256, 64, device=cuda)
    ids = (torch.arange(256 * 4, device=cuda, dtype=torch.int32) % 64).view(256, 4)
    for kind in ("softmax", "sqrtsoftplus"):
        loss, counts, dl = run(l, ids, kind, torch.tensor(1.0, device=cuda))
        assert abs(float(loss) - 1) <= 1e-5 and bool((counts == 16).all()) and float(dl.abs().max()) <= 1e-8


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignments(dtype, cuda):
    l, ids = data(200, 64, 2, dtype, cuda)
    g = torch.tensor(1.0, device=cuda)
    for pad, off in ((4, 0), (4, 4), (1, 0), (3, 1), (64, 2)):
        big = torch.full((200, 64 + pad), float("nan"), dtype=dtype, device=cuda)
        big[:, off:off + 64] = l
        check(big[:, off:off + 64], ids, "softmax", g)
    check(l.t().contiguous().t(), ids.t().contiguous().t(), "sqrtsoftplus", g)
    valid = torch.zeros(400, dtype=torch.bool, device=cuda)
    valid[::2] = torch.arange(200, device=cuda) % 3 > 0
    check(l, ids, "softmax", g, valid=valid[::2])
    off = torch.tensor([0, 9, 50, 9, 200, 9], dtype=torch.int32, device=cuda)[::2]
    check(l, ids, "softmax", torch.ones(1, device=cuda).expand(2), offsets=off)


def test_empty(cuda):
    l, ids = data(4, 16, 2, F32, cuda)
    loss, counts, dl = run(l[:0], ids[:0], "softmax", torch.tensor(1.0, device=cuda))
    assert float(loss) == 0 and not counts.any() and dl.shape == (0, 16)
    none = torch.zeros(4, dtype=torch.bool, device=cuda)
    loss, counts, dl = run(l, ids, "softmax", torch.tensor(1.0, device=cuda), valid=none)
    assert float(loss) == 0 and not counts.any() and not dl.any()


def test_offsets_outside_the_rows(cuda):
    """Offsets that leave the matrix or descend stay inside memory; sequences that are in order keep their results."""
    l, ids = data(100, 32, 2, F32, cuda)
    off = torch.tensor([0, 60, 1000, -5, 7], dtype=torch.int32, device=cuda)
    loss, counts, dl = run(l, ids, "softmax", torch.ones(4, device=cuda), offsets=off)
    want = definition(l, ids, "softmax", torch.ones(2), offsets=torch.tensor([0, 60, 100]))
    close(loss[:2], *want[0])
    assert torch.equal(counts[:2], want[1]) and dl.shape == l.shape


def test_against_differences(cuda):
    """Central differences of the 64-bit loss at steps of 2^-12, whose own error is far below 1e-5 here."""
    for kind in ("softmax", "sqrtsoftplus"):
        l, ids = data(5, 6, 2, F32, cuda, seed=3)
        g = torch.tensor(1.0, device=cuda)
        dl = run(l, ids, kind, g)[2].double()
        num = torch.zeros_like(dl)
        for i in range(l.numel()):
            for sign in (1, -1):
                x = l.double()
                x.view(-1)[i] += sign * 2.0 ** -12
                num.view(-1)[i] += sign * definition(x, ids, kind, g)[0][0] * 2.0 ** 11
        assert float((dl - num).abs().max()) <= 1e-5 * max(1.0, float(num.abs().max()))


@pytest.mark.parametrize("kind", ["softmax", "sqrtsoftplus"])
def test_with_the_router(kind, cuda):
    l, _ = data(640, 96, 6, F32, cuda)
    if kind == "softmax":
        _, ids = moe.route_softmax_topk(l, 6)
    else:
        _, ids = moe.route_sqrtsoftplus(l, torch.zeros(96, device=cuda), 6)
    loss, counts, _ = check(l, ids, kind, torch.tensor(1.0, device=cuda))
    assert int(counts.sum()) == 640 * 6 and float(loss) > 1.0            # what is chosen has the larger shares


def test_streams_and_graph(cuda):
    l, ids = data(900, 128, 8, F32, cuda)
    off = torch.tensor([0, 100, 900], dtype=torch.int32, device=cuda)
    g = torch.tensor([0.5, 2.0], device=cuda)
    want = run(l, ids, "softmax", g, offsets=off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(l, ids, "softmax", g, offsets=off)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaf = l.clone().requires_grad_()
    held, held_off = ids.clone(), off.clone()
    with torch.cuda.stream(side):
        torch.autograd.grad(balance.balance_loss(leaf, held, offsets=held_off)[0], leaf, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with moe.graph_capture(graph):
        loss, counts = balance.balance_loss(leaf, held, offsets=held_off)
        dl, = torch.autograd.grad(loss, leaf, g)
    for seed, mid in ((5, 100), (6, 0), (7, 899)):
        l2, ids2 = data(900, 128, 8, F32, cuda, seed=seed)
        with torch.no_grad():
            leaf.copy_(l2)
        held.copy_(ids2)
        held_off[1] = mid
        graph.replay()
        want = run(l2, ids2, "softmax", g, offsets=held_off)
        assert all(torch.equal(a, b) for a, b in zip((loss, counts, dl), want))


def test_calls_at_once(cuda):
    cases = []
    for T, E, k, ends in ((3000, 128, 8, [0, 5, 2000, 3000]), (61, 16, 2, None), (900, 1024, 4, [0, 900])):
        l, ids = data(T, E, k, F32, cuda, seed=T)
        off = None if ends is None else torch.tensor(ends, device=cuda)
        cases.append((l, ids, "sqrtsoftplus", torch.ones((), device=cuda) if off is None else torch.ones(len(ends) - 1, device=cuda),
                      off))
    want = [run(*c[:4], offsets=c[4]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run(*c[:4], offsets=c[4]))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))


def test_counts_alone_and_loss_alone(cuda):
    """Either result may be left unused; a loss in a larger sum gets its own gradient."""
    l, ids = data(50, 20, 3, F32, cuda)
    leaf = l.clone().requires_grad_()
    loss, counts = balance.balance_loss(leaf, ids)
    total = loss * 0.25 + leaf.sum() * 0.0
    total.backward()
    want = run(l, ids, "softmax", torch.tensor(0.25, device=cuda))
    assert torch.equal(leaf.grad, want[2]) and torch.equal(counts, want[1])
    leaf.grad = None
    for _ in range(2):                                                  # the same graph twice
        loss, _ = balance.balance_loss(leaf, ids)
        loss.backward(retain_graph=True)
        loss.backward()
    assert bool((leaf.grad - 4 * run(l, ids, "softmax", torch.tensor(1.0, device=cuda))[2]).abs().max() <= 1e-7)


def test_refusals(cuda):
    l, ids = data(8, 16, 2, F32, cuda)
    ok = dict(valid=torch.ones(8, dtype=torch.bool, device=cuda), offsets=torch.tensor([0, 8], device=cuda))
    balance.balance_loss(l, ids, **ok)
    for a in ((l.double(), ids), (l.cpu(), ids), (l[0], ids), (l, ids.long()), (l, ids[:7]), (l, ids[:, :0]),
              (l, ids.cpu()), (torch.zeros(8, 1025, device=cuda), ids), (l, ids.repeat(1, 17)), (l[:, :0], ids)):
        with pytest.raises(ValueError):
            balance.balance_loss(*a)
    for kw in (dict(kind="sigmoid"), dict(valid=ok["valid"][:7]), dict(valid=ok["valid"].int()),
               dict(valid=ok["valid"].cpu()), dict(offsets=ok["offsets"].float()), dict(offsets=ok["offsets"].cpu()),
               dict(offsets=ok["offsets"][:0]), dict(offsets=ok["offsets"][None])):
        with pytest.raises(ValueError):
            balance.balance_loss(l, ids, **kw)
    a = l.clone().requires_grad_()
    g, = torch.autograd.grad(balance.balance_loss(a, ids)[0], a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            balance.balance_loss(torch.autograd.forward_ad.make_dual(l, torch.ones_like(l)), ids)
