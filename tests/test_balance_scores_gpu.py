"""Scores of the balance loss (deepseeker.balance) far from a row's largest one.

Tolerances, derived before the first run, u = 2^-24.  A score far from the row's largest is 2^t e^r: 4 u for the
instruction 2^t (2^-22), a unit for the product with e^r, and 4 u for what f32 leaves out of log 2 (1.9e-9 |t|,
|t| <= 126).  A row's sum Z of 16 scores of one lane is off by 9 u for its additions and by the error of its largest
score, 4 u; 1 / Z, the products with the upstream gradient, with the score and with the coefficient's difference,
the coefficient and that difference round once each, 6 u.  Where the largest score's expert was not chosen, d =
sum p c is below 1e-8 c, so nothing cancels: 28 u of the gradient's size, rounded up to 32 u.
"""
from __future__ import annotations

import pytest
import torch

from deepseeker import balance

pytestmark = pytest.mark.gpu
F32 = torch.float32
U = 2.0 ** -24


def gradient(l, ids, kind, g):
    """dlogits of one sequence by the formula in 64 bits, and what its two terms add up to without their signs."""
    x, (T, E), k = l.double(), l.shape, ids.shape[1]
    c = torch.bincount(ids.reshape(-1).long(), minlength=E).double() * E / (k * T * T)
    if kind == "softmax":
        p = torch.softmax(x, 1)
        slope = p
    else:
        a = torch.logaddexp(x, torch.zeros_like(x)).sqrt()
        z = a.sum(1, keepdim=True)
        p, slope = a / z, torch.sigmoid(x) / (2 * a) / z
    d = (p * c).sum(1, keepdim=True)
    return g * slope * (c - d), abs(g) * slope * (c + d)


def grad(l, ids, kind, g):
    leaf = l.clone().requires_grad_()
    loss, _ = balance.balance_loss(leaf, ids, kind=kind)
    return torch.autograd.grad(loss, leaf, torch.tensor(g, device=l.device))[0]


@pytest.mark.parametrize("g", [1.0, 1e6, -1e30])
def test_low_rows_and_large_gradients(g, cuda):
    """Rows whose scores are all near the smallest numbers of f32: 1 / Z times the upstream gradient leaves f32, the
    gradient of the logits does not."""
    l = torch.linspace(-170, -150, 5 * 16, device=cuda).view(5, 16).clone()
    l[4] = 1.0
    ids = torch.tensor([[0, 1], [2, 3], [0, 7], [9, 0], [1, 15]], dtype=torch.int32, device=cuda)
    got = grad(l, ids, "sqrtsoftplus", g).double()
    want, size = gradient(l, ids, "sqrtsoftplus", g)
    # as above, and the differences c - d cancel: the errors of p in d (28 u) count in full
    assert bool(((got - want).abs() <= 64 * U * size).all())


def test_infinite_gradient_leaves_masked_rows_alone(cuda):
    l = torch.randn(40, 16, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).requires_grad_()
    ids = torch.zeros(40, 2, dtype=torch.int32, device=cuda)
    valid = torch.arange(40, device=cuda) % 3 > 0
    for kind in ("softmax", "sqrtsoftplus"):
        for g in (float("inf"), float("nan")):
            loss, _ = balance.balance_loss(l, ids, kind=kind, valid=valid)
            dl, = torch.autograd.grad(loss, l, torch.tensor(g, device=cuda))
            assert not dl[~valid].any() and not torch.isfinite(dl[valid]).any()


@pytest.mark.parametrize("kind,top,least,most", [("softmax", 0.0, -80.0, -20.0), ("sqrtsoftplus", 3.0, -160.0, -40.0)])
def test_far_scores(kind, top, least, most, cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    l = least + (most - least) * torch.rand(3000, 16, generator=g, device=cuda)
    l[:, 5] = top                                                       # never chosen
    ids = torch.randint(6, 21, (3000, 2), generator=g, device=cuda, dtype=torch.int32) % 16
    got = grad(l, ids, kind, 1.0).double()
    want, size = gradient(l, ids, kind, 1.0)
    far = torch.arange(16, device=cuda) != 5
    assert bool(((got - want).abs() <= 32 * U * size)[:, far].all()), float(((got - want).abs() / size)[:, far].max() / U)


def test_bound_of_low_rows(cuda):
    """exp(l / 2) is a number of f32 (2^-126 and above) down to -174.67: rows above have their shares, rows below none."""
    ids = torch.tensor([[0, 1], [2, 3], [0, 7]], dtype=torch.int32, device=cuda)
    l = torch.full((3, 16), -173.5, device=cuda)
    l[1] += torch.linspace(-1, 0, 16, device=cuda)
    want, size = gradient(l, ids, "sqrtsoftplus", 1.0)
    got = grad(l, ids, "sqrtsoftplus", 1.0).double()
    assert bool(((got - want).abs() <= 64 * U * size).all())
    loss, counts = balance.balance_loss(l, ids, kind="sqrtsoftplus")
    # even shares where the logits are even: loss = sum over rows and experts of c / E
    p = torch.softmax(l.double() / 2, 1)
    c = counts.double() * 16 / (2 * 9)
    assert abs(float(loss) - float((p.sum(0) * c).sum())) <= 64 * U * float(loss)
    l = torch.full((3, 16), -175.5, device=cuda)
    loss, counts = balance.balance_loss(l, ids, kind="sqrtsoftplus")
    assert float(loss) == 0 and int(counts.sum()) == 6 and not grad(l, ids, "sqrtsoftplus", 1.0).any()


@pytest.mark.parametrize("offsets", [None, [0, 100, 20000]])
def test_what_is_kept_for_the_backward_pass(offsets, cuda):
    """The logits and E coefficients a sequence, not the forward pass's workspace."""
    l = torch.randn(20000, 64, device=cuda).requires_grad_()
    ids = torch.zeros(20000, 2, dtype=torch.int32, device=cuda)
    off = None if offsets is None else torch.tensor(offsets, device=cuda)
    loss, _ = balance.balance_loss(l, ids, offsets=off)
    held = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in loss.grad_fn.saved_tensors if t is not None}
    del held[l.data_ptr()]
    assert sum(held.values()) <= (4 * 64 if off is None else 2 * 4 * 64 + 3 * 8)


def test_low_rows_of_long_sequences(cuda):
    """Coefficients of a long sequence are small: their products with the smallest scores leave f32, d does not."""
    g = torch.Generator(device=cuda).manual_seed(4)
    l = -172 + 12 * torch.rand(60000, 16, generator=g, device=cuda)
    ids = torch.randint(0, 16, (60000, 2), generator=g, device=cuda, dtype=torch.int32)
    for up in (1.0, 1e5, 1e-25):
        got = grad(l, ids, "sqrtsoftplus", up).double()
        want, size = gradient(l, ids, "sqrtsoftplus", up)
        # as for low rows; and half the smallest number where the result itself is that small
        assert bool(((got - want).abs() <= 64 * U * size + 2.0 ** -149).all()), float(((got - want).abs() / size).max() / U)
