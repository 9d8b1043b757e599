"""Layer norm of rows whose mean is far larger than their deviation (deepseeker.norm).

Rows of one value each, an eighth of a whole number below 2^11: every sum of up to 8192 of them is exact in f32, and
so is the mean.  Then x - mean is 0, so y is the bias and the weight's gradient 0, both exactly, whatever r is
(316 here, 1 / sqrt(eps)).
"""
from __future__ import annotations

import pytest
import torch

from deepseeker import norm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def flat(rows, cols, gap, dtype, device):
    """Rows of one value, exact in `dtype`, `gap` values that are no numbers apart."""
    big = torch.full((rows, cols + gap), float("nan"), device=device)
    big[:, :cols] = (129 + torch.arange(rows, device=device) % 126)[:, None] / 8   # eight bits: exact in bf16
    return big.to(dtype)[:, :cols]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [1, 8, 64, 512, 1024, 4096, 8192])
def test_gradients_of_flat_rows(cols, dtype, cuda):
    """Widths whose inverse is a number of f32."""
    for rows, gap in ((1, 0), (126, 0), (1300, 3)):
        x = flat(rows, cols, gap, dtype, cuda).requires_grad_()
        g = torch.Generator(device=cuda).manual_seed(cols)
        w = (1 + 0.3 * torch.randn(cols, generator=g, device=cuda)).requires_grad_()
        b = torch.randn(cols, generator=g, device=cuda)
        dy = torch.randn(rows, cols, generator=g, device=cuda).to(dtype)
        y = norm.layer_norm(x, w, b)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        assert torch.equal(y.detach(), b.to(dtype).expand(rows, cols))
        assert not dw.any()
        # dx = r (g - mean g): r off by 4 u, the sum by 64 u of mean|g| (chain of 16 values, the tree), the product,
        # the mean, the difference and the last product u each, then the result's rounding
        v = dy.double() * w.detach().double()
        r = 1e-5 ** -0.5
        want = r * (v - v.mean(1, keepdim=True))
        bound = r * (64 * U * v.abs().mean(1, keepdim=True) + 8 * U * (v.abs() + v.mean(1, keepdim=True).abs()))
        unit = torch.finfo(dtype).eps / 2
        bound = bound + unit * (want.abs() + bound) + (2.0 ** -25 if dtype == F16 else 0.0)
        assert bool(((dx.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [7, 56, 328, 984, 1000, 1968, 4095, 7872, 8191])
def test_flat_rows_of_any_width(cols, dtype, cuda):
    """The mean is the quotient of the sum, not a product with an inverse that was rounded."""
    for rows, gap in ((1, 0), (126, 0), (1300, 3)):
        x = flat(rows, cols, gap, dtype, cuda).requires_grad_()
        g = torch.Generator(device=cuda).manual_seed(cols)
        w = (1 + 0.3 * torch.randn(cols, generator=g, device=cuda)).requires_grad_()
        b = torch.randn(cols, generator=g, device=cuda)
        y = norm.layer_norm(x, w, b)
        dw, = torch.autograd.grad(y, w, torch.randn(rows, cols, generator=g, device=cuda).to(dtype))
        assert torch.equal(y.detach(), b.to(dtype).expand(rows, cols))
        assert not dw.any()
