"""What the dense gated block does where h leaves f16's range, as its documentation says."""
from __future__ import annotations

import pytest
import torch

from deepseeker import gated

pytestmark = pytest.mark.gpu


def block(T, dtype, device, big):
    """One row of x is `big` times as large as the others; h is about big^2 there, y about 2^-6 of it."""
    g = torch.Generator(device=device).manual_seed(4)
    n = lambda r, c, s: torch.randn(r, c, generator=g, device=device) * s  # noqa: E731
    H, I = 128, 96
    x = n(T, H, 1.0)
    x[3] *= big
    return [t.to(dtype) for t in (x, n(I, H, H ** -0.5), n(I, H, H ** -0.5), n(H, I, I ** -0.5 * 2.0 ** -6))]


@pytest.mark.parametrize("T", [20, 300])
def test_range_of_h(T, cuda):
    for dtype in (torch.float16, torch.bfloat16):
        ins = block(T, dtype, cuda, 400.0)
        x, w1, w3, w2 = (t.double() for t in ins)
        g, u = x @ w1.T, x @ w3.T
        h = g * torch.sigmoid(g) * u
        want = h @ w2.T
        assert float(h.abs().max()) > 65504 and float(want.abs().max()) < 65504
        y = gated.gated_ffn(*ins)
        others = [i for i in range(T) if i != 3]
        assert torch.isfinite(y[others]).all()
        if dtype == torch.float16:                   # the infinity shows: every value of that row has it as a term
            assert not torch.isfinite(y[3]).any()
        else:
            assert float((y[3].double() - want[3]).norm()) <= 2.0 ** -7 * float(want[3].norm())
        # clamps up to 255 keep |h| below 255^2 = 65,025
        hc = g.clamp(max=255) * torch.sigmoid(g) * u.clamp(-255, 255)
        y = gated.gated_ffn(*ins, limit=255.0)
        want = hc @ w2.T
        assert float((y.double() - want).norm()) <= 2.0 ** -7 * float(want.norm()) and torch.isfinite(y).all()
    clean = block(T, torch.float16, cuda, 1.0)
    assert torch.equal(gated.gated_ffn(*clean)[others], gated.gated_ffn(*block(T, torch.float16, cuda, 400.0))[others])
