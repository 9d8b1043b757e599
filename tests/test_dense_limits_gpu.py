"""Limits of the dense operators' arguments that a 32-bit field of the C ABI would change silently."""
from __future__ import annotations

import pytest
import torch

from deepseeker import gated, mx4

pytestmark = pytest.mark.gpu


def operands(device, T=4, H=64, I=32):
    g = torch.Generator(device=device).manual_seed(2)
    return [torch.randn(r, c, generator=g, device=device).bfloat16() for r, c in ((T, H), (I, H), (I, H), (H, I))]


def test_a_limit_that_f32_rounds_to_zero(cuda):
    """0 stands for no clamps, so a limit below f32's smallest value is refused; that value clamps."""
    x, *ws = operands(cuda)
    q = [mx4.quantize(w) for w in ws]
    for limit in (1e-46, 2.0 ** -150, 5e-324):
        with pytest.raises(ValueError, match="limit"):
            gated.gated_ffn(x, *ws, limit=limit)
        with pytest.raises(ValueError, match="limit"):
            mx4.gated_ffn(x, *q, limit=limit)
    for limit in (2.0 ** -149, 1.0001 * 2.0 ** -150):
        # |h| <= limit times silu(limit), nothing in 16 bits
        assert float(gated.gated_ffn(x, *ws, limit=limit).abs().max()) == 0
        assert float(mx4.gated_ffn(x, *q, limit=limit).abs().max()) == 0
    assert torch.equal(gated.gated_ffn(x, *ws, limit=1e300), gated.gated_ffn(x, *ws))


def test_sizes_that_32_bits_would_wrap(cuda):
    """2^32 + 64 columns are not 64 (broadcast operands: nothing of that size is allocated)."""
    one = torch.zeros(1, 1, dtype=torch.bfloat16, device=cuda)
    for n in (2 ** 32 + 64, 2 ** 31, 2 ** 17 + 1):
        with pytest.raises(ValueError, match="2.17"):
            gated.gated_ffn(one.expand(1, n), one.expand(1, n), one.expand(1, n), one.expand(n, 1))
        with pytest.raises(ValueError, match="2.17"):
            gated.gated_ffn(one, one.expand(n, 1), one.expand(n, 1), one.expand(1, n))
