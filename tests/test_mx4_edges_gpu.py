"""Microscaled 4-bit operators (deepseeker.mx4) at their edges."""
from __future__ import annotations

import pytest
import torch

from deepseeker import mx4

pytestmark = pytest.mark.gpu


def weights(H, I, device):
    g = torch.Generator(device=device).manual_seed(1)
    return [mx4.quantize(torch.randn(r, c, generator=g, device=device) * c ** -0.5) for r, c in ((I, H), (I, H), (H, I))]


def test_no_rows_quantised(cuda):
    ws = weights(128, 64, cuda)
    for shape in ((0, 128), (3, 0, 128)):
        q = mx4.quantize(torch.empty(shape, device=cuda))
        y = mx4.linear(q, ws[0])
        assert y.shape == (*shape[:-1], 64) and y.dtype == torch.bfloat16
        z = mx4.gated_ffn(q, *ws, out_dtype=torch.float32)
        assert z.shape == shape and z.dtype == torch.float32
