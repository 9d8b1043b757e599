"""Handles of the 8-bit operators (deepseeker.int8) that quantisation itself does not make: no rows, scales of either
sign; and what decides between the kernels of few rows.

A product's tolerance: the sum is exact, its conversion to f32 and each scale round once (u = 2^-24 each).
"""
from __future__ import annotations

import pytest
import torch

from deepseeker import int8

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def normal(rows, cols, device, seed=0, dtype=F32):
    return torch.randn(rows, cols, generator=torch.Generator(device=device).manual_seed(seed), device=device).to(dtype)


def product(q, w):
    sums = q.codes.double() @ w.codes.double().T                        # whole numbers below 2^53
    return sums * q.scales.double()[:, None] * w.scales.double()


def close(y, want):
    assert y.dtype == F32 and y.shape == want.shape
    assert bool(((y.double() - want).abs() <= (4 * U + 8 * U * U) * want.abs()).all())   # and the result's own rounding


@pytest.mark.parametrize("rows", [1, 3, 12, 40, 300, 2000])
def test_scales_of_either_sign(rows, cuda):
    """Scales of stored codes whose product with the sum leaves f32 on the way unless the one nearer to 0 comes first."""
    codes = (normal(rows, 96, cuda, rows) * 40).clamp(-128, 127).to(torch.int8)
    wide = (normal(520, 96, cuda, 1) * 40).clamp(-128, 127).to(torch.int8)
    for a, b in ((-1e36, 1e-30), (1e-30, -1e36), (-1e36, -1e-30), (-1e-30, -1e36), (1e36, 1e-30), (-3.0, 2.0)):
        q = int8.from_codes(codes, torch.full((rows,), a, device=cuda))
        w = int8.from_codes(wide, torch.full((520,), b, device=cuda))
        close(int8.linear(q, w, out_dtype=F32), product(q, w))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_weights_of_no_rows(dtype, cuda):
    x = normal(6, 40, cuda, dtype=dtype)
    none = int8.quantize(normal(3, 40, cuda)[:0])
    for rows in (x, x[:1], x[:0], x[0], x.view(2, 3, 40), int8.quantize(x), int8.quantize(x[:0])):
        y = int8.linear(rows, none)
        assert y.shape == (*rows.shape[:-1], 0) and y.dtype == (BF16 if isinstance(rows, int8.Int8Tensor) else dtype)
    assert int8.linear(x, none, out_dtype=F16).dtype == F16
    for bad in (x[:, :39], x.double(), x.cpu()):
        with pytest.raises(ValueError):
            int8.linear(bad, none)


def test_scales_that_ask_for_a_derivative(cuda):
    codes = torch.ones(3, 16, dtype=torch.int8, device=cuda)
    scales = torch.ones(3, device=cuda, requires_grad=True)
    with pytest.raises(ValueError, match="backward"):
        int8.from_codes(codes, scales)
    with torch.no_grad():
        assert torch.equal(int8.from_codes(codes, scales).dequantize(), torch.ones(3, 16, device=cuda))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones(3, device=cuda), torch.ones(3, device=cuda))
        with pytest.raises(ValueError, match="forward-mode"):
            int8.from_codes(codes, dual)


@pytest.mark.parametrize("K", [33, 300, 1001, 4096])
@pytest.mark.parametrize("rows", [1, 2, 3, 4])
def test_few_rows_by_every_width(rows, K, cuda):
    """Each number of features that a block takes (4, 8 or 16, by how many there are for an SM), whole and with a rest."""
    wave = 2 * torch.cuda.get_device_properties(cuda).multi_processor_count
    x = normal(rows, K, cuda, K, BF16)
    q = int8.quantize(x)
    for n in (1, 4 * wave, 4 * wave - 3, 4 * wave + 7, 8 * wave, 8 * wave - 5, 8 * wave + 9, 16 * wave + 8):
        w = int8.quantize(normal(n, K, cuda, n))
        want = product(q, w)
        y = int8.linear(x, w, out_dtype=F32)
        close(y, want)
        assert torch.equal(int8.linear(q, w, out_dtype=F32), y)
    assert int8.status() == 0


def test_the_scale_is_a_product(cuda):
    """A row's scale is max * (1 / 127), factor and product rounded to f32.  It can be a unit of the last place from
    the rounded quotient max / 127, and half of the maximum, next to the middle of two codes, then has another code."""
    x = torch.tensor([[143.0, 71.5], [144.0, -72.0], [254.0, 127.0], [127.0, 63.5]], device=cuda)
    for dtype in (F32, BF16, F16):
        q = int8.quantize(x.to(dtype))
        assert torch.equal(q.scales, x[:, 0] * torch.tensor(1 / 127, device=cuda))
        assert q.codes.tolist() == [[127, 64], [127, -64], [127, 64], [127, 64]]
    quotient = torch.tensor([143 / 127, 144 / 127], dtype=torch.float64).float()     # rounded once: one unit above
    assert bool((q.scales[:2].cpu() < quotient).all())
    by_quotient = torch.round(x[:2].cpu().double() / quotient.double()[:, None])
    assert by_quotient.tolist() == [[127, 63], [127, -63]]
    # stored codes are taken as they are, whichever rule made them
    held = int8.from_codes(by_quotient.to(torch.int8).to(cuda), quotient.to(cuda))
    assert torch.equal(held.dequantize().cpu(), by_quotient.float() * quotient[:, None])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [4096, 4095])
def test_values_of_matrices_beyond_l2(cols, dtype, cuda):
    """Results on both sides of the size from which they are written past L2."""
    least = 126 * 2 ** 20 // (cols * torch.finfo(dtype).bits // 8)
    for rows in (least, least + 1):
        codes = torch.randint(-128, 128, (rows, cols), device=cuda, dtype=torch.int8)
        scales = torch.rand(rows, device=cuda) + 0.5
        got = int8.from_codes(codes, scales).dequantize(dtype)
        assert torch.equal(got, (codes.float() * scales[:, None]).to(dtype))
