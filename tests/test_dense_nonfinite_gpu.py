"""Extreme and non-finite values through the dense operators, in every type and on both kernels (few rows, many)."""
from __future__ import annotations

import math

import pytest
import torch

from deepseeker import gated, mx4
from test_gated_gpu import both, formula, make
from test_mx4_gpu import data, emulate, unpack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 17])
def test_quantize_extremes_of_16_bits(rows, dtype, cuda):
    """The types' subnormals, smallest and largest values, zeros of both signs, ties, infinities and NaN."""
    f = torch.finfo(dtype)
    sub, tiny, top = f.smallest_normal * f.eps, f.smallest_normal, f.max
    lines = [[sub, 3 * sub, 0.0, -sub], [2 * sub, 5 * sub, -7 * sub, 6 * sub], [tiny, -tiny / 2, tiny / 4, 0.0], [6 * tiny, tiny, -tiny, 1.5 * tiny],
             [top, -top, top / 4, 1.0], [top, top / 2, top / 3, top / 16], [top * 0.75, -top / 8, 0.0, 1.0], [-0.0, 0.0, -0.0, 0.0],
             [2.5, -3.5, 1.25, 1.75], [6.0, -6.0, 0.25, -0.25], [0.75, 5.0, -0.75, 7.0], [0.0, math.inf, 1.0, 2.0],
             [math.nan, 1.0, 2.0, 3.0], [-math.inf, math.nan, 0.0, 1.0]]
    for first in range(0, len(lines), rows):
        some = lines[first:first + rows]
        x = torch.zeros(len(some), 72, device=cuda, dtype=dtype)
        x[:, 5:9] = torch.tensor(some, device=cuda, dtype=torch.float64).to(dtype)
        x[:, 40] = 1.0
        code, byte, vals = emulate(x)
        # magnitudes that round to 2^128 stand for a value outside f32
        vals = torch.where(vals.abs() >= 2.0 ** 128, torch.sign(vals) * math.inf, vals)
        for view in (x, x[:, 1:], x[:, :70]):       # whole groups, unaligned rows, an uneven end
            q = mx4.quantize(view)
            if view.data_ptr() != x.data_ptr():
                code_v, byte_v, vals_v = emulate(view)
                vals_v = torch.where(vals_v.abs() >= 2.0 ** 128, torch.sign(vals_v) * math.inf, vals_v)
            else:
                code_v, byte_v, vals_v = code, byte, vals[:, : view.shape[1]]
            assert torch.equal(unpack(q.packed), code_v) and torch.equal(q.scales.cpu().long(), byte_v)
            for to in (torch.float32, torch.bfloat16):
                got = q.dequantize(to).cpu().double()
                assert torch.equal(torch.isnan(got), torch.isnan(vals_v)) and torch.equal(got.nan_to_num(7), vals_v.nan_to_num(7))


@pytest.mark.parametrize("T", [9, 40, 300])
def test_4bit_rows(T, cuda):
    """A NaN or an infinity in a row of x makes that row of the result NaN, one in a weight's block its column."""
    x = data(T, 200, cuda, seed=3)
    w = mx4.quantize(data(130, 200, cuda, seed=4))
    clean = mx4.linear(x, w)
    x2 = x.clone()
    x2[4, 199], x2[6, 0], x2[T - 1, 77] = math.inf, math.nan, -math.inf
    bad = [4, 6, T - 1]
    keep = [i for i in range(T) if i not in bad]
    for given in (x2, mx4.quantize(x2)):
        y = mx4.linear(given, w, out_dtype=torch.float32)
        assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[bad]).all()
    scales = w.scales.clone()
    scales[77, 2] = 255
    y = mx4.linear(x, mx4.from_packed(w.packed, scales, 200))
    others = [i for i in range(130) if i != 77]
    assert torch.isnan(y[:, 77]).all() and torch.equal(y[:, others], clean[:, others])
    ws = [mx4.quantize(data(r, c, cuda, seed=s) * c ** -0.5) for r, c, s in ((70, 200, 1), (70, 200, 2), (200, 70, 3))]
    for limit in (None, 1.0):
        clean = mx4.gated_ffn(x, *ws, limit=limit)
        y = mx4.gated_ffn(x2, *ws, limit=limit)
        assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[bad]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [40, 100, 300])
def test_gated_rows(T, dtype, cuda):
    """Non-finite values of x and dy stay in their rows of y and dx, and reach the weight gradients as in the formula."""
    ins, dy = make(T, 72, 56, dtype, cuda)
    x, gy = ins[0].clone(), dy.clone()
    x[7, 3], x[T - 1, 5] = math.nan, math.inf
    gy[9, 70], gy[11, 0] = math.nan, -math.inf
    for limit in (None, 1.0):
        clean = both(ins, dy, limit)[0]
        for a, g, bad in ((x, dy, [7, T - 1]), (ins[0], gy, [9, 11])):
            got = both((a, *ins[1:]), g, limit)[0]
            keep = [i for i in range(T) if i not in bad]
            assert torch.equal(got[1][keep], clean[1][keep])
            if a is x:
                assert torch.equal(got[0][keep], clean[0][keep]) and torch.isnan(got[0][7]).all()
                want = formula(a.double(), *[t.double() for t in ins[1:]], limit)
                assert torch.equal(torch.isnan(got[0][T - 1]), torch.isnan(want[T - 1]))
            else:
                assert torch.equal(got[0], clean[0])
            assert torch.isnan(got[1][bad[0]]).all()                # every value of dx's row has the NaN as a term
            if a is x:                                              # every weight's gradient has row 7 as a term
                assert limit or not any(torch.isfinite(t).any() for t in got[2:4])
            else:
                b = [t.detach().double().requires_grad_() for t in ins]
                want = torch.autograd.grad(formula(*b, limit), b, g.double())
                assert all(torch.equal(torch.isfinite(p), torch.isfinite(w)) for p, w in zip(got[2:], want[1:]))
