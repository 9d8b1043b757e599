"""Microscaled 4-bit dense operators (deepseeker.mx4) against their definition in 64 bits.

Tolerances, derived before the first run:
  * codes and scales: exact (every step of the definition is exact in 64 bits);
  * product: operands are exact, so only the f32 accumulation is off.  A sum of
    K products is K / 64 additions of 64-wide dot products; allowing each
    addition 2^-22 of the largest partial sum and each dot product 64 dropped
    parts of 2^-24 of its largest term, |error| <= (K / 64 * 2^-22 + 2^-18)
    sum |a b|, plus the rounding of the output (u |y| with the type's unit
    roundoff u, and 2^-24 in f16);
  * gated block: h is quantised from f32 sums, so an h within about 1e-6 of
    the middle between two codes may go the other way: about 1e-5 of the
    elements by at most half their size, a relative L2 of 2e-3 of y at most;
    asserted 5e-3 plus the output's unit roundoff.
"""
from __future__ import annotations

import math

import pytest
import torch

from deepseeker import metal_fp4, mx4, synthetic

pytestmark = pytest.mark.gpu
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def emulate(x):
    """(codes [rows, 32 nb], scale bytes [rows, nb], values [rows, cols]) of the definition, on the CPU in float64."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    nb = -(-cols // 32)
    b = torch.zeros(rows, nb * 32, dtype=torch.float64)
    b[:, :cols] = x
    b = b.view(rows, nb, 32)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(top)
    m, ex = torch.frexp(torch.where(bad, torch.ones_like(top), top))
    e = torch.where(m <= 0.75, ex - 3, ex - 2).clamp(min=-127)
    e = torch.where((top == 0) | bad, torch.zeros_like(e), e)
    a = torch.where(bad[..., None], torch.zeros_like(b), b) / torch.exp2(e.double())[..., None]
    dist = (a.abs()[..., None] - GRID).abs()
    near = dist == dist.amin(-1, keepdim=True)
    idx = torch.arange(8)
    # the nearest code, the even one of two
    code = torch.where(near, idx + 100 * (idx % 2), torch.full_like(idx, 1000)).amin(-1) % 100
    sign = (a < 0) & (code > 0)
    vals = torch.where(sign, -1.0, 1.0) * GRID[code] * torch.exp2(e.double())[..., None]
    vals = torch.where(bad[..., None], torch.full_like(vals, math.nan), vals)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    return (code + 8 * sign).view(rows, -1), byte, vals.view(rows, -1)[:, :cols]


def unpack(packed):
    p = packed.cpu().long()
    return torch.stack([p & 15, p >> 4], -1).view(p.shape[0], -1)


def data(rows, cols, device, seed=0, dtype=torch.float32):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=device) * torch.exp(torch.randn(1, cols, generator=g, device=device))
    half = torch.rand(rows, cols, generator=g, device=device) < 0.2
    x = torch.where(half, torch.round(x * 4) / 4, x)             # ties and exact codes
    if rows > 3:
        x[3] = 0
    return x.to(dtype)


SHAPES = [(1, 1), (1, 32), (2, 33), (3, 64), (5, 31), (8, 4096), (127, 130), (128, 256), (129, 999), (300, 72),
          (1, 5000), (4097, 40)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(rows, cols, dtype, cuda):
    x = data(rows, cols, cuda, seed=rows + cols, dtype=dtype)
    q = mx4.quantize(x)
    code, byte, vals = emulate(x)
    assert torch.equal(unpack(q.packed), code)
    assert torch.equal(q.scales.cpu().long(), byte)
    assert torch.equal(q.dequantize().cpu().double(), vals)
    assert torch.equal(q.dequantize(torch.bfloat16).cpu().double(), vals)
    again = mx4.from_packed(q.packed, q.scales, cols)             # atoms of both ways: the rows and blocks that exist
    nb, nc = -(-cols // 32), -(-cols // 128)
    r, b = torch.meshgrid(torch.arange(rows), torch.arange(nc * 4), indexing="ij")
    at = ((r // 128) * nc + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
    a0, a1 = q.atoms.cpu()[at], again.atoms.cpu()[at]
    assert torch.equal(a0, a1) and torch.equal(a0[:, :nb].long(), byte) and int(a0[:, nb:].long().sum()) == 0


def test_quantize_extremes(cuda):
    tiny = 2.0 ** -149
    rows = [[tiny, 3 * tiny, 0.0, -tiny], [2.0 ** -126, -2.0 ** -127, 2.0 ** -128, 0.0], [6.0, -6.0, 0.25, -0.25],
            [6.0000005, 1.0, -0.75, 5.0], [1e38, -1e37, 1.0, 0.0], [-0.0, 0.0, -0.0, 0.0], [2.5, -3.5, 1.25, 1.75],
            [0.0, float("inf"), 1.0, 2.0], [float("nan"), 1.0, 2.0, 3.0], [-float("inf"), float("nan"), 0.0, 1.0]]
    x = torch.zeros(len(rows), 70, device=cuda)
    x[:, :4] = torch.tensor(rows, device=cuda)
    x[:, 40] = 1.0                                                # the next block is not touched by a NaN
    q = mx4.quantize(x)
    code, byte, vals = emulate(x)
    assert torch.equal(unpack(q.packed), code) and torch.equal(q.scales.cpu().long(), byte)
    got = q.dequantize().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(vals)) and torch.equal(got.nan_to_num(), vals.nan_to_num())
    assert torch.isnan(got[7:, :32]).all() and torch.isfinite(got[:, 32:]).all()


def test_quantize_agrees_with_the_bank_quantiser(cuda):
    w = data(96, 512, cuda, seed=4)
    packed, scales = synthetic.quantize_fp4(w)
    q = mx4.quantize(w)
    assert torch.equal(q.packed, packed) and torch.equal(q.scales, scales)
    assert torch.equal(metal_fp4.dequant(packed, scales).view(96, 512), q.dequantize())


def test_quantize_strides_and_shapes(cuda):
    x = data(60, 150, cuda, seed=6, dtype=torch.bfloat16)
    want = mx4.quantize(x).dequantize()
    for pad, off in ((8, 0), (10, 2), (1, 1), (3, 3)):
        big = torch.full((60, 150 + pad), float("nan"), dtype=x.dtype, device=cuda)
        big[:, off:off + 150] = x
        assert torch.equal(mx4.quantize(big[:, off:off + 150]).dequantize(), want)
    assert torch.equal(mx4.quantize(x.t().contiguous().t()).dequantize(), want)
    q = mx4.quantize(x.view(5, 12, 150))
    assert q.shape == (5, 12, 150) and torch.equal(q.dequantize(), want.view(5, 12, 150))
    assert mx4.quantize(x[:0]).dequantize().shape == (0, 150)


def product_check(y, xv, wv, K, dtype):
    want = xv @ wv.T
    mass = xv.abs() @ wv.abs().T
    bound = (K / 64 * 2.0 ** -22 + 2.0 ** -18) * mass + UNIT[dtype] * want.abs() + (2.0 ** -24 if dtype == torch.float16 else 0)
    err = (y.double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


PRODUCTS = [(1, 32, 128), (1, 4096, 4096), (2, 64, 1), (15, 33, 40), (16, 256, 128), (17, 999, 513), (33, 160, 264),
            (64, 1, 7), (65, 288, 640), (100, 1001, 777), (128, 512, 128), (129, 544, 200), (300, 2560, 136),
            (1111, 96, 1280), (1, 20000, 24), (257, 384, 256), (2048, 128, 384)]


@pytest.mark.parametrize("dtype,to", [(torch.bfloat16, None), (torch.float32, torch.float32), (torch.float16, torch.float32),
                                      (torch.float16, torch.float16)])
@pytest.mark.parametrize("T,K,N", PRODUCTS)
def test_linear(T, K, N, dtype, to, cuda):
    x = data(T, K, cuda, seed=T, dtype=dtype)
    g = torch.Generator(device=cuda).manual_seed(N)
    w = mx4.quantize(torch.randn(N, K, generator=g, device=cuda) * 0.02)
    y = mx4.linear(x, w, out_dtype=to)
    assert y.shape == (T, N) and y.dtype == (to or dtype)
    q = mx4.quantize(x)
    product_check(y, q.dequantize().double(), w.dequantize().double(), K, y.dtype)
    assert torch.equal(mx4.linear(q, w, out_dtype=to or dtype), y)          # quantised before or on the way
    assert mx4.status() == 0


def test_linear_large(cuda):
    x = data(2500, 4096, cuda, seed=1, dtype=torch.bfloat16)
    w = mx4.quantize(data(4096, 4096, cuda, seed=2))
    xv, wv = mx4.quantize(x).dequantize().double(), w.dequantize().double()
    for to in (torch.bfloat16, torch.float32):
        product_check(mx4.linear(x, w, out_dtype=to), xv, wv, 4096, to)


def test_linear_non_finite_rows(cuda):
    x = data(20, 200, cuda, seed=3)
    w = mx4.quantize(data(130, 200, cuda, seed=4))
    clean = mx4.linear(x, w)
    x[4, 199], x[6, 0] = float("inf"), float("nan")
    y = mx4.linear(x, w)
    keep = [i for i in range(20) if i not in (4, 6)]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[[4, 6]]).all()
    scales = w.scales.clone()
    scales[77, 2] = 255                                                      # a weight block that is NaN
    bad = mx4.linear(x[:4], mx4.from_packed(w.packed, scales, 200))
    assert torch.isnan(bad[:, 77]).all()
    others = [i for i in range(130) if i != 77]
    assert torch.equal(bad[:, others], clean[:4][:, others])


def block(x, w1, w3, w2, limit):
    g, u = x @ w1.T, x @ w3.T
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    h = g * torch.sigmoid(g) * u
    return emulate(h)[2].to(x.device) @ w2.T


BLOCKS = [(1, 64, 32), (1, 4096, 2048), (2, 96, 40), (17, 999, 200), (40, 256, 128), (70, 72, 711), (128, 512, 96),
          (130, 1000, 520), (300, 33, 1000), (515, 640, 256)]


@pytest.mark.parametrize("T,H,I", BLOCKS)
def test_gated_block(T, H, I, cuda):
    for limit, dtype in ((None, torch.bfloat16), (1.0, torch.float32), (10.0, torch.float16)):
        x = data(T, H, cuda, seed=T, dtype=dtype)
        ws = [mx4.quantize(data(r, c, cuda, seed=s) * c ** -0.5) for r, c, s in ((I, H, 1), (I, H, 2), (H, I, 3))]
        y = mx4.gated_ffn(x, *ws, limit=limit)
        q = mx4.quantize(x)
        want = block(q.dequantize().double(), *[w.dequantize().double() for w in ws], limit)
        assert y.shape == (T, H) and y.dtype == dtype
        err, norm = float((y.double() - want).norm()), float(want.norm())
        assert err <= (5e-3 + UNIT[dtype]) * norm + 2.0 ** -24 * (T * H) ** 0.5, (limit, dtype, err / max(norm, 1e-30))
        assert torch.equal(mx4.gated_ffn(q, *ws, limit=limit, out_dtype=dtype), y)
    assert mx4.status() == 0


def test_gated_block_non_finite_rows(cuda):
    x = data(9, 130, cuda, seed=3, dtype=torch.bfloat16)
    ws = [mx4.quantize(data(r, c, cuda, seed=s) * c ** -0.5) for r, c, s in ((70, 130, 1), (70, 130, 2), (130, 70, 3))]
    clean = mx4.gated_ffn(x, *ws)
    x[5, 129] = float("nan")
    y = mx4.gated_ffn(x, *ws, limit=None)
    keep = [i for i in range(9) if i != 5]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[5]).all()


def test_shapes_streams_and_graphs(cuda):
    x = data(24, 128, cuda, seed=1, dtype=torch.bfloat16)
    ws = [mx4.quantize(data(r, c, cuda, seed=s) * c ** -0.5) for r, c, s in ((64, 128, 1), (64, 128, 2), (128, 64, 3))]
    want = mx4.gated_ffn(x, *ws)
    assert torch.equal(mx4.gated_ffn(x.view(2, 3, 4, 128), *ws), want.view(2, 3, 4, 128))
    assert torch.equal(mx4.linear(x[0], ws[0]), mx4.linear(x[:1], ws[0])[0])
    assert mx4.linear(x[:0], ws[0]).shape == (0, 64) and mx4.gated_ffn(x[:0], *ws).shape == (0, 128)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = mx4.gated_ffn(x, *ws)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx4.gated_ffn(x, *ws)
        lin = mx4.linear(x, ws[0])
    out.zero_(), lin.zero_()
    graph.replay()
    assert torch.equal(out, want) and torch.equal(lin, mx4.linear(x, ws[0]))


def test_repeats_bit_for_bit(cuda):
    for T in (1, 50, 400):
        x = data(T, 2048, cuda, seed=1, dtype=torch.bfloat16)
        ws = [mx4.quantize(data(r, c, cuda, seed=s) * c ** -0.5) for r, c, s in ((640, 2048, 1), (640, 2048, 2), (2048, 640, 3))]
        first = mx4.gated_ffn(x, *ws)
        assert all(torch.equal(mx4.gated_ffn(x, *ws), first) for _ in range(3))


def test_refusals(cuda):
    x = data(4, 64, cuda)
    w = mx4.quantize(data(32, 64, cuda))
    for bad in (x.cpu(), x.double(), x.long(), x[:, :0], torch.tensor(1.0, device=cuda), x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            mx4.quantize(bad)
        with pytest.raises(ValueError):
            mx4.linear(bad, w)
    with torch.no_grad():
        assert mx4.linear(x.clone().requires_grad_(), w).shape == (4, 32)
    for args in ((x[:, :63], w), (x, x), (mx4.quantize(x[:, :32]), w)):
        with pytest.raises(ValueError):
            mx4.linear(*args)
    with pytest.raises(ValueError):
        mx4.linear(x, w, out_dtype=torch.float64)
    w2 = mx4.quantize(data(64, 32, cuda))
    for ws in ((w, w, w), (w, w2, w2), (w, w, w2.packed)):
        with pytest.raises(ValueError):
            mx4.gated_ffn(x, *ws)
    for limit in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            mx4.gated_ffn(x, w, w, w2, limit=limit)
    for p, s, c in ((w.packed, w.scales, 65), (w.packed, w.scales, 32), (w.packed[:31], w.scales, None),
                    (w.packed.int(), w.scales, None), (w.packed, w.scales[0], None), (w.packed.cpu(), w.scales, None)):
        with pytest.raises(ValueError):
            mx4.from_packed(p, s, c)
    with pytest.raises(ValueError):
        w.dequantize(torch.float16)
