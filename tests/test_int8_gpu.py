"""8-bit integer dense operators (deepseeker.int8) against their definition in 64 bits.

Tolerances, derived before the first run, u = 2^-24:
  * codes and scales: exact;
  * values: code * scale rounded to f32, then to the result's type: (u + v) |y|, v the type's unit roundoff;
  * product: the sum is exact, its conversion to f32 and each scale round once: (3 u + v (1 + 3 u)) |y|,
    and half the smallest number of the type (f16: 2^-25, f32: three times 2^-150) where results leave its
    normal range.  From 65520, half a step above 65504, f16 rounds to infinity.
"""
from __future__ import annotations

import math

import pytest
import torch

from deepseeker import int8, moe

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def emulate(x):
    """(codes, scales f32) of the definition, on the CPU in float64."""
    x = x.detach().cpu().double()
    top = x.abs().amax(1)
    bad = ~torch.isfinite(top)
    scale = torch.where(bad, torch.full_like(top, math.nan), top).float() * torch.tensor(1 / 127)   # f32 throughout
    s = torch.where(bad | (scale == 0), torch.ones_like(top), scale.double())
    q = torch.round((x / s[:, None]).nan_to_num(0, 0, 0)).clamp(-127, 127)
    return torch.where((bad | (scale == 0))[:, None], torch.zeros_like(q), q).to(torch.int8), scale


def data(rows, cols, device, seed=0, dtype=F32):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=device) * torch.exp(torch.randn(1, cols, generator=g, device=device))
    x[: rows // 3] = torch.round(x[: rows // 3] * 8) / 16          # many quotients in the middle of two codes
    if rows > 2:
        x[0, 0] = 127.0 / 2
        x[0].clamp_(-63.5, 63.5)                                   # scale 1 / 2
    if rows > 3:
        x[3] = 0
    return x.to(dtype)


def same(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


SHAPES = [(1, 1), (1, 16), (2, 33), (3, 64), (5, 31), (8, 4096), (127, 130), (9, 255), (129, 999), (300, 72), (1, 5000),
          (4097, 40), (2, 16384), (2, 32768), (3, 32769), (2, 131071)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(rows, cols, dtype, cuda):
    x = data(rows, cols, cuda, seed=rows + cols, dtype=dtype)
    q = int8.quantize(x)
    codes, scales = emulate(x)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    want = codes.double() * scales.double()[:, None]
    for to in (F32, BF16, F16):
        got = q.dequantize(to).cpu().double()
        assert bool(((got - want).abs() <= (U + torch.finfo(to).eps / 2) * want.abs() + 2.0 ** -25 * (to == F16)).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [1, 5, 1900])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 17, 64, 255, 257, 1022, 1025, 2049, 4095, 8191, 20001])
def test_rows_anywhere(cols, rows, dtype, cuda):
    """Rows that begin and end between 16-byte boundaries, among values that are no numbers; several turns a block."""
    x = data(rows, cols, cuda, seed=cols, dtype=dtype)
    codes, scales = emulate(x)
    want = codes.float() * scales[:, None]
    for pad, off in ((0, 1), (5, 0), (3, 6)):
        big = torch.full((rows * (cols + pad) + 2 * off,), float("nan"), dtype=dtype, device=cuda)
        view = big[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        view.copy_(x)
        q = int8.quantize(view)
        assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
    for to in (F32, BF16, F16):
        assert torch.equal(q.dequantize(to).cpu(), want.to(to))   # one product, rounded once more


def test_every_tie(cuda):
    """Scale 1: all multiples of 1 / 2, and their neighbours in f32."""
    half = torch.arange(-254, 255, device=cuda).float() / 2
    x = torch.stack([half, torch.nextafter(half, half + 1), torch.nextafter(half, half - 1)])
    x = torch.cat([x.clamp(-127, 127), torch.full((3, 1), 127.0, device=cuda)], 1)
    for factor in (1.0, 3.0, 1 / 3, 1.1e-5, 7e20):                 # and what a scale that rounds makes of them
        y = x * factor
        q = int8.quantize(y)
        codes, scales = emulate(y)
        assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_random_quotients(dtype, cuda):
    """Millions of values with scales of every mantissa."""
    g = torch.Generator(device=cuda).manual_seed(5)
    x = (torch.rand(4096, 1024, generator=g, device=cuda) * 2 - 1).to(dtype)
    q = int8.quantize(x)
    codes, scales = emulate(x)
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)


def test_extremes(cuda):
    tiny, least = 2.0 ** -149, 2.0 ** -126
    rows = [[0.0, -0.0, 0.0, 0.0], [tiny, -tiny, 0.0, 0.0], [63 * tiny, tiny, 0.0, 0.0], [64 * tiny, -3 * tiny, tiny, 0.0],
            [190 * tiny, 100 * tiny, -190 * tiny, tiny], [least, -least / 3, 5 * tiny, 0.0],
            [127 * least, least / 2, -least * 1.5, least], [126.9 * least, least / 2, 3.0 * tiny, 0.0],
            [3.4028234663852886e38, -1e38, 1.0, 0.0], [2.0 ** 127, -(2.0 ** 126), 2.0 ** 120, 1e38],
            [math.inf, 1.0, 2.0, 0.0], [-math.inf, math.nan, 0.0, 1.0], [math.nan, 1.0, 0.0, 3.0], [1.0, -1.0, 0.5, -0.5]]
    for cols in (4, 70, 33000):
        x = torch.zeros(len(rows), cols, device=cuda)
        x[:, -4:] = torch.tensor(rows, device=cuda)
        q = int8.quantize(x)
        codes, scales = emulate(x)
        assert torch.equal(q.codes.cpu(), codes) and same(q.scales.cpu(), scales)
        assert torch.isnan(q.dequantize()[10:13]).all() and torch.isfinite(q.dequantize()[13]).all()
        one = int8.quantize(torch.ones(3, cols, device=cuda))
        y = int8.linear(x, one)
        assert torch.isnan(y[10:13]).all() and torch.isfinite(y[:10]).all() and not y[:3].any()


def test_strides_and_shapes(cuda):
    x = data(60, 150, cuda, seed=6, dtype=BF16)
    want = int8.quantize(x)
    for pad, off in ((8, 0), (10, 2), (1, 1), (3, 3)):
        big = torch.full((60, 150 + pad), float("nan"), dtype=x.dtype, device=cuda)
        big[:, off:off + 150] = x
        got = int8.quantize(big[:, off:off + 150])
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    assert torch.equal(int8.quantize(x.t().contiguous().t()).codes, want.codes)
    q = int8.quantize(x.view(5, 12, 150))
    assert q.shape == q.codes.shape == (5, 12, 150) and q.scales.shape == (5, 12)
    assert torch.equal(q.codes.reshape(60, 150), want.codes) and q.dequantize(F16).shape == (5, 12, 150)
    one = int8.quantize(x[7])
    assert one.shape == one.codes.shape == (150,) and one.scales.shape == () and torch.equal(one.codes, want.codes[7])
    w = int8.quantize(data(24, 150, cuda, seed=1))
    y = int8.linear(x, w)
    assert torch.equal(int8.linear(x.view(5, 12, 150), w), y.view(5, 12, 24))
    assert torch.equal(int8.linear(q, w), y.view(5, 12, 24)) and torch.equal(int8.linear(one, w), y[7])
    assert torch.equal(int8.linear(x[7], w), y[7])
    assert int8.quantize(x[:0]).dequantize().shape == (0, 150) and int8.linear(x[:0], w).shape == (0, 24)
    assert int8.linear(int8.quantize(x[:0]), w).shape == (0, 24)


def product(q, w):
    """Exact sums and the product of two Int8Tensors' values, in float64 (whole numbers below 2^53 are exact)."""
    sums = q.codes.double() @ w.codes.double().T
    return sums * q.scales.double()[:, None] * w.scales.double()[None, :]


def check(y, want):
    v = torch.finfo(y.dtype).eps / 2
    bound = (3 * U + v * (1 + 3 * U)) * want.abs() + (2.0 ** -25 if y.dtype == F16 else 3 * 2.0 ** -150)
    err = (y.double() - want).abs()
    if y.dtype == F16:
        err = torch.where((want.abs() * (1 + 3 * U) >= 65520) & torch.isinf(y) & (y.sign() == want.sign()),
                          torch.zeros_like(err), err)
    assert y.shape == want.shape and bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


PRODUCTS = [(1, 1, 1), (2, 15, 9), (3, 17, 5), (4, 500, 1300), (5, 4096, 300), (7, 10000, 33), (8, 64, 5000),
            (9, 100, 130), (12, 1100, 257), (1, 32, 128), (1, 4096, 4096), (2, 64, 1), (15, 33, 40), (16, 256, 128), (17, 999, 513),
            (32, 130, 96), (33, 160, 264), (64, 1, 7), (65, 288, 640), (100, 1001, 777), (128, 512, 128), (129, 544, 200),
            (200, 2000, 72), (300, 2560, 136), (1111, 96, 1280), (1, 20000, 24), (257, 384, 256), (2048, 128, 384),
            (520, 1024, 4096), (3000, 257, 2049)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,N", PRODUCTS)
def test_linear(M, K, N, dtype, cuda):
    x, w = data(M, K, cuda, seed=M, dtype=dtype), int8.quantize(data(N, K, cuda, seed=N + 1) * K ** -0.5)
    q = int8.quantize(x)
    want = product(q, w)
    for to in (None, F32, BF16, F16):
        y = int8.linear(x, w, out_dtype=to)
        assert y.dtype == (to or dtype)
        check(y, want)
        assert torch.equal(int8.linear(q, w, out_dtype=to or dtype), y)
    assert int8.status() == 0


def test_largest_sums(cuda):
    """K = 2^17 - 1 products of -128 with itself end 16384 below 2^31; of 127 with -127 above -2^31."""
    K = (1 << 17) - 1
    for rows in (1, 130):
        a = torch.full((rows, K), -128, dtype=torch.int8, device=cuda)
        b = torch.full((3, K), -128, dtype=torch.int8, device=cuda)
        b[1], b[2] = 127, 0
        q, w = (int8.from_codes(t, torch.ones(t.shape[0], device=cuda)) for t in (a, b))
        y = int8.linear(q, w, out_dtype=F32)
        want = torch.tensor([K * 128 * 128, -K * 127 * 128, 0], dtype=torch.float64, device=cuda).float()
        assert torch.equal(y, want.expand(rows, 3))


def test_scales_of_every_size(cuda):
    """Scales whose product, or whose product with the sum, leaves f32 while the result does not."""
    x = torch.tensor([[1.0], [1e38], [1e-36], [2.0 ** -120], [3e-44]], device=cuda) * data(5, 64, cuda, seed=2).sign().add(0.5)
    for rows in (x, x.repeat(60, 1)):
        w = torch.tensor([[1.0], [1e-38], [1e37], [1e-10], [1e20]], device=cuda) * data(5, 64, cuda, seed=4).clamp(-1, 1)
        w = w.repeat(8, 1)
        q, p = int8.quantize(rows), int8.quantize(w)
        want = product(q, p)
        got = int8.linear(rows, p)
        fine = want.abs() < 3.4e38
        check(torch.where(fine, got, torch.zeros_like(got)), torch.where(fine, want, torch.zeros_like(want)))
        assert torch.isinf(got[~fine]).all()


def test_from_codes(cuda):
    g = torch.Generator(device=cuda).manual_seed(3)
    codes = torch.randint(-128, 128, (200, 300), generator=g, device=cuda, dtype=torch.int8)
    scales = torch.rand(200, generator=g, device=cuda) + 0.1
    x = int8.quantize(data(40, 300, cuda))
    want = int8.linear(x, int8.from_codes(codes, scales), out_dtype=F32)
    assert torch.equal(int8.from_codes(codes, scales).codes, codes)
    for pad, off in ((20, 0), (20, 16), (20, 3), (1, 0), (4, 4)):
        big = torch.full((200, 300 + pad), 99, dtype=torch.int8, device=cuda)
        big[:, off:off + 300] = codes
        held = int8.from_codes(big[:, off:off + 300], scales)
        assert torch.equal(held.codes, codes) and torch.equal(int8.linear(x, held, out_dtype=F32), want)
        if (300 + pad) % 16 == 0 and off % 16 == 0:
            assert held.codes.data_ptr() == big.data_ptr() + off    # in place
    held = int8.from_codes(codes.t().contiguous().t(), scales.repeat_interleave(2)[::2])
    assert torch.equal(int8.linear(x, held, out_dtype=F32), want) and torch.equal(held.scales, scales)
    assert torch.equal(held.dequantize(), codes.float() * scales[:, None])


def test_results_past_the_matrix_are_left(cuda):
    """Neither the rows nor the columns behind a result are written, whatever the tile."""
    w = int8.quantize(data(72, 256, cuda, seed=1))
    for rows in (1, 17, 100, 300):
        x = data(rows, 256, cuda, seed=rows, dtype=BF16)
        n = rows * 72
        pool = torch.full((n + 4096,), 7.0, dtype=BF16, device=cuda)
        want = int8.linear(x, w)
        from deepseeker import _abi

        ws = torch.empty(int8._workspace_bytes(rows, 256), dtype=torch.uint8, device=cuda)
        for off in (0, 1):                                          # boxes, and row by row
            pool.fill_(7.0)
            _abi.call("ds_int8_linear", x.data_ptr(), None, _abi.DS_BF16, rows, 256, w._ref(), pool[off:].data_ptr(),
                      _abi.DS_BF16, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(pool[off:off + n].view(rows, 72), want) and bool((pool[off + n:] == 7.0).all())
            assert off == 0 or float(pool[0]) == 7.0


def test_streams_and_graphs(cuda):
    w = int8.quantize(data(512, 640, cuda, seed=1))
    xs = [data(r, 640, cuda, seed=r, dtype=BF16) for r in (1, 40, 200)]
    want = [int8.linear(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):                                             # three calls at once
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(int8.linear(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = [x.clone() for x in xs]
    graphs, outs = [], []
    for x in held:
        int8.linear(x, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with moe.graph_capture(graph):
            outs.append(int8.linear(x, w))
        graphs.append(graph)
    for seed in (5, 6):
        for x in held:
            x.copy_(data(*x.shape, cuda, seed=seed + x.shape[0], dtype=BF16))
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, int8.linear(x, w)) for o, x in zip(outs, held))
    assert int8.status() == 0


def test_many_values(cuda):
    """Results past 2^32 elements."""
    rows, N = (1 << 20) + 200, 4104
    x = data(256, 32, cuda, seed=1, dtype=BF16).repeat(rows // 256 + 1, 1)[:rows]
    w = int8.quantize(data(N, 32, cuda, seed=2))
    y = int8.linear(x, w)
    want = int8.linear(x[:256], w)
    for r in (0, 1 << 19, (1 << 20) - 256, 1 << 20):
        n = min(256, rows - r)
        assert torch.equal(y[r:r + n], want[:n])


def test_refusals(cuda):
    x, w = data(4, 64, cuda, dtype=BF16), int8.quantize(data(8, 64, cuda))
    for bad in (x.double(), x.cpu(), x.int(), x[:, :0], x[0, 0], "x"):
        with pytest.raises(ValueError):
            int8.quantize(bad)
        with pytest.raises(ValueError):
            int8.linear(bad, w)
    with pytest.raises(ValueError):
        int8.quantize(torch.zeros(1, 1 << 17, device=cuda))
    for a in ((x, x), (x[:, :63], w), (x, int8.quantize(x.view(1, 4, 64))), (x, w, torch.int8), (int8.quantize(x[:, :8]), w)):
        with pytest.raises(ValueError):
            int8.linear(*a)
    codes, scales = torch.zeros(4, 8, dtype=torch.int8, device=cuda), torch.ones(4, device=cuda)
    for a in ((codes.int(), scales), (codes[0], scales), (codes.cpu(), scales), (codes, scales[:3]), (codes, scales.half()),
              (codes, scales.cpu()), (codes[:0], scales[:0]), (codes[:, :0], scales)):
        with pytest.raises(ValueError):
            int8.from_codes(*a)
    with pytest.raises(ValueError):
        w.dequantize(torch.int8)
    g = x.float().requires_grad_()
    for call in (lambda: int8.quantize(g), lambda: int8.linear(g, w)):
        with pytest.raises(ValueError, match="backward"):
            call()
    with torch.no_grad():
        assert torch.equal(int8.linear(g, w), int8.linear(g.detach(), w))
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x.float(), x.float())
        for call in (lambda: int8.quantize(d), lambda: int8.linear(d, w)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
