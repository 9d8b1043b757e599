"""Dense operators where element offsets pass 32 bits: the last rows of a
matrix of more than 2^32 elements against the same rows alone."""
from __future__ import annotations

import pytest
import torch

from deepseeker import gated, mx4

pytestmark = pytest.mark.gpu


def need(gib: float) -> None:
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


ROWS, LAST = 2 ** 21 + 37, 700


def test_quantise_and_product(cuda):
    need(60)
    cols, out = 2080, 2064
    x = torch.empty(ROWS, cols, dtype=torch.bfloat16, device=cuda)
    x.normal_(generator=torch.Generator(device=cuda).manual_seed(1))
    assert ROWS * cols > 2 ** 32 and ROWS * out > 2 ** 32
    q = mx4.quantize(x)
    tail = mx4.quantize(x[-LAST:])
    assert torch.equal(q.packed[-LAST:], tail.packed) and torch.equal(q.scales[-LAST:], tail.scales)
    v = q.dequantize(torch.bfloat16)
    assert torch.equal(v[-LAST:], tail.dequantize(torch.bfloat16)) and torch.equal(v[:5], mx4.quantize(x[:5]).dequantize(torch.bfloat16))
    del v
    w = mx4.quantize(torch.randn(out, cols, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda))
    y = mx4.linear(q, w)
    assert torch.equal(y[-LAST:], mx4.linear(tail, w)) and torch.equal(y[:130], mx4.linear(x[:130], w))
    assert mx4.status() == 0


def test_gated_block(cuda):
    need(120)
    H, I = 64, 2064
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.empty(ROWS, H, dtype=torch.bfloat16, device=cuda).normal_(generator=g).requires_grad_()
    w1, w3, w2 = ((torch.randn(r, c, generator=g, device=cuda) * c ** -0.5).bfloat16().requires_grad_()
                  for r, c in ((I, H), (I, H), (H, I)))
    dy = torch.empty(ROWS, H, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    assert ROWS * I > 2 ** 32
    y = gated.gated_ffn(x, w1, w3, w2, limit=2.0)
    dx, dw1, dw3, dw2 = torch.autograd.grad(y, (x, w1, w3, w2), dy)
    xt = x.detach()[-LAST:].requires_grad_()
    yt = gated.gated_ffn(xt, w1, w3, w2, limit=2.0)
    dxt, = torch.autograd.grad(yt, xt, dy[-LAST:])
    # the same sums; another tile width may round them in another order (2^-8: one bf16 step)
    assert rel(y.detach()[-LAST:], yt.detach()) <= 2.0 ** -8 and rel(dx[-LAST:], dxt) <= 2.0 ** -8
    del y, dx
    # weight gradients are sums over the rows: three parts, each rounded to bf16, against the whole
    total = [torch.zeros_like(t, dtype=torch.float64) for t in (w1, w3, w2)]
    for part in torch.arange(ROWS, device="cpu").tensor_split(3):
        a, b = int(part[0]), int(part[-1]) + 1
        yp = gated.gated_ffn(x.detach()[a:b], w1, w3, w2, limit=2.0)
        for t, d in zip(total, torch.autograd.grad(yp, (w1, w3, w2), dy[a:b])):
            t += d.double()
        del yp
    # f32 sums of 2 M terms: 32768 additions of 64, each off by 2^-24 of a partial sum at most, beside the roundings
    assert all(rel(d, t) <= 2.0 ** -7 for d, t in zip((dw1, dw3, dw2), total))
    assert gated.status() == 0


def test_gated_4bit_block(cuda):
    need(60)
    H, I = 64, 2080
    g = torch.Generator(device=cuda).manual_seed(4)
    x = torch.empty(ROWS, H, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    ws = [mx4.quantize(torch.randn(r, c, generator=g, device=cuda) * c ** -0.5) for r, c in ((I, H), (I, H), (H, I))]
    y = mx4.gated_ffn(x, *ws)
    assert torch.equal(y[-LAST:], mx4.gated_ffn(x[-LAST:], *ws))
    assert mx4.status() == 0
