"""Quantisation to the 4-bit format and back (deepseeker.mx4) where a thread takes several groups (millions of
values), on rows of every kind: whole, aligned with an uneven end or a gap, and unaligned."""
from __future__ import annotations

import pytest
import torch

from deepseeker import mx4
from test_mx4_gpu import data, emulate, unpack

pytestmark = pytest.mark.gpu
#: rows, columns, gap behind a row, offset of its first value.  A thread takes
#: several groups of 16 values from 303,104 of them on (148 SMs); its groups are
#: 256 apart, within a row of more than 256 groups (4,096 values) or rows apart.
CASES = [(8192, 1024, 0, 0), (8192, 1288, 0, 0), (8200, 1001, 0, 0), (8192, 1024, 8, 0), (8192, 1024, 5, 3), (2000, 5000, 0, 0),
         (2003, 5001, 0, 0), (1500, 8192, 24, 16), (20001, 264, 0, 0), (40000, 100, 4, 0), (160000, 17, 0, 0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,gap,off", CASES)
def test_quantise_and_back(rows, cols, gap, off, dtype, cuda):
    wide = torch.full((rows, cols + gap), float("nan"), dtype=dtype, device=cuda)
    x = wide[:, off:off + cols]
    x.copy_(data(rows, cols, cuda, seed=rows, dtype=dtype))
    nb, nc = -(-cols // 32), -(-cols // 128)
    assert rows * nb * 2 >= torch.cuda.get_device_properties(cuda).multi_processor_count * 2048
    q = mx4.quantize(x)
    back, back16 = q.dequantize(), q.dequantize(torch.bfloat16)
    # the definition, at both ends and in between
    g = torch.Generator().manual_seed(0)
    some = torch.cat([torch.arange(40), torch.randint(rows, (120,), generator=g), torch.arange(rows - 40, rows)])
    code, byte, vals = emulate(x[some.to(cuda)])
    pick = lambda t: t[some.to(cuda)].cpu()  # noqa: E731
    assert torch.equal(unpack(pick(q.packed)), code) and torch.equal(pick(q.scales).long(), byte)
    assert torch.equal(pick(back).double(), vals) and torch.equal(pick(back16).double(), vals)
    # every row: as in parts small enough for one group a thread
    part = max(1, 300000 // (2 * nb))
    for a in range(0, rows, part):
        p = mx4.quantize(x[a:a + part])
        b = a + p.rows
        assert torch.equal(p.packed, q.packed[a:b]) and torch.equal(p.scales, q.scales[a:b])
        assert torch.equal(p.dequantize(), back[a:b]) and torch.equal(p.dequantize(torch.bfloat16), back16[a:b])
    # the scale of every row and block in the tensor cores' order, 0 behind the last block
    r, blk = torch.arange(rows, device=cuda)[:, None], torch.arange(nc * 4, device=cuda)[None, :]
    at = ((r // 128) * nc + blk // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + blk % 4
    assert torch.equal(q.atoms[at], torch.nn.functional.pad(q.scales, (0, nc * 4 - nb)))
