"""The dense operators have no forward-mode derivatives and say so: a result without a tangent would read as a zero one."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from deepseeker import gated, mx4

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused(cuda):
    gen = torch.Generator(device=cuda).manual_seed(0)
    ins = [torch.randn(r, c, generator=gen, device=cuda).bfloat16() for r, c in ((4, 64), (32, 64), (32, 64), (64, 32))]
    q = [mx4.quantize(t) for t in ins[1:]]
    want = gated.gated_ffn(*ins), mx4.gated_ffn(ins[0], *q), mx4.linear(ins[0], q[0])
    with forward_ad.dual_level():
        for i in range(4):
            for grad in (False, True):               # an ordinary gradient asked for beside it or not
                a = [t.clone().requires_grad_(grad) for t in ins]
                a[i] = forward_ad.make_dual(ins[i], torch.ones_like(ins[i]))
                with pytest.raises(ValueError, match="forward-mode"):
                    gated.gated_ffn(*a)
        x = forward_ad.make_dual(ins[0], torch.ones_like(ins[0]))
        for call in (lambda: mx4.quantize(x), lambda: mx4.linear(x, q[0]), lambda: mx4.gated_ffn(x, *q)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call()
        # plain tensors inside a level, and the primal of a dual one, are served
        x = forward_ad.unpack_dual(x).primal
        got = gated.gated_ffn(x, *ins[1:]), mx4.gated_ffn(x, *q), mx4.linear(x, q[0])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
