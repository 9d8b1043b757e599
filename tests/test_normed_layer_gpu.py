"""Norm, router with its balance loss, dense block and 8-bit projection in one run, as a layer uses them."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "deepseeker-v4.1_b200" / "examples" / "normed_layer.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("normed_layer_example", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_runs(example, cuda):
    r = example.main(hidden=256, inter=384, experts=12, top_k=3, tokens=400, out=130, steps=3)
    assert r["status"] == 0 and r["counted"] == 3 * (400 - 5)
    # codes are off by half a step of max / 127, each operand: normal rows of 256 have a maximum of about 3 standard
    # deviations, so 3 / 127 / sqrt(12) = 7e-3 of a value each, 1e-2 together; twice that for rows with larger maxima
    assert r["projection_off"] <= 2e-2
    assert r["single_tokens_equal"]                # sums of codes are exact, whichever kernel forms them


def test_gradients(example, cuda):
    """The whole step's gradients against the same formulas by autograd in 64 bits, on the operands as stored.

    The norm's 16-bit output (2^-9 of its size, root mean square, as are the block's h, g and u gradients and
    the gradient that enters the norm) carries through a handful of such roundings: 8 of 2^-9 in quadrature is 6e-3,
    and each parameter's gradient is asserted to 1e-2 of its norm.  The balance loss alone sees one rounding."""
    p = example.make_params(128, 192, 10, cuda)
    p = {k: v.bfloat16() if k[0] == "w" else v for k, v in p.items()}
    g = torch.Generator(device=cuda).manual_seed(4)
    x, target = ((torch.randn(333, 128, generator=g, device=cuda) + 0.5).bfloat16() for _ in range(2))
    offsets = torch.tensor([0, 100, 100, 330], dtype=torch.int32, device=cuda)
    a = {k: v.clone().requires_grad_() for k, v in p.items()}
    a["x"] = x.clone().requires_grad_()
    loss, fit, even, counts, ids = example.loss_of({k: v for k, v in a.items() if k != "x"}, a["x"], target, offsets, 3)
    got = dict(zip(a, torch.autograd.grad(loss, list(a.values()))))

    b = {k: v.detach().double().requires_grad_() for k, v in a.items()}
    z = b["x"]
    xh = (z - z.mean(1, keepdim=True)) / torch.sqrt(z.var(1, unbiased=False, keepdim=True) + 1e-5)
    n = xh * b["scale"] + b["shift"]
    logits = n @ b["router"].t()
    u, v = (n @ b["w1"].t()).clamp(max=example.LIMIT), (n @ b["w3"].t()).clamp(-example.LIMIT, example.LIMIT)
    out = (u * torch.sigmoid(u) * v) @ b["w2"].t()
    share = torch.softmax(logits, 1)
    want_even = []
    for i, (lo, hi) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        c = torch.bincount(ids[lo:hi].reshape(-1).long(), minlength=10)
        assert torch.equal(counts[i].long(), c)
        want_even.append((c * 10 / (3 * max(hi - lo, 1)) * share[lo:hi].sum(0) / max(hi - lo, 1)).sum())
    want_even = torch.stack(want_even)
    want_fit = (out - target.double()).square().mean()
    want = dict(zip(b, torch.autograd.grad(want_fit + example.SHARE * want_even.mean(), list(b.values()))))
    even, fit, want_even, want_fit = (t.detach() for t in (even, fit, want_even, want_fit))
    assert float((even.double() - want_even).abs().max()) <= 2.0 ** -8 * float(want_even.max())
    assert abs(float(fit) - float(want_fit)) <= 2.0 ** -7 * float(want_fit)
    for k in got:
        err = float((got[k].double() - want[k]).norm() / want[k].norm())
        assert err <= 1e-2, (k, err)
