"""Train a layer's norm, router and dense block together, then serve its output projection in 8 bits.

    python deepseeker-v4.1_b200/examples/normed_layer.py [--steps 50]

A layer as a model holds it: the layer norm in front (``deepseeker.norm``), the
router behind it with its balance loss per sequence (``moe.route_softmax_topk``,
``deepseeker.balance``), the dense gated block (``deepseeker.gated``).  They
learn with plain gradient steps on f32 masters; the trained layer's output then
goes through a projection quantised to 8-bit integers (``deepseeker.int8``), for
a batch and for single tokens.  Synthetic data; prints the losses, how evenly the
experts are used and how far the quantised projection is off.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from deepseeker import balance, gated, int8, moe, norm  # noqa: E402

LIMIT, SHARE = 10.0, 0.05   # the block's clamp, the balance loss's share of the loss


def rel(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a.float() - b.float()).norm() / b.float().norm())


def make_params(hidden: int, inter: int, experts: int, device, seed: int = 0) -> dict[str, torch.Tensor]:
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    # a few experts are liked better at the start
    return {"scale": torch.ones(hidden, device=device), "shift": 0.1 * normal(hidden),
            "router": normal(experts, hidden) * hidden ** -0.5 + 0.5 * normal(experts, 1) * normal(1, hidden) * hidden ** -0.5,
            "w1": normal(inter, hidden) * hidden ** -0.5, "w3": normal(inter, hidden) * hidden ** -0.5,
            "w2": normal(hidden, inter) * inter ** -0.5}


def layer(p: dict[str, torch.Tensor], x: torch.Tensor):
    """The norm's output, the router's logits, and the block's output: p holds 16-bit block weights, f32 others."""
    n = norm.layer_norm(x, p["scale"], p["shift"])
    logits = n.float() @ p["router"].t()
    return n, logits, gated.gated_ffn(n, p["w1"], p["w3"], p["w2"], limit=LIMIT)


def loss_of(p, x, target, offsets, top_k: int):
    """The loss, its parts, and the counts per sequence and expert."""
    _, logits, out = layer(p, x)
    _, ids = moe.route_softmax_topk(logits.detach(), top_k)
    even, counts = balance.balance_loss(logits, ids, offsets=offsets)
    fit = (out.float() - target.float()).square().mean()
    return fit + SHARE * even.mean(), fit, even, counts, ids


def main(hidden: int = 512, inter: int = 1024, experts: int = 32, top_k: int = 4, tokens: int = 2048, out: int = 1000,
         steps: int = 50) -> dict:
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(1)
    master, teacher = make_params(hidden, inter, experts, device), make_params(hidden, inter, experts, device, seed=2)
    wide = {k: v.bfloat16() if k[0] == "w" else v for k, v in teacher.items()}
    params = {k: (v.bfloat16() if k[0] == "w" else v.clone()).requires_grad_() for k, v in master.items()}
    rates = {"scale": 0.5, "shift": 0.5, "router": 2.0, "w1": 20.0, "w3": 20.0, "w2": 20.0}
    # packed sequences of different lengths, the last rows padding
    offsets = torch.tensor([0, tokens // 8, tokens // 2, tokens // 2, tokens - 5], dtype=torch.int32, device=device)
    fits, evens, used = [], [], None
    for _ in range(steps):
        x = (torch.randn(tokens, hidden, generator=g, device=device) + 0.5).bfloat16()
        with torch.no_grad():
            target = layer(wide, x)[2]
        loss, fit, even, used, _ = loss_of(params, x, target, offsets, top_k)
        grads = torch.autograd.grad(loss, list(params.values()))
        with torch.no_grad():
            for (k, p), gr in zip(params.items(), grads):
                master[k] -= rates[k] * gr.float()
                p.copy_(master[k])
        fits.append(fit.detach()), evens.append(even.detach().max())
    # serving: the output projection in 8 bits
    with torch.no_grad():
        proj = torch.randn(out, hidden, generator=g, device=device) * hidden ** -0.5
        held = int8.quantize(proj)
        h = layer(params, (torch.randn(tokens, hidden, generator=g, device=device) + 0.5).bfloat16())[2]
        exact = h.float() @ proj.t()
        batch = int8.linear(h, held, out_dtype=torch.float32)
        ones = torch.cat([int8.linear(h[i:i + 1], held, out_dtype=torch.float32) for i in range(4)])
    return {"first_fit": float(fits[0]) if steps else None, "last_fit": float(fits[-1]) if steps else None,
            "first_balance": float(evens[0]) if steps else None, "last_balance": float(evens[-1]) if steps else None,
            "counted": int(used.sum()) if steps else 0, "projection_off": rel(batch, exact),
            "single_tokens_equal": torch.equal(ones, batch[:4]), "status": gated.status() | int8.status()}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=50)
    for name, value in main(steps=ap.parse_args().steps).items():
        print(f"{name:20s} {value}")
