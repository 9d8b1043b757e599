"""Train a layer's dense (shared) expert, quantise it and serve it next to the routed experts.

    python deepseeker-v4.1_b200/examples/dense_block.py [--steps 200]

A 16-bit gated block (``deepseeker.gated``) learns to imitate another one with
plain gradient steps on f32 master weights; its weights then go to the 4-bit
format (``deepseeker.mx4``), and the quantised block serves a prompt and single
tokens, alone and as the ``shared_fn`` of ``moe_layer`` over FP4 experts.
Synthetic data; prints the losses and how far the quantised block is off.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from deepseeker import gated, moe, mx4, synthetic  # noqa: E402


def rel(a: torch.Tensor, b: torch.Tensor) -> float:
    return float((a.float() - b.float()).norm() / b.float().norm())


def main(hidden: int = 512, inter: int = 1024, tokens: int = 1024, steps: int = 200, limit: float = 10.0) -> dict:
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(0)

    def weights(gain: float) -> list[torch.Tensor]:
        return [torch.randn(r, c, generator=g, device=device) * (gain * c ** -0.5)
                for r, c in ((inter, hidden), (inter, hidden), (hidden, inter))]

    # training: 16-bit weights in the block, f32 masters in the optimiser
    teacher = [w.bfloat16() for w in weights(1.0)]
    master = [t.float() + 0.5 * n for t, n in zip(teacher, weights(1.0))]
    params = [m.bfloat16().requires_grad_() for m in master]
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, hidden, generator=g, device=device).bfloat16()
        with torch.no_grad():
            target = gated.gated_ffn(x, *teacher, limit=limit)
        out = gated.gated_ffn(x, *params, limit=limit)
        loss = (out.float() - target.float()).square().mean()
        grads = torch.autograd.grad(loss, params)
        with torch.no_grad():
            for m, p, gr in zip(master, params, grads):
                m -= 20.0 * gr.float()
                p.copy_(m)
        losses.append(loss)
    losses = torch.stack(losses).tolist() if losses else []

    # serving: the same block in 4 bits
    params = [p.detach() for p in params]
    with torch.no_grad():
        block = [mx4.quantize(p) for p in params]
        prompt = torch.randn(tokens, hidden, generator=g, device=device).bfloat16()
        exact = gated.gated_ffn(prompt, *params, limit=limit)
        served = mx4.gated_ffn(prompt, *block, limit=limit)
        one = torch.cat([mx4.gated_ffn(prompt[i:i + 1], *block, limit=limit) for i in range(4)])
        kept = [w.dequantize(torch.bfloat16) for w in block]
        # the projections alone, x quantised once for both
        q = mx4.quantize(prompt)
        gate, up = mx4.linear(q, block[0], out_dtype=torch.float32), mx4.linear(q, block[1], out_dtype=torch.float32)

        # the shared expert of a mixture layer
        layer = synthetic.make_layer("fp4", hidden, inter, 8, seed=1, shared_inter=None, device=device)
        router = torch.randn(8, hidden, generator=g, device=device) * hidden ** -0.5
        routed = moe.moe_layer(prompt[:4], router, None, layer.resident(), None, top_k=2, limit=limit)
        mixed = moe.moe_layer(prompt[:4], router, None, layer.resident(),
                              lambda t: mx4.gated_ffn(t, *block, limit=limit), top_k=2, limit=limit)
        # a routed expert's stored matrix is the same format
        expert = mx4.from_packed(layer.w1.data[3], layer.w1.scales[3])
        logits = mx4.linear(prompt[:4], expert)
    result = {
        "first_loss": losses[0] if losses else None, "last_loss": losses[-1] if losses else None,
        "weights_off": max(rel(k, p) for k, p in zip(kept, params)),
        "block_off": rel(served, exact), "single_tokens_off": rel(one, served[:4]),
        "gate_off": rel(torch.nn.functional.silu(gate.clamp(max=limit)) * up.clamp(-limit, limit),
                        _hidden(prompt, params, limit)),
        "mixture_off": rel(mixed, routed.float() + served[:4].float()),
        "expert_rows": tuple(logits.shape), "status": gated.status() | mx4.status(),
    }
    return result


def _hidden(x, params, limit):
    g, u = x.float() @ params[0].float().t(), x.float() @ params[1].float().t()
    return torch.nn.functional.silu(g.clamp(max=limit)) * u.clamp(-limit, limit)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    for name, value in main(steps=ap.parse_args().steps).items():
        print(f"{name:18s} {value}")
