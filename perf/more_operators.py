"""Cases of the operators around the expert layer: what is measured, on what data, against which plain form.

Operators (``op`` of a case):

  norm_forward    layer norm of a token's features, y = (x - mean) / sqrt(var + eps) * w + b
  norm_train      the same with its backward pass: y and the gradients of x, w and b
  balance         the router's balance loss of every sequence, the counts per expert, and the gradient of the
                  logits for given gradients of the losses
  int8_quantize   quantisation of rows to 8-bit integers with one scale a row (max / 127); what comes back is the
                  values that the codes stand for, and the scales
  int8_linear     product of activations quantised by token with weights quantised by channel

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits (64 where sums of products of
codes, or sums over many tokens, need them), rounded once at the end; with ``own`` true it calls this repository's
operators.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5


def _package():
    path = str(Path(__file__).resolve().parents[1] / "deepseeker-v4.1_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from deepseeker import balance, int8, norm

    return norm, balance, int8


# ---------------------------------------------------------------- cases

def listed():
    return [
        # the norm in front of a layer while one token is decoded
        {"name": "norm one token", "op": "norm_forward", "tokens": 1, "hidden": 4096, "dtype": "bf16",
         "weights": "bf16", "gap": 0},
        # the same over a prefill batch
        {"name": "norm prefill", "op": "norm_forward", "tokens": 16384, "hidden": 4096, "dtype": "bf16",
         "weights": "bf16", "gap": 0},
        # a training step on a few rows of uneven width, a slice of a wider activation
        {"name": "norm ragged step", "op": "norm_train", "tokens": 333, "hidden": 711, "dtype": "f16",
         "weights": "f32", "gap": 24},
        # a training step on one device's share of a batch
        {"name": "norm training step", "op": "norm_train", "tokens": 8192, "hidden": 4096, "dtype": "bf16",
         "weights": "f32", "gap": 0},
        # the router of a small mixture on a short batch: launch latency counts
        {"name": "balance small step", "op": "balance", "tokens": 61, "experts": 16, "top_k": 2, "kind": "softmax",
         "sequences": 0, "masked": False, "dtype": "f32"},
        # the router of a layer of 256 experts on one device's share of a batch, one loss for all of it
        {"name": "balance training step", "op": "balance", "tokens": 16384, "experts": 256, "top_k": 8,
         "kind": "softmax", "sequences": 0, "masked": False, "dtype": "f32"},
        # packed sequences with padding between and behind them, one loss for each, sqrt-softplus scores
        {"name": "balance sequences", "op": "balance", "tokens": 65536, "experts": 384, "top_k": 6,
         "kind": "sqrtsoftplus", "sequences": 24, "masked": True, "dtype": "f32"},
        # the activations of a decode batch
        {"name": "int8 quantise eight rows", "op": "int8_quantize", "tokens": 8, "hidden": 4096, "dtype": "bf16",
         "gap": 0},
        # the activations of a prefill batch
        {"name": "int8 quantise prefill", "op": "int8_quantize", "tokens": 16384, "hidden": 4096, "dtype": "bf16",
         "gap": 0},
        # a projection while one token is decoded
        {"name": "int8 product one token", "op": "int8_linear", "tokens": 1, "hidden": 4096, "out": 4096,
         "dtype": "bf16", "to": "bf16", "gap": 0},
        # a verification batch through uneven widths
        {"name": "int8 product ragged", "op": "int8_linear", "tokens": 100, "hidden": 1001, "out": 777,
         "dtype": "f16", "to": "f32", "gap": 0},
        # a projection of a prefill batch: the largest case
        {"name": "int8 product prefill", "op": "int8_linear", "tokens": 16384, "hidden": 4096, "out": 4096,
         "dtype": "bf16", "to": "bf16", "gap": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature width: a power of two or five quarters of one, an odd multiple of 8, or any odd number."""
    v, kind = _log(rng, lo, hi), rng.choice("222255888o")
    if kind in "25":
        p = 1 << int(round(math.log2(v)))
        return min(hi, max(lo, p if kind == "2" else p * 5 // 4))
    return min(hi // 8 - 1, v // 8) * 8 | 8 if kind == "8" else min(hi - 1, v) | 1


def draw(rng):
    op = rng.choice(["norm_forward", "norm_train", "balance", "int8_quantize", "int8_linear"])
    c = {"op": op, "tokens": _log(rng, 1, 65536 if op == "balance" else 16384)}
    if op == "balance":
        c["experts"] = rng.choice([8, 16, 60, 64, 128, 160, 256, 384, 2 * _log(rng, 4, 256) + 1])
        c["top_k"] = rng.randint(1, 8)
        c["kind"] = rng.choice(["softmax", "sqrtsoftplus"])
        c["sequences"] = rng.choice([0, 0, 1, _log(rng, 2, 64)])
        c["masked"] = rng.choice([False, True])
        c["dtype"] = rng.choice(["f32", "f32", "bf16", "f16"])
        c["tokens"] = max(1, min(c["tokens"], 65536 * 384 // c["experts"]))
        return c
    c["hidden"] = _width(rng, 16 if op.startswith("norm") else 64, 8192)
    most = 16384 * 4096 if op != "norm_train" else 8192 * 4096
    c["tokens"] = max(1, min(c["tokens"], most // c["hidden"]))
    if op == "int8_linear":
        c["out"] = _width(rng, 64, 8192)
        c["tokens"] = max(1, min(c["tokens"], 16384 * 4096 * 4096 // (c["hidden"] * c["out"])))
        c["to"] = rng.choice(["bf16", "f16", "f32"])
    c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("norm"):
        c["weights"] = rng.choice([c["dtype"], "f32"])
    c["gap"] = rng.choice([0, 0, 8, 5])
    return c


def work(case):
    op, T, e = case["op"], case["tokens"], BYTES[case["dtype"]]
    if op == "balance":
        E = case["experts"]
        # logits and ids in, gradient and counts out
        return {"bytes": 2 * T * E * e + 4 * T * case["top_k"] + 4 * E * max(1, case["sequences"]), "flops": 12 * T * E}
    H = case["hidden"]
    if op == "norm_forward":
        return {"bytes": 2 * T * H * e + 2 * H * BYTES[case["weights"]], "flops": 8 * T * H}
    if op == "norm_train":
        # x, dy, w, b in; y, dx and the gradients of w and b out
        return {"bytes": 4 * T * H * e + 4 * H * BYTES[case["weights"]], "flops": 24 * T * H}
    if op == "int8_quantize":
        # x in, codes and scales out; then codes and scales in, their values out
        return {"bytes": T * H * (2 * e + 2) + 8 * T, "flops": 4 * T * H}
    N = case["out"]
    return {"bytes": T * H * e + N * H + 4 * N + T * N * BYTES[case["to"]], "flops": 2 * T * H * N}


# ---------------------------------------------------------------- inputs

def _balance_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, E, S = case["tokens"], case["experts"], case["sequences"]
    # some experts are liked better than others, some tokens are surer than others
    logits = torch.randn(T, E, generator=g, device="cuda") + 0.7 * torch.randn(1, E, generator=g, device="cuda")
    logits = logits * torch.exp(0.5 * torch.randn(T, 1, generator=g, device="cuda"))
    s = {"logits": logits.to(DTYPES[case["dtype"]])}
    s["ids"] = s["logits"].float().topk(case["top_k"], dim=1).indices.int()
    s["dloss"] = 0.01 * (1 + torch.rand(S, generator=g, device="cuda")) if S else torch.tensor(0.01, device="cuda")
    if S:
        # sequences of every length, none or one token long among them, and rows behind the last
        cuts = torch.randint(0, T + 1, (S + 1,), generator=g, device="cuda").sort().values
        cuts[0] = 0
        s["offsets"] = cuts.int()
    if case["masked"]:
        s["valid"] = torch.rand(T, generator=g, device="cuda") > 0.05
        # what a masked row holds is nobody's business
        s["logits"][~s["valid"]] = math.nan
    return s


def _inputs(case, seed):
    if case["op"] == "balance":
        return _balance_inputs(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, H = case["tokens"], case["hidden"]
    dtype = DTYPES[case["dtype"]]

    def normal(rows, cols, std):
        return torch.randn(rows, cols, generator=g, device="cuda") * std

    wide = normal(T, H + case["gap"], 1.0)
    if case["op"].startswith("norm"):
        # a residual stream: channels with means of their own, tokens of different size
        wide = (wide + normal(1, H + case["gap"], 0.5)) * torch.exp(normal(T, 1, 0.5))
        s = {"x": wide.to(dtype)[:, :H]}
        s["w"] = (1 + normal(1, H, 0.2))[0].to(DTYPES[case["weights"]])
        s["b"] = normal(1, H, 0.2)[0].to(DTYPES[case["weights"]])
        if case["op"] == "norm_train":
            s["dy"] = normal(T, H, 1.0).to(dtype)
        return s
    # activations have channels of very different size, and padding rows of zeros
    wide *= torch.exp(normal(1, H + case["gap"], 1.0))
    wide *= torch.rand(T, 1, generator=g, device="cuda") > (0.05 if T > 4 else 0.0)
    s = {"x": wide.to(dtype)[:, :H]}
    if case["op"] == "int8_linear":
        s["w"] = normal(case["out"], H, H ** -0.5)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"] = case["op"]
    if case["op"] == "norm_train":
        for k in ("x", "w", "b"):
            s[k].requires_grad_(own)
    elif case["op"] == "balance":
        s["kind"] = case["kind"]
        s["logits"].requires_grad_(own)
    elif case["op"] == "int8_linear":
        # the weights as a checkpoint holds them, and the handle that a program keeps
        codes, scales = _quantized(s.pop("w"))
        s["w"] = _package()[2].from_codes(codes.to(torch.int8), scales) if own else (codes.to(torch.int8), scales)
        s["to"] = DTYPES[case["to"]]
    return s


# ---------------------------------------------------------------- plain forms

def _quantized(x):
    """Whole numbers of x's rows in 32 bits and their scales: the nearest number to x / scale, ties to the even one.
    The quotient is taken in 64 bits: in 32 it can fall on a tie that is none."""
    x = x.float()
    scale = x.abs().amax(1) / 127
    q = torch.round(x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[:, None])
    return q.clamp(-127, 127).float(), scale


def _scores(s):
    """Each row's share of every expert in 32 bits, and what else its gradient needs."""
    l = s["logits"].float()
    if "valid" in s:
        l = torch.where(s["valid"][:, None], l, torch.zeros_like(l))
    if s["kind"] == "softmax":
        a = torch.exp(l - l.amax(1, keepdim=True))
        return a / a.sum(1, keepdim=True), None
    soft = torch.clamp(l, min=0) + torch.log1p(torch.exp(-l.abs()))
    a = torch.sqrt(soft)
    z = a.sum(1, keepdim=True)
    return a / z, 1 / (1 + torch.exp(-l)) / (2 * a * z)


def _plain_balance(s):
    p, slope = _scores(s)
    T, E = p.shape
    S, k = s["dloss"].numel(), s["ids"].shape[1]
    rows = torch.arange(T, device=p.device)
    if "offsets" in s:
        seq = (rows[:, None] >= s["offsets"][None, :]).sum(1) - 1       # S: behind the last sequence
    else:
        seq = torch.zeros_like(rows)
    if "valid" in s:
        seq = torch.where(s["valid"], seq, torch.full_like(seq, S))
    counts = torch.zeros((S + 1) * E, dtype=torch.int32, device=p.device)
    at = (seq[:, None] * E + s["ids"].long()).reshape(-1)
    counts.index_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    counts = counts.view(S + 1, E)[:S]
    n = torch.zeros(S + 1, dtype=torch.int32, device=p.device).index_add_(0, seq, torch.ones_like(seq, dtype=torch.int32))
    n = n[:S].double().clamp(min=1)[:, None]
    mean = torch.zeros(S + 1, E, dtype=torch.float64, device=p.device).index_add_(0, seq, p.double())[:S] / n
    f = counts.double() * E / (k * n)
    loss = (f * mean).sum(1)
    c = torch.cat([s["dloss"].view(S, 1) * (f / n).float(), torch.zeros(1, E, device=p.device)])[seq]
    d = c - (p * c).sum(1, keepdim=True)
    d = d * (p if slope is None else slope)
    d = torch.where(seq[:, None] < S, d, torch.zeros_like(d))
    return {"loss": loss.float().view(s["dloss"].shape), "counts": counts.view(*s["dloss"].shape, E),
            "dlogits": d.to(s["logits"].dtype)}


def _plain(s):
    op = s["op"]
    if op == "balance":
        return _plain_balance(s)
    x = s["x"]
    if op == "int8_quantize":
        q, scale = _quantized(x)
        return {"values": (q * scale[:, None]).to(x.dtype), "scales": scale}
    if op == "int8_linear":
        q, scale = _quantized(x)
        # whole numbers past 2^24: 64 bits hold the sums
        sums = q.double() @ s["w"][0].double().t()
        return (sums * scale.double()[:, None] * s["w"][1].double()[None, :]).float().to(s["to"])
    w, b = s["w"].float(), s["b"].float()
    xf = x.float()
    off = xf - xf.mean(1, keepdim=True)
    r = 1 / torch.sqrt((off * off).mean(1, keepdim=True) + EPS)
    xh = off * r
    y = (xh * w + b).to(x.dtype)
    if op == "norm_forward":
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dw": (dy * xh).sum(0, dtype=torch.float64).to(s["w"].dtype),
            "db": dy.sum(0, dtype=torch.float64).to(s["b"].dtype)}


def run(state):
    if not own:
        return _plain(state)
    norm, balance, int8 = _package()
    op = state["op"]
    if op == "balance":
        loss, counts = balance.balance_loss(state["logits"], state["ids"], kind=state["kind"],
                                            valid=state.get("valid"), offsets=state.get("offsets"))
        dlogits, = torch.autograd.grad(loss, state["logits"], state["dloss"])
        return {"loss": loss.detach(), "counts": counts, "dlogits": dlogits}
    x = state["x"]
    if op == "int8_quantize":
        q = int8.quantize(x)
        return {"values": q.dequantize(x.dtype), "scales": q.scales}
    if op == "int8_linear":
        return int8.linear(x, state["w"], out_dtype=state["to"])
    w, b = state["w"], state["b"]
    y = norm.layer_norm(x, w, b, eps=EPS)
    if op == "norm_forward":
        return y
    dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


# ---------------------------------------------------------------- 64 bits

def _codes(x):
    """Codes and scales of x's rows [rows, cols] (64 bits holding 32-bit values), from the definition: the scale is
    the 32-bit number nearest to max / 127, a code the whole number nearest to x / scale, the even one of two."""
    scale = (x.abs().max(dim=1).values / 127.0).float().double()
    t = x / torch.where(scale == 0, torch.ones_like(scale), scale).unsqueeze(1)
    low = torch.floor(t)
    rest = t - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.clip(low + up.double(), -127, 127), scale


def _exact_balance(case, seed):
    s = _inputs(case, seed)
    T, E = s["logits"].shape
    k, many = case["top_k"], case["sequences"]
    ends = s["offsets"].tolist() if many else [0, T]
    up = s["dloss"].double().reshape(-1)
    grad = torch.zeros(T, E, dtype=torch.float64, device="cuda")
    losses, counts = [], []
    for i in range(len(ends) - 1):
        rows = torch.arange(ends[i], ends[i + 1], device="cuda")
        if case["masked"]:
            rows = rows[s["valid"][rows]]
        n = len(rows)
        c = torch.bincount(s["ids"][rows].reshape(-1).long(), minlength=E)
        counts.append(c.int())
        if n == 0:
            losses.append(torch.zeros((), dtype=torch.float64, device="cuda"))
            continue
        l = s["logits"][rows].double().requires_grad_()
        a = torch.exp(torch.log_softmax(l, 1)) if case["kind"] == "softmax" else torch.sqrt(torch.logaddexp(
            l, torch.zeros_like(l)))
        share = a / torch.einsum("te->t", a).unsqueeze(1)
        loss = torch.einsum("e,te->", c.double() * (E / (k * n)), share) / n
        losses.append(loss.detach())
        grad[rows], = torch.autograd.grad(loss, l, up[i])
    if not many:
        return {"loss": losses[0], "counts": counts[0], "dlogits": grad}
    return {"loss": torch.stack(losses), "counts": torch.stack(counts), "dlogits": grad}


def exact(case, seed):
    if case["op"] == "balance":
        return _exact_balance(case, seed)
    d = {k: v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "int8_quantize":
        code, scale = _codes(d["x"])
        return {"values": torch.einsum("tk,t->tk", code, scale), "scales": scale}
    if case["op"] == "int8_linear":
        (a, sa), (b, sb) = _codes(d["x"]), _codes(d["w"])
        return torch.einsum("tk,nk->tn", a, b) * torch.outer(sa, sb)
    v, m = torch.var_mean(d["x"], dim=1, correction=0)
    dev = (v + EPS).sqrt().unsqueeze(1)
    z = (d["x"] - m.unsqueeze(1)) / dev
    y = torch.addcmul(d["b"].expand_as(z), z, d["w"].expand_as(z))
    if case["op"] == "norm_forward":
        return y
    t = d["dy"] * d["w"]
    H = z.shape[1]
    dx = (H * t - torch.einsum("th->t", t).unsqueeze(1) - z * torch.einsum("th,th->t", t, z).unsqueeze(1)) / (H * dev)
    return {"y": y, "dx": dx, "dw": torch.einsum("th,th->h", d["dy"], z), "db": torch.einsum("th->h", d["dy"])}
