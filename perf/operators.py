"""Cases of the dense feed-forward operators: what is measured, on what data, against which plain form.

Operators (``op`` of a case):

  gated_forward   the gated feed-forward block y = (silu(min(x W1^T, L)) * clip(x W3^T, -L, L)) W2^T
                  over 16-bit weights (no clamps where ``limit`` is 0)
  gated_train     the same block with its backward pass: y and the gradients of x, W1, W3, W2
  mx4_quantize    microscaled 4-bit quantisation (e2m1 codes, one power-of-two scale per 32 values of a
                  row); what comes back is the values that the codes stand for
  mx4_linear      product of quantised activations with quantised weights
  mx4_block       the gated block over quantised weights, x and h quantised on the way

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits, rounded once at the end;
with ``own`` true it calls this repository's operators.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _package():
    path = str(Path(__file__).resolve().parents[1] / "deepseeker-v4.1_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from deepseeker import gated, mx4

    return gated, mx4


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a layer's dense (shared) expert while one token is decoded
        {"name": "gated one token", "op": "gated_forward", "tokens": 1, "hidden": 4096, "inter": 2048,
         "dtype": "bf16", "limit": 10.0, "gap": 0},
        # a short prompt through a small block of uneven widths, x a slice of a wider activation
        {"name": "gated ragged prompt", "op": "gated_forward", "tokens": 333, "hidden": 1000, "inter": 711,
         "dtype": "f16", "limit": 0.0, "gap": 24},
        # a training step on a few rows of a small block: launch latency counts
        {"name": "gated small step", "op": "gated_train", "tokens": 37, "hidden": 512, "inter": 256,
         "dtype": "bf16", "limit": 10.0, "gap": 0},
        # a training step of the dense expert on one device's share of a batch: the largest case
        {"name": "gated training step", "op": "gated_train", "tokens": 8192, "hidden": 4096, "inter": 2048,
         "dtype": "bf16", "limit": 0.0, "gap": 0},
        # the activations of a decode batch
        {"name": "quantise eight rows", "op": "mx4_quantize", "tokens": 8, "hidden": 4096, "dtype": "bf16", "gap": 0},
        # the activations of a prefill batch
        {"name": "quantise prefill", "op": "mx4_quantize", "tokens": 16384, "hidden": 4096, "dtype": "bf16", "gap": 0},
        # a projection while one token is decoded
        {"name": "product one token", "op": "mx4_linear", "tokens": 1, "hidden": 4096, "out": 4096,
         "dtype": "bf16", "to": "bf16", "gap": 0},
        # a verification batch through uneven widths
        {"name": "product ragged", "op": "mx4_linear", "tokens": 100, "hidden": 1001, "out": 777,
         "dtype": "f16", "to": "f32", "gap": 0},
        # a projection of a prefill batch
        {"name": "product prefill", "op": "mx4_linear", "tokens": 16384, "hidden": 4096, "out": 4096,
         "dtype": "bf16", "to": "bf16", "gap": 0},
        # the quantised dense expert while one token is decoded
        {"name": "block one token", "op": "mx4_block", "tokens": 1, "hidden": 4096, "inter": 2048,
         "dtype": "bf16", "limit": 10.0, "gap": 0},
        # the quantised dense expert over a prompt
        {"name": "block prompt", "op": "mx4_block", "tokens": 2048, "hidden": 4096, "inter": 2048,
         "dtype": "bf16", "limit": 10.0, "gap": 0},
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
    op = rng.choice(["gated_forward", "gated_train", "mx4_quantize", "mx4_linear", "mx4_block"])
    c = {"op": op, "tokens": _log(rng, 1, 16384), "hidden": _width(rng, 64, 4096)}
    if op == "mx4_linear":
        c["out"] = _width(rng, 64, 4096)
    elif op != "mx4_quantize":
        c["inter"] = _width(rng, 64, 4096)
        c["limit"] = rng.choice([0.0, 1.5, 10.0])
    if op == "gated_train":
        # no dearer than the largest listed step
        c["tokens"] = max(1, min(c["tokens"], 8192 * 4096 * 2048 // (c["hidden"] * c["inter"])))
    c["dtype"] = rng.choice(["bf16", "f16", "f32"] if op in ("mx4_quantize", "mx4_linear") else ["bf16", "f16"])
    if op == "mx4_linear":
        c["to"] = rng.choice(["bf16", "f16", "f32"])
    c["gap"] = rng.choice([0, 0, 8, 5])
    return c


def work(case):
    T, H, e = case["tokens"], case["hidden"], BYTES[case["dtype"]]
    op = case["op"]
    packed = lambda rows, cols: rows * (-(-cols // 32) * 17)  # noqa: E731  16 bytes of codes and one scale per 32
    if op == "mx4_quantize":
        # x in, codes and scales out; then codes and scales in, their values out
        return {"bytes": T * H * e + 2 * packed(T, H) + T * H * 2, "flops": 0}
    if op == "mx4_linear":
        N = case["out"]
        return {"bytes": T * H * e + packed(N, H) + T * N * BYTES[case["to"]], "flops": 2 * T * H * N}
    I = case["inter"]
    if op == "mx4_block":
        return {"bytes": 2 * T * H * e + 2 * packed(I, H) + packed(H, I), "flops": 6 * T * H * I}
    if op == "gated_forward":
        return {"bytes": (2 * T * H + 3 * H * I) * e, "flops": 6 * T * H * I}
    # x, dy and three weights in; y, dx and three gradients out; nine products
    return {"bytes": (4 * T * H + 6 * H * I) * e, "flops": 18 * T * H * I}


# ---------------------------------------------------------------- inputs

def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, H = case["tokens"], case["hidden"]
    dtype = DTYPES[case["dtype"]]

    def normal(rows, cols, std):
        return torch.randn(rows, cols, generator=g, device="cuda") * std

    wide = normal(T, H + case["gap"], 1.0)
    if case["op"].startswith("mx4"):
        # activations have channels of very different size, and padding rows of zeros
        wide *= torch.exp(normal(1, H + case["gap"], 1.0))
        wide *= torch.rand(T, 1, generator=g, device="cuda") > (0.05 if T > 4 else 0.0)
    s = {"x": wide.to(dtype)[:, :H]}
    if case["op"] == "mx4_linear":
        s["w"] = normal(case["out"], H, H ** -0.5)
    elif case["op"] != "mx4_quantize":
        I = case["inter"]
        s["w1"], s["w3"], s["w2"] = normal(I, H, H ** -0.5), normal(I, H, H ** -0.5), normal(H, I, I ** -0.5)
    if case["op"].startswith("gated"):
        s = {k: v.to(dtype) for k, v in s.items()}
    if case["op"] == "gated_train":
        s["dy"] = normal(T, H, 1.0).to(dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"], s["limit"] = case["op"], case.get("limit", 0.0)
    if case["op"] == "gated_train":
        for k in ("x", "w1", "w3", "w2"):
            s[k].requires_grad_(own)
    if case["op"] in ("mx4_linear", "mx4_block"):
        # the weights as a checkpoint holds them, and the handle that a program keeps of each
        for k in [k for k in s if k in ("w", "w1", "w3", "w2")]:
            packed, scales, cols = _pack(s.pop(k))
            s[k] = _package()[1].from_packed(packed, scales, cols) if own else (packed, scales, cols)
        s["to"] = DTYPES[case.get("to", case["dtype"])]
    return s


# ---------------------------------------------------------------- plain forms

def _blocks(x):
    """Blocks of 32 of x's rows in 32 bits, zeros behind an uneven end; and each block's exponent: the smallest
    power of two that brings the block's largest magnitude to 6 or less (1 for a block of zeros)."""
    x = x.float()
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.75, e - 3, e - 2).clamp(min=-127)
    return x, torch.where(top == 0, torch.zeros_like(e), e)


def _power(e):
    """2^e in 32 bits, e from -127 to 127."""
    return torch.where(e == -127, torch.full_like(e, 0x00400000), (e + 127) << 23).view(torch.float32)


def _grid(x, e):
    """Magnitudes of x / 2^e rounded to 0, 0.5, 1, 1.5, 2, 3, 4, 6; ties to the even code."""
    a = x.abs() * _power(-e)
    step = 0.5 + 0.5 * (a >= 2) + (a >= 4)
    return torch.round(a / step) * step


def _rounded(x):
    """The values that x's rows keep in the 4-bit format, in 32 bits."""
    b, e = _blocks(x)
    v = torch.where(b < 0, -1.0, 1.0) * _grid(b, e) * _power(e)
    return v.view(x.shape[0], -1)[:, : x.shape[1]]


def _pack(w):
    """Codes [rows, 16 per block of 32] and scale bytes [rows, blocks] of w, and its columns."""
    b, e = _blocks(w)
    v = _grid(b, e)
    code = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4)).int()
    code = torch.where((b < 0) & (code > 0), code + 8, code).view(w.shape[0], -1)
    return ((code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8).contiguous(),
            (e + 127).to(torch.uint8).view(w.shape[0], -1).contiguous(), w.shape[1])


def _unpacked(packed, scales, cols):
    code = torch.stack([packed & 15, packed >> 4], -1).view(packed.shape[0], -1, 32).int()
    m = (code & 7).float()
    v = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
    v = torch.where(code > 7, -v, v) * _power(scales.int()[:, :, None] - 127)
    return v.view(packed.shape[0], -1)[:, :cols]


def _bend(x, w1, w3, limit):
    """Both projections of x and their clamped forms."""
    g, u = x @ w1.t(), x @ w3.t()
    return (g, u, g.clamp(max=limit), u.clamp(-limit, limit)) if limit else (g, u, g, u)


def _plain(s):
    op, x, limit = s["op"], s["x"], s["limit"]
    if op == "mx4_quantize":
        return _rounded(x).to(torch.bfloat16)
    if op == "mx4_linear":
        return (_rounded(x) @ _unpacked(*s["w"]).t()).to(s["to"])
    if op == "mx4_block":
        w1, w3, w2 = (_unpacked(*s[k]) for k in ("w1", "w3", "w2"))
        _, _, g, u = _bend(_rounded(x), w1, w3, limit)
        return (_rounded(g / (1 + torch.exp(-g)) * u) @ w2.t()).to(s["to"])
    xf, w1, w3, w2 = (s[k].float() for k in ("x", "w1", "w3", "w2"))
    g0, u0, g, u = _bend(xf, w1, w3, limit)
    sig = 1 / (1 + torch.exp(-g))
    h = g * sig * u
    y = h @ w2.t()
    if op == "gated_forward":
        return y.to(x.dtype)
    dy = s["dy"].float()
    dh = dy @ w2
    dg, du = dh * u * sig * (1 + g * (1 - sig)), dh * g * sig
    if limit:
        dg, du = dg * (g0 <= limit), du * (u0.abs() <= limit)
    out = {"y": y, "dx": dg @ w1 + du @ w3, "dw1": dg.t() @ xf, "dw3": du.t() @ xf, "dw2": dy.t() @ h}
    return {k: v.to(x.dtype) for k, v in out.items()}


def run(state):
    if not own:
        return _plain(state)
    gated, mx4 = _package()
    op, x, limit = state["op"], state["x"], state["limit"] or None
    if op == "mx4_quantize":
        return mx4.quantize(x).dequantize(torch.bfloat16)
    if op == "mx4_linear":
        return mx4.linear(x, state["w"], out_dtype=state["to"])
    if op == "mx4_block":
        return mx4.gated_ffn(x, state["w1"], state["w3"], state["w2"], limit=limit)
    w1, w3, w2 = state["w1"], state["w3"], state["w2"]
    y = gated.gated_ffn(x, w1, w3, w2, limit=limit)
    if op == "gated_forward":
        return y
    dx, dw1, dw3, dw2 = torch.autograd.grad(y, (x, w1, w3, w2), state["dy"])
    return {"y": y.detach(), "dx": dx, "dw1": dw1, "dw3": dw3, "dw2": dw2}


# ---------------------------------------------------------------- 64 bits

#: Magnitudes of the eight codes, and the points half way between them.
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
HALF = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _kept(x):
    """What x's rows keep in the 4-bit format, from the definition: the code whose magnitude is nearest, the even
    one of two that are as near."""
    rows, cols = x.shape
    b = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    b[:, :cols] = x
    b = b.view(rows, -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -150) / 6))
    e = e + (top > 6 * torch.exp2(e)).double() - (top <= 3 * torch.exp2(e)).double()
    scale = torch.where(top > 0, torch.exp2(e.clamp(min=-127)), torch.ones_like(e))
    a = b.abs() / scale
    half = torch.tensor(HALF, dtype=torch.float64, device=x.device)
    low, high = torch.bucketize(a, half), torch.bucketize(a, half, right=True)
    code = torch.where(low % 2 == 0, low, high)  # low < high only half way: the even one of the two
    v = torch.tensor(CODES, dtype=torch.float64, device=x.device)[code] * scale * torch.sign(b)
    return v.view(rows, -1)[:, :cols]


def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: v.double() for k, v in s.items()}
    L = case.get("limit") or math.inf
    if case["op"] == "mx4_quantize":
        return _kept(d["x"])
    if case["op"] == "mx4_linear":
        return torch.einsum("tk,nk->tn", _kept(d["x"]), _kept(d["w"]))
    if case["op"] == "mx4_block":
        d = {k: _kept(v) for k, v in d.items()}
    a, b = torch.einsum("th,ih->ti", d["x"], d["w1"]), torch.einsum("th,ih->ti", d["x"], d["w3"])
    ga, gb = torch.minimum(a, torch.full_like(a, L)), torch.maximum(torch.minimum(b, torch.full_like(b, L)),
                                                                   torch.full_like(b, -L))
    p = torch.sigmoid(ga)
    h = ga * p * gb
    if case["op"] == "mx4_block":
        h = _kept(h)
    y = torch.einsum("ti,hi->th", h, d["w2"])
    if case["op"] != "gated_train":
        return y
    dh = torch.einsum("th,hi->ti", d["dy"], d["w2"])
    da = torch.where(a <= L, dh * gb * (p + ga * p * (1 - p)), torch.zeros_like(dh))
    db = torch.where(b.abs() <= L, dh * ga * p, torch.zeros_like(dh))
    return {"y": y, "dx": torch.einsum("ti,ih->th", da, d["w1"]) + torch.einsum("ti,ih->th", db, d["w3"]),
            "dw1": torch.einsum("ti,th->ih", da, d["x"]), "dw3": torch.einsum("ti,th->ih", db, d["x"]),
            "dw2": torch.einsum("th,ti->hi", d["dy"], h)}
