"""The example that trains the dense block, quantises it and serves it beside routed experts."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "deepseeker-v4.1_b200" / "examples" / "dense_block.py"


def test_example(cuda):
    spec = importlib.util.spec_from_file_location("dense_block_example", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    r = m.main(hidden=256, inter=384, tokens=300, steps=40)
    assert r["last_loss"] < 0.5 * r["first_loss"]
    # e2m1 keeps a block maximum in (3, 6] and rounds to a relative step of at
    # most 1/4 below it: 0.1 for normal weights, and three such roundings
    # (x, W, h) in the block
    assert r["weights_off"] <= 0.15 and r["block_off"] <= 0.4 and r["gate_off"] <= 0.4
    # one token and a prompt accumulate in different orders: an h code in ten thousand may differ
    assert r["single_tokens_off"] <= 2e-2
    # moe_layer adds the shared output in f32 and rounds once to bf16
    assert r["mixture_off"] <= 2.0 ** -7
    assert r["expert_rows"] == (4, 384) and r["status"] == 0
