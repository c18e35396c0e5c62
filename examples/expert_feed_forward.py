"""An encoder block's feed-forward module with experts in place of its two linears.

A chunk's tokens go through an INT8 router (QuantizedLinear), each to its two
best experts of eight, whose e4m3 weights are made here from random f32 ones; the
module's call and the same steps one by one give the same rows.

    python examples/expert_feed_forward.py [--streams 64] [--tokens 14]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "catcher-tippi_b200"))
import nemotron_cuda as cq  # noqa: E402
from nemotron_cuda.experts import ExpertFeedForward, ExpertLinear, combine, route  # noqa: E402
from nemotron_cuda.fp8 import quantize_weight  # noqa: E402

HIDDEN, FF, EXPERTS, TOP = 1024, 4096, 8, 2


def expert_linear(outputs: int, inputs: int, seed: int) -> ExpertLinear:
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes, scales = zip(*(quantize_weight(torch.randn(outputs, inputs, generator=g, device="cuda") * inputs ** -0.5)
                          for _ in range(EXPERTS)))
    return ExpertLinear.from_codes(torch.stack(codes), torch.stack(scales))


def run(streams: int = 1, tokens: int = 14) -> dict:
    g = torch.Generator().manual_seed(7)
    weight = torch.randn(EXPERTS, HIDDEN, generator=g) * HIDDEN ** -0.5
    router = cq.QuantizedLinear.from_f32(weight.numpy(), EXPERTS, HIDDEN, np.zeros(EXPERTS), group_size=64, dtype="bf16")
    up, down = expert_linear(FF, HIDDEN, 8), expert_linear(HIDDEN, FF, 9)
    module = ExpertFeedForward(up, down, top=TOP, act="silu")

    x = torch.randn(streams * tokens, HIDDEN, generator=g).to("cuda", torch.bfloat16)
    logits = router.forward(x)
    y = module.forward(x, logits)

    r = route(logits, TOP)
    h = up.forward(x[r.token.long()], r.offsets, act="silu")
    stepwise = combine(down.forward(h, r.offsets), r.position, r.weight)
    difference = (y.float() - stepwise.float()).norm() / stepwise.float().norm()
    return {"rows": x.shape[0], "rows of each expert": r.offsets.diff().tolist(), "difference": difference.item(), "y": y}


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--streams", type=int, default=1)
    p.add_argument("--tokens", type=int, default=14, help="of each stream's chunk")
    a = p.parse_args()
    out = run(a.streams, a.tokens)
    print(f"{out['rows']} tokens, rows of each expert {out['rows of each expert']}")
    print(f"module against its steps one by one (h and z rounded to bf16 there): relative difference {out['difference']:.4f}")


if __name__ == "__main__":
    main()
