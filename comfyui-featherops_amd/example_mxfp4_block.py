#!/usr/bin/env python3
"""A transformer feed-forward block under adaptive norms, its layers in MXFP4: the operators together.

    x, y = gated_residual_norm(x, h, gate, scale, shift) -> 4 bits -> up -> GELU -> down -> the next block's h

The norm leaves its result in 4 bits for the up projection, whose output is quantized on its way into the
down projection. Prints the time of a block against the same block in bf16 library calls, and how far its
output is from the bf16 block's.

    python3 example_mxfp4_block.py [--tokens 4096] [--width 5120] [--hidden 13824]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent))
from _bench_common import load_plugin  # noqa: E402

load_plugin()
from featherops_amd.comfy_feather.mxfp4 import mxfp4_ops  # noqa: E402
from featherops_amd.kernel.hip.norm import gated_residual_norm  # noqa: E402


class AdaptiveFeedForward(nn.Module):
    """One block's feed-forward half. forward takes the stream x, the attention's output h with its gate, and
    this half's scale and shift; it returns the stream and the half's own output, for the next norm."""

    def __init__(self, width: int, hidden: int, linear=nn.Linear):
        super().__init__()
        self.up = linear(width, hidden)
        self.down = linear(hidden, width)

    def forward(self, x, h, gate, scale, shift):
        x, y = gated_residual_norm(x, h, gate, scale=scale, shift=shift, kind="layer", out_dtype="mxfp4")
        return x, self.down(F.gelu(self.up(y), approximate="tanh"))


class PlainFeedForward(AdaptiveFeedForward):
    """The same with library calls."""

    def forward(self, x, h, gate, scale, shift):
        x = x + gate * h
        y = F.layer_norm(x, x.shape[-1:], eps=1e-6) * (1 + scale) + shift
        return x, self.down(F.gelu(self.up(y), approximate="tanh"))


def build(width: int, hidden: int, device="cuda", seed: int = 0):
    """(the plain block, the MXFP4 block with the same weights)."""
    torch.manual_seed(seed)
    plain = PlainFeedForward(width, hidden).to(device=device, dtype=torch.bfloat16)
    with torch.device("meta"):
        block = AdaptiveFeedForward(width, hidden, mxfp4_ops(torch.bfloat16).Linear)
    block.load_state_dict(plain.state_dict())
    return plain, block


def inputs(tokens: int, width: int, device="cuda", seed: int = 1):
    g = torch.Generator(device=device).manual_seed(seed)

    def r(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=device) * std).to(torch.bfloat16)

    return r(1, tokens, width, std=3.0), r(1, tokens, width), *(r(1, 1, width, std=0.3) for _ in range(3))


def _time(fn, reps: int = 20) -> float:
    for _ in range(3):
        fn()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(reps):
        fn()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / reps


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=4096)
    parser.add_argument("--width", type=int, default=5120)
    parser.add_argument("--hidden", type=int, default=13824)
    args = parser.parse_args()
    with torch.inference_mode():
        plain, block = build(args.width, args.hidden)
        args_in = inputs(args.tokens, args.width)
        x, y = block(*args_in)
        x_ref, y_ref = plain(*args_in)
        off = (y.float() - y_ref.float()).norm() / y_ref.float().norm()
        same = torch.equal(x, x_ref)
        t, t_plain = _time(lambda: block(*args_in)), _time(lambda: plain(*args_in))
    print(f"tokens {args.tokens} width {args.width} hidden {args.hidden}: MXFP4 {t:.3f} ms, bf16 library {t_plain:.3f} ms "
          f"({t_plain / t:.2f}x); stream {'equal' if same else 'differs by roundings'}, output {off:.3f} off (2-norm)")


if __name__ == "__main__":
    main()
