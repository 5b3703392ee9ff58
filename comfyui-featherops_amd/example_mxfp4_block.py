#!/usr/bin/env python3
"""A transformer block under adaptive norms, its layers in MXFP4: the operators together.

    x, y = gated_residual_norm(x, h, gate, scale, shift) -> 4 bits -> q, k, v -> norm and positions -> attention -> out
    x, y = gated_residual_norm(x, h, gate, scale, shift) -> 4 bits -> up -> GELU -> down -> the next block's h

The norms leave their results in 4 bits for the projections behind them; what goes into the out and down projections
is quantized on its way. Queries and keys are normed and turned where the joint projection left them, and attention
reads its values there. Prints the time of each half against the same half in bf16 library calls, and how far
its output is from theirs.

    python3 example_mxfp4_block.py [--tokens 4096] [--width 5120] [--hidden 13824] [--head-dim 128]
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
from featherops_amd.kernel.hip.attention import attention  # noqa: E402
from featherops_amd.kernel.hip.norm import gated_residual_norm  # noqa: E402
from featherops_amd.kernel.hip.rope import qk_norm_rope, rope_table  # noqa: E402


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


class AdaptiveSelfAttention(nn.Module):
    """One block's attention half, of tokens with positions whose table rope_table() made: like AdaptiveFeedForward."""

    def __init__(self, width: int, head_dim: int, linear=nn.Linear):
        super().__init__()
        self.head_dim = head_dim
        self.qkv = linear(width, 3 * width)
        self.out = linear(width, width)
        self.q_norm = nn.Parameter(torch.ones(head_dim))
        self.k_norm = nn.Parameter(torch.ones(head_dim))

    def forward(self, x, h, gate, scale, shift, table):
        x, y = gated_residual_norm(x, h, gate, scale=scale, shift=shift, kind="layer", out_dtype="mxfp4")
        q, k, v = self.qkv(y).unflatten(-1, (3, -1, self.head_dim)).unbind(2)
        q, k = qk_norm_rope(q, k, table, q_weight=self.q_norm, k_weight=self.k_norm, norm="head")
        return x, self.out(attention(q, k, v).flatten(2))


class PlainSelfAttention(AdaptiveSelfAttention):
    """The same with library calls."""

    def forward(self, x, h, gate, scale, shift, table):
        x = x + gate * h
        y = F.layer_norm(x, x.shape[-1:], eps=1e-6) * (1 + scale) + shift
        q, k, v = self.qkv(y).unflatten(-1, (3, -1, self.head_dim)).unbind(2)
        q, k = (turned(F.rms_norm(t, t.shape[-1:], w, eps=1e-6), table) for t, w in ((q, self.q_norm), (k, self.k_norm)))
        o = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)))
        return x, self.out(o.transpose(1, 2).flatten(2))


def turned(x, table):
    a, b = x.float().unflatten(-1, (-1, 2)).unbind(-1)
    cos, sin = table[:, None].unbind(-1)
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).to(x.dtype)


def positions(tokens: int, device="cuda"):
    """(tokens, 3): a picture's tokens, row by row, of a video's first frame."""
    n = torch.arange(tokens, device=device)
    side = max(1, round(tokens ** 0.5))
    return torch.stack((torch.zeros_like(n), n // side, n % side), -1)


def build_attention(width: int, head_dim: int, device="cuda", seed: int = 0):
    """(the plain half, the MXFP4 half with the same weights)."""
    torch.manual_seed(seed)
    plain = PlainSelfAttention(width, head_dim).to(device=device, dtype=torch.bfloat16)
    with torch.device("meta"):
        half = AdaptiveSelfAttention(width, head_dim, mxfp4_ops(torch.bfloat16).Linear)
    half.load_state_dict(plain.state_dict(), assign=True)
    return plain, half


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
    parser.add_argument("--head-dim", type=int, default=128)
    args = parser.parse_args()
    sizes = f"tokens {args.tokens} width {args.width}"
    with torch.inference_mode():
        args_in = inputs(args.tokens, args.width)
        report(f"{sizes} hidden {args.hidden}", *build(args.width, args.hidden), args_in)
        if args.width % args.head_dim:
            print(f"{sizes}: no heads of {args.head_dim} in this width, no attention half")
            return
        rest = args.head_dim // 8 * 3 // 2 * 2  # the two directions of a picture; time has what is left
        table = rope_table(positions(args.tokens), (args.head_dim - 2 * rest, rest, rest))
        report(f"{sizes} heads {args.width // args.head_dim}", *build_attention(args.width, args.head_dim), (*args_in, table))


def report(sizes: str, plain, block, args_in) -> None:
    x, y = block(*args_in)
    x_ref, y_ref = plain(*args_in)
    off = (y.float() - y_ref.float()).norm() / y_ref.float().norm()
    same = torch.equal(x, x_ref)
    t, t_plain = _time(lambda: block(*args_in)), _time(lambda: plain(*args_in))
    print(f"{sizes}: MXFP4 {t:.3f} ms, bf16 library {t_plain:.3f} ms "
          f"({t_plain / t:.2f}x); stream {'equal' if same else 'differs by roundings'}, output {off:.3f} off (2-norm)")


if __name__ == "__main__":
    main()
