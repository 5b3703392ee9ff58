"""example_mxfp4_block.py on the GPU: as it is started, and its attention half against float64."""

import importlib
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import attention_oracle as A
from oracle import block_oracle as B

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "comfyui-featherops_amd" / "example_mxfp4_block.py"


@pytest.mark.parametrize("options,halves", [(("--width", "192"), 1), (("--width", "250", "--head-dim", "64"), 1),
                                            (("--width", "192", "--head-dim", "64"), 2)], ids=str)
def test_widths(cuda, options, halves):
    """A width that holds no whole number of heads has the feed-forward half alone."""
    out = subprocess.run([sys.executable, str(EXAMPLE), "--tokens", "40", "--hidden", "320", *options], capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    assert out.stdout.count("MXFP4") == halves and ("no attention half" in out.stdout) == (halves == 1), out.stdout


def test_attention_half(pkg, cuda):
    """Against the same run in float64 on the quantised values. What attention returns is off by two roundings to bf16, 2^-7 of a
    value at most: with 4-bit steps of a quarter of a value at least, up to one in 32 then falls on the other side of a
    rounding in front of the out projection and moves by up to half of itself: sqrt(1 / 32) / 2 of the norm, 0.09."""
    sys.path.insert(0, str(EXAMPLE.parent))
    try:
        example = importlib.import_module("example_mxfp4_block")
    finally:
        sys.path.pop(0)
    rope = importlib.import_module("featherops_amd.kernel.hip.rope")
    tokens, width, head = 201, 256, 64
    axes = (16, 24, 24)
    with torch.inference_mode():
        plain, half = example.build_attention(width, head)
        x, h, gate, scale, shift = example.inputs(tokens, width)
        places = example.positions(tokens)
        s, y = half(x, h, gate, scale, shift, rope.rope_table(places, axes))
    d = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    bf16 = lambda a: torch.from_numpy(a).bfloat16().double().numpy()  # noqa: E731
    quantised = lambda v: B.mxfp4_values(*B.mxfp4_quantize(v), v.shape[1])  # noqa: E731
    want_s, n = B.gated_norm(d(x), d(h), d(gate), scale=d(scale), shift=d(shift), layer=True)
    assert np.abs(d(s) - want_s).max() <= (2.0 ** -8 * np.abs(want_s)).max()
    qkv = bf16(quantised(n[0]) @ quantised(d(plain.qkv.weight)).T + d(plain.qkv.bias)).reshape(tokens, 3, width // head, head)
    angles = A.rope_angles(places.cpu().numpy(), axes)
    q, k = (bf16(A.norm_rope(qkv[:, i], angles, d(w), "head")) for i, w in ((0, plain.q_norm), (1, plain.k_norm)))
    o = bf16(A.attention_one(q, k, qkv[:, 2])[0]).reshape(tokens, width)
    want = quantised(o) @ quantised(d(plain.out.weight)).T + d(plain.out.bias)
    off = np.linalg.norm(d(y)[0] - want) / np.linalg.norm(want)
    print("attention half off by", off)
    assert off <= 0.1
