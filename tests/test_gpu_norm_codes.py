"""The norms' 4-bit results of 16-bit blocks, and wide 16-bit streams with two vectors a thread, against float64."""

import importlib

import numpy as np
import pytest
import torch

from oracle import block_oracle as B
from test_gpu_block_norm import ALL, BF16, F16, F32, check, d, inputs

pytestmark = pytest.mark.gpu
TYPES = [(BF16, BF16, BF16), (F16, F16, F16), (BF16, BF16, F32), (F16, F16, F32), (F32, BF16, BF16), (F32, F16, F32)]


@pytest.fixture(scope="module")
def nm(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.norm")


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


def bounds(t, use, layer, eps):
    """(y, err): the fp32 result in float64, and how far fp32 arithmetic may take it: 16 roundings of 2^-24 on a value's
    way and 2^-24 (8 + log2 D) for the statistics, relative to the largest terms that meet (|x| + |gate h'|), divided by
    the row's norm and amplified by the affine factors; the added vectors' own roundings beside it."""
    v = {k: d(t[k]) for k in use}
    h, gate, post = v.pop("h", None), v.pop("gate", None), v.pop("post_weight", None)
    x = d(t["x"])
    s, y = B.gated_norm(x, h, gate, post, **v, layer=layer, eps=eps)
    u = 2.0 ** -24 * (24 + np.log2(max(2, x.shape[-1])))
    mags = np.abs(x)
    if h is not None:
        hh = np.abs(h)
        if post is not None:
            mean = h.mean(-1, keepdims=True) * layer
            hh = (hh + np.abs(mean)) / np.sqrt(((h - mean) ** 2).mean(-1, keepdims=True) + eps) * np.abs(post)
        mags = mags + (hh if gate is None else np.abs(gate) * hh)
    mean = s.mean(-1, keepdims=True) * layer
    sd = np.sqrt(((s - mean) ** 2).mean(-1, keepdims=True) + eps)
    up = 1.0 + v["scale"] if "scale" in v else 1.0
    amp = np.abs(v.get("weight", 1.0)) * np.abs(up)
    err = u * (mags + np.sqrt((mags ** 2).mean(-1, keepdims=True)) + np.abs(mean)) / sd * (1.0 + np.abs(s - mean) / sd) * amp
    for k in ("bias", "shift"):
        if k in v:
            err = err + u * np.abs(v[k]) * (np.abs(up) if k == "bias" else 1.0)
    return y, err + u * np.abs(y)


def nearest(v, step):
    """The 4-bit value nearest to v under the given scale, ties to the even code."""
    a, code = np.abs(v) / step, np.zeros(v.shape, dtype=int)
    for i, m in enumerate((B.VALUES[:-1] + B.VALUES[1:]) / 2):
        code += (a > m) | ((a == m) & (i % 2 == 1))
    return np.sign(v) * B.VALUES[code] * step


def check_codes(mx, q, y, err, label):
    """Each block's scale is that of a largest magnitude within the error; each value lies between the 4-bit values
    nearest to the error's ends, which for all but a few are the same."""
    rows, D = int(np.prod(y.shape[:-1])), y.shape[-1]
    blocks = -(-D // 32)

    def split(v):
        return np.pad(v.reshape(rows, D), ((0, 0), (0, blocks * 32 - D))).reshape(rows, blocks, 32)

    y, err = split(y), split(np.broadcast_to(err, y.shape))
    codes, scales = (t.cpu().numpy() for t in mx.unprepack_mxfp4(q))
    got = B.mxfp4_values(codes, scales, blocks * 32).reshape(rows, blocks, 32)

    def byte(amax):
        return np.where(amax == 0, 0, np.maximum(np.frexp(amax)[1] - 3 + 127, 0))

    low, high = byte(np.maximum(np.abs(y) - err, 0).max(2)), byte((np.abs(y) + err).max(2))
    assert ((low <= scales) & (scales <= high)).all(), f"{label}: scales"
    step = np.ldexp(1.0, scales.astype(int) - 127)[:, :, None]
    a, b = nearest(y - err, step), nearest(y + err, step)
    bad = (got < a) | (got > b)
    assert not bad.any(), f"{label}: {bad.sum()} of {rows * D} values, the first at {np.argwhere(bad)[0]}"
    assert ((a != b) & (y != 0)).mean() < 0.01, label


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x)[6:] for x in t))
@pytest.mark.parametrize("rows,D", [(7, 7), (2, 33), (5, 500), (3, 1160), (130, 2081), (20, 4097), (1030, 5120), (12, 9000)])
def test_codes(nm, mx, cuda, rows, D, types):
    t = inputs(cuda, 1, rows, D, *types, seed=rows + D)
    for use in (ALL, ("h", "gate", "scale", "shift")):
        for kind in ("layer", "rms"):
            args = {k: t[k] for k in use}
            h, gate = args.pop("h"), args.pop("gate")
            s, q = nm.gated_residual_norm(t["x"], h, gate, kind=kind, eps=1e-3, out_dtype="mxfp4", **args)
            y, err = bounds(t, use, kind == "layer", 1e-3)
            check_codes(mx, q, y, err, f"{rows} {D} {types} {kind} {use}")
            assert torch.equal(s, nm.gated_residual_norm(t["x"], h, gate, kind=kind, eps=1e-3, **args)[0])
    use = ("weight", "bias", "scale", "shift")
    q = nm.modulated_norm(t["x"], **{k: t[k] for k in use}, kind="layer", eps=1e-3, out_dtype="mxfp4")
    check_codes(mx, q, *bounds(t, use, True, 1e-3), f"{rows} {D} {types} modulated")


@pytest.mark.parametrize("types", [(BF16, BF16, BF16), (F16, F16, F32)], ids=lambda t: "-".join(str(x)[6:] for x in t))
@pytest.mark.parametrize("rows,D", [(1030, 5120), (1025, 4099), (1100, 8190)])
def test_two_vectors_a_thread(nm, cuda, rows, D, types):
    """Wide 16-bit streams of many rows, with a last vector that ends with the row."""
    t = inputs(cuda, 1, rows, D, *types, seed=D)
    for kind in ("layer", "rms"):
        check(nm, t, ALL, kind, eps=1e-3, label=f"{rows} {D}")
