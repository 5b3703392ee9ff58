"""Inputs and the error bound of the attention tests."""

import numpy as np
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


def d(t):
    if t is None:
        return None
    return t.cpu().numpy() if t.dtype == torch.bool else t.double().cpu().numpy()


def normal(gen, *shape, dtype=BF16, std=1.0, dev="cuda"):
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(dev)


def qkv(gen, B, Sq, Sk, H, Hk, D, dtype, std=1.0, dev="cuda"):
    return (normal(gen, B, Sq, H, D, dtype=dtype, std=std, dev=dev), normal(gen, B, Sk, Hk, D, dtype=dtype, std=std, dev=dev),
            normal(gen, B, Sk, Hk, D, dtype=dtype, dev=dev))


def check(got, want, mags, reach, keys, label="", added=0.0):
    """got against the 64-bit result. The weights are rounded to the tensors' type (u, relative, and in fp16 at most 2^-25
    in absolute terms where the largest is 2^7 or more) and so is the result: u (sum p |v| + |o|). Everything else is
    fp32: scores are sums of D products (2^-24 D sum |q k|), their factor and distance from the maximum (8 roundings
    of at most |score| 1.45 + 130 each, in units of an exponent, and one of |mask|), the exponential (2^-22), and the two
    sums over the keys (2^-24 keys, relative to sum p |v| and |o|)."""
    u = HALF[got.dtype]
    D = want.shape[-1]
    e = 2.0 ** -24 * ((D + 8) * 1.45 * reach + 8 * 130.0 + 4.0 * added) + 2.0 ** -22 + 2.0 ** -24 * (keys + 8)
    tol = u * (mags + np.abs(want)) + 2.0 * e * (mags + np.abs(want)) + 2.0 ** -25
    if got.dtype == F16:
        tol = tol + keys * 2.0 ** -32 * 8.0
    off = np.abs(d(got) - want)
    assert np.isfinite(d(got)).all(), f"{label}: not finite"
    worst = float((off / tol).max()) if off.size else 0.0
    assert worst <= 1.0, f"{label}: {worst:.3g} times the bound"
    return worst
