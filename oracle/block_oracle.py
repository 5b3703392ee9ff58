"""Plain 64-bit evaluations of the MXFP4 operators and the block norms: test infrastructure only.

Written from the definitions in numpy, independent of the kernels and of their layout:
  * MXFP4: a block of 32 values has the scale 2^max(floor(log2 amax) - 2, -127) and for each value the
    nearest of the fifteen numbers 0, +-0.5 .. +-6 times it, ties to the even code, NaN as a whole if any
    value is not finite;
  * the norms: statistics, affine terms, gate and residual in float64.
"""

from __future__ import annotations

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mxfp4_quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(rows, cols) float values -> row-major codes (rows, blocks * 16) and scales (rows, blocks), uint8."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    finite = np.isfinite(v).all(axis=2)
    amax = np.where(finite, np.abs(np.where(np.isfinite(v), v, 0.0)).max(axis=2), 1.0)
    _, e = np.frexp(amax)  # amax in [2^(e-1), 2^e)
    exponent = np.where(amax == 0.0, -127, np.maximum(e - 3, -127))
    with np.errstate(over="ignore", invalid="ignore"):
        a = np.abs(v) * np.ldexp(1.0, -exponent)[:, :, None]
    # the code counts the midpoints below the value; on a midpoint it goes to the even neighbour
    mids = (VALUES[:-1] + VALUES[1:]) / 2
    code = np.zeros(v.shape, dtype=np.uint8)
    for i, m in enumerate(mids):
        code += (a > m) | ((a == m) & (i % 2 == 1))
    code = code | (np.signbit(v).astype(np.uint8) << 3)
    scales = np.where(finite, exponent + 127, 255).astype(np.uint8)
    code = code.reshape(rows, blocks * 32)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def mxfp4_values(codes: np.ndarray, scales: np.ndarray, cols: int) -> np.ndarray:
    """Row-major codes and scales -> the float64 values they stand for."""
    rows = codes.shape[0]
    code = np.stack((codes & 15, codes >> 4), axis=2).reshape(rows, -1)
    v = VALUES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(rows, -1, 32) * s[:, :, None]).reshape(rows, -1)[:, :cols]


def norm(v: np.ndarray, layer: bool, eps: float) -> np.ndarray:
    if layer:
        v = v - v.mean(axis=-1, keepdims=True)
    return v / np.sqrt((v * v).mean(axis=-1, keepdims=True) + eps)


def gated_norm(x, h=None, gate=None, post_weight=None, weight=None, bias=None, scale=None, shift=None, layer=False,
               eps=1e-6, residual_scale=1.0):
    """(stream, y) in float64; arguments are float64 arrays that broadcast against x."""
    s = x
    if h is not None:
        if post_weight is not None:
            h = norm(h, layer, eps) * post_weight
        s = residual_scale * x + (h if gate is None else gate * h)
    y = norm(s, layer, eps)
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    if scale is not None:
        y = y * (1.0 + scale)
    if shift is not None:
        y = y + shift
    return s, y
