"""Plain 64-bit evaluations of rotary positions and attention: test infrastructure only.

Written from the definitions in numpy, independent of the kernels and of their layout.
"""

from __future__ import annotations

import numpy as np


def rope_angles(positions: np.ndarray, axes, theta: float = 10000.0, shared: bool = False) -> np.ndarray:
    """(..., pairs) angles for (..., axes) positions."""
    pairs = sum(axes) // 2
    out = np.empty((*positions.shape[:-1], pairs))
    p = 0
    for axis, d in enumerate(axes):
        for j in range(d // 2):
            power = -2.0 * p / sum(axes) if shared else -2.0 * j / d
            out[..., p] = positions[..., axis].astype(np.float64) * theta ** power
            p += 1
    return out


def norm_rope(x: np.ndarray, angles=None, weight=None, norm=None, eps: float = 1e-6, halves: bool = False) -> np.ndarray:
    """x (..., tokens, heads, dim); angles (tokens, pairs) or (batch, tokens, pairs)."""
    heads, dim = x.shape[-2:]
    if norm == "head":
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if weight is not None:
            x = x * weight
    elif norm == "row":
        x = x / np.sqrt((x * x).mean((-2, -1), keepdims=True) + eps)
        if weight is not None:
            x = x * weight.reshape(heads, dim)
    if angles is None:
        return x
    pairs = angles.shape[-1]
    c, s = np.cos(angles)[..., None, :], np.sin(angles)[..., None, :]
    y = x.copy()
    first = slice(0, pairs) if halves else slice(0, 2 * pairs, 2)
    second = slice(pairs, 2 * pairs) if halves else slice(1, 2 * pairs, 2)
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def attention_one(q, k, v, causal=False, scale=None, mask=None):
    """One sample: q (n, heads, dim), k and v (m, kv heads, dim), mask (1 or heads, 1 or n, m), bool or added. Returns the
    result and, for error bounds, sum_j p |v| and the largest sum_d |q k| * scale of a query's seen keys."""
    n, heads, dim = q.shape
    m, shared, _ = k.shape
    scale = dim ** -0.5 if scale is None else scale
    out, mags, reach = np.zeros((n, heads, dim)), np.zeros((n, heads, dim)), np.zeros((n, heads, 1))
    if n == 0 or m == 0:
        return out, mags, reach
    seen = np.ones((n, m), dtype=bool)
    if causal:
        seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + (m - n)
    for h in range(heads):
        kh, vh = k[:, h * shared // heads], v[:, h * shared // heads]
        s = scale * (q[:, h] @ kh.T)
        see = seen
        if mask is not None:
            mh = np.broadcast_to(mask[h % mask.shape[0]], (n, m))
            if mh.dtype == bool:
                see = see & mh
            else:
                s = s + mh
                see = see & ~np.isneginf(mh)
        s = np.where(see, s, -np.inf)
        top = s.max(1, keepdims=True)
        some = see.any(1, keepdims=True)
        p = np.where(see, np.exp(s - np.where(some, top, 0.0)), 0.0)
        p = p / np.where(some, p.sum(1, keepdims=True), 1.0)
        # what a query does not see takes no part, whatever it holds
        vs = np.where(see.any(0)[:, None], vh, 0.0)
        out[:, h], mags[:, h] = p @ vs, p @ np.abs(vs)
        reach[:, h, 0] = np.where(see, scale * (np.abs(q[:, h]) @ np.abs(kh).T), 0.0).max(1)
    return out, mags, reach


def attention(q, k, v, causal=False, scale=None, lengths=None, mask=None):
    """Samples (batch, tokens, heads, dim); mask broadcast to (batch, heads, n, m)."""
    parts = []
    for b in range(q.shape[0]):
        m = k.shape[1] if lengths is None else int(np.clip(lengths[b], 0, k.shape[1]))
        mb = None
        if mask is not None:
            mb = mask.reshape((1,) * (4 - mask.ndim) + mask.shape)
            mb = np.broadcast_to(mb[b % mb.shape[0]], (*mb.shape[1:3], k.shape[1]))[..., :m]
        parts.append(attention_one(q[b], k[b, :m], v[b, :m], causal, scale, mb))
    return tuple(np.stack(x) for x in zip(*parts))


def packed_attention(q, k, v, q_offsets, k_offsets, causal=False, scale=None):
    out = [np.zeros(q.shape), np.zeros(q.shape), np.zeros((*q.shape[:2], 1))]
    for s in range(len(q_offsets) - 1):
        qs, ks = slice(q_offsets[s], q_offsets[s + 1]), slice(k_offsets[s], k_offsets[s + 1])
        for whole, part in zip(out, attention_one(q[qs], k[ks], v[ks], causal, scale)):
            whole[qs] = part
    return tuple(out)
