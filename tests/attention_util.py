"""Inputs and the error bound of the attention tests."""

import ctypes

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


class AttentionArgs(ctypes.Structure):
    """feather_attention_args of include/featherops_amd.h."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "mask", "q_offsets", "k_offsets", "k_lengths")]
                + [(n, ctypes.c_int64) for n in ("batch", "q_tokens", "k_tokens", "heads", "kv_heads", "head_dim",
                                                 "q_batch_stride", "q_token_stride", "q_head_stride", "k_batch_stride",
                                                 "k_token_stride", "k_head_stride", "v_batch_stride", "v_token_stride",
                                                 "v_head_stride", "mask_batch_stride", "mask_head_stride", "mask_query_stride")]
                + [(n, ctypes.c_int) for n in ("dtype", "mask_dtype", "causal")] + [("scale", ctypes.c_float)])


def attention_args(B, Sq, Sk, H, Hk, D, **kw):
    """Of contiguous bf16 tensors; the pointers stand for some until they are set."""
    P = 4096
    a = AttentionArgs(q=P, k=P, v=P, out=P, batch=B, q_tokens=Sq, k_tokens=Sk, heads=H, kv_heads=Hk, head_dim=D, dtype=1, mask_dtype=1,
                      q_batch_stride=Sq * H * D, q_token_stride=H * D, q_head_stride=D, k_batch_stride=Sk * Hk * D,
                      k_token_stride=Hk * D, k_head_stride=D, v_batch_stride=Sk * Hk * D, v_token_stride=Hk * D, v_head_stride=D,
                      scale=0.1)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def plan_of(lib, args):
    """(waves, splits, blocks), see feather_attention_plan."""
    plan = (ctypes.c_int64 * 3)()
    assert lib.feather_attention_plan(ctypes.byref(args), plan) == 0
    return tuple(plan)


# Shapes that each form takes where there is no mask, and some with one: ((waves, whether workgroups share a block's keys), (batch, q tokens, k tokens,
# heads, kv heads, head_dim)). test_attention_host.py checks that they do.
FORMS = [((0, False), (3, 1101, 140, 16, 2, 64)), ((0, False), (2, 777, 1300, 24, 8, 64)), ((0, False), (3, 1101, 157, 16, 16, 40)),
         ((4, False), (3, 7, 77, 16, 2, 64)), ((4, True), (2, 1, 2111, 8, 2, 64)), ((8, False), (2, 142, 300, 8, 2, 64)),
         ((8, True), (1, 33, 9011, 8, 8, 56)), ((0, False), (3, 1101, 140, 16, 2, 96)), ((0, False), (2, 777, 1300, 24, 8, 88)),
         ((4, False), (3, 35, 77, 16, 2, 96)), ((4, True), (1, 1100, 5003, 8, 8, 96)), ((8, False), (1, 77, 301, 24, 24, 72)),
         ((8, True), (2, 7, 9001, 8, 2, 96)), ((0, False), (3, 1101, 140, 16, 2, 128)), ((0, False), (2, 777, 1300, 24, 8, 128)),
         ((0, False), (1, 1500, 459, 21, 7, 104)), ((4, False), (3, 7, 300, 15, 3, 128)), ((4, True), (1, 2, 1100, 24, 24, 128)),
         ((8, False), (1, 77, 513, 24, 24, 128)), ((8, True), (2, 33, 5001, 5, 5, 120)), ((0, False), (3, 1101, 140, 16, 2, 256)),
         ((0, False), (2, 777, 1300, 24, 8, 136)), ((4, False), (3, 35, 140, 16, 2, 256)), ((4, True), (2, 7, 9001, 8, 2, 256)),
         ((4, True), (1, 65, 1100, 24, 24, 200))]
