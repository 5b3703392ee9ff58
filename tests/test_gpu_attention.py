"""Attention on the GPU against float64 (oracle/attention_oracle.py)."""

import importlib

import numpy as np
import pytest
import torch

from attention_util import BF16, F16, F32, check, d, normal, qkv
from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def at(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.attention")


def run(at, q, k, v, label="", added=0.0, **kw):
    o = at.attention(q, k, v, **kw)
    assert o.shape == q.shape and o.dtype == q.dtype and o.is_contiguous()
    lengths = kw.get("k_lengths")
    want = A.attention(d(q), d(k), d(v), kw.get("causal", False), kw.get("scale"), None if lengths is None else lengths.tolist(),
                       d(kw.get("mask")))
    check(o, *want, k.shape[1], label, added)
    return o


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 96, 104, 128, 136, 256])
def test_head_dims(at, cuda, D, dtype, causal):
    g = torch.Generator().manual_seed(D)
    run(at, *qkv(g, 2, 150, 203, 3, 3, D, dtype), causal=causal)


SIZES = [(1, 1), (1, 2), (2, 1), (1, 63), (1, 64), (1, 65), (3, 31), (31, 33), (32, 32), (33, 64), (64, 128), (127, 129), (128, 128),
         (129, 127), (200, 7), (257, 300), (500, 64), (64, 1000)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_lengths(at, cuda, sizes, causal):
    """Causal with fewer keys than queries: the first queries see none."""
    for dtype, D in ((BF16, 128), (F16, 64)):
        g = torch.Generator().manual_seed(sum(sizes))
        run(at, *qkv(g, 1, *sizes, 2, 2, D, dtype), f"{D}", causal=causal)


@pytest.mark.parametrize("heads", [(1, 1), (4, 1), (7, 1), (6, 2), (40, 8), (16, 16)])
def test_shared_heads(at, cuda, heads):
    g = torch.Generator().manual_seed(heads[0])
    for Sq in (1, 5, 140):
        run(at, *qkv(g, 3, Sq, 170, *heads, 80, BF16), f"{Sq}", causal=True)


def counting(cuda, B, Sk, H, D, dtype, seed=0):
    """Values of which each key has a one in one column: with equal weights a result is a small count over the keys."""
    v = torch.zeros(B, Sk, H, D, dtype=dtype)
    col = (torch.arange(Sk)[None, :] * 7 + torch.arange(B)[:, None] * 3 + seed) % D
    v.scatter_(3, col[:, :, None, None].expand(B, Sk, H, 1), 1.0)
    return v.to(cuda), col


@pytest.mark.parametrize("Sk", [1, 64, 65, 200, 1000, 3000])
@pytest.mark.parametrize("Sq", [1, 4, 129])
def test_every_key_counts_once(at, cuda, Sq, Sk):
    """Equal scores: the result is exactly a count over the number of keys, rounded once (and the count's own quotient in
    fp32)."""
    D, dtype = 128, BF16
    q, k = torch.zeros(2, Sq, 4, D, dtype=dtype, device=cuda), normal(torch.Generator().manual_seed(1), 2, Sk, 2, D)
    v, col = counting(cuda, 2, Sk, 2, D, dtype)
    lengths = torch.tensor([Sk, max(1, Sk - 37)], dtype=torch.int32, device=cuda)
    o = d(at.attention(q, k, v, k_lengths=lengths))
    for b in range(2):
        n = int(lengths[b])
        want = np.bincount(col[b, :n].numpy(), minlength=D) / n
        assert (np.abs(o[b] - want) <= want * (2.0 ** -8 + 2.0 ** -20)).all()


def test_causal_counts(at, cuda):
    D, S = 64, 300
    for Sk in (S, 250, 427):
        q, k = torch.zeros(1, S, 1, D, dtype=F16, device=cuda), torch.ones(1, Sk, 1, D, dtype=F16, device=cuda)
        v, col = counting(cuda, 1, Sk, 1, D, F16)
        o = d(at.attention(q, k, v, causal=True))[0, :, 0]
        for i in range(S):
            n = max(0, i + 1 + Sk - S)
            want = np.bincount(col[0, :n].numpy(), minlength=D) / max(n, 1)
            assert (np.abs(o[i] - want) <= want * (2.0 ** -11 + 2.0 ** -20)).all(), (Sk, i)


@pytest.mark.parametrize("Sq", [1, 77])
def test_k_lengths(at, cuda, Sq):
    """Keys and values behind a sample's length are not read: they hold NaN."""
    lengths = [0, 1, 63, 64, 65, 128, 300, 299, 400, -5]  # (400 and -5 are clamped)
    g = torch.Generator().manual_seed(3)
    q, k, v = qkv(g, len(lengths), Sq, 300, 4, 2, 96, BF16)
    for b, n in enumerate(lengths):
        k[b, max(n, 0):] = float("nan")
        v[b, max(n, 0):] = float("inf")
    for causal in (False, True):
        o = run(at, q, k, v, k_lengths=torch.tensor(lengths, dtype=torch.int32, device=cuda), causal=causal)
        assert not o[0].any() and not o[-1].any()


MASKS = [(1, 1, 1, 0), (2, 1, 1, 0), (1, 3, 0, 0), (2, 3, 0, 0), (2, 1, 0, 0), (2, 3, 0, 1)]


@pytest.mark.parametrize("shape", MASKS, ids=str)
@pytest.mark.parametrize("kind", ["bool", "half", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_masks(at, cuda, D, kind, shape):
    """Broadcast over any of the dimensions (0: the whole one), rows that see nothing among them."""
    Sq, Sk = 139, 205
    g = torch.Generator().manual_seed(D + sum(shape))
    q, k, v = qkv(g, 2, Sq, Sk, 3, 3, D, BF16)
    full = (shape[0], shape[1], shape[2] or Sq, shape[3] or Sk)
    if kind == "bool":
        mask = torch.rand(full, generator=g) < 0.6
        if full[2] > 1:
            mask[..., 5:9, :] = False
    else:
        mask = torch.randn(full, generator=g) * 3.0
        mask = torch.where(torch.rand(full, generator=g) < 0.2, float("-inf"), mask).to(BF16 if kind == "half" else F32)
        if full[2] > 1:
            mask[..., 5:9, :] = float("-inf")
    for causal in (False, True):
        run(at, q, k, v, f"{causal}", 8.0, mask=mask.to(cuda), causal=causal)


def test_mask_of_lowest_values(at, cuda):
    """The type's lowest value is added, not taken for -inf: a row of nothing else has weights by its scores' rounding
    beside it (all alike), and one key without it takes all."""
    g = torch.Generator().manual_seed(5)
    q, k, v = qkv(g, 1, 130, 150, 2, 2, 64, BF16)
    mask = torch.zeros(1, 1, 130, 150)
    low = torch.finfo(F32).min
    mask[:, :, 3] = low
    mask[:, :, 4] = low
    mask[:, :, 4, 77] = 0.0
    mask[:, :, 5, 100:] = low
    o = d(at.attention(q, k, v, mask=mask.to(cuda)))
    vd = d(v)
    tol = 2.0 ** -7 * np.abs(vd[0]).max()
    assert (np.abs(o[0, 3] - vd[0].mean(0)) <= tol).all()
    assert (np.abs(o[0, 4] - vd[0, 77]) <= 2.0 ** -8 * np.abs(vd[0, 77])).all()
    short = A.attention(d(q)[:, 5:6], d(k)[:, :100], vd[:, :100])
    assert (np.abs(o[0, 5] - short[0][0, 0]) <= 2.0 ** -7 * (short[1][0, 0] + 2.0 ** -10)).all()


def test_mask_views(at, cuda):
    """Strided, expanded and transposed masks, keys at odd offsets."""
    g = torch.Generator().manual_seed(6)
    q, k, v = qkv(g, 2, 50, 61, 4, 4, 64, F16)
    big = torch.randn(2, 4, 61, 50, generator=g).half().to(cuda)
    run(at, q, k, v, "transposed", 8.0, mask=big.transpose(2, 3))
    wide = torch.randn(50, 200, generator=g).to(cuda)
    run(at, q, k, v, "slice", 8.0, mask=wide[:, 3:64])
    run(at, q, k, v, "expanded", 8.0, mask=wide[:, 5:66].expand(2, 4, 50, 61))
    run(at, q, k, v, "one dimension", 8.0, mask=wide[0, 7:68])
    keep = torch.rand(2, 1, 1, 64, generator=g) < 0.5
    run(at, q, k, v, "bool slice", mask=keep.to(cuda)[..., 2:63])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens,k_lens", [
    ([1], None), ([77, 154, 1, 0, 333, 512], None), ([128, 128, 0, 0, 64], None), ([5] * 70, None),
    ([10, 0, 300, 1, 4], [0, 5, 1, 300, 129]), ([1] * 9, [64, 1, 0, 65, 200, 3, 128, 127, 1000])])
def test_packed(at, cuda, q_lens, k_lens, causal):
    g = torch.Generator().manual_seed(len(q_lens))
    k_lens = k_lens or q_lens
    qo, ko = np.concatenate(([0], np.cumsum(q_lens))), np.concatenate(([0], np.cumsum(k_lens)))
    for dtype, H, Hk, D in ((BF16, 4, 2, 128), (F16, 3, 3, 72)):
        q, k, v = (normal(g, n, h, D, dtype=dtype) for n, h in ((qo[-1], H), (ko[-1], Hk), (ko[-1], Hk)))
        offsets = [torch.tensor(o, dtype=torch.int32, device=cuda) for o in (qo, ko)]
        o = at.packed_attention(q, k, v, *(offsets[:1] if k_lens is q_lens else offsets), causal=causal)
        check(o, *A.packed_attention(d(q), d(k), d(v), qo, ko, causal), max(k_lens))


def test_packed_outside_and_wrong_offsets(at, cuda):
    """Tokens outside every sequence get zeros; offsets beyond the tensors are clamped, falling ones give empty sequences."""
    g = torch.Generator().manual_seed(8)
    q, k, v = (normal(g, 500, 2, 64) for _ in range(3))
    off = np.array([130, 200, 200, 333])
    o = at.packed_attention(q, k, v, torch.tensor(off, dtype=torch.int32, device=cuda))
    check(o, *A.packed_attention(d(q), d(k), d(v), off, off), 133)
    assert not o[:130].any() and not o[333:].any() and o[130:333].any()
    for bad in ([-7, 200, 5000], [0, 2 ** 31 - 1], [-2 ** 31, 600]):
        clamped = np.clip(bad, 0, 500)
        o = at.packed_attention(q, k, v, torch.tensor(bad, dtype=torch.int32, device=cuda))
        check(o, *A.packed_attention(d(q), d(k), d(v), clamped, clamped), 500)
    at.packed_attention(q, k, v, torch.tensor([300, 100, 400, 0], dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()


def test_layouts(at, cuda):
    """A joint output's slices, heads in front of tokens, a slice of a cache, expanded samples, unaligned and strided views."""
    g = torch.Generator().manual_seed(9)
    B, S, H, D = 2, 147, 4, 64
    joint = normal(g, B, S, 3, H, D)
    want = run(at, *(joint[:, :, i].contiguous() for i in range(3)))
    assert torch.equal(at.attention(*(joint[:, :, i] for i in range(3))), want)
    front = [joint[:, :, i].transpose(1, 2).contiguous().transpose(1, 2) for i in range(3)]
    assert torch.equal(at.attention(*front), want)
    cache = torch.full((2, B, 400, H, D), float("nan"), dtype=BF16, device=cuda)
    cache[0, :, 100:100 + S], cache[1, :, 100:100 + S] = joint[:, :, 1], joint[:, :, 2]
    assert torch.equal(at.attention(joint[:, :, 0], cache[0, :, 100:100 + S], cache[1, :, 100:100 + S]), want)
    odd = torch.empty(B * S * H * D + 3, dtype=BF16, device=cuda)[3:].view(B, S, H, D).copy_(joint[:, :, 1])
    assert torch.equal(at.attention(joint[:, :, 0], odd, joint[:, :, 2]), want)
    spread = torch.empty(B, S, H, D, 2, dtype=BF16, device=cuda)[..., 1].copy_(joint[:, :, 2])
    assert torch.equal(at.attention(joint[:, :, 0], joint[:, :, 1], spread), want)
    one = joint[:1, :, 1].expand(B, S, H, D)
    assert torch.equal(at.attention(joint[:, :, 0], one, one), at.attention(joint[:, :, 0], one.contiguous(), one.contiguous()))


@pytest.mark.parametrize("std", [0.05, 3.0, 8.0])
def test_score_ranges(at, cuda, std):
    """Nearly equal weights and weights that one key takes."""
    g = torch.Generator().manual_seed(10)
    for dtype in (F16, BF16):
        run(at, *qkv(g, 1, 140, 700, 2, 2, 128, dtype, std=std), f"{dtype}")


def test_rising_scores(at, cuda):
    """Each tile of keys has a larger maximum than the one before: by less and by more than the lag that is allowed."""
    for step in (0.5, 3.0, 20.0):
        k = torch.zeros(1, 640, 1, 64)
        k[0, :, 0, 0] = torch.arange(640).float() // 32 * step
        q = torch.ones(1, 130, 1, 64)
        v = normal(torch.Generator().manual_seed(1), 1, 640, 1, 64)
        run(at, q.to(BF16).to(cuda), k.to(BF16).to(cuda), v, f"{step}", scale=1.0)
        run(at, q.to(BF16).to(cuda), -k.to(BF16).to(cuda), v, f"-{step}", scale=1.0)


def test_scale(at, cuda):
    g = torch.Generator().manual_seed(11)
    q, k, v = qkv(g, 1, 70, 90, 2, 2, 64, BF16)
    for scale in (1e-30, 0.03, 1.0, 4.0):
        run(at, q, k, v, f"{scale}", scale=scale)


def test_special_values(at, cuda):
    """NaN and infinite scores and values reach the queries that see them, and no other."""
    g = torch.Generator().manual_seed(12)
    q, k, v = qkv(g, 1, 200, 200, 2, 1, 64, BF16)
    q[0, 7, 0, 3] = float("nan")
    o = at.attention(q, k, v)
    bad = torch.isnan(o).flatten(3).any(3)[0]
    assert bad[7, 0] and bad.sum() == 1
    q[0, 7, 0, 3] = 0.0
    v[0, 150, 0, 5] = float("inf")
    o = at.attention(q, k, v)
    assert torch.isinf(o[..., 5]).all() and torch.isfinite(o[..., :5]).all() and torch.isfinite(o[..., 6:]).all()


def test_empty(at, cuda):
    q = torch.zeros(2, 0, 4, 64, dtype=BF16, device=cuda)
    k = torch.zeros(2, 5, 4, 64, dtype=BF16, device=cuda)
    assert at.attention(q, k, k).shape == q.shape
    assert not at.attention(k + 1, q, q).any()
    assert at.attention(q[:0], k[:0], k[:0]).shape == (0, 0, 4, 64)
    off = torch.zeros(3, dtype=torch.int32, device=cuda)
    assert at.packed_attention(q[0], q[0], q[0], off).shape == (0, 4, 64)
    assert not at.packed_attention(k[0] + 1, q[0], q[0], off, off).any()
