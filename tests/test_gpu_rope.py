"""Rotary positions and the norm of queries and keys on the GPU against float64 (oracle/attention_oracle.py)."""

import importlib

import numpy as np
import pytest
import torch

from attention_util import BF16, F16, F32, HALF, d, normal
from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rp(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.rope")


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, F32, torch.float64])
@pytest.mark.parametrize("axes", [(128,), (16, 56, 56), (44, 42, 42), (2,), (0, 6), (10, 2, 4, 8), (128, 128)], ids=str)
@pytest.mark.parametrize("ladder", ["axis", "shared"])
def test_table(rp, cuda, axes, ladder, dtype):
    """fp32 cosines and sines of fp64 angles: half a step of 1 (2^-24), and an angle of up to 1e6 that fp64 roundings (a
    handful of 2^-53) move by less than 2^-30."""
    g = torch.Generator().manual_seed(sum(axes))
    pos = torch.randint(0, 10 ** 6, (3, 50, len(axes)), generator=g)
    pos = pos.to(dtype) if dtype in (torch.int32, torch.int64) else (pos.double() / 7.0 - 30000.0).to(dtype)
    table = rp.rope_table(pos.to(cuda), axes, 10000.0, ladder=ladder)
    assert table.shape == (3, 50, sum(axes) // 2, 2) and table.dtype == F32
    angles = A.rope_angles(pos.double().numpy(), axes, 10000.0, ladder == "shared")
    for i, want in enumerate((np.cos(angles), np.sin(angles))):
        assert np.abs(d(table[..., i]) - want).max() <= 2.0 ** -25 + 2.0 ** -30, i


def test_table_far_positions_and_theta(rp, cuda):
    pos = torch.tensor([[0.0], [-3.5], [2.0 ** 24 + 1], [1e9]], dtype=torch.float64, device=cuda)
    for theta in (1.0, 256.0, 1e6):
        angles = A.rope_angles(d(pos), (64,), theta)
        table = d(rp.rope_table(pos, (64,), theta))
        # (1e9 radians: fp64 keeps them to 2^-23)
        off = np.abs(np.stack((np.cos(angles), np.sin(angles)), -1) - table)
        assert off[:3].max() <= 2.0 ** -24 and off[3].max() <= 2.0 ** -20


def check(got, x, table, weight, norm, halves, eps=1e-6, label=""):
    """Half a step of the type for the one rounding, and fp32 arithmetic before it: the sum of squares (a tree of at most
    8 + 8 + 12 additions), division, root, weight, and the turn's two products and sum, 2^-24 each, relative to |a| + |b|
    of the pair. The table is taken as it is."""
    xd, wd = d(x), d(weight)
    angles = None
    if table is not None:
        t = d(table)
        angles = np.arctan2(t[..., 1], t[..., 0])
    want = A.norm_rope(xd, angles, wd, norm, eps, halves)
    plain = A.norm_rope(xd, None, wd, norm, eps)
    pair = np.abs(plain)
    if table is not None:
        P = angles.shape[-1]
        a, b = (slice(0, P), slice(P, 2 * P)) if halves else (slice(0, 2 * P, 2), slice(1, 2 * P, 2))
        pair = pair.copy()
        pair[..., a] = pair[..., b] = np.abs(plain[..., a]) + np.abs(plain[..., b])
    # (2^-23: cosine and sine of the table, which are rounded, on a circle that is off by as much)
    tol = HALF[got.dtype] * np.abs(want) + 2.0 ** -24 * (28 + 8) * pair + 2.0 ** -25 * (got.dtype == F16) + 2.0 ** -22 * pair
    off = np.abs(d(got) - want)
    worst = float((off / (tol + 1e-300)).max()) if off.size else 0.0
    assert worst <= 1.0, f"{label}: {worst:.3g} times the bound"


CASES = [(128, (16, 56, 56)), (128, (128,)), (64, (16, 24, 24)), (72, (36, 36)), (80, (40, 40)), (80, (20,)), (96, (18, 18)),
         (256, (64, 96, 96)), (40, (2,)), (8, (4, 4)), (136, (68, 68)), (16, (8,))]


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("norm", [None, "head", "row"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rope(rp, cuda, case, norm, halves):
    D, axes = case
    g = torch.Generator().manual_seed(D + len(axes))
    pos = torch.randint(0, 5000, (37, len(axes)), generator=g).to(cuda)
    table = rp.rope_table(pos, axes)
    for dtype, H, Hk in ((BF16, 5, 5), (F16, 6, 2), (F32, 3, 1)):
        q, k = normal(g, 2, 37, H, D, dtype=dtype, std=2.0), normal(g, 2, 37, Hk, D, dtype=dtype, std=0.3)
        qw = kw = None
        if norm:
            qw = (torch.randn(H * D if norm == "row" else D, generator=g) * 0.3 + 1).to(dtype).to(cuda)
            kw = (torch.randn(Hk * D if norm == "row" else D, generator=g) * 0.3 + 1).to(cuda)  # fp32 beside 16 bits
        qo, ko = rp.qk_norm_rope(q, k, table, q_weight=qw, k_weight=kw, norm=norm, pairs="halves" if halves else "adjacent")
        check(qo, q, table, qw, norm, halves, label=f"q {dtype}")
        check(ko, k, table, kw, norm, halves, label=f"k {dtype}")
        one = rp.norm_rope(q, table, weight=qw, norm=norm, pairs="halves" if halves else "adjacent")
        assert torch.equal(one, qo)


@pytest.mark.parametrize("norm,heads", [("head", 1), ("head", 24), ("head", 70), ("row", 24), ("row", 40), ("row", 128), ("row", 17)])
@pytest.mark.parametrize("tokens", [1, 3, 257, 600])
def test_heads_and_tokens(rp, cuda, tokens, norm, heads):
    """One pass and several of a wave's or workgroup's heads, few tokens and many."""
    g = torch.Generator().manual_seed(heads + tokens)
    pos = torch.randint(0, 100, (tokens, 2), generator=g).to(cuda)
    table = rp.rope_table(pos, (64, 64))
    x = normal(g, tokens, heads, 128)
    w = (torch.randn(heads * 128 if norm == "row" else 128, generator=g) * 0.3 + 1).to(BF16).to(cuda)
    check(rp.norm_rope(x, table, weight=w, norm=norm), x, table, w, norm, False)
    check(rp.norm_rope(x, None, weight=w, norm=norm), x, None, w, norm, False)


def test_tables_of_samples_and_views(rp, cuda):
    g = torch.Generator().manual_seed(2)
    B, S, H, D = 3, 50, 4, 96
    joint = normal(g, B, S, H + 2, D, dtype=F16)
    q, k = joint[:, :, :H], joint[:, :, H:H + 1]
    pos = torch.randint(0, 999, (B, S, 2), generator=g).to(cuda)
    table = rp.rope_table(pos, (48, 48))
    qo, ko = rp.qk_norm_rope(q, k, table, norm="head")
    check(qo, q, table, None, "head", False)
    check(ko, k, table, None, "head", False)
    assert qo.is_contiguous() and ko.is_contiguous()
    one = rp.qk_norm_rope(q, k, table[:1], norm="head")
    assert torch.equal(one[0], rp.qk_norm_rope(q, k, table[0], norm="head")[0])
    front = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(rp.norm_rope(front, table, norm="head"), qo)
    odd = torch.empty(q.numel() + 1, dtype=F16, device=cuda)[1:].view(q.shape).copy_(q)
    assert torch.equal(rp.norm_rope(odd, table, norm="head"), qo)
    apart = torch.empty(*q.shape, 2, dtype=F16, device=cuda)[..., 0].copy_(q)
    assert torch.equal(rp.norm_rope(apart, table, norm="head"), qo)


def test_turn_is_exact_where_it_can_be(rp, cuda):
    """Position 0 changes nothing; a NaN stays in its pair, or with a norm in its head."""
    x = normal(torch.Generator().manual_seed(3), 40, 3, 64)
    table = rp.rope_table(torch.zeros(40, 1, dtype=torch.int32, device=cuda), (64,))
    for pairs in ("adjacent", "halves"):
        assert torch.equal(rp.norm_rope(x, table, pairs=pairs), x)
    x[5, 1, 10] = float("nan")
    table = rp.rope_table(torch.arange(40, device=cuda)[:, None], (64,))
    bad = torch.isnan(rp.norm_rope(x, table))
    assert bad[5, 1, 10:12].all() and bad.sum() == 2
    bad = torch.isnan(rp.norm_rope(x, table, pairs="halves"))
    assert bad[5, 1, 10] and bad[5, 1, 42] and bad.sum() == 2
    bad = torch.isnan(rp.norm_rope(x, table, norm="head"))
    assert bad[5, 1].all() and bad.sum() == 64


def test_zero_rows_and_empty(rp, cuda):
    table = rp.rope_table(torch.arange(4, device=cuda)[:, None], (64,))
    x = torch.zeros(4, 2, 64, dtype=BF16, device=cuda)
    assert not rp.norm_rope(x, table, norm="head").any() and not rp.norm_rope(x, table, norm="row").any()
    none = torch.zeros(0, 1, dtype=torch.int64, device=cuda)
    table = rp.rope_table(none, (64,))
    assert table.shape == (0, 32, 2)
    assert rp.norm_rope(x[:0], table).shape == (0, 2, 64)
