"""Block norms of more rows than one grid holds threads for."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def nm(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.norm")


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


def test_narrow_rows(nm, cuda):
    """More than 2^26 rows of 8 columns in three samples, whose ends are no launch's: the bits of the same rows in pieces."""
    B, S, D = 3, 2 ** 26 // 3 + 7, 8
    assert B * S > 2 ** 26
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(B, S, D, generator=g, device=cuda, dtype=BF16)
    gate, scale = (torch.randn(B, 1, D, generator=g, device=cuda, dtype=BF16) for _ in range(2))
    got = nm.gated_residual_norm(x, x, gate, scale=scale, kind="layer")
    piece = 2 ** 20 - 3
    for b in range(B):
        for at in range(0, S, piece):
            part = x[b, at:at + piece]
            want = nm.gated_residual_norm(part, part, gate[b, 0], scale=scale[b, 0], kind="layer")
            for t, w in zip(got, want):
                assert torch.equal(t[b, at:at + piece], w), (b, at)


def test_wide_rows_to_four_bits(nm, mx, cuda):
    """Rows of several waves, the packed result's rows behind the first launch's."""
    rows, D, first = 2 ** 21 + 75, 520, 2 ** 21 - 64
    x = torch.randn(rows, D, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda, dtype=BF16)
    q = nm.modulated_norm(x, out_dtype="mxfp4")
    got = mx.dequantize_mxfp4(q, BF16)[first:]
    want = mx.dequantize_mxfp4(nm.modulated_norm(x[first:], out_dtype="mxfp4"), BF16)
    assert torch.equal(got, want)
    assert torch.equal(nm.modulated_norm(x)[first:], nm.modulated_norm(x[first:]))
