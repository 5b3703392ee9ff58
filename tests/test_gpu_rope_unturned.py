"""Values of a head behind those that turn, on the GPU: they stay as they are, whatever they and their neighbours hold."""

import importlib

import pytest
import torch

from attention_util import BF16, F16, F32, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rp(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.rope")


# heads and turned values: whole groups of eight, a part of one, groups of four, pairs of two halves that lie in one group
SIZES = [(96, 64), (96, 36), (80, 20), (128, 120), (40, 2), (256, 130), (16, 8)]


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,turned", SIZES)
def test_they_stay(rp, cuda, D, turned, dtype, pairs):
    g = torch.Generator().manual_seed(D + turned)
    inf, nan = float("inf"), float("nan")
    for tokens, heads in ((7, 3), (300, 21)):  # a pass of heads a wave, and two
        table = rp.rope_table(torch.arange(5, 5 + tokens, device=cuda)[:, None], (turned,))
        x = normal(g, tokens, heads, D, dtype=dtype)
        rest = x[..., turned:]
        want = rp.norm_rope(x, table, pairs=pairs)[..., :turned].clone()
        for at, value in ((0, inf), (1, nan), (2, -inf), (5, -0.0)):
            rest[:, at % heads, at] = value
        rest[3, 1, -1], rest[4, 1] = inf, nan
        got = rp.norm_rope(x, table, pairs=pairs)
        assert torch.equal(got[..., :turned], want)
        assert torch.equal(torch.isnan(got[..., turned:]), torch.isnan(rest))
        bits = torch.int32 if dtype == F32 else torch.int16
        seen = ~torch.isnan(rest)
        assert torch.equal(got[..., turned:].contiguous().view(bits)[seen], rest.contiguous().view(bits)[seen])
