"""Masked attention on the GPU against float64 (oracle/attention_oracle.py). In blocks of 128 queries with keys and values that no
cache holds and that differ from call to call: what a workgroup copies then comes late, and what lies in LDS from another call is
not the same. Far scales."""

import importlib

import pytest
import torch

from attention_util import BF16, F16, F32, attention_args, check, d, plan_of, qkv
from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def at(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.attention")


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


@pytest.fixture(scope="module")
def caches_are_emptied(cuda):
    """A call that writes 1 GiB, four times what the last cache before the memory holds."""
    space = torch.empty(1 << 30, dtype=torch.uint8, device=cuda)
    yield lambda n: space.fill_(n)


def mask_of(kind, g, B, Sq, Sk, dtype):
    """Shared by all heads; the last query sees nothing where each has values of its own."""
    if kind == "keys":
        return (torch.rand(B, 1, 1, Sk, generator=g) < 0.7).cuda()
    keep = torch.rand(B, 1, Sq, Sk, generator=g) < 0.7
    keep[:, :, -1] = False
    if kind == "bool":
        return keep.cuda()
    m = torch.randn(B, 1, Sq, Sk, generator=g) * 2.0
    return torch.where(keep, m, float("-inf")).to(dtype if kind == "half" else F32).cuda()


def run(at, lib, empty, B, Sq, Sk, H, Hk, D, kind, dtype, seed):
    """Against float64 for the heads of the first and the last key head."""
    code = {"keys": 4, "bool": 4, "half": 0 if dtype == F16 else 1, "fp32": 2}[kind]
    args = attention_args(B, Sq, Sk, H, Hk, D, mask=4096, mask_dtype=code, mask_query_stride=Sk, dtype=0 if dtype == F16 else 1)
    assert plan_of(lib, args)[0] == 0
    g = torch.Generator().manual_seed(seed)
    q, k, v = qkv(g, B, Sq, Sk, H, Hk, D, dtype)
    mask = mask_of(kind, g, B, Sq, Sk, dtype)
    for causal in (False, True):
        empty(seed % 251)
        o = at.attention(q, k, v, mask=mask, causal=causal)
        for shared in {0, Hk - 1}:
            heads = slice(shared * H // Hk, (shared + 1) * H // Hk)
            some = (t[:, :, h] for t, h in ((q, heads), (k, slice(shared, shared + 1)), (v, slice(shared, shared + 1))))
            want = A.attention(*map(d, some), causal, None, None, d(mask))
            check(o[:, :, heads], *want, Sk, f"{Sk} keys, causal {causal}, key head {shared}", 8.0)


@pytest.mark.parametrize("kind", ["keys", "bool", "half", "fp32"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_new_keys_every_call(at, lib, caches_are_emptied, D, kind):
    """One unit of 32 keys to several, odd and even, the last one full or not; the last block's rows end inside it."""
    for i, Sk in enumerate((77, 1, 33, 96, 64, 300, 130)):
        run(at, lib, caches_are_emptied, 2, 2100, Sk, 24, 24, D, kind, BF16 if i % 2 else F16, 100 * D + i)


@pytest.mark.parametrize("kind", ["half", "fp32"])
@pytest.mark.parametrize("D", [72, 88, 128, 136, 256])
def test_added_masks_of_many_keys(at, lib, caches_are_emptied, D, kind):
    run(at, lib, caches_are_emptied, 2, 2900, 1300, 24, 8, D, kind, BF16, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [3, 1500])
def test_far_scales(at, cuda, Sq, D):
    """Scales up to the largest, with queries as small, and one that is a subnormal number, beside keys that are masked or behind
    a query's own."""
    g = torch.Generator().manual_seed(D + Sq)
    q, k, v = qkv(g, 2, Sq, 300, 8, 8, D, BF16)
    keep = (torch.rand(2, 1, 1, 300, generator=g) < 0.7).cuda()
    for t, scale in ((q * 2.0 ** -100, 2.0 ** 100), (q * 2.0 ** -115, 2.0 ** 127), (q, 1e-44)):
        for causal in (False, True):
            o = at.attention(t, k, v, mask=keep, causal=causal, scale=scale)
            check(o, *A.attention(d(t), d(k), d(v), causal, scale, None, d(keep)), 300, f"{scale} {causal}")
