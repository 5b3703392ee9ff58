"""The MXFP4 product on every kernel that the plan takes: each tile, strip and K split, and results of two launches on
either side of the seam (mxfp4_shapes.py). The operands are numbers that 4 bits hold under block scales of 1, 2 and 4, so
every sum is a whole number below 2^24, exact in fp32 in any order, and a wrong scale, row, column, step or seam shows."""

import ctypes
import importlib

import pytest
import torch

from mxfp4_shapes import PLANS

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


def whole(rows, cols, g, cuda):
    """-3 to 3, each block of 32 with a 4 or -4, times 1, 2 or 4: at most 16, quantised without an error."""
    blocks = -(-cols // 32)
    v = torch.randint(-3, 4, (rows, blocks, 32), generator=g, device=cuda, dtype=torch.int32)
    v[:, :, 0] = 8 * torch.randint(0, 2, (rows, blocks), generator=g, device=cuda, dtype=torch.int32) - 4
    v <<= torch.randint(0, 3, (rows, blocks, 1), generator=g, device=cuda, dtype=torch.int32)
    return v.view(rows, -1)[:, :cols]


def check(got, want, label):
    """want: float64 whole numbers, rounded once to got's type."""
    want = want.to(got.dtype)
    if not torch.equal(got, want):
        wrong = (got != want).nonzero()
        raise AssertionError(f"{label}: {len(wrong)} of {got.numel()} wrong, from {wrong[0].tolist()} to {wrong[-1].tolist()}")


@pytest.mark.parametrize("shape", list(PLANS), ids=lambda s: "x".join(map(str, s)))
def test_exact(mx, lib, cuda, shape):
    M, N, K = shape
    plan = (ctypes.c_int64 * 8)()
    assert lib.feather_mxfp4_mm_plan(M, N, K, plan) == 0 and tuple(plan) == PLANS[shape]
    assert K * 16 * 16 < 2 ** 24
    g = torch.Generator(device=cuda).manual_seed(M + N + K)
    x, w = whole(M, K, g, cuda), whole(N, K, g, cuda)
    bias = torch.randint(-8, 9, (N,), generator=g, device=cuda)
    sums = x.double() @ w.double().t()
    q = mx.quantize_mxfp4(w.to(BF16))
    for dtype in (F16, BF16):
        a = x.to(dtype)
        check(mx.mxfp4_mm(a, q, bias.to(dtype)), sums + bias, f"{shape} {dtype}")
        packed = mx.quantize_mxfp4(a)
        check(mx.mxfp4_mm(packed, q, None, dtype), sums, f"{shape} packed, {dtype}")
    check(mx.mxfp4_mm(x.to(BF16), q, bias.to(F16), F16), sums + bias, f"{shape} bf16 in, fp16 out")


@pytest.mark.parametrize("shape", [(1, 521, 8200), (27, 301, 6003), (622, 993, 12643), (4377, 197, 10255), (2699, 641, 10310),
                                   (1683, 2543, 19510), (3308, 5238, 11662), (4758, 3534, 9205)],
                         ids=lambda s: "x".join(map(str, s)))
def test_splits_repeat_and_replay(mx, cuda, shape):
    """A K split's workspace is left ready: the same bits call after call, with other splits in between, and in a graph
    replayed among eager calls on changed operands."""
    M, N, K = shape
    g = torch.Generator(device=cuda).manual_seed(K)
    x = torch.randn(M, K, generator=g, device=cuda, dtype=BF16)
    q = mx.quantize_mxfp4(torch.randn(N, K, generator=g, device=cuda, dtype=BF16))
    other, q_other = x[:40, :7000], mx.quantize_mxfp4(torch.randn(200, min(K, 7000), generator=g, device=cuda, dtype=BF16))
    first = mx.mxfp4_mm(x, q)
    for _ in range(4):
        mx.mxfp4_mm(other, q_other)
        assert torch.equal(mx.mxfp4_mm(x, q), first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx.mxfp4_mm(x, q)
    for i in range(3):
        x.neg_() if i % 2 else x.mul_(2)
        graph.replay()
        want = mx.mxfp4_mm(x, q)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
