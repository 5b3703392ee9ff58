"""CPU tests of which kernels of the MXFP4 operators and the block norms the library holds, and which of them calls reach.
No kernel runs."""

import ctypes
import importlib
import random
import re

import pytest

from conftest import REPO
from mxfp4_shapes import PLANS

LIB = REPO / "comfyui-featherops_amd" / "lib" / "libfeatherops_amd.so"


def test_norm_kernels_are_reached(pkg):
    """Two vectors a thread are for rows of more than 512 vectors, which no single wave holds."""
    names = set(re.findall(rb"norm_kernelILi(\d)ELi(\d)ELb([01])ELi(\d)ELb([01])ELb([01])ELb([01])E", LIB.read_bytes()))
    assert len(names) >= 50
    for x, y, mods, vectors, one_wave, codes, tiny in names:
        assert not (vectors == b"2" and (one_wave == b"1" or tiny == b"1"))
        assert not (tiny == b"1" and one_wave == b"0")


@pytest.fixture(scope="module")
def plan(pkg):
    lib = importlib.import_module("featherops_amd.kernel.hip._lib").lib()

    def query(M, N, K):
        out = (ctypes.c_int64 * 8)(*[-1] * 8)
        assert lib.feather_mxfp4_mm_plan(M, N, K, out) == 0
        return tuple(out)

    query.lib = lib
    return query


def test_product_shapes_take_their_kernels(plan):
    """The GPU tests' shapes run the kernels that they stand for: one that the plan has moved needs a new shape."""
    assert {shape: plan(*shape) for shape in PLANS} == PLANS


def test_every_product_kernel_has_a_shape(plan):
    """All tiles, alone and behind a seam of columns and of rows, with and without a K split where the plan takes one."""
    few = {(p[0], p[1], p[2] > 1) for s, p in PLANS.items() if s[0] <= 32}
    assert few == {(m, n, False) for m in (16, 32) for n in (16, 32, 64)} | {(16, 16, True), (32, 16, True)}
    tiles = [(64, 64), (64, 128), (128, 128), (128, 256)]
    kinds = {(p[:2], p[2] > 1, p[3:5], p[5] > 1, p[6] > 0, p[7] > 0) for s, p in PLANS.items() if s[0] > 32}
    want = {(t, split, (0, 0), False, False, False) for t in tiles for split in (False, True)}
    want |= {((256, 256), split, (0, 0), False, False, False) for split in (False, True)}
    want |= {((256, 256), False, t, split, rows, not rows) for t in tiles for split in (False, True) for rows in (False, True)}
    want |= {((256, 256), False, (256, 256), True, rows, not rows) for rows in (False, True)}
    assert kinds == want
    rng = random.Random(0)
    for _ in range(20000):  # no other kind comes up
        M, N, K = (int(2 ** rng.uniform(0, hi)) for hi in (14, 14, 15))
        p = plan(M, N, K)
        if M <= 32:
            assert (p[0], p[1], p[2] > 1) in few and p[3:] == (0,) * 5, (M, N, K, p)
        else:
            assert (p[:2], p[2] > 1, p[3:5], p[5] > 1, p[6] > 0, p[7] > 0) in want, (M, N, K, p)


def test_split_counters_and_workspace(plan):
    """A split's arrival counters, one for each tile of the launch, fit the workspace's first 64 KB, and the rest of it
    holds one fp32 tile for each workgroup."""
    rng = random.Random(1)
    shapes = [tuple(int(2 ** rng.uniform(0, hi)) for hi in (15, 15, 15)) for _ in range(5000)] + list(PLANS)
    split = 0
    for M, N, K in shapes:
        p = plan(M, N, K)
        need = 0
        for bm, bn, ks, m0, n0 in ((*p[:3], 0, 0), (*p[3:6], *p[6:])):
            if ks > 1:
                tiles = -(-(M - m0) // bm) * -(-(N - n0) // bn)
                assert 4 * tiles <= 65536, (M, N, K, p)
                need, split = max(need, 65536 + tiles * ks * bm * bn * 4), split + 1
        assert plan.lib.feather_mxfp4_mm_workspace_size(M, N, K, 3) == need, (M, N, K, p)
    assert split > 100


def test_plan_refuses(plan):
    out = (ctypes.c_int64 * 8)()
    for sizes in ((-1, 4, 4), (4, 0, 4), (4, 4, 0), (4, 4, 1 << 24)):
        assert plan.lib.feather_mxfp4_mm_plan(*sizes, out) == 1
    assert plan.lib.feather_mxfp4_mm_plan(4, 4, 4, None) == 1
    assert plan(0, 4, 4) == (0,) * 8
