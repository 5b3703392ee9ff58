"""MXFP4 and the block norms where offsets pass 32 bits, where a result is composed of parts, and without scratch."""

import ctypes
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


@pytest.fixture(scope="module")
def nm(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.norm")


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


def some(rows, cols, dtype, cuda, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, cols, generator=g).to(dtype).to(cuda)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [3, 20, 40])
def test_rows_far_apart(mx, nm, cuda, rows, dtype):
    """Rows whose offsets pass 2^32 bytes and 2^31 elements: the same bits as rows next to each other."""
    stride = (2 ** 32 // (rows - 1)) // 8 * 8 + 24
    store = torch.empty((rows - 1) * stride + 520, dtype=dtype, device=cuda)
    far = store.as_strided((rows, 520), (stride, 1))
    near = some(rows, 520, dtype, cuda, rows)
    far.copy_(near)
    # (in the row-major form: what the packed one holds beyond its rows is not specified)
    got, want = (mx.unprepack_mxfp4(mx.quantize_mxfp4(t)) for t in (far, near))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    y, want = nm.gated_residual_norm(far, far, kind="layer"), nm.gated_residual_norm(near, near, kind="layer")
    assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])
    if dtype == BF16:
        w = mx.quantize_mxfp4(some(48, 520, dtype, cuda))
        assert torch.equal(mx.mxfp4_mm(far, w), mx.mxfp4_mm(near, w))


def test_many_rows(mx, nm, cuda):
    """More than 2^31 elements: the last rows equal the same rows on their own."""
    rows, cols = 64 * 1093 + 81, 32768
    x = torch.empty(rows, cols, dtype=BF16, device=cuda)
    tail = some(81, cols, BF16, cuda)  # from a multiple of 64 rows on
    first = rows - 81
    assert first % 64 == 0
    x[first:] = tail
    x[:64] = tail[:64]
    q, alone = mx.quantize_mxfp4(x), mx.quantize_mxfp4(tail)
    groups = alone.codes.shape[0]
    assert torch.equal(q.codes[-groups], alone.codes[0]) and torch.equal(q.scales[-groups], alone.scales[0])
    assert torch.equal(q.codes[0], alone.codes[0])
    back = mx.dequantize_mxfp4(q, BF16)
    assert torch.equal(back[first:], mx.dequantize_mxfp4(alone, BF16))
    del back, q
    flat = x.view(-1, cols // 2)  # 16384 columns
    y = nm.modulated_norm(flat, kind="rms")
    assert torch.equal(y[2 * first:], nm.modulated_norm(tail.view(-1, cols // 2), kind="rms"))


def test_large_result(mx, cuda):
    """A result of more than 2^31 elements: its corners equal those of the product of their rows and columns."""
    M, N, K = 70001, 32768, 64
    a, b = some(M, K, BF16, cuda, 1), some(N, K, BF16, cuda, 2)
    w = mx.quantize_mxfp4(b)
    y = mx.mxfp4_mm(a, w)
    for rows in (slice(0, 40), slice(M - 40, M)):
        for cols in (slice(0, 200), slice(N - 200, N)):
            assert torch.equal(y[rows, cols], mx.mxfp4_mm(a[rows], mx.quantize_mxfp4(b[cols])))


@pytest.mark.parametrize("M,N", [(4096, 5120), (5120, 4096), (4100, 4610), (8200, 2304), (6000, 5000)])
def test_result_of_two_launches(mx, lib, cuda, M, N):
    """Results whose last round of large tiles would leave the chip idle are composed of two launches. The
    operands are whole numbers that 4 bits hold, so every element is exact and any seam shows."""
    K = 640
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-2, 3, (M, K), generator=g).to(BF16).to(cuda)
    w = torch.randint(-2, 3, (N, K), generator=g).to(BF16).to(cuda)
    bias = torch.randint(-8, 9, (N,), generator=g).to(BF16).to(cuda)
    x[:, ::32], w[:, ::32] = 4, 4  # every block's scale 1
    y = mx.mxfp4_mm(x, mx.quantize_mxfp4(w), bias)
    want = (x.float() @ w.float().t() + bias.float()).to(BF16)  # whole numbers below 2^24: exact
    assert torch.equal(y, want)


@pytest.mark.parametrize("M,N,K", [(1, 512, 8192), (40, 200, 7000), (130, 260, 4200)])
def test_without_scratch(mx, lib, cuda, M, N, K):
    """Packed operands and no workspace: K is not split, the sums differ by their order alone."""
    x, b = some(M, K, BF16, cuda, 3), some(N, K, BF16, cuda, 4)
    qa, qb = mx.quantize_mxfp4(x), mx.quantize_mxfp4(b)
    split = mx.mxfp4_mm(qa, qb, None, BF16)
    out = torch.empty(M, N, dtype=BF16, device=cuda)
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    st = lib.feather_mxfp4_mm(p(qa.codes), p(qa.scales), 3, 0, p(qb.codes), p(qb.scales), None, p(out), M, N, K, 1, None, 0,
                              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert st == 0
    # on either side one rounding to bf16 (2^-8) and K fp32 additions
    sums = mx.dequantize_mxfp4(qa, F32).abs().double() @ mx.dequantize_mxfp4(qb, F32).abs().double().t()
    bound = 2.0 ** -7 * split.double().abs() + 2 * K * 2.0 ** -24 * sums
    assert ((out.double() - split.double()).abs() <= bound).all()


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("D", [1, 3, 7, 31, 127, 161])
def test_narrow_quantised_norm(mx, nm, cuda, rows, D):
    x = some(rows, D, F32, cuda, D)
    scale, shift = some(1, D, F32, cuda, 1), some(1, D, F32, cuda, 2)
    for kind in ("rms", "layer"):
        q = nm.modulated_norm(x, scale=scale, shift=shift, kind=kind, eps=1e-2, out_dtype="mxfp4")
        want = mx.quantize_mxfp4(nm.modulated_norm(x, scale=scale, shift=shift, kind=kind, eps=1e-2))
        got, want = mx.unprepack_mxfp4(q), mx.unprepack_mxfp4(want)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w = mx.quantize_mxfp4(some(40, D, BF16, cuda, 3))
    assert mx.mxfp4_mm(q, w, None, BF16).shape == (rows, 40)
