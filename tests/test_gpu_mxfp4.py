"""MXFP4 on the GPU: quantisation and layouts bit for bit against the definition in 64 bits, the product against
64-bit sums of the operands' values."""

import importlib

import numpy as np
import pytest
import torch

from oracle import block_oracle as B

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


def mixed(rows, cols, dtype, seed=0):
    """Values whose magnitudes differ from block to block by many binades, with zeros, rows of zeros and values on
    the midpoints between codes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    lo, hi = {torch.float16: (-18, 12), torch.bfloat16: (-120, 120), torch.float32: (-130, 120)}[dtype]
    blocks = -(-cols // 32)
    e = torch.randint(lo, hi, (rows, blocks), generator=g).repeat_interleave(32, 1)[:, :cols]
    on_grid = torch.randint(-24, 25, (rows, cols), generator=g) * 0.25
    x = torch.where(torch.rand(rows, cols, generator=g) < 0.3, on_grid, x)
    x = torch.ldexp(x.double(), e).to(dtype)
    x[torch.rand(rows, cols, generator=g) < 0.05] = 0
    if rows > 2:
        x[rows // 2] = 0
    return x


def row_major(mx, q):
    codes, scales = mx.unprepack_mxfp4(q)
    return codes.cpu().numpy(), scales.cpu().numpy()


def check_codes(mx, q, x, cols):
    codes, scales = row_major(mx, q)
    want, want_scales = B.mxfp4_quantize(x.double().reshape(-1, cols).cpu().numpy())
    np.testing.assert_array_equal(scales, want_scales)
    live = np.repeat(want_scales != 255, 16, axis=1)  # a NaN block's codes stand for nothing
    np.testing.assert_array_equal(codes[live], want[live])
    return want, want_scales


SHAPES = [(1, 1), (1, 31), (3, 33), (16, 128), (17, 129), (64, 256), (65, 160), (130, 1000), (1, 8197), (2, 5120)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_and_back(mx, cuda, rows, cols, dtype):
    x = mixed(rows, cols, dtype, seed=rows + cols)
    q = mx.quantize_mxfp4(x.to(cuda))
    codes, scales = check_codes(mx, q, x, cols)
    back = mx.dequantize_mxfp4(q, dtype)
    want = torch.from_numpy(B.mxfp4_values(codes, scales, cols)).to(dtype)
    assert back.dtype == dtype and torch.equal(back.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_16_bit_value(mx, cuda, dtype):
    """Each bit pattern as a whole block, and as one value under each larger power of two of its block."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    finite = bits[torch.isfinite(bits)]
    x = finite[:, None].expand(-1, 32).contiguous()
    check_codes(mx, mx.quantize_mxfp4(x.to(cuda)), x, 32)
    for over in (0, 1, 2, 3, 4, 6):
        _, e = torch.frexp(finite.double())
        big = torch.ldexp(torch.full_like(finite, 1.5, dtype=torch.float64), e + over - 1).to(dtype)
        big = torch.where(torch.isfinite(big), big, finite)
        x = torch.zeros(finite.numel(), 32, dtype=dtype)
        x[:, 0], x[:, 13], x[:, 31] = big, finite, -finite
        check_codes(mx, mx.quantize_mxfp4(x.to(cuda)), x, 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_blocks(mx, cuda, dtype):
    x = mixed(20, 160, dtype, seed=5)
    x[3, 40], x[7, 159], x[8, 0], x[19, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    q = mx.quantize_mxfp4(x.to(cuda))
    codes, scales = check_codes(mx, q, x, 160)
    assert (scales == 255).sum() == 4
    back = mx.dequantize_mxfp4(q, dtype).cpu()
    want = torch.from_numpy(B.mxfp4_values(codes, scales, 160)).to(dtype)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(back.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_views(mx, cuda, dtype):
    """Rows with a stride, rows that start off any vector's alignment, more dimensions, a transposed tensor."""
    base = mixed(40, 333, dtype, seed=7).to(cuda)
    for view in (base[:, :200], base[1::3, 5:5 + 165], base[:, 1:], base.t(), base[:24].view(4, 6, 333)[:, :3, 7:]):
        q = mx.quantize_mxfp4(view)
        assert q.shape == tuple(view.shape)
        check_codes(mx, q, view, view.shape[-1])
        back = mx.dequantize_mxfp4(q, torch.float32)
        assert back.shape == view.shape
        assert torch.equal(back, mx.dequantize_mxfp4(mx.quantize_mxfp4(view.contiguous()), torch.float32))


@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 100), (64, 128), (200, 4096), (129, 1056)])
def test_prepack_layout_and_back(mx, cuda, rows, cols):
    rng = np.random.default_rng(rows)
    blocks = -(-cols // 32)
    codes = rng.integers(0, 256, (rows, blocks * 16), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, blocks), dtype=np.uint8)
    q = mx.prepack_mxfp4(torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda), cols)
    got, got_scales = row_major(mx, q)
    np.testing.assert_array_equal(got, codes)
    np.testing.assert_array_equal(got_scales, scales)
    # the documented place of every block
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    packed, packed_scales = q.codes.cpu().numpy(), q.scales.cpu().numpy()
    lane = 16 * (b % 4) + r % 16
    np.testing.assert_array_equal(packed[r // 64, b // 4, r // 16 % 4, lane], codes.reshape(rows, blocks, 16))
    np.testing.assert_array_equal(packed_scales[r // 64, b // 4, lane, r // 16 % 4], scales)
    # steps are padded with zero codes
    assert not packed[:, blocks // 4:, :, 16 * (blocks % 4):].any() or blocks % 4 == 0


def operands(mx, cuda, M, N, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * (1 + 7 * (torch.rand(K, generator=g) < 0.02))).to(dtype)
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype)
    bias = (torch.randn(N, generator=g) * 0.1).to(dtype)
    return x.to(cuda), mx.quantize_mxfp4(w.to(cuda)), w, bias.to(cuda)


def check_product(y, x, w, bias, label):
    """y against 64-bit sums of the quantised operands: half an ulp of the output type for the one rounding, and
    8 sqrt(K) 2^-24 of the sum of magnitudes for the fp32 sums (a probabilistic bound on their rounding errors,
    with room for another order of the sums)."""
    qa = B.mxfp4_values(*B.mxfp4_quantize(x.double().cpu().numpy()), x.shape[1])
    qw = B.mxfp4_values(*B.mxfp4_quantize(w.double().cpu().numpy()), w.shape[1])
    want = qa @ qw.T
    mags = np.abs(qa) @ np.abs(qw).T
    if bias is not None:
        want = want + bias.double().cpu().numpy()
        mags = mags + np.abs(bias.double().cpu().numpy())
    half = 2.0 ** -11 if y.dtype == torch.float16 else 2.0 ** -8
    got = y.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{label}: NaN pattern"
    fine = ~np.isnan(want)
    tol = half * np.abs(want) + 8 * x.shape[1] ** 0.5 * 2.0 ** -24 * mags + 2.0 ** -24
    worst = (np.abs(got - want) / tol)[fine].max() if fine.any() else 0.0
    assert worst <= 1.0, f"{label}: {worst:.3g} times the bound"


MM_SHAPES = [(1, 1, 1), (1, 16, 128), (1, 1000, 513), (2, 65, 4100), (3, 17, 31), (15, 250, 1024), (16, 256, 96),
             (16, 48, 8192), (17, 64, 128), (33, 100, 129), (48, 3, 640), (64, 64, 1000), (65, 65, 65), (100, 1000, 260),
             (128, 256, 512), (257, 130, 2100), (300, 515, 333), (1, 5120, 640), (40, 2048, 1152)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", MM_SHAPES)
def test_product(mx, cuda, M, N, K, dtype):
    x, q, w, bias = operands(mx, cuda, M, N, K, dtype, M + N + K)
    y = mx.mxfp4_mm(x, q, bias)
    assert y.shape == (M, N) and y.dtype == dtype
    check_product(y, x, w, bias, f"{M} {N} {K}")
    # activations quantised beforehand: the same sums
    assert torch.equal(mx.mxfp4_mm(mx.quantize_mxfp4(x), q, bias, dtype), y)
    plain = mx.mxfp4_mm(x, q)
    check_product(plain, x, w, None, f"{M} {N} {K} without a bias")


@pytest.mark.parametrize("M,N,K", [(512, 4096, 256), (2048, 2048, 384), (4096, 4160, 200), (1025, 4097, 1030)])
def test_product_large_tiles(mx, cuda, M, N, K):
    x, q, w, bias = operands(mx, cuda, M, N, K, torch.bfloat16, K)
    check_product(mx.mxfp4_mm(x, q, bias), x, w, bias, f"{M} {N} {K}")


@pytest.mark.parametrize("M", [4, 80])
def test_product_other_types_and_views(mx, cuda, M):
    x, q, w, bias = operands(mx, cuda, M, 200, 320, torch.float16, 3)
    y = mx.mxfp4_mm(x, q, bias.to(torch.bfloat16), torch.bfloat16)
    assert y.dtype == torch.bfloat16
    check_product(y, x, w, bias.to(torch.bfloat16), "fp16 activations, bf16 result")
    wide = torch.zeros(M, 333, dtype=torch.float16, device=cuda)
    wide[:, 5:325] = x
    assert torch.equal(mx.mxfp4_mm(wide[:, 5:325], q, bias), mx.mxfp4_mm(x, q, bias))
    y3 = mx.mxfp4_mm(x.view(2, M // 2, 320), q, bias)
    assert y3.shape == (2, M // 2, 200) and torch.equal(y3.view(M, 200), mx.mxfp4_mm(x, q, bias))
    assert mx.mxfp4_mm(x[:0], q, bias).shape == (0, 200)
    q0 = mx.quantize_mxfp4(x[:0])
    assert mx.mxfp4_mm(q0, q, bias, torch.float16).shape == (0, 200)


@pytest.mark.parametrize("M", [5, 70])
def test_product_keeps_rows_apart(mx, cuda, M):
    """NaN and infinite activations reach their own row's results alone, a NaN weight its own column's; what lies in
    the packed operand beyond its rows reaches none."""
    x, q, w, bias = operands(mx, cuda, M, 90, 260, torch.bfloat16, 11)
    x[1, 3], x[M - 1, 200] = float("nan"), float("inf")
    w[7, 100] = float("nan")
    q = mx.quantize_mxfp4(w.to(cuda))
    y = mx.mxfp4_mm(x, q, bias)
    check_product(y, x, w, bias, "non-finite")
    a = mx.quantize_mxfp4(x)
    codes = a.codes.view(*a.codes.shape[:3], 4, 16, 16)
    codes[-1, :, M % 64 // 16, :, M % 16:] = 0xFF
    codes[-1, :, M % 64 // 16 + 1:] = 0xFF
    a.scales.view(-1, a.scales.shape[1], 4, 16, 4)[-1, :, :, M % 16:, M % 64 // 16] = 0xFF
    if M % 64 // 16 < 3:
        a.scales.view(-1, a.scales.shape[1], 4, 16, 4)[-1, :, :, :, M % 64 // 16 + 1:] = 0xFF
    y2 = mx.mxfp4_mm(a, q, bias, torch.bfloat16)
    assert torch.equal(y2.isnan(), y.isnan()) and torch.equal(y2.nan_to_num(0.0), y.nan_to_num(0.0))


@pytest.mark.parametrize("M,N,K", [(1, 512, 8192), (16, 300, 6000), (40, 200, 7000), (130, 260, 4200)])
def test_product_split_over_k(mx, cuda, M, N, K):
    """Shapes whose K is split over workgroups: the same bits each time, eagerly, on another stream and in a graph
    replayed between other work."""
    x, q, w, bias = operands(mx, cuda, M, N, K, torch.bfloat16, 2)
    lib = importlib.import_module("featherops_amd.kernel.hip._lib").lib()
    assert lib.feather_mxfp4_mm_workspace_size(M, N, K, 3) > 0
    y = mx.mxfp4_mm(x, q, bias)
    check_product(y, x, w, bias, f"{M} {N} {K}")
    for _ in range(3):
        assert torch.equal(mx.mxfp4_mm(x, q, bias), y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = mx.mxfp4_mm(x, q, bias)
    side.synchronize()
    assert torch.equal(z, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx.mxfp4_mm(x, q, bias)
    for i in range(4):
        x.copy_(x.flip(0))
        graph.replay()
        want = mx.mxfp4_mm(x, q, bias)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_operands_from_another_stream(mx, cuda):
    """A chain on a stream that is not the default one."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = torch.randn(200, 640, device=cuda).to(torch.bfloat16)
        w = torch.randn(130, 640, device=cuda).to(torch.bfloat16)
        y = mx.mxfp4_mm(x, mx.quantize_mxfp4(w))
    side.synchronize()
    check_product(y, x, w.cpu(), None, "side stream")


def test_refusals(mx, cuda):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    w = mx.quantize_mxfp4(torch.zeros(8, 64, dtype=torch.bfloat16, device=cuda))
    for call, message in [
        (lambda: mx.quantize_mxfp4(x.double()), "float16, bfloat16 or float32"),
        (lambda: mx.quantize_mxfp4(x[:, :0]), "at least one column"),
        (lambda: mx.dequantize_mxfp4(w, torch.float64), "float16, bfloat16 or float32"),
        (lambda: mx.dequantize_mxfp4(w._replace(shape=(80, 64))), "packed for"),
        (lambda: mx.mxfp4_mm(x.float(), w), "float16 or bfloat16"),
        (lambda: mx.mxfp4_mm(x[:, :32], w), "b's 64 columns"),
        (lambda: mx.mxfp4_mm(mx.quantize_mxfp4(x[:, :32]), w), "columns"),
        (lambda: mx.mxfp4_mm(x, w, torch.zeros(8, device=cuda)), "output's dtype"),
        (lambda: mx.mxfp4_mm(x, w, torch.zeros(9, dtype=x.dtype, device=cuda)), "N (8) elements"),
        (lambda: mx.mxfp4_mm(x, w, None, torch.float32), "out_dtype"),
        (lambda: mx.mxfp4_mm(x, w._replace(data=w.data.cpu())), "device"),
        (lambda: mx.mxfp4_mm(x, w._replace(data=w.data.repeat_interleave(2)[::2])), "contiguous"),
        (lambda: mx.mxfp4_mm(x, w._replace(data=w.data[:-1])), "packed for"),
        (lambda: mx.mxfp4_mm(x, w._replace(data=torch.cat((w.data[:8], w.data))[8:])), "aligned"),
        (lambda: mx.prepack_mxfp4(w.codes.view(-1, 16)[:8], w.scales.view(-1, 1)[:9]), "rows"),
        (lambda: mx.prepack_mxfp4(torch.zeros(8, 32, dtype=torch.uint8, device=cuda),
                                  torch.zeros(8, 2, dtype=torch.uint8, device=cuda), 65), "for 65 columns"),
    ]:
        with pytest.raises(RuntimeError, match=message.replace("(", r"\(").replace(")", r"\)")):
            call()
