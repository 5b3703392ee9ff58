"""CPU tests of the MXFP4 operators and the block norms: the C entries refuse what no kernel takes before anything is
launched, fake tensors have the results' shapes, CPU tensors raise, and the 64-bit oracle is what the format's
definition says. No kernel runs."""

import ctypes
import importlib

import numpy as np
import pytest
import torch

from oracle import block_oracle as B


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


@pytest.fixture(scope="module")
def nm(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.norm")


class NormArgs(ctypes.Structure):
    """feather_block_norm_args of include/featherops_amd.h."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "h", "gate", "post_weight", "weight", "bias", "scale", "shift",
                                                "x_out", "y", "codes", "scales")]
                + [(n, ctypes.c_int64) for n in ("rows", "cols", "x_row_stride", "h_row_stride", "gate_group",
                                                 "gate_row_stride", "mod_group", "scale_row_stride", "shift_row_stride")]
                + [(n, ctypes.c_int) for n in ("x_dtype", "y_dtype", "mod_dtype", "norm")]
                + [("eps", ctypes.c_float), ("residual_scale", ctypes.c_float)])


def test_c_entries_refuse_without_launching(lib):
    P = 4096  # stands for a pointer: every call below ends at a check before it is used
    bad = [
        lib.feather_mxfp4_quantize(P, 0, -1, 64, 64, P, P, None), lib.feather_mxfp4_quantize(P, 0, 4, 0, 64, P, P, None),
        lib.feather_mxfp4_quantize(P, 3, 4, 64, 64, P, P, None), lib.feather_mxfp4_quantize(P, 0, 4, 64, -64, P, P, None),
        lib.feather_mxfp4_quantize(None, 0, 4, 64, 64, P, P, None), lib.feather_mxfp4_quantize(P, 0, 4, 64, 64, None, P, None),
        lib.feather_mxfp4_quantize(P, 0, 4, 1 << 24, 64, P, P, None),
        lib.feather_mxfp4_quantize(P, 0, 1 << 30, 1 << 23, 64, P, P, None),
        lib.feather_mxfp4_dequantize(P, P, P, 7, 4, 64, None), lib.feather_mxfp4_dequantize(P, None, P, 0, 4, 64, None),
        lib.feather_mxfp4_prepack(P, P, None, P, 4, 64, None), lib.feather_mxfp4_unprepack(P, P, P, None, 4, 64, None),
        lib.feather_mxfp4_mm(P, P, 2, 64, P, P, None, P, 4, 64, 64, 0, None, 0, None),  # fp32 activations
        lib.feather_mxfp4_mm(P, P, 3, 64, P, P, None, P, 4, 64, 64, 2, None, 0, None),  # fp32 result
        lib.feather_mxfp4_mm(P, None, 3, 64, P, P, None, P, 4, 64, 64, 0, None, 0, None),  # packed without scales
        lib.feather_mxfp4_mm(P, P, 3, 64, P, P, None, P, 4, 0, 64, 0, None, 0, None),
        lib.feather_mxfp4_mm(P, P, 0, -1, P, P, None, P, 4, 64, 64, 0, None, 0, None),
        lib.feather_mxfp4_mm(P, P, 3, 64, P, P, None, None, 4, 64, 64, 0, None, 0, None),
    ]
    assert bad == [1] * len(bad)
    # more 16-bit rows than the product quantises itself
    assert not lib.feather_mxfp4_mm_takes_16bit(4096, 4096, 4096, 4096)
    assert lib.feather_mxfp4_mm_takes_16bit(4, 4096, 4096, 1 << 27) and not lib.feather_mxfp4_mm_takes_16bit(4, 4096, 4096, 1 << 28)
    assert lib.feather_mxfp4_mm(P, None, 1, 4096, P, P, None, P, 4096, 4096, 4096, 1, None, 0, None) == 2
    # nothing to do
    assert lib.feather_mxfp4_quantize(None, 0, 0, 64, 64, None, None, None) == 0
    assert lib.feather_mxfp4_mm(None, None, 3, 0, None, None, None, None, 0, 64, 64, 0, None, 0, None) == 0
    assert lib.feather_mxfp4_codes_bytes(65, 129) == 2 * 4 * 2 * 1024 and lib.feather_mxfp4_scales_bytes(65, 129) == 2 * 2 * 256
    assert lib.feather_mxfp4_codes_bytes(4, 0) == 0


def test_norm_entry_refuses_without_launching(lib):
    P = 4096
    good = dict(x=P, y=P, rows=4, cols=64, x_row_stride=64, x_dtype=1, y_dtype=1, mod_dtype=1, gate_group=1, mod_group=1)
    cases = [dict(rows=-1), dict(cols=0), dict(cols=16385), dict(x_dtype=3), dict(x_dtype=0), dict(mod_dtype=0),
             dict(norm=2), dict(x=None), dict(y=None), dict(h=P), dict(gate=P), dict(post_weight=P), dict(codes=P),
             dict(codes=P, scales=P), dict(y=None, codes=P), dict(h=P, x_out=P, gate=P, gate_group=0),
             dict(scale=P, mod_group=0)]
    for case in cases:
        assert lib.feather_block_norm(ctypes.byref(NormArgs(**{**good, **case})), None) == 1, case
    assert lib.feather_block_norm(None, None) == 1
    assert lib.feather_block_norm(ctypes.byref(NormArgs(**{**good, "rows": 0})), None) == 0


def test_splits_fit_their_counters(lib):
    """Every K split's arrival counters fit the workspace's first 64 KB, and few rows need little scratch."""
    rng = np.random.default_rng(0)
    for _ in range(3000):
        M, N, K = (int(2 ** rng.uniform(0, hi)) for hi in (15, 15, 15))
        ws = lib.feather_mxfp4_mm_workspace_size(M, N, K, 3)
        assert ws == 0 or 65536 < ws <= 65536 + (64 << 20), (M, N, K, ws)


def test_fake_tensors(mx, nm):
    x = torch.empty(3, 5, 200, dtype=torch.bfloat16, device="meta")
    q = mx.quantize_mxfp4(x)
    assert q.codes.shape == (1, 2, 4, 64, 16) and q.scales.shape == (1, 2, 64, 4) and q.shape == (3, 5, 200)
    assert (q.rows, q.cols) == (15, 200)
    assert mx.dequantize_mxfp4(q, torch.float32).shape == (3, 5, 200)
    w = mx.prepack_mxfp4(torch.empty(70, 112, dtype=torch.uint8, device="meta"),
                         torch.empty(70, 7, dtype=torch.uint8, device="meta"), 200)
    assert w.codes.shape == (2, 2, 4, 64, 16) and w.shape == (70, 200)
    assert [t.shape for t in mx.unprepack_mxfp4(w)] == [(70, 112), (70, 7)]
    assert mx.mxfp4_mm(x, w).shape == (3, 5, 70) and mx.mxfp4_mm(q, w).dtype == torch.bfloat16
    s, y = nm.gated_residual_norm(x.float(), x, x[0, 0])
    assert s.dtype == torch.float32 and y.dtype == torch.bfloat16 and y.shape == x.shape
    assert nm.gated_residual_norm(x, x, out_dtype="mxfp4")[1].codes.shape == q.codes.shape
    assert nm.modulated_norm(x.float(), out_dtype=torch.float16).dtype == torch.float16
    assert nm.modulated_norm(x, out_dtype="mxfp4").shape == (3, 5, 200)


def test_cpu_tensors_raise(mx, nm):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        mx.quantize_mxfp4(x)
    with pytest.raises(NotImplementedError):
        nm.modulated_norm(x)
    with pytest.raises(ValueError, match="kind"):
        nm.gated_residual_norm(x, x, kind="none")


def test_oracle_is_the_definition():
    """The codes by a search over all sixteen, the scale by its inequality, ties and saturation by hand."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 64)) * np.exp(rng.uniform(-20, 20, (50, 1)))
    codes, scales = B.mxfp4_quantize(x)
    back = B.mxfp4_values(codes, scales, 64)
    s = np.ldexp(1.0, scales.astype(int) - 127).repeat(32, axis=1)
    amax = np.abs(x).reshape(50, 2, 32).max(axis=2).repeat(32, axis=1)
    assert ((4 * s <= amax) & (amax < 8 * s)).all()
    all_values = np.concatenate((B.VALUES, -B.VALUES))
    best = np.abs(x[:, :, None] - s[:, :, None] * all_values).min(axis=2)
    assert np.array_equal(np.abs(x - back), best)
    row = np.zeros((1, 32))
    row[0, :11] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7.9, -0.25, -5]
    codes, scales = B.mxfp4_quantize(row)
    assert scales[0, 0] == 127
    assert B.mxfp4_values(codes, scales, 32)[0, :11].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 0, -4]
    row[0, 3] = np.inf
    assert B.mxfp4_quantize(row)[1][0, 0] == 255
    assert B.mxfp4_quantize(np.zeros((1, 5)))[1][0, 0] == 0
