"""CPU tests: the C entries of the MXFP4 operators and the block norms refuse packed buffers off a 16-byte boundary, which
the kernels' copies could not read. No kernel runs."""

import ctypes
import importlib

import pytest

from test_block_host import NormArgs


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_packed_buffers_off_a_boundary(lib, off):
    P, Q = 4096, 4096 + off  # stand for pointers: every call ends at a check before they are used
    results = [
        lib.feather_mxfp4_quantize(P, 0, 4, 64, 64, Q, P, None), lib.feather_mxfp4_quantize(P, 0, 4, 64, 64, P, Q, None),
        lib.feather_mxfp4_dequantize(Q, P, P, 0, 4, 64, None), lib.feather_mxfp4_dequantize(P, Q, P, 0, 4, 64, None),
        lib.feather_mxfp4_prepack(P, P, Q, P, 4, 64, None), lib.feather_mxfp4_prepack(P, P, P, Q, 4, 64, None),
        lib.feather_mxfp4_unprepack(Q, P, P, P, 4, 64, None), lib.feather_mxfp4_unprepack(P, Q, P, P, 4, 64, None),
    ]
    for M in (4, 400):  # either kernel
        for a, a_scales, b, b_scales in ((Q, P, P, P), (P, Q, P, P), (P, P, Q, P), (P, P, P, Q)):
            results.append(lib.feather_mxfp4_mm(a, a_scales, 3, 0, b, b_scales, None, P, M, 64, 64, 0, None, 0, None))
    results.append(lib.feather_mxfp4_mm(P, None, 0, 64, Q, P, None, P, 4, 64, 64, 0, None, 0, None))
    good = dict(x=P, rows=4, cols=64, x_row_stride=64, x_dtype=1, y_dtype=1, mod_dtype=1, gate_group=1, mod_group=1)
    for codes, scales in ((Q, P), (P, Q)):
        results.append(lib.feather_block_norm(ctypes.byref(NormArgs(**good, codes=codes, scales=scales)), None))
    assert results == [1] * len(results)
