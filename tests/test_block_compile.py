"""The MXFP4 operators and the block norms on fake tensors: compiled once for any number of tokens, and refusing what the
kernels refuse. No kernel runs."""

import importlib

import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


@pytest.fixture(scope="module")
def nm(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.norm")


def meta(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def calls(mx, nm):
    """By name: a function of x (tokens, 64) and the result shapes at n tokens."""
    w = mx.quantize_mxfp4(meta(32, 64))
    v = meta(64)

    def packed(n, cols=64):
        return (-(-n // 64) * -(-cols // 128) * 4352,)

    return {
        "quantize": (lambda x: (mx.quantize_mxfp4(x).data,), lambda n: [packed(n)]),
        "there and back": (lambda x: (mx.dequantize_mxfp4(mx.quantize_mxfp4(x), F32),), lambda n: [(n, 64)]),
        "unprepack": (lambda x: mx.unprepack_mxfp4(mx.quantize_mxfp4(x)), lambda n: [(n, 32), (n, 2)]),
        "prepack": (lambda x: (mx.prepack_mxfp4(x[:, :32].to(torch.uint8), x[:, :2].to(torch.uint8)).data,), lambda n: [packed(n)]),
        "mm": (lambda x: (mx.mxfp4_mm(x, w),), lambda n: [(n, 32)]),
        "mm with leading dimensions": (lambda x: (mx.mxfp4_mm(x[None], w, None, F16),), lambda n: [(1, n, 32)]),
        "mm packed": (lambda x: (mx.mxfp4_mm(mx.quantize_mxfp4(x), w),), lambda n: [(n, 32)]),
        "norm": (lambda x: (nm.modulated_norm(x, weight=v, scale=v, shift=x),), lambda n: [(n, 64)]),
        "norm to 4 bits": (lambda x: (nm.modulated_norm(x, out_dtype="mxfp4").data,), lambda n: [packed(n)]),
        "gated norm": (lambda x: nm.gated_residual_norm(x, x, v, post_weight=v), lambda n: [(n, 64), (n, 64)]),
        "gated norm to 4 bits, product": (
            lambda x: (mx.mxfp4_mm(nm.gated_residual_norm(x, x, out_dtype="mxfp4")[1], w),), lambda n: [(n, 32)]),
    }


NAMES = ["quantize", "there and back", "unprepack", "prepack", "mm", "mm with leading dimensions", "mm packed", "norm",
         "norm to 4 bits", "gated norm", "gated norm to 4 bits, product"]


@pytest.mark.parametrize("name", NAMES)
def test_token_counts_under_compile(mx, nm, name):
    """One graph for the first count and one for every other: no count is compiled for itself."""
    fn, shapes = calls(mx, nm)[name]
    torch._dynamo.reset()
    graphs = []

    def backend(gm, _):
        graphs.append(gm)
        return gm.forward

    compiled = torch.compile(fn, backend=backend, fullgraph=True)
    for n in (5, 9, 70, 333):
        assert [tuple(t.shape) for t in compiled(meta(n, 64))] == shapes(n), n
    assert len(graphs) <= 2
    torch._dynamo.reset()


def test_names_are_all():
    class Any:
        def __getattr__(self, name):
            return lambda *a, **k: None

    assert list(calls(Any(), Any())) == NAMES


def test_fake_tensors_are_checked(mx, nm):
    """What the kernels refuse does not trace."""
    x, v = meta(4, 64), meta(64)
    w = mx.quantize_mxfp4(meta(8, 64))
    q = mx.quantize_mxfp4(x)
    for call, message in [
        (lambda: mx.quantize_mxfp4(meta(4, 0)), "at least one column"),
        (lambda: mx.quantize_mxfp4(meta()), "at least one column"),
        (lambda: mx.quantize_mxfp4(meta(4, 64, dtype=torch.float64)), "float16, bfloat16 or float32"),
        (lambda: mx.dequantize_mxfp4(q, torch.float64), "float16, bfloat16 or float32"),
        (lambda: mx.dequantize_mxfp4(q._replace(shape=(4, 0))), "at least one column"),
        (lambda: mx.dequantize_mxfp4(q._replace(shape=(65, 64))), "packed for"),
        (lambda: mx.unprepack_mxfp4(q._replace(shape=(65, 64))), "packed for"),
        (lambda: mx.prepack_mxfp4(meta(4, 32, dtype=torch.uint8), meta(5, 2, dtype=torch.uint8)), "rows"),
        (lambda: mx.prepack_mxfp4(meta(4, 32), meta(4, 2)), "1-byte"),
        (lambda: mx.mxfp4_mm(meta(4, 64, dtype=F32), w), "float16 or bfloat16"),
        (lambda: mx.mxfp4_mm(meta(4, 32), w), "b's 64 columns"),
        (lambda: mx.mxfp4_mm(x, w, v), "elements"),
        (lambda: mx.mxfp4_mm(x, w, None, F32), "out_dtype"),
        (lambda: mx.mxfp4_mm(x, w._replace(shape=(70, 64))), "packed for"),
        (lambda: mx.mxfp4_mm(q._replace(shape=(4, 32)), w), "columns"),
        (lambda: mx.mxfp4_mm(q._replace(shape=(65, 64)), w), "packed for"),
        (lambda: nm.modulated_norm(meta(4, 0)), "columns"),
        (lambda: nm.modulated_norm(meta(4, 0), out_dtype="mxfp4"), "columns"),
        (lambda: nm.modulated_norm(meta(4, 16385)), "16384 columns"),
        (lambda: nm.modulated_norm(meta(4, 64, dtype=torch.float64)), "float16, bfloat16 or float32"),
        (lambda: nm.modulated_norm(x, out_dtype=F16), "block's dtype"),
        (lambda: nm.modulated_norm(x, weight=v[:63]), "64 columns"),
        (lambda: nm.modulated_norm(x, scale=meta(3, 64)), "broadcast"),
        (lambda: nm.gated_residual_norm(x, meta(3, 64)), "shape"),
        (lambda: nm.gated_residual_norm(x, x.to(F16)), "block's dtype"),
        (lambda: nm.gated_residual_norm(x, x, out_dtype=F32), "h's dtype"),
        (lambda: nm.gated_residual_norm(x, meta(5, 64), out_dtype="mxfp4"), "shape"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
