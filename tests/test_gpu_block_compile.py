"""The MXFP4 operators and the block norms under torch.compile on the GPU: the eager results at every token count."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_compiled_block(pkg, cuda):
    mx = importlib.import_module("featherops_amd.kernel.hip.mxfp4")
    nm = importlib.import_module("featherops_amd.kernel.hip.norm")
    g = torch.Generator().manual_seed(0)

    def r(*shape):
        return torch.randn(*shape, generator=g).to(torch.bfloat16).to(cuda)

    w, bias, gate = mx.quantize_mxfp4(r(96, 320)), r(96), r(320)

    def block(x, h):
        x, y = nm.gated_residual_norm(x, h, gate, scale=gate, shift=gate, kind="layer", out_dtype="mxfp4")
        y = mx.mxfp4_mm(y, w, bias)
        return x, y, mx.mxfp4_mm(x, w), mx.dequantize_mxfp4(mx.quantize_mxfp4(y)), nm.modulated_norm(x)

    torch._dynamo.reset()
    graphs = []

    def backend(gm, _):
        graphs.append(gm)
        return gm.forward

    compiled = torch.compile(block, backend=backend, fullgraph=True)
    for n in (3, 5, 40, 200):
        x, h = r(2, n, 320), r(2, n, 320)
        for got, want in zip(compiled(x, h), block(x, h)):
            assert got.shape == want.shape and torch.equal(got, want), n
    assert len(graphs) <= 2
    torch._dynamo.reset()
