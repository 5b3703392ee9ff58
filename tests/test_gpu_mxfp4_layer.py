"""The MXFP4 Linear and the example block on the GPU."""

import importlib
import subprocess
import sys
from types import SimpleNamespace

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from conftest import REPO
from oracle import block_oracle as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module("featherops_amd.comfy_feather.mxfp4").mxfp4_ops


def layer(ops, state, n, k, out=torch.bfloat16, excluded=(), prefix="blocks.0.up."):
    model = torch.nn.Module()
    with torch.device("meta"):
        linear = ops(out, excluded).Linear(k, n, bias="bias" in state)
    model.add_module("up", linear)
    blocks = torch.nn.Module()
    blocks.add_module("0", model)
    top = torch.nn.Module()
    top.add_module("blocks", blocks)
    top.load_state_dict({prefix + key: v for key, v in state.items()})
    return linear


def weight(n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, k, generator=g) * k ** -0.5).bfloat16(), (torch.randn(n, generator=g) * 0.1).bfloat16()


@pytest.mark.parametrize("n,k", [(200, 320), (96, 1000)])
@pytest.mark.parametrize("x_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_forward(ops, mx, cuda, n, k, x_dtype):
    w, bias = weight(n, k)
    linear = layer(ops, {"weight": w, "bias": bias.float()}, n, k)
    linear.to(cuda)
    q = mx.quantize_mxfp4(w.to(cuda))
    for shape in ((k,), (1, k), (2, 3, k), (50, k), (0, k)):
        x = torch.randn(shape, device=cuda).to(x_dtype)
        y = linear(x)
        a = x.to(torch.bfloat16) if x_dtype == torch.float32 else x
        want = mx.mxfp4_mm(a, q, bias.to(cuda), torch.bfloat16).to(x_dtype)
        assert y.shape == (*shape[:-1], n) and y.dtype == x_dtype and torch.equal(y, want)
    q4 = mx.quantize_mxfp4(torch.randn(7, k, device=cuda))
    assert torch.equal(linear(q4), mx.mxfp4_mm(q4, q, bias.to(cuda)))


def test_checkpoint_in_mxfp4_and_back(ops, mx, cuda):
    """A row-major MXFP4 checkpoint loads without a change and leaves as it came; a 16-bit one leaves as its codes."""
    w, _ = weight(70, 200, 3)
    codes, scales = B.mxfp4_quantize(w.double().numpy())
    state = {"weight": torch.from_numpy(codes), "weight_scale": torch.from_numpy(scales)}
    a, b = layer(ops, dict(state), 70, 200), layer(ops, {"weight": w}, 70, 200)
    x = torch.randn(5, 200, device=cuda).bfloat16()
    assert torch.equal(a(x), b(x))
    for linear in (a, b):
        out = linear.state_dict()
        assert set(out) == {"weight", "weight_scale"}
        assert torch.equal(out["weight"].cpu(), state["weight"]) and torch.equal(out["weight_scale"].cpu(), state["weight_scale"])
    a.to(torch.float16)
    assert a.mx_weight.data.dtype == torch.uint8 and torch.equal(a(x), b(x))


def test_excluded_and_missing(ops, cuda):
    w, _ = weight(40, 64)
    linear = layer(ops, {"weight": w.to(cuda)}, 40, 64, excluded=("up",))
    assert linear.mx_weight is None
    x = torch.randn(3, 64, device=cuda).bfloat16()
    assert torch.equal(linear(x), F.linear(x, w.to(cuda)))
    with pytest.raises(RuntimeError, match="Missing key"):
        layer(ops, {}, 40, 64)
    with pytest.raises(ValueError, match="expected a"):
        layer(ops, {"weight": weight(40, 96)[0]}, 40, 64)


def test_merge_and_lora(ops, mx, cuda):
    w, _ = weight(64, 128, 5)
    linear = layer(ops, {"weight": w}, 64, 128)
    plain = linear.convert_weight(linear.weight)
    values = B.mxfp4_values(*B.mxfp4_quantize(w.double().numpy()), 128)
    assert plain.dtype == torch.bfloat16 and np.array_equal(plain.double().cpu().numpy(), values)
    delta = torch.randn(64, 128, device=cuda).bfloat16() * 0.02
    merged = linear.set_weight(plain + delta, return_weight=True)
    assert torch.equal(merged.data, mx.quantize_mxfp4(plain + delta).data)
    x = torch.randn(9, 128, device=cuda).bfloat16()
    before = linear(x)
    up, down = torch.randn(64, 4, device=cuda).bfloat16(), torch.randn(4, 128, device=cuda).bfloat16()
    entry = (0.5, SimpleNamespace(weights=(up, down, 2.0, None)), 1.0, None, None)
    linear.weight_function = [SimpleNamespace(patches={"w": [entry]}, key="w")]
    want = before.clone()
    want += F.linear(F.linear(x, down), up) * 0.25
    assert torch.equal(linear(x), want)
    with pytest.raises(NotImplementedError):
        linear(mx.quantize_mxfp4(x))
    linear.weight_function = []
    linear.set_weight(plain + delta)
    assert torch.equal(linear.mx_weight.data, merged.data)


def test_example_block(pkg, cuda):
    """The block's stream and output against float64 on the quantised values, and the script's own report."""
    sys.path.insert(0, str(REPO / "comfyui-featherops_amd"))
    try:
        example = importlib.import_module("example_mxfp4_block")
    finally:
        sys.path.pop(0)
    plain, block = example.build(256, 640)
    x, h, gate, scale, shift = example.inputs(33, 256)
    s, y = block(x, h, gate, scale, shift)
    d = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    want_s, n = B.gated_norm(d(x), d(h), d(gate), scale=d(scale), shift=d(shift), layer=True)
    assert np.abs(d(s) - want_s).max() <= (2.0 ** -8 * np.abs(want_s)).max()
    q = lambda v: B.mxfp4_values(*B.mxfp4_quantize(v), v.shape[1])  # noqa: E731
    u = q(n[0]) @ q(d(plain.up.weight)).T + d(plain.up.bias)
    u = torch.from_numpy(u).bfloat16()
    u = F.gelu(u, approximate="tanh").double().numpy()
    want = q(u) @ q(d(plain.down.weight)).T + d(plain.down.bias)
    # a value that lands on the other side of a 4-bit rounding moves the result by far less than a layer's error
    assert np.linalg.norm(d(y)[0] - want) <= 0.02 * np.linalg.norm(want)
    print("run example_mxfp4_block.py", flush=True)
    out = subprocess.run([sys.executable, str(REPO / "comfyui-featherops_amd" / "example_mxfp4_block.py"), "--tokens", "128",
                          "--width", "512", "--hidden", "1024"], capture_output=True, text=True, timeout=110, check=True).stdout
    assert "MXFP4" in out and "off (2-norm)" in out
