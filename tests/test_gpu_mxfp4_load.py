"""How weights and biases get into the MXFP4 Linear and out of it, on the GPU."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module("featherops_amd.comfy_feather.mxfp4").mxfp4_ops


def load(ops, state, n, k, out=torch.bfloat16):
    with torch.device("meta"):
        linear = ops(out).Linear(k, n, bias="bias" in state)
    top = torch.nn.Module()
    top.add_module("up", linear)
    top.load_state_dict({"up." + key: v for key, v in state.items()})
    return linear


def some(*shape, dtype=torch.bfloat16, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize("where", ["cpu", "cuda"])
@pytest.mark.parametrize("dtype", [F8, torch.bfloat16, torch.float32])
def test_scaled_checkpoint(ops, mx, cuda, dtype, where):
    """One scale, and one per row: the layer's weight is the quantised product."""
    weight = some(70, 200, dtype=dtype)
    x = some(5, 200, seed=1).to(cuda)
    for scale in (torch.tensor(0.003), some(70, 1, dtype=torch.float32, seed=2).abs()):
        linear = load(ops, {"weight": weight.to(where), "weight_scale": scale.to(where)}, 70, 200)
        want = mx.quantize_mxfp4((weight.float() * scale).to(cuda))
        assert torch.equal(linear(x), mx.mxfp4_mm(x, want))


def test_layer_in_host_memory(ops, mx, cuda):
    """Saved, converted and given a merged weight where it lies, with the values of the layer on the GPU."""
    weight = some(70, 200)
    here, off = load(ops, {"weight": weight}, 70, 200), load(ops, {"weight": weight}, 70, 200).to("cpu")
    assert off.weight.device.type == "cpu" and here.weight.is_cuda
    want = here.state_dict()
    for name, t in off.state_dict().items():
        assert t.device.type == "cpu" and want[name].is_cuda and torch.equal(t, want[name].cpu())
    again = load(ops, off.state_dict(), 70, 200).state_dict()  # (a packed operand's bytes beyond its rows are not specified)
    assert all(torch.equal(again[name], want[name]) for name in want)
    values = off.convert_weight(off.weight)
    assert values.device.type == "cpu" and torch.equal(values, here.convert_weight().cpu())
    merged = values + some(70, 200, seed=3, std=0.02)
    assert torch.equal(off.convert_weight(off.set_weight(merged, return_weight=True)).cpu(),
                       mx.dequantize_mxfp4(mx.quantize_mxfp4(merged.to(cuda))).cpu())
    off.set_weight(merged)
    here.set_weight(merged.to(cuda))
    assert off.weight.device.type == "cpu" and torch.equal(off.state_dict()["weight"], here.state_dict()["weight"].cpu())


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
def test_cpu_checkpoint_and_offloaded_layer(ops, mx, cuda, out):
    """A layer from a checkpoint in host memory runs as it is, and so does one that was moved back there."""
    weight, bias = some(70, 200), some(70, seed=4)
    x = some(5, 200, seed=1).to(cuda)
    q = mx.quantize_mxfp4(x)
    want = mx.mxfp4_mm(x, mx.quantize_mxfp4(weight.to(cuda)), bias.to(cuda, out), out)
    linear = load(ops, {"weight": weight, "bias": bias}, 70, 200, out)
    assert linear.weight.is_cuda and linear.bias.is_cuda
    for move in (lambda m: m, lambda m: m.to("cpu"), lambda m: m.to(cuda), lambda m: m.to(torch.float16), lambda m: m.to(torch.bfloat16)):
        move(linear)
        assert torch.equal(linear(x), want.to(x.dtype)) and torch.equal(linear(q), want)
        assert linear.weight.device == linear.bias.device
