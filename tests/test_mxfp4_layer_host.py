"""CPU tests of the MXFP4 Linear's bookkeeping, with the library's kernels replaced by stand-ins that record what they
are given. No kernel runs."""

import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def layer_module(pkg):
    return importlib.import_module("featherops_amd.comfy_feather.mxfp4")


@pytest.fixture
def seen(layer_module, monkeypatch):
    """What quantize_mxfp4 was given, in order; its result is a packed operand of zeros."""
    given = []

    def quantize(x):
        given.append(x)
        rows, cols = x.shape
        data = torch.zeros(-(-rows // 64) * -(-cols // 128) * 4352, dtype=torch.uint8)
        return layer_module.MXFP4Tensor(data, tuple(x.shape))

    monkeypatch.setattr(layer_module, "quantize_mxfp4", quantize)
    monkeypatch.setattr(layer_module, "_on_gpu", lambda t: t)
    return given


def load(layer_module, state, n, k, out=torch.bfloat16, excluded=(), strict=True):
    with torch.device("meta"):
        linear = layer_module.mxfp4_ops(out, excluded).Linear(k, n, bias="bias" in state)
    top = torch.nn.Module()
    top.add_module("up", linear)
    top.load_state_dict({"up." + key: v for key, v in state.items()}, strict=strict)
    return linear


F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("key", ["weight_scale", "scale_weight"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, F8, torch.float8_e5m2])
def test_checkpoint_scale_reaches_the_quantiser(layer_module, seen, key, dtype):
    g = torch.Generator().manual_seed(0)
    weight = torch.randn(5, 64, generator=g).to(dtype)
    for scale in (torch.tensor(0.0125), torch.tensor([0.0125]), torch.rand(5, 1, generator=g)):
        load(layer_module, {"weight": weight, key: scale}, 5, 64)
        assert torch.equal(seen.pop(), weight.float() * scale)  # as the 8-bit layer: in fp32, one rounding


@pytest.mark.parametrize("dtype", [F8, torch.float8_e5m2])
def test_unscaled_fp8_weight(layer_module, seen, dtype):
    weight = torch.randn(4, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    load(layer_module, {"weight": weight}, 4, 64)
    assert torch.equal(seen.pop().float(), weight.float())


def test_scale_of_an_excluded_layer(layer_module, seen):
    weight, scale = torch.randn(4, 64, generator=torch.Generator().manual_seed(2)), torch.tensor(0.25)
    for dtype, held in ((F8, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32)):
        linear = load(layer_module, {"weight": weight.to(dtype), "weight_scale": scale}, 4, 64, excluded=("up",))
        assert linear.weight.dtype == held
        assert torch.equal(linear.weight.data.float(), weight.to(dtype).float() * scale)  # (a power of two: exact)
    linear = load(layer_module, {"weight": weight.half()}, 4, 64, excluded=("up",))
    assert torch.equal(linear.weight.data, weight.half()) and not seen


def test_scale_refusals(layer_module, seen):
    weight = torch.zeros(4, 64, dtype=torch.bfloat16)
    for scale in (torch.ones(4), torch.ones(1, 64), torch.ones(3, 1), torch.ones(4, 2)):
        with pytest.raises(ValueError, match="weight scale must be"):
            load(layer_module, {"weight": weight, "weight_scale": scale}, 4, 64)
    assert not seen


@pytest.fixture
def codec(layer_module, seen, monkeypatch):
    """Dequantisation that marks its result with the operand's first byte."""
    monkeypatch.setattr(layer_module, "dequantize_mxfp4",
                        lambda q, dtype: torch.full(q.shape, float(q.data[0]), dtype=dtype, device="cpu"))


def test_weight_is_the_packed_operand(layer_module, seen):
    """Whatever reads, sizes, moves or restores a parameter finds the packed bytes."""
    linear = load(layer_module, {"weight": torch.zeros(70, 200)}, 70, 200)
    assert isinstance(linear.weight, torch.nn.Parameter) and dict(linear.named_parameters())["weight"] is linear.weight
    assert linear.weight.dtype == torch.uint8 and linear.weight.shape == (2 * 2 * 4352,) and not linear.weight.requires_grad
    assert linear.mx_weight.shape == (70, 200) and linear.mx_weight.data.data_ptr() == linear.weight.data_ptr()
    backup = linear.weight.detach().clone()
    backup[0] = 7
    linear.weight = torch.nn.Parameter(backup, requires_grad=False)
    assert linear.mx_weight.data[0] == 7
    for cast in (lambda m: m.to(torch.float16), lambda m: m.half(), lambda m: m.float(), lambda m: m.type(torch.float64)):
        cast(linear)
        assert linear.weight.dtype == torch.uint8 and linear.weight[0] == 7
    assert linear.to("meta").weight.device.type == "meta"


def test_convert_weight_converts_its_argument(layer_module, codec):
    linear = load(layer_module, {"weight": torch.zeros(4, 64)}, 4, 64)
    new = linear.set_weight(torch.ones(4, 64), return_weight=True)
    new.data[0] = 3
    for weight, first in ((new, 3), (new.data, 3), (linear.weight, 0), (linear.mx_weight, 0), (None, 0)):
        values = linear.convert_weight(weight)
        assert values.dtype == torch.bfloat16 and values.shape == (4, 64) and (values == first).all()
    for other in (torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.uint8), "weight"):
        with pytest.raises(TypeError, match="packed MXFP4 weight"):
            linear.convert_weight(other)
    with pytest.raises(ValueError, match="expected a"):
        linear.convert_weight(new._replace(shape=(64, 4)))


def test_conversions_of_a_layer_in_host_memory(layer_module, codec, monkeypatch):
    """The kernels get the operand on the GPU (here: another device than the layer's), results come back from it."""
    there = []

    def on_gpu(t):
        there.append(t)
        return t

    def unprepack(q):
        return torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)

    monkeypatch.setattr(layer_module, "_on_gpu", on_gpu)
    monkeypatch.setattr(layer_module, "unprepack_mxfp4", unprepack)
    linear = load(layer_module, {"weight": torch.zeros(4, 64)}, 4, 64)
    for convert in (linear.state_dict, lambda: linear.convert_weight(linear.weight)):
        there.clear()
        convert()
        assert any(t is linear.weight for t in there)


def test_layer_without_storage(layer_module, seen):
    state = load(layer_module, {"weight": torch.zeros(4, 64)}, 4, 64).to("meta").state_dict()
    assert {k: (t.shape, t.device.type) for k, t in state.items()} == {"weight": ((4, 32), "meta"), "weight_scale": ((4, 2), "meta")}


@pytest.fixture
def product(layer_module, monkeypatch):
    """Stands for mxfp4_mm: the operands it was given, a result of zeros."""
    calls = []

    def mm(a, w, bias=None, out_dtype=None):
        calls.append((a, w, bias))
        return torch.zeros(*a.shape[:-1], w.shape[0], dtype=out_dtype, device=w.data.device)

    monkeypatch.setattr(layer_module, "mxfp4_mm", mm)
    return calls


def test_offloaded_layer_comes_to_the_activations(layer_module, seen, product):
    """Weight and bias elsewhere than the activations (here: those on the meta device) are brought to them for the call;
    a bias of another type, as .to(float16) leaves it, is cast."""
    linear = load(layer_module, {"weight": torch.zeros(4, 64), "bias": torch.ones(4)}, 4, 64)
    for x in (torch.zeros(3, 64, dtype=torch.bfloat16, device="meta"),
              layer_module.MXFP4Tensor(torch.zeros(4352, dtype=torch.uint8, device="meta"), (3, 64))):
        linear(x)
        _, weight, bias = product.pop()
        assert weight.data.device.type == bias.device.type == "meta" and weight.shape == (4, 64)
        assert linear.weight.device.type == linear.bias.device.type == "cpu"
    linear.to(torch.float16)
    linear(torch.zeros(3, 64, dtype=torch.float16))
    assert product[-1][2].dtype == torch.bfloat16 and product[-1][1].data is linear.weight
    linear.to(torch.bfloat16)
    linear(torch.zeros(3, 64, dtype=torch.bfloat16))
    assert product[-1][1].data is linear.weight and product[-1][2] is linear.bias
    plain = load(layer_module, {"weight": torch.zeros(4, 64)}, 4, 64)
    plain(torch.zeros(3, 64, dtype=torch.bfloat16, device="meta"))
    assert product[-1][1].data.device.type == "meta" and product[-1][2] is None


def test_bias_patches(layer_module, seen, product):
    """bias_function runs on the bias in the output's type, in order, and leaves the stored one as it is."""
    linear = load(layer_module, {"weight": torch.zeros(4, 64), "bias": torch.ones(4)}, 4, 64)
    linear.bias_function = [lambda b: b + 1, lambda b: b * 3]
    linear(torch.zeros(3, 64, dtype=torch.bfloat16))
    assert torch.equal(product[-1][2], torch.full((4,), 6, dtype=torch.bfloat16)) and (linear.bias == 1).all()
    linear.bias_function = []
    linear(torch.zeros(3, 64, dtype=torch.bfloat16))
    assert product[-1][2] is linear.bias


def test_assigned_weight(layer_module, seen, product):
    linear = load(layer_module, {"weight": torch.zeros(4, 64, dtype=torch.bfloat16)}, 4, 64, excluded=("up",))
    assert linear.mx_weight is None
    operand = layer_module.MXFP4Tensor(torch.full((4352,), 5, dtype=torch.uint8), (4, 64))
    linear.mx_weight = operand
    assert linear.is_quantized and torch.equal(linear.weight, operand.data)
    linear(torch.zeros(3, 64, dtype=torch.bfloat16))
    assert product[-1][1].data is linear.weight
    with pytest.raises(ValueError, match="expected a"):
        linear.mx_weight = operand._replace(shape=(64, 4))


def test_forward_under_compile(layer_module, seen):
    """One graph for the first token count, one for every other, with 16-bit and with 4-bit activations."""
    linear = load(layer_module, {"weight": torch.zeros(4, 64), "bias": torch.zeros(4)}, 4, 64).to("meta")
    quantise = importlib.import_module("featherops_amd.kernel.hip.mxfp4").quantize_mxfp4
    graphs = []

    def backend(gm, _):
        graphs.append(gm)
        return gm.forward

    for fn in (linear, lambda x: linear(quantise(x))):
        torch._dynamo.reset()
        graphs.clear()
        compiled = torch.compile(fn, backend=backend, fullgraph=True)
        for n in (3, 5, 200):
            assert compiled(torch.empty(n, 64, dtype=torch.bfloat16, device="meta")).shape == (n, 4)
        assert len(graphs) <= 2
    torch._dynamo.reset()
