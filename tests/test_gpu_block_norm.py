"""The fused block norms on the GPU against float64 (oracle/block_oracle.py)."""

import importlib

import numpy as np
import pytest
import torch

from oracle import block_oracle as B

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def nm(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.norm")


@pytest.fixture(scope="module")
def mx(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.mxfp4")


def d(t):
    return None if t is None else t.double().cpu().numpy()


def inputs(cuda, B_, S, D, x_type, block, mods, seed, mean=0.0):
    g = torch.Generator().manual_seed(seed)

    def r(*shape, std=1.0, m=0.0, dtype=mods):
        return (torch.randn(*shape, generator=g) * std + m).to(dtype).to(cuda)

    return {"x": r(B_, S, D, std=3.0, m=mean, dtype=x_type), "h": r(B_, S, D, dtype=block),
            "post_weight": r(D, std=0.2, m=1.0), "weight": r(D, std=0.2, m=1.0), "bias": r(D, std=0.2),
            "gate": r(B_, 1, D, std=0.5), "scale": r(B_, 1, D, std=0.3), "shift": r(B_, 1, D, std=0.3)}


def check(nm, t, use, kind, eps=1e-6, rs=1.0, block=None, label=""):
    """Both results within half an ulp of their type for the one rounding, plus the fp32 arithmetic's: 16 roundings
    of 2^-24 on a value's way (gate, residual, centring, the norm, affine terms) and the statistics' relative error,
    2^-24 (8 + log2 D) for sums over a tree whose leaves are at most 16 in a row, all of them relative to the largest
    terms that meet: |x| + |h| for the stream, and for y the same divided by the row's norm and amplified by the
    affine factors."""
    args = {k: t[k] for k in use}
    h = args.pop("h", None)
    gate, post = args.pop("gate", None), args.pop("post_weight", None)
    if h is not None:
        stream, y = nm.gated_residual_norm(t["x"], h, gate, post_weight=post, kind=kind, eps=eps, residual_scale=rs, **args)
        assert stream.dtype == t["x"].dtype and y.dtype == h.dtype
    else:
        stream, y = t["x"], nm.modulated_norm(t["x"], kind=kind, eps=eps, out_dtype=block, **args)
    layer = kind == "layer"
    x64 = d(t["x"])
    want_s, want_y = B.gated_norm(x64, d(h), d(gate), d(post), **{k: d(v) for k, v in args.items()}, layer=layer, eps=eps,
                                  residual_scale=rs)
    D = x64.shape[-1]
    u = 2.0 ** -24 * (16 + 8 + np.log2(max(2, D)))
    mags = np.abs(rs * x64)
    if h is not None:
        hh = np.abs(d(h))
        if post is not None:
            hh = (hh + np.abs(d(h).mean(-1, keepdims=True)) * layer) / np.sqrt(
                (B.norm(d(h), layer, eps) * 0 + ((d(h) - d(h).mean(-1, keepdims=True) * layer) ** 2).mean(-1, keepdims=True)) + eps) * np.abs(d(post))
        mags = mags + (hh if gate is None else np.abs(d(gate)) * hh)
    if h is not None:
        tol = HALF[stream.dtype] * np.abs(want_s) + u * mags + 2.0 ** -25 * (stream.dtype == F16)
        worst = (np.abs(d(stream) - want_s) / tol).max()
        assert worst <= 1.0, f"{label} stream: {worst:.3g} times the bound"
    centre = want_s - want_s.mean(-1, keepdims=True) * layer
    sd = np.sqrt((centre ** 2).mean(-1, keepdims=True) + eps)
    rms_mags = np.sqrt((mags ** 2).mean(-1, keepdims=True))
    amp = np.abs(1.0 if "weight" not in args else d(args["weight"])) * np.abs(1.0 if "scale" not in args else 1.0 + d(args["scale"]))
    # a value's own error, and the statistics' on the normalised value
    err = u * (mags + rms_mags + np.abs(want_s.mean(-1, keepdims=True)) * layer) / sd * (1.0 + np.abs(centre) / sd) * amp
    for k in ("bias", "shift"):
        if k in args:
            err = err + u * np.abs(d(args[k])) * (1.0 if "scale" not in args else np.abs(1.0 + d(args["scale"])))
    tol = HALF[y.dtype] * np.abs(want_y) + err + 2.0 ** -25 * (y.dtype == F16)
    worst = (np.abs(d(y) - want_y) / tol).max()
    assert worst <= 1.0, f"{label} y: {worst:.3g} times the bound"
    return stream, y


ALL = ("h", "gate", "post_weight", "weight", "bias", "scale", "shift")
USES = [(), ("weight",), ("scale", "shift"), ("weight", "bias", "scale", "shift"), ("h",), ("h", "gate", "scale", "shift"),
        ("h", "post_weight", "weight"), ALL]
TYPES = [(F16, F16, F16), (BF16, BF16, BF16), (BF16, BF16, F32), (F16, F16, F32), (F32, BF16, F32), (F32, BF16, BF16),
         (F32, F16, F16), (F32, F32, F32)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x)[6:] for x in t))
@pytest.mark.parametrize("use", USES, ids=lambda u: "+".join(u) or "plain")
def test_types_and_terms(nm, cuda, use, types, kind):
    x, block, mods = types
    t = inputs(cuda, 2, 5, 1160, x, block, mods, len(use))
    check(nm, t, use, kind, block=block)


@pytest.mark.parametrize("D", [1, 2, 7, 8, 9, 63, 64, 65, 500, 512, 513, 1027, 4096, 4097, 5120, 8191, 16384])
def test_widths(nm, cuda, D):
    for types in ((BF16, BF16, BF16), (F32, BF16, F32)):
        t = inputs(cuda, 1, 3, D, *types, seed=D)
        check(nm, t, ALL, "layer", eps=1e-3, label=f"{D}")
        check(nm, t, ALL, "rms", eps=1e-3, label=f"{D}")


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 127, 129])
def test_row_counts(nm, cuda, rows):
    for D in (96, 1500):
        t = inputs(cuda, 1, rows, D, BF16, BF16, F32, rows)
        check(nm, t, ("h", "gate", "scale", "shift"), "layer")


def test_large_mean(nm, cuda):
    """A mean a thousand times the deviation: the variance is summed about the mean."""
    t = inputs(cuda, 1, 4, 2048, F32, F32, F32, 1, mean=3000.0)
    check(nm, t, ("scale", "shift"), "layer", block=F32)


def test_residual_scale_and_eps(nm, cuda):
    t = inputs(cuda, 2, 3, 640, BF16, BF16, BF16, 9)
    check(nm, t, ALL, "rms", eps=0.5, rs=0.125)
    check(nm, t, ALL, "layer", eps=1e-5, rs=-2.0)


def test_constant_and_zero_rows(nm, cuda):
    x = torch.zeros(3, 700, dtype=BF16, device=cuda)
    x[1] = 5.0
    y = nm.modulated_norm(x, kind="layer")
    assert torch.equal(y, torch.zeros_like(x))
    y = nm.modulated_norm(x, kind="rms", eps=1e-6)
    assert torch.equal(y[0], x[0]) and torch.equal(y[1], torch.ones_like(x[1])) and torch.equal(y[2], x[2])


def test_non_finite_rows_stay_apart(nm, mx, cuda):
    t = inputs(cuda, 1, 20, 300, BF16, BF16, BF16, 4)
    clean = nm.gated_residual_norm(t["x"], t["h"], t["gate"])[1]
    t["x"][0, 3, 10], t["h"][0, 8, 299] = float("nan"), float("inf")
    s, y = nm.gated_residual_norm(t["x"], t["h"], t["gate"])
    bad = torch.zeros(20, dtype=torch.bool, device=cuda)
    bad[3] = bad[8] = True
    assert torch.equal(y[0, ~bad], clean[0, ~bad])
    assert y[0, 3].isnan().all() and y[0, 8, 299].isnan() and s[0, 3, 10].isnan()
    q = nm.gated_residual_norm(t["x"], t["h"], t["gate"], out_dtype="mxfp4")[1]
    v = mx.dequantize_mxfp4(q, F32)
    assert v[0, 3].isnan().all() and not v[0, ~bad].isnan().any()


def test_broadcast_forms(nm, cuda):
    """Vectors for all rows, a sample's, a token's, a leading dimension's own, slices of a modulation tensor: the
    same bits as written out for every row."""
    B_, S, D = 3, 7, 416
    t = inputs(cuda, B_, S, D, BF16, BF16, BF16, 6)
    g = torch.Generator().manual_seed(1)
    six = (torch.randn(B_, 1, 6 * D, generator=g) * 0.4).to(BF16).to(cuda)
    chunks = six.chunk(6, dim=-1)
    forms = [t["gate"][0, 0], t["gate"][:1], t["gate"], chunks[2], chunks[5].expand(B_, S, D),
             (torch.randn(B_, S, D, generator=g)).to(BF16).to(cuda), (torch.randn(S, D, generator=g)).to(BF16).to(cuda),
             (torch.randn(1, S, D, generator=g)).to(BF16).to(cuda)]
    for i, a in enumerate(forms):
        b = forms[(i + 3) % len(forms)]
        got = nm.gated_residual_norm(t["x"], t["h"], a, scale=b, shift=a, kind="layer")
        full = [v.expand(B_, S, D).contiguous() for v in (a, b)]
        want = nm.gated_residual_norm(t["x"], t["h"], full[0], scale=full[1], shift=full[0], kind="layer")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


def test_views(nm, cuda):
    t = inputs(cuda, 1, 12, 450, F16, F16, F16, 8)
    x, h = t["x"][0], t["h"][0]
    for view in (lambda v: v[:, 3:403], lambda v: v[::2, 1:], lambda v: v.t()):
        got = nm.gated_residual_norm(view(x), view(h), kind="layer")
        want = nm.gated_residual_norm(view(x).contiguous(), view(h).contiguous(), kind="layer")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert got[0].is_contiguous() and got[1].is_contiguous()
    assert nm.modulated_norm(x[:0]).shape == (0, 450)
    assert nm.modulated_norm(x[0]).shape == (450,)


@pytest.mark.parametrize("rows,D", [(1, 32), (1, 5120), (2, 33), (5, 513), (17, 1000), (130, 640), (64, 4128), (200, 8200)])
def test_mxfp4_output(nm, mx, cuda, rows, D):
    """The quantised result is that of the same norm's fp32 result, and the stream's bits do not change."""
    for types in ((F32, F32, F32), (F32, BF16, F32)):
        t = inputs(cuda, 1, rows, D, *types, seed=rows + D)
        use = {k: t[k] for k in ("weight", "scale", "shift")}
        s, q = nm.gated_residual_norm(t["x"], t["h"], t["gate"], kind="layer", out_dtype="mxfp4", **use)
        s2, y = nm.gated_residual_norm(t["x"], t["h"], t["gate"], kind="layer", **use)
        assert torch.equal(s, s2) and q.shape == (1, rows, D)
        if types[1] == F32:
            want = mx.quantize_mxfp4(y)
            got_rows, want_rows = mx.unprepack_mxfp4(q), mx.unprepack_mxfp4(want)
            assert torch.equal(got_rows[0], want_rows[0]) and torch.equal(got_rows[1], want_rows[1])
            # columns beyond D are zero codes
            v = mx.dequantize_mxfp4(q._replace(shape=(rows, -(-D // 128) * 128)), F32)
            assert not v[:, D:].any()
        q2 = nm.modulated_norm(t["x"], kind="rms", out_dtype="mxfp4", weight=t["weight"])
        y2 = nm.modulated_norm(t["x"], kind="rms", weight=t["weight"].float(), out_dtype=F32)
        a, b = mx.unprepack_mxfp4(q2), mx.unprepack_mxfp4(mx.quantize_mxfp4(y2))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_graph_and_stream(nm, cuda):
    t = inputs(cuda, 2, 40, 1600, BF16, BF16, BF16, 3)
    call = lambda: nm.gated_residual_norm(t["x"], t["h"], t["gate"], scale=t["scale"], shift=t["shift"], kind="layer")
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        t["x"].copy_(t["x"].flip(1))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals(nm, cuda):
    x = torch.zeros(2, 3, 64, dtype=BF16, device=cuda)
    h = torch.zeros_like(x)
    v = torch.zeros(64, dtype=BF16, device=cuda)
    for call, message in [
        (lambda: nm.modulated_norm(x.double()), "float16, bfloat16 or float32"),
        (lambda: nm.modulated_norm(torch.zeros(2, 16385, device=cuda)), "16384 columns"),
        (lambda: nm.modulated_norm(x[..., :0]), "columns"),
        (lambda: nm.modulated_norm(x, out_dtype=F16), "block's dtype"),
        (lambda: nm.modulated_norm(x, weight=v[:63]), "64 columns"),
        (lambda: nm.modulated_norm(x, weight=v.double()), "weight"),
        (lambda: nm.modulated_norm(x, scale=v.expand(3, 2, 64)), "broadcast"),
        (lambda: nm.modulated_norm(x, scale=v.cpu()), "device"),
        (lambda: nm.gated_residual_norm(x, h[:1]), "shape"),
        (lambda: nm.gated_residual_norm(x, h.to(F16)), "block's dtype"),
        (lambda: nm.gated_residual_norm(x, h, out_dtype=F32), "h's dtype"),
        (lambda: nm.gated_residual_norm(x, h.cpu()), "device"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
    with pytest.raises(ValueError, match="kind"):
        nm.modulated_norm(x, kind="batch")
