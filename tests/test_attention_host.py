"""CPU tests of rotary positions and attention: the C entries refuse what no kernel takes before anything is launched, fake
tensors have the results' shapes and are checked like real ones, CPU tensors raise, and the 64-bit oracle is what the
definitions say. No kernel runs."""

import ctypes
import importlib

import numpy as np
import pytest
import torch

from attention_util import AttentionArgs, attention_args, plan_of
from oracle import attention_oracle as A

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = torch.int32


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


@pytest.fixture(scope="module")
def rp(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.rope")


@pytest.fixture(scope="module")
def at(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.attention")


class RopeArgs(ctypes.Structure):
    """feather_rope_args of include/featherops_amd.h."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "q_out", "k_out", "q_weight", "k_weight", "table")]
                + [(n, ctypes.c_int64) for n in ("batch", "tokens", "q_heads", "k_heads", "head_dim", "pairs", "q_batch_stride",
                                                 "q_token_stride", "q_head_stride", "k_batch_stride", "k_token_stride",
                                                 "k_head_stride", "table_batch_stride")]
                + [(n, ctypes.c_int) for n in ("dtype", "weight_dtype", "norm", "pairs_of_halves")] + [("eps", ctypes.c_float)])


P = 4096  # stands for a pointer: every call below ends at a check before it is used


def test_table_entry_refuses(lib):
    def call(pos=P, code=1, rows=4, dims=(16, 24, 24), axes=None, theta=1e4, table=P):
        arr = (ctypes.c_int * 9)(*dims)
        return lib.feather_rope_table(pos, code, rows, arr, len(dims) if axes is None else axes, theta, 0, table, None)

    bad = [call(pos=None), call(table=None), call(table=P + 4), call(code=4), call(code=-1), call(rows=-1), call(rows=1 << 31),
           call(axes=0), call(axes=9), call(dims=(3,)), call(dims=(-2, 8)), call(dims=(0, 0)), call(dims=(128, 130)),
           call(dims=(258,)), call(theta=0.0), call(theta=-1.0), call(theta=float("inf")), call(theta=float("nan")),
           lib.feather_rope_table(P, 1, 4, None, 1, 1e4, 0, P, None)]
    assert bad == [1] * len(bad)
    assert call(rows=0, pos=None, table=None) == 0


def test_rope_entry_refuses(lib):
    good = dict(q=P, k=P, q_out=P, k_out=P, table=P, batch=2, tokens=5, q_heads=8, k_heads=2, head_dim=128, pairs=64,
                q_batch_stride=5120, q_token_stride=1024, q_head_stride=128, k_batch_stride=1280, k_token_stride=256,
                k_head_stride=128, dtype=1, weight_dtype=1, norm=1, eps=1e-6)
    cases = [dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(batch=-1), dict(tokens=-1), dict(tokens=1 << 31),
             dict(batch=1 << 20, tokens=1 << 20), dict(q_heads=0), dict(k_heads=-1), dict(q_heads=1 << 17), dict(head_dim=0),
             dict(head_dim=12), dict(head_dim=264), dict(pairs=0), dict(pairs=65), dict(dtype=3), dict(weight_dtype=0),
             dict(norm=3), dict(norm=-1), dict(norm=0, q_weight=P), dict(norm=0, k_weight=P), dict(norm=2, q_heads=129),
             dict(norm=2, k_heads=257, head_dim=40, pairs=20), dict(pairs_of_halves=2), dict(table=P + 2), dict(table_batch_stride=-1)]
    for case in cases:
        assert lib.feather_qk_norm_rope(ctypes.byref(RopeArgs(**{**good, **case})), None) == 1, case
    assert lib.feather_qk_norm_rope(None, None) == 1
    for case in (dict(tokens=0), dict(batch=0)):
        assert lib.feather_qk_norm_rope(ctypes.byref(RopeArgs(**{**good, **case, "q": None, "q_out": None})), None) == 0


GOOD = dict(q=P, k=P, v=P, out=P, batch=2, q_tokens=5, k_tokens=7, heads=8, kv_heads=2, head_dim=128, q_batch_stride=5120,
            q_token_stride=1024, q_head_stride=128, k_batch_stride=1792, k_token_stride=256, k_head_stride=128,
            v_batch_stride=1792, v_token_stride=256, v_head_stride=128, dtype=1, mask_dtype=1, scale=0.1)


def test_attention_entry_refuses(lib):
    cases = [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=P + 8), dict(k=P + 2), dict(v=P + 4), dict(out=P + 8),
             dict(batch=-1), dict(batch=65537), dict(q_tokens=-1), dict(k_tokens=-1), dict(q_tokens=1 << 31), dict(k_tokens=1 << 31),
             dict(q_tokens=(1 << 28) + 1),  # times 4 heads of a group
             dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(kv_heads=16), dict(heads=1 << 17), dict(head_dim=0),
             dict(head_dim=100), dict(head_dim=264), dict(dtype=2), dict(dtype=4), dict(scale=0.0), dict(scale=-1.0),
             dict(scale=float("inf")), dict(scale=float("nan")), dict(causal=2), dict(q_token_stride=1028), dict(k_head_stride=4),
             dict(v_batch_stride=-8), dict(k_token_stride=1 << 23), dict(q_batch_stride=12), dict(mask=P, mask_dtype=0),
             dict(mask=P, mask_dtype=3), dict(mask=P + 1), dict(mask=P + 2, mask_dtype=2), dict(mask=P, mask_head_stride=-1),
             dict(q_offsets=P), dict(k_offsets=P), dict(q_offsets=P, k_offsets=P, k_lengths=P),
             dict(q_offsets=P, k_offsets=P, mask=P), dict(q_offsets=P, k_offsets=P, batch=0)]
    for case in cases:
        assert lib.feather_attention(ctypes.byref(AttentionArgs(**{**GOOD, **case})), None, 0, None) == 1, case
    assert lib.feather_attention(None, None, 0, None) == 1
    for case in (dict(q_tokens=0), dict(batch=0)):
        assert lib.feather_attention(ctypes.byref(AttentionArgs(**{**GOOD, **case, "q": None, "out": None})), None, 0, None) == 0


def meta(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_fake_tensors(rp, at):
    assert rp.rope_table(meta(3, 7, 3, dtype=torch.int64), (16, 56, 56)).shape == (3, 7, 64, 2)
    q, k = meta(2, 7, 6, 64), meta(2, 7, 3, 64)
    assert [t.shape for t in rp.qk_norm_rope(q, k, meta(7, 32, 2, dtype=F32), norm="row")] == [q.shape, k.shape]
    assert rp.norm_rope(q, meta(2, 7, 20, 2, dtype=F32), weight=meta(64), norm="head").dtype == BF16
    kv = meta(2, 9, 3, 64)
    assert at.attention(q, kv, kv, causal=True, mask=meta(7, 9, dtype=torch.bool), k_lengths=meta(2, dtype=I32)).shape == q.shape
    assert at.packed_attention(q[0], k[0], k[0], meta(4, dtype=I32), scale=2.0).shape == q[0].shape


REFUSED_TABLES = [(dict(axes=()), "1 to 8 axes"), (dict(axes=(2,) * 9), "1 to 8 axes"), (dict(axes=(16, 56, 55)), "even number"),
                  (dict(axes=(0, 0, 0)), "2 to 256"), (dict(axes=(128, 128, 2)), "2 to 256"), (dict(axes=(16, 56)), "end in 2 axes"),
                  (dict(theta=0.0), "theta"), (dict(positions=meta(7, 3, dtype=F16)), "positions must be"),
                  (dict(ladder="each"), "ladder must be")]


@pytest.mark.parametrize("change,message", REFUSED_TABLES)
def test_tables_are_refused(rp, change, message):
    args = {"positions": meta(7, 3, dtype=I32), "axes": (16, 56, 56), "theta": 1e4, "ladder": "axis", **change}
    with pytest.raises((RuntimeError, ValueError), match=message):
        rp.rope_table(args["positions"], args["axes"], args["theta"], ladder=args["ladder"])


REFUSED_ROPES = [
    (dict(q=meta(7, 64)), "must be \\(tokens"), (dict(q=meta(2, 7, 6, 60), k=meta(2, 7, 3, 60)), "multiple of 8"),
    (dict(q=meta(2, 7, 6, 264), k=meta(2, 7, 3, 264)), "multiple of 8"), (dict(q=meta(2, 7, 6, 64, dtype=torch.float64)), "q must be"),
    (dict(k=meta(2, 7, 3, 64, dtype=F16)), "q's dtype"), (dict(k=meta(2, 8, 3, 64)), "q's batch"), (dict(k=meta(7, 3, 64)), "q's batch"),
    (dict(k=meta(2, 7, 0, 64)), "1 to 65536 heads"), (dict(table=meta(7, 32, 2)), "float32"),
    (dict(table=meta(7, 33, 2, dtype=F32)), "table must be"), (dict(table=meta(8, 32, 2, dtype=F32)), "table must be"),
    (dict(table=meta(3, 7, 32, 2, dtype=F32)), "table must be"), (dict(table=meta(7, 64, dtype=F32)), "table must be"),
    (dict(q_weight=meta(64)), "needs a norm"), (dict(q_weight=meta(63), norm="head"), "64 elements"),
    (dict(k_weight=meta(64), norm="row"), "192 elements"), (dict(k_weight=meta(64, dtype=torch.int8), norm="head"), "a weight must be"),
    (dict(norm="layer"), "norm must be"), (dict(pairs="quarters"), "pairs must be"),
    (dict(q=meta(2, 7, 300, 64), norm="row"), "16384")]


@pytest.mark.parametrize("change,message", REFUSED_ROPES)
def test_ropes_are_refused(rp, change, message):
    args = {"q": meta(2, 7, 6, 64), "k": meta(2, 7, 3, 64), "table": meta(7, 32, 2, dtype=F32), **change}
    with pytest.raises((RuntimeError, ValueError), match=message):
        rp.qk_norm_rope(**args)


REFUSED = [
    (dict(q=meta(2, 5, 8, 64, dtype=F32)), "q must be float16"), (dict(k=meta(2, 7, 2, 64, dtype=F16)), "q's dtype"),
    (dict(q=meta(5, 8, 64)), "must be \\(batch"), (dict(v=meta(2, 7, 2, 72)), "one shape"), (dict(k=meta(2, 7, 2, 72)), "one shape"),
    (dict(v=meta(2, 8, 2, 64)), "one shape"), (dict(k=meta(2, 7, 3, 64), v=meta(2, 7, 3, 64)), "multiple of k's"),
    (dict(k=meta(3, 7, 2, 64), v=meta(3, 7, 2, 64)), "q's batch"), (dict(scale=0.0), "positive"), (dict(scale=-0.1), "positive"),
    (dict(scale=1e-60), "positive"), (dict(scale=float("nan")), "positive"), (dict(k_lengths=meta(2, dtype=torch.int64)), "int32"),
    (dict(k_lengths=meta(3, dtype=I32)), "int32"), (dict(mask=meta(5, 7, dtype=F16)), "mask must be bool"),
    (dict(mask=meta(5, 7, dtype=torch.uint8)), "mask must be bool"), (dict(mask=meta(5, 8)), "broadcast"),
    (dict(mask=meta(2, 3, 5, 7)), "broadcast"), (dict(mask=meta(1, 2, 8, 5, 7)), "broadcast"), (dict(mask=meta()), "broadcast"),
    (dict(q=meta(2, (1 << 28) + 1, 8, 64)), "2\\^30"), (dict(k=meta(2, (1 << 30) + 1, 2, 64), v=meta(2, (1 << 30) + 1, 2, 64)), "2\\^30")]


@pytest.mark.parametrize("change,message", REFUSED)
def test_attentions_are_refused(at, change, message):
    args = {"q": meta(2, 5, 8, 64), "k": meta(2, 7, 2, 64), "v": meta(2, 7, 2, 64), **change}
    with pytest.raises(RuntimeError, match=message):
        at.attention(**args)


@pytest.mark.parametrize("change,message", [
    (dict(q=meta(1, 5, 8, 64)), "must be \\(tokens"), (dict(q_offsets=meta(4, dtype=torch.int64)), "int32"),
    (dict(q_offsets=meta(1, dtype=I32)), "int32"), (dict(q_offsets=meta(2, 2, dtype=I32)), "int32"),
    (dict(k_offsets=meta(5, dtype=I32)), "q_offsets' size"), (dict(k_offsets=None), "q's tokens"), (dict(scale=0.0), "positive")])
def test_packed_attentions_are_refused(at, change, message):
    args = {"q": meta(5, 8, 64), "k": meta(7, 2, 64), "v": meta(7, 2, 64), "q_offsets": meta(4, dtype=I32),
            "k_offsets": meta(4, dtype=I32), **change}
    with pytest.raises(RuntimeError, match=message):
        at.packed_attention(**args)


def test_cpu_tensors_raise(rp, at):
    x = torch.zeros(1, 4, 2, 64, dtype=BF16)
    for call in (lambda: rp.rope_table(torch.zeros(4, 1), (64,)), lambda: rp.norm_rope(x), lambda: rp.qk_norm_rope(x, x),
                 lambda: at.attention(x, x, x), lambda: at.packed_attention(x[0], x[0], x[0], torch.zeros(2, dtype=I32))):
        with pytest.raises(NotImplementedError):
            call()


def test_token_counts_under_compile(rp, at):
    """One graph for the first count and one for every other."""
    w = meta(64)

    def fn(q, k, pos):
        table = rp.rope_table(pos, (32, 32))
        a, b = rp.qk_norm_rope(q, k, table, q_weight=w, k_weight=w, norm="head")
        return at.attention(a[None], b[None], k[None], causal=True)

    torch._dynamo.reset()
    graphs = []

    def backend(gm, _):
        graphs.append(gm)
        return gm.forward

    compiled = torch.compile(fn, backend=backend, dynamic=None)
    for n in (5, 70, 4096, 9):
        assert compiled(meta(n, 4, 64), meta(n, 2, 64), meta(n, 2, dtype=I32)).shape == (1, n, 4, 64)
    assert len(graphs) <= 2


def test_oracle_is_the_definition():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 8))
    angles = A.rope_angles(np.array([[2, 5], [0, 1], [7, 0]]), (4, 4), 100.0)
    assert np.allclose(angles[0], [2, 0.2, 5, 0.5]) and np.allclose(A.rope_angles(np.array([[2, 5]]), (4, 4), 16.0, True), [[2, 1, 1.25, 0.625]])
    y = A.norm_rope(x, angles)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * angles)[:, None]
    assert np.allclose(y[..., 0::2], z.real) and np.allclose(y[..., 1::2], z.imag)
    h = A.norm_rope(x, angles, halves=True)
    z = (x[..., :4] + 1j * x[..., 4:]) * np.exp(1j * angles)[:, None]
    assert np.allclose(h[..., :4], z.real) and np.allclose(h[..., 4:], z.imag)
    q, k, v = rng.standard_normal((4, 2, 8)), rng.standard_normal((3, 1, 8)), rng.standard_normal((3, 1, 8))
    o, mags, _ = A.attention_one(q, k, v, causal=True)
    assert not o[0].any()  # 4 queries, 3 keys: the first sees none
    assert np.allclose(o[1], v[0]) and (mags >= np.abs(o) - 1e-12).all()
    w = np.exp(q[3, 1] @ k[:, 0].T / np.sqrt(8))
    assert np.allclose(o[3, 1], w @ v[:, 0] / w.sum())


def test_plans(lib):
    """Every form has shapes that take it, with and without a mask; keys are shared only as far as there are counters, and
    the workspace holds what is written."""
    from attention_util import FORMS

    wide = lambda D: next(w for w in (64, 96, 128, 256) if D <= w)  # noqa: E731
    every = {((w, s), D) for D in (64, 96, 128, 256) for w, s in ((0, False), (4, False), (4, True), (8, False), (8, True))
             if D < 256 or w < 8}
    for mask in (None, P):
        got = [(*plan_of(lib, attention_args(*shape, mask=mask))[:2], form, shape) for form, shape in FORMS]
        assert {((waves, splits > 1), wide(shape[5])) for waves, splits, _, shape in got} == every
        assert mask or all((waves, splits > 1) == form for waves, splits, form, _ in got), got
    rng = np.random.default_rng(1)
    for _ in range(4000):
        B, Hk, G, D = (int(rng.choice(c)) for c in ((1, 2, 7, 64, 4000), (1, 2, 5, 8, 40), (1, 2, 8), (8, 64, 96, 104, 128, 256)))
        Sq, Sk = (int(2 ** rng.uniform(0, 17)) for _ in range(2))
        args = attention_args(B, Sq, Sk, Hk * G, Hk, D, causal=int(rng.integers(2)), mask=None if rng.integers(2) else P)
        if rng.integers(2):
            args.mask, args.q_offsets, args.k_offsets = None, P, P
        waves, splits, blocks = plan_of(lib, args)
        size = lib.feather_attention_workspace_size(ctypes.byref(args))
        assert waves in (0, 4, 8) and 1 <= splits <= 64 and blocks >= 1
        if splits == 1:
            assert size == 0
        else:
            assert waves and blocks <= 16384 and size == 65536 + blocks * splits * 32 * (wide(D) + 4) * 4
        if args.q_offsets is None:
            assert blocks == (B * Hk * -(-Sq * G // 32) if waves else B * Hk * G * -(-Sq // 128))


def test_more_workgroups_than_a_launch_holds(lib):
    """2^32 threads and more are refused before a launch, in every form: few rows of 4 and of 8 waves, blocks of 128 queries."""
    for waves, shape in ((4, (65536, 1, 8, 256, 256, 64)), (8, (32768, 1, 9000, 256, 256, 64)), (0, (65536, 33, 8, 256, 256, 128))):
        args = attention_args(*shape)
        form, splits, blocks = plan_of(lib, args)
        threads = splits * blocks * 64 * (form or 4)
        assert threads >= 2 ** 32, (form, splits, blocks)
        assert form == waves
        assert lib.feather_attention(ctypes.byref(args), None, 0, None) == 2


@pytest.mark.parametrize("scale,status", [(2.0 ** 127, 0), (1e-44, 0), (2.4e38, 1), (float("inf"), 1), (float("nan"), 1), (0.0, 1)])
def test_scales(lib, at, scale, status):
    """The scale times log2(e) is an fp32 number, too: from 2^127.5 on it would be infinite, and every weight NaN."""
    plan = (ctypes.c_int64 * 3)()
    assert lib.feather_attention_plan(ctypes.byref(attention_args(1, 5, 7, 2, 2, 64, scale=scale)), plan) == status
    q = meta(1, 5, 2, 64)
    if status:
        with pytest.raises(RuntimeError, match="positive and at most"):
            at.attention(q, q, q, scale=scale)
    else:
        assert at.attention(q, q, q, scale=scale).shape == q.shape
