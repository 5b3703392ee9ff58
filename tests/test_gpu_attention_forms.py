"""Attention's forms on the GPU: blocks of 128 queries, and few rows whose keys are shared by waves and workgroups, each
against float64 with every mask; the same results every time; streams, captured graphs, caches past 32-bit offsets; and
the operators one behind the other, as a layer runs them."""

import ctypes
import importlib

import numpy as np
import pytest
import torch

from attention_util import BF16, F16, F32, FORMS, HALF, AttentionArgs, attention_args, check, d, normal, plan_of, qkv
from oracle import attention_oracle as A

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.fixture(scope="module")
def at(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.attention")


@pytest.fixture(scope="module")
def rp(pkg):
    return importlib.import_module("featherops_amd.kernel.hip.rope")


@pytest.fixture(scope="module")
def lib(pkg):
    return importlib.import_module("featherops_amd.kernel.hip._lib").lib()


def mask_of(kind, g, B, H, Sq, Sk, dtype):
    if kind == "none":
        return None
    if kind == "keys":
        return (torch.rand(B, 1, 1, Sk, generator=g) < 0.7).cuda()
    if kind == "bool":
        return (torch.rand(B, 1, Sq, Sk, generator=g) < 0.7).cuda()
    m = torch.randn(B, H, Sq, Sk, generator=g) * 2.0
    m = torch.where(torch.rand(B, H, Sq, Sk, generator=g) < 0.2, float("-inf"), m)
    m[:, :, -1] = float("-inf")
    return m.to(dtype if kind == "half" else F32).cuda()


@pytest.mark.parametrize("kind", ["none", "keys", "bool", "half", "fp32"])
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(map(str, f[0])) + f"-D{f[1][5]}")
def test_forms(at, cuda, form, kind):
    B, Sq, Sk, H, Hk, D = form[1]
    if kind in ("half", "fp32") and B * H * Sq * Sk > 1 << 25:
        pytest.skip("a mask of over 100 MB")
    dtype = F16 if H % 2 else BF16
    g = torch.Generator().manual_seed(D + Sk)
    q, k, v = qkv(g, B, Sq, Sk, H, Hk, D, dtype)
    mask = mask_of(kind, g, B, H, Sq, Sk, dtype)
    lengths = torch.tensor([Sk - 41 * b for b in range(B)], dtype=I32, device=cuda)
    for causal in (False, True):
        o = at.attention(q, k, v, causal=causal, mask=mask, k_lengths=lengths)
        want = A.attention(d(q), d(k), d(v), causal, None, lengths.tolist(), d(mask))
        check(o, *want, Sk, f"{causal}", 8.0)
        for _ in range(3):
            assert torch.equal(at.attention(q, k, v, causal=causal, mask=mask, k_lengths=lengths), o)


@pytest.mark.parametrize("first", [0, 1, 2, 3])
@pytest.mark.parametrize("kind", ["bool", "half", "fp32"])
@pytest.mark.parametrize("shape", [(3, 1101, 157, 16, 16, 40), (2, 9, 301, 4, 2, 128)], ids=["tiles", "rows"])
def test_mask_alignment(at, cuda, shape, kind, first):
    """Rows that begin at any element, odd and even distances between them, and what lies around them of another sign."""
    B, Sq, Sk, H, Hk, D = shape
    g = torch.Generator().manual_seed(first)
    q, k, v = qkv(g, B, Sq, Sk, H, Hk, D, F16)
    for width in (Sk + 4, Sk + 7):
        if kind == "bool":
            whole = torch.zeros(Sq, width, dtype=torch.bool)
            whole[:, first:first + Sk] = torch.rand(Sq, Sk, generator=g) < 0.7
        else:
            whole = torch.full((Sq, width), float("nan"))
            whole[:, first:first + Sk] = torch.randn(Sq, Sk, generator=g) * 2.0
            whole = whole.to(F16 if kind == "half" else F32)
        mask = whole.cuda()[:, first:first + Sk]
        for causal in (False, True):
            o = at.attention(q, k, v, mask=mask, causal=causal)
            check(o, *A.attention(d(q), d(k), d(v), causal, None, None, d(mask[None, None])), Sk, f"{width} {causal}", 8.0)


@pytest.mark.parametrize("D", [64, 128, 200])
def test_packed_tokens_over_long_caches(at, cuda, D):
    """One and few queries a sequence, whose keys workgroups share; a sequence without keys, one without queries."""
    g = torch.Generator().manual_seed(D)
    for q_lens, k_lens in (([1, 1, 0, 1], [5000, 0, 3, 9000]), ([3, 1, 2], [8192, 31, 4097])):
        qo, ko = np.concatenate(([0], np.cumsum(q_lens))), np.concatenate(([0], np.cumsum(k_lens)))
        q, k, v = (normal(g, n, h, D) for n, h in ((qo[-1], 8), (ko[-1], 2), (ko[-1], 2)))
        offsets = [torch.tensor(o, dtype=I32, device=cuda) for o in (qo, ko)]
        for causal in (False, True):
            o = at.packed_attention(q, k, v, *offsets, causal=causal)
            check(o, *A.packed_attention(d(q), d(k), d(v), qo, ko, causal), max(k_lens), f"{causal}")
            assert torch.equal(at.packed_attention(q, k, v, *offsets, causal=causal), o)


def test_entry_with_and_without_workspace(lib, cuda):
    """The C entry: without a workspace, or with one that is too small, no keys are shared; with one its counters are zero
    again behind every call."""
    B, Sq, Sk, H, Hk, D = 2, 1, 9000, 8, 2, 128
    g = torch.Generator().manual_seed(2)
    q, k, v = qkv(g, B, Sq, Sk, H, Hk, D, BF16)
    args = attention_args(B, Sq, Sk, H, Hk, D)
    want = A.attention(d(q), d(k), d(v), scale=args.scale)
    out = torch.empty_like(q)
    args.q, args.k, args.v, args.out = (t.data_ptr() for t in (q, k, v, out))
    size = lib.feather_attention_workspace_size(ctypes.byref(args))
    assert size > 65536 and plan_of(lib, args)[1] > 1
    ws = torch.zeros(size, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    for space, n in ((None, 0), (ws.data_ptr(), size), (ws.data_ptr(), size - 1), (ws.data_ptr(), size)):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        assert lib.feather_attention(ctypes.byref(args), space, n, None) == 0
        torch.cuda.synchronize()
        check(out, *want, Sk, f"{n}")
        assert not ws[:65536].any()


def test_streams(at, cuda):
    """Calls on other streams than the default one, two at once, each with a workspace of its own."""
    g = torch.Generator().manual_seed(4)
    sets = [qkv(g, 1, 2, 12000, 8, 2, 128, BF16) for _ in range(2)]
    want = [at.attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(at.attention(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_captured(at, rp, cuda):
    """A step of a decoder in a graph: positions of new tokens, attention over the cache up to lengths that lie in memory,
    twice; another graph of the same stream beside it; eager calls between the replays."""
    g = torch.Generator().manual_seed(5)
    B, H, Hk, D, room = 3, 8, 2, 128, 6000
    x = normal(g, B, 1, H + 2 * Hk, D)
    cache = normal(g, 2, B, room, Hk, D)
    lengths = torch.tensor([17, 3500, 6000], dtype=I32, device=cuda)

    def step():
        table = rp.rope_table((lengths - 1).view(B, 1, 1), (D,))
        q, k = rp.qk_norm_rope(x[:, :, :H], x[:, :, H:H + Hk], table, norm="head")
        index = (lengths.long() - 1).view(B, 1, 1, 1).expand(B, 1, Hk, D)
        cache[0].scatter_(1, index, k)
        cache[1].scatter_(1, index, x[:, :, H + Hk:])
        first = at.attention(q, cache[0], cache[1], k_lengths=lengths)
        return first, at.attention(first, cache[0], cache[1], k_lengths=lengths)

    def prompt():
        return at.attention(x[:, :, :H].expand(B, 300, H, D), cache[0], cache[1], k_lengths=lengths)

    before = cache.clone()
    for fn in (step, prompt):
        fn()
    graphs = []
    for fn in (step, prompt):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn()
        graphs.append((graph, out if isinstance(out, tuple) else (out,), fn))
    for i in range(4):
        x.copy_(normal(g, B, 1, H + 2 * Hk, D))
        lengths.copy_(torch.tensor([18 + i, 3000 + 700 * i, 6000 - 1500 * i], dtype=I32))  # (1 to room)
        cache.copy_(before)
        for graph, out, fn in graphs:
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in out]
            want = fn()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want if isinstance(want, tuple) else (want,)))
    streams = [torch.cuda.Stream() for _ in graphs]
    want = [[o.clone() for o in out] for _, out, _ in graphs]
    torch.cuda.synchronize()
    for (graph, _, _), s in zip(graphs[:1], streams):  # a replay beside eager calls of the same form on another stream
        with torch.cuda.stream(s):
            for _ in range(5):
                graph.replay()
    other = qkv(g, 1, 1, 9000, 8, 2, 128, BF16)
    beside = [at.attention(*other) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], want[0]))
    assert all(torch.equal(b, beside[0]) for b in beside)


@pytest.mark.parametrize("Sq", [1, 130])
def test_cache_past_32_bits(at, cuda, Sq):
    """Keys and values of 4.9 GB, a token's beside each other: two keys far back take all the weight, each half of it."""
    tokens, Hk, D = 1_200_003, 8, 128
    cache = torch.zeros(1, tokens, 2, Hk, D, dtype=BF16, device=cuda)
    k, v = cache[:, :, 0], cache[:, :, 1]
    q = torch.full((1, Sq, Hk, D), 4.0, dtype=BF16, device=cuda)
    k[:, tokens - 3], k[:, tokens - 70_000] = 4.0, 4.0  # scores of 181, the others 0
    v[:, tokens - 3], v[:, tokens - 70_000] = 3.0, 5.0
    o = at.attention(q, k, v)
    assert (o == 4.0).all()
    o = at.attention(q, k, v, k_lengths=torch.tensor([tokens - 3], dtype=I32, device=cuda))
    assert (o == 5.0).all()
    offsets = [torch.tensor(t, dtype=I32, device=cuda) for t in ([0, Sq], [tokens - 50_000, tokens])]
    o = at.packed_attention(q[0], k[0], v[0], *offsets)
    assert (o == 3.0).all()


def test_mask_past_32_bits(at, cuda):
    """A mask of 2.4 GB that leaves one key to each query."""
    Sq, Sk = 4000, 600_000
    g = torch.Generator().manual_seed(6)
    q, k, v = qkv(g, 1, Sq, Sk, 1, 1, 64, BF16)
    key = torch.randint(0, Sk, (Sq,), generator=g).cuda()
    mask = torch.zeros(1, 1, Sq, Sk, dtype=torch.bool, device=cuda)
    mask[0, 0].scatter_(1, key[:, None], True)
    o = at.attention(q, k, v, mask=mask)
    assert torch.equal(o[0, :, 0], v[0, key, 0])


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_layer(at, rp, cuda, dtype, halves):
    """A layer's run of them: the joint projection's slices normed and turned, attended where they lie; then token by token
    over a cache that is filled as they come, against the whole causal sequence."""
    g = torch.Generator().manual_seed(8)
    B, S, H, Hk, D = 2, 133, 6, 2, 64
    joint = normal(g, B, S, H + 2 * Hk, D, dtype=dtype)
    q, k, v = joint.split((H, Hk, Hk), 2)
    qw, kw = (normal(g, D, dtype=dtype, std=0.2) + 1 for _ in range(2))
    positions = torch.arange(S, device=cuda)[:, None]
    table, angles = rp.rope_table(positions, (D,)), A.rope_angles(d(positions), (D,))
    pairs = "halves" if halves else "adjacent"
    u = HALF[dtype]
    for causal in (False, True):
        nq, nk = rp.qk_norm_rope(q, k, table, q_weight=qw, k_weight=kw, norm="head", pairs=pairs)
        o = at.attention(nq, nk, v, causal=causal)
        want_q, want_k = (A.norm_rope(d(t), angles, d(w), "head", 1e-6, halves) for t, w in ((q, qw), (k, kw)))
        want, mags, reach = A.attention(want_q, want_k, d(v), causal)
        # q and k are off by u each (and their fp32 arithmetic by far less than 2^-18), so a score by 2.1 u |q||k|,
        # a weight and the sum of them by a factor exp of that each, at most
        slack = np.expm1(2 * 2.1 * (u + 2.0 ** -18) * reach) * (mags + np.abs(want))
        off = np.abs(d(o) - want)
        assert (off <= slack + (2 * u + 2.0 ** -12) * (mags + np.abs(want)) + 2.0 ** -20).all()
    cache = torch.full((2, B, S + 20, Hk, D), float("nan"), dtype=dtype, device=cuda)
    for t in range(S):
        nq, nk = rp.qk_norm_rope(q[:, t:t + 1], k[:, t:t + 1], table[t:t + 1], q_weight=qw, k_weight=kw, norm="head", pairs=pairs)
        cache[0, :, t:t + 1], cache[1, :, t:t + 1] = nk, v[:, t:t + 1]
        one = at.attention(nq, cache[0], cache[1], k_lengths=torch.full((B,), t + 1, dtype=I32, device=cuda))
        off = np.abs(d(one[:, 0]) - want[:, t])
        assert (off <= slack[:, t] + (2 * u + 2.0 ** -12) * (mags[:, t] + np.abs(want[:, t])) + 2.0 ** -20).all(), t


def test_example_attention_half(pkg, cuda):
    """The example block's attention half runs, near its bf16 library form."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "comfyui-featherops_amd"))
    try:
        example = importlib.import_module("example_mxfp4_block")
    finally:
        sys.path.pop(0)
    rope = importlib.import_module("featherops_amd.kernel.hip.rope")
    with torch.inference_mode():
        plain, half = example.build_attention(256, 64)
        table = rope.rope_table(example.positions(33), (16, 24, 24))
        x, h, gate, scale, shift = example.inputs(33, 256)
        s, y = half(x, h, gate, scale, shift, table)
        want_s, want = plain(x, h, gate, scale, shift, table)
    # 4 bits a value: an error of 2^-3 of a value at most in either operand of each of two products, most of it averaged away
    assert torch.allclose(s.float(), want_s.float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    assert (y.float() - want.float()).norm() <= 0.5 * want.float().norm()
