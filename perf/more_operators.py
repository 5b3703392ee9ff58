"""What the attention operators are timed on: rotary positions with the norm of queries and keys, and attention.

Two kinds of pass:

* "rope": queries and keys of a layer, normalised (each head by itself, or a token's heads together) and turned by their
          positions (`qk_norm_rope`). A position has one coordinate for text, two or three (time, height, width) for
          images and video; each turns its own part of a head. The cosines and sines are kept between layers and
          steps ("kept"), or made in the pass for positions that are new (`rope_table`; "made");
* "attn": attention of queries over keys and values (`attention`), or over packed sequences that lie one behind the
          other (`packed_attention`). Query heads share key heads in groups; keys are limited by causality, by a sample's
          length, by a mask of truth values or by a bias on the scores.

Tokens: one for a decoded token or a pooling query, tens to hundreds for prompts, thousands and tens of thousands for
image and video latents.
"""

import importlib
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = "featherops_amd"
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6
#: the most that a drawn case may cost: products of the largest listed attention, values of the largest listed rope
_MOST_PAIRS = 12 * 32760 * 32760 * 128
_MOST_VALUES = 2 * 32760 * 40 * 128


def _module(name):
    """A module of the plugin package (its folder's name is not a Python identifier)."""
    if _PKG not in sys.modules:
        folder = Path(__file__).resolve().parents[1] / "comfyui-featherops_amd"
        spec = importlib.util.spec_from_file_location(_PKG, folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        package = importlib.util.module_from_spec(spec)
        sys.modules[_PKG] = package
        spec.loader.exec_module(package)
    return importlib.import_module(f"{_PKG}.{name}")


def listed():
    return [
        # one decoded token's queries and keys, its position new in every step
        {"name": "rope_token", "kind": "rope", "B": 1, "S": 1, "H": 32, "G": 4, "D": 128, "axes": "128", "x": "bf16",
         "norm": "head", "weight": True, "pairs": "halves", "table": "made"},
        # an image's patches in a vision encoder: two coordinates, no norm, odd sizes, positions of a new picture
        {"name": "rope_ragged", "kind": "rope", "B": 3, "S": 1003, "H": 15, "G": 1, "D": 80, "axes": "40,40", "x": "fp16",
         "norm": "", "weight": False, "pairs": "halves", "table": "made"},
        # an image model's joint tokens, each head normalised, three coordinates
        {"name": "rope_image", "kind": "rope", "B": 2, "S": 4250, "H": 24, "G": 1, "D": 128, "axes": "16,56,56", "x": "bf16",
         "norm": "head", "weight": True, "pairs": "adjacent", "table": "kept"},
        # a video's tokens, all heads of a token normalised together
        {"name": "rope_video", "kind": "rope", "B": 1, "S": 32760, "H": 40, "G": 1, "D": 128, "axes": "44,42,42", "x": "bf16",
         "norm": "row", "weight": True, "pairs": "adjacent", "table": "kept"},
        # a pooling query over one picture's patches: the smallest attention
        {"name": "attn_pool", "kind": "attn", "form": "batch", "B": 1, "Sq": 1, "Sk": 729, "H": 16, "G": 1, "D": 72,
         "x": "fp16", "causal": False, "lens": "", "mask": ""},
        # one decoded token over a long cache
        {"name": "attn_token", "kind": "attn", "form": "batch", "B": 1, "Sq": 1, "Sk": 32768, "H": 32, "G": 4, "D": 128,
         "x": "bf16", "causal": True, "lens": "32001", "mask": ""},
        # several prompts, each with its own next token
        {"name": "attn_tokens", "kind": "attn", "form": "batch", "B": 8, "Sq": 1, "Sk": 4096, "H": 40, "G": 5, "D": 128,
         "x": "bf16", "causal": True, "lens": "4096,1,333,2048,4001,77,1003,0", "mask": ""},
        # prompts of different lengths through a text encoder, packed, an empty one among them
        {"name": "attn_prompts", "kind": "attn", "form": "packed", "H": 28, "G": 7, "D": 128, "x": "bf16", "causal": True,
         "q_lens": "77,154,1,0,333,512", "k_lens": ""},
        # a text encoder with a learned bias on the scores, sizes that are multiples of no tile
        {"name": "attn_bias", "kind": "attn", "form": "batch", "B": 2, "Sq": 1003, "Sk": 1003, "H": 16, "G": 1, "D": 64,
         "x": "bf16", "causal": False, "lens": "", "mask": "bias"},
        # a video's tokens over two padded prompts
        {"name": "attn_cross", "kind": "attn", "form": "batch", "B": 2, "Sq": 8190, "Sk": 512, "H": 40, "G": 1, "D": 128,
         "x": "bf16", "causal": False, "lens": "", "mask": "keys"},
        # long documents, packed, causal, grouped heads
        {"name": "attn_packed", "kind": "attn", "form": "packed", "H": 32, "G": 4, "D": 128, "x": "fp16", "causal": True,
         "q_lens": "8191,1,4096,2047,1000", "k_lens": ""},
        # every token of a video over every other
        {"name": "attn_video", "kind": "attn", "form": "batch", "B": 1, "Sq": 32760, "Sk": 32760, "H": 12, "G": 1, "D": 128,
         "x": "bf16", "causal": False, "lens": "", "mask": ""},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _numbers(text):
    return [int(n) for n in text.split(",")] if text else []


def _draw_rope(rng):
    D = rng.choice([64, 72, 80, 96, 128, 128, 128, 256])
    quarter = D // 8 * 2
    axes = rng.choice([[D], [D // 2, D - D // 2], [D - 2 * quarter, quarter, quarter], [quarter, quarter]])
    case = {"kind": "rope", "B": rng.choice([1, 1, 2, 3]), "S": _log_int(rng, 1, 32768), "G": rng.choice([1, 1, 2, 4, 7]),
            "D": D, "axes": ",".join(str(a) for a in axes), "x": rng.choice(["fp16", "bf16", "bf16", "fp32"]),
            "norm": rng.choice(["", "head", "head", "row"]), "pairs": rng.choice(["adjacent", "halves"]),
            "table": rng.choice(["made", "kept", "kept"])}
    case["H"] = case["G"] * rng.randint(1, max(1, 40 // case["G"]))
    case["weight"] = case["norm"] != "" and rng.random() < 0.8
    return case


def _draw_attn(rng):
    case = {"kind": "attn", "form": rng.choice(["batch", "batch", "packed"]), "G": rng.choice([1, 1, 2, 4, 7, 8]),
            "D": rng.choice([40, 64, 72, 80, 96, 128, 128, 128, 128, 256]), "x": rng.choice(["fp16", "bf16", "bf16"]),
            "causal": rng.random() < 0.4}
    case["H"] = case["G"] * rng.randint(1, max(1, 40 // case["G"]))
    if case["form"] == "packed":
        count = rng.randint(1, 9)
        lengths = [rng.choice([0, 1, _log_int(rng, 1, 8192), _log_int(rng, 16, 2048)]) for _ in range(count)]
        case["q_lens"] = ",".join(str(n) for n in lengths + [_log_int(rng, 1, 4096)])
        case["k_lens"] = ""
        if rng.random() < 0.3:  # other lengths on the other side: a prompt for each picture, or a prefix in front
            case["k_lens"] = ",".join(str(rng.choice([0, n, _log_int(rng, 1, 4096)])) for n in _numbers(case["q_lens"]))
        return case
    B = case["B"] = rng.choice([1, 1, 2, 3, 8])
    case["Sk"] = _log_int(rng, 1, 32768)
    case["Sq"] = rng.choice([1, case["Sk"], case["Sk"], _log_int(rng, 1, 32768)])
    case["lens"] = ",".join(str(rng.choice([0, case["Sk"], rng.randint(0, case["Sk"])])) for _ in range(B)) if rng.random() < 0.3 else ""
    case["mask"] = rng.choice(["", "", "", "keys", "bias"])
    return case


def _cost_fits(case):
    if case["kind"] == "rope":
        return 2 * case["B"] * case["S"] * case["H"] * case["D"] <= _MOST_VALUES
    # (a bias is held for every pair: no more than 2 GiB of it)
    if case.get("mask") == "bias" and case["H"] * case["Sq"] * case["Sk"] > 1 << 30:
        return False
    return work(case)["flops"] <= 4 * _MOST_PAIRS and work(case)["bytes"] <= 1 << 31


def draw(rng):
    one = rng.choice([_draw_rope, _draw_attn, _draw_attn])
    case = one(rng)
    while not _cost_fits(case):
        case = one(rng)
    return case


# ---- inputs ----

def _positions(case, gen, dev):
    """(S, axes) whole numbers: a text's places, or the places of patches in a picture or a video, row by row."""
    S, count = case["S"], len(_numbers(case["axes"]))
    start = torch.randint(0, 4096, (1,), generator=gen, device=dev)
    n = torch.arange(S, device=dev)
    if count == 1:
        return (n + start)[:, None]
    width = max(1, int(S ** (1.0 / count)))
    at = [n // width ** (count - 1 - i) % (width if i else 1 << 30) for i in range(count)]
    at[0] = at[0] + start
    return torch.stack(at, dim=1)


def _inputs(case, seed):
    """Plain tensors on the GPU, from the seed alone. Queries and keys as a layer leaves them: a few channels of a head
    louder than the others, keys off centre; values of a layer's size."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, H, G, D = _DTYPES[case["x"]], case["H"], case["G"], case["D"]

    def loud(*shape, std=1.0, centre=0.0):
        channels = 1.0 + 3.0 * (torch.rand(shape[-1], generator=gen, device=dev) < 0.05)
        mean = torch.randn(shape[-1], generator=gen, device=dev) * centre
        t = torch.empty(shape, dtype=dtype, device=dev)
        for part in t.flatten(0, -3).split(max(1, (1 << 27) // (shape[-1] * shape[-2]))):
            part.copy_(torch.randn(part.shape, generator=gen, device=dev).mul_(channels).add_(mean).mul_(std))
        return t

    if case["kind"] == "rope":
        B, S = case["B"], case["S"]
        heads = H + 2 * (H // G)  # what one layer makes for queries, keys and values lies together
        qkv = loud(B, S, heads, D, std=1.5, centre=0.3)
        t = {"q": qkv[:, :, :H], "k": qkv[:, :, H:H + H // G], "positions": _positions(case, gen, dev)}
        width = {"": D, "head": D, "row": H * D}[case["norm"]]
        for name, n in (("q_weight", width), ("k_weight", width if case["norm"] != "row" else H // G * D)):
            weight = (torch.randn(n, generator=gen, device=dev) * 0.2 + 1.0).to(dtype)
            t[name] = weight if case["weight"] else None
        return t
    if case["form"] == "packed":
        q_lens = _numbers(case["q_lens"])
        k_lens = _numbers(case["k_lens"]) or q_lens
        t = {"q": loud(sum(q_lens), H, D), "k": loud(sum(k_lens), H // G, D, centre=0.5), "v": loud(sum(k_lens), H // G, D)}
        for name, lens in (("q_offsets", q_lens), ("k_offsets", k_lens)):
            ends = torch.tensor([0, *lens], dtype=torch.int64).cumsum(0)
            t[name] = ends.to(device=dev, dtype=torch.int32)
        return t
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    t = {"q": loud(B, Sq, H, D), "k": loud(B, Sk, H // G, D, centre=0.5), "v": loud(B, Sk, H // G, D), "mask": None,
         "k_lengths": None}
    if case["lens"]:
        t["k_lengths"] = torch.tensor(_numbers(case["lens"]), dtype=torch.int32, device=dev)
    if case["mask"] == "keys":  # padded prompts: keys up to a length of its own for every sample
        kept = torch.randint(Sk // 4, Sk + 1, (B, 1, 1, 1), generator=gen, device=dev)
        t["mask"] = torch.arange(Sk, device=dev).view(1, 1, 1, Sk) < kept
    elif case["mask"] == "bias":  # learned, by head and by distance, the same for all samples
        near = torch.randn(H, 64, generator=gen, device=dev)
        far = (torch.arange(Sq, device=dev)[:, None] - torch.arange(Sk, device=dev)[None, :]).abs().add_(1).float().log2_()
        t["mask"] = near.to(dtype)[:, (far * 4.0).long().clamp_(max=63)][None]
    return t


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case, kind=case["kind"])
    if case["kind"] == "rope":
        state["axes"] = tuple(_numbers(case["axes"]))
        if case["table"] == "kept":
            state["table"] = _plain_table(state["positions"], state["axes"])
    if own:
        state["rope"], state["attention"] = _module("kernel.hip.rope"), _module("kernel.hip.attention")
        if "table" in state:
            state["table"] = state["rope"].rope_table(state["positions"], state["axes"])
    elif case["kind"] == "attn" and case["form"] == "packed":
        state["q_lens"] = _numbers(case["q_lens"])
        state["k_lens"] = _numbers(case["k_lens"]) or state["q_lens"]
    return state


# ---- plain forms ----

def _plain_table(positions, axes):
    """(S, pairs, 2): cosine and sine of each pair's angle; angles in 64 bits."""
    angles = []
    for i, d in enumerate(axes):
        ladder = torch.arange(0, d, 2, dtype=torch.float64, device=positions.device) / d
        angles.append(positions[:, i:i + 1].double() * torch.exp(ladder * -math.log(10000.0)))
    angles = torch.cat(angles, dim=1)
    return torch.stack((angles.cos(), angles.sin()), dim=2).float()


def _plain_rope(x, weight, table, case):
    v = x.float()
    if case["norm"] == "row":
        v = v.flatten(2)
    if case["norm"]:
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
        if weight is not None:
            v = v * weight.float()
    v = v.view(x.shape)
    pairs = table.shape[-2]
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]  # against (B, S, heads, pairs)
    if case["pairs"] == "adjacent":
        a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, v[..., 2 * pairs:]), dim=-1).to(x.dtype)


def _plain_attention(q, k, v, causal, length=None, mask=None):
    """One sample or sequence: q (Sq, H, D), k and v (Sk, heads that groups share, D), mask (1 or H, 1 or Sq, Sk)."""
    Sq, H, D = q.shape
    Sk, shared, _ = k.shape
    out = torch.zeros_like(q)
    if Sq == 0 or Sk == 0:
        return out
    G = H // shared
    places = torch.arange(Sk, device=q.device)
    if length is None:
        length = Sk
    rows_at_once = max(1, min(Sq, (1 << 30) // (G * Sk)))
    heads_at_once = max(1, (1 << 30) // (G * rows_at_once * Sk))
    for h in range(0, shared, heads_at_once):
        n = min(heads_at_once, shared - h)
        kt = k[:, h:h + n].float().permute(1, 2, 0).contiguous()
        vs = v[:, h:h + n].float().transpose(0, 1).contiguous()
        for r in range(0, Sq, rows_at_once):
            rows = min(rows_at_once, Sq - r)
            qs = q[r:r + rows, h * G:(h + n) * G].float().transpose(0, 1).reshape(n, G * rows, D)
            s = torch.bmm(qs, kt).view(n * G, rows, Sk) * D ** -0.5
            seen = None
            if mask is not None:
                part = mask[h * G:(h + n) * G] if mask.shape[0] > 1 else mask
                part = part[:, r:r + rows] if part.shape[1] > 1 else part
                if part.dtype == torch.bool:
                    seen = part
                else:
                    s = s + part.float()
            if causal:
                last = torch.arange(r, r + rows, device=q.device)[:, None] + length - Sq
                below = (places <= last)[None]
                seen = below if seen is None else seen & below
            if not isinstance(length, int):
                seen = (places < length) if seen is None else seen & (places < length)
            if seen is not None:
                s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            s = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = s.sum(-1, keepdim=True)
            o = torch.bmm(s.view(n, G * rows, Sk), vs).view(n * G, rows, D) / torch.where(total == 0.0, 1.0, total)
            out[r:r + rows, h * G:(h + n) * G] = o.transpose(0, 1).to(q.dtype)
    return out


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["kind"] == "rope":
        table = state["table"] if case["table"] == "kept" else _plain_table(state["positions"], state["axes"])
        return [_plain_rope(state["q"], state["q_weight"], table, case), _plain_rope(state["k"], state["k_weight"], table, case)]
    q, k, v = state["q"], state["k"], state["v"]
    if case["form"] == "packed":
        parts = zip(q.split(state["q_lens"]), k.split(state["k_lens"]), v.split(state["k_lens"]))
        return torch.cat([_plain_attention(*part, case["causal"]) for part in parts])
    out = torch.empty_like(q)
    for b in range(case["B"]):
        mask = state["mask"]
        if mask is not None:
            mask = mask[b if mask.shape[0] > 1 else 0]
        length = state["k_lengths"][b] if case["lens"] else None
        out[b] = _plain_attention(q[b], k[b], v[b], case["causal"], length, mask)
    return out


def _run_own(state, case):
    if case["kind"] == "rope":
        rope = state["rope"]
        table = state["table"] if case["table"] == "kept" else rope.rope_table(state["positions"], state["axes"])
        return list(rope.qk_norm_rope(state["q"], state["k"], table, q_weight=state["q_weight"], k_weight=state["k_weight"],
                                      norm=case["norm"] or None, eps=_EPS, pairs=case["pairs"]))
    q, k, v = state["q"], state["k"], state["v"]
    if case["form"] == "packed":
        offsets = (state["q_offsets"], state["k_offsets"]) if case["k_lens"] else (state["q_offsets"],)
        return state["attention"].packed_attention(q, k, v, *offsets, causal=case["causal"])
    return state["attention"].attention(q, k, v, causal=case["causal"], k_lengths=state["k_lengths"], mask=state["mask"])


# ---- what a pass cannot do without ----

def _seen_pairs(Sq, Sk, length, causal):
    """Pairs of a query and a key that it may see."""
    if not causal:
        return Sq * length
    first = length - Sq + 1  # what the first query sees
    if first >= 0:
        return Sq * (first + length) // 2
    return length * (length + 1) // 2


def work(case):
    size, H, shared, D = _DTYPES[case["x"]].itemsize, case["H"], case["H"] // case["G"], case["D"]
    if case["kind"] == "rope":
        tokens, pairs = case["B"] * case["S"], sum(_numbers(case["axes"])) // 2
        table = case["S"] * (pairs * 8 if case["table"] == "kept" else 8 * len(_numbers(case["axes"])))
        return {"bytes": 2 * tokens * (H + shared) * D * size + table, "flops": 10 * tokens * (H + shared) * D}
    if case["form"] == "packed":
        q_lens = _numbers(case["q_lens"])
        k_lens = _numbers(case["k_lens"]) or q_lens
        pairs = sum(_seen_pairs(q, k, k, case["causal"]) for q, k in zip(q_lens, k_lens))
        queries, keys, extra = sum(q_lens), sum(k_lens), 0
    else:
        B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
        lens = _numbers(case["lens"]) or [Sk] * B
        pairs = sum(_seen_pairs(Sq, Sk, n, case["causal"]) for n in lens)
        queries, keys = B * Sq, sum(lens)
        extra = {"": 0, "keys": B * Sk, "bias": H * Sq * Sk * size}[case["mask"]]
    return {"bytes": 2 * queries * H * D * size + 2 * keys * shared * D * size + extra, "flops": 4 * pairs * H * D}


# ---- the definitions, in 64 bits ----

def _exact_rope(x, weight, positions, case):
    B, S, H, D = x.shape
    y = x.double().clone()
    if case["norm"] == "head":
        y /= (y.pow(2).sum(3, keepdim=True) / D + _EPS).sqrt()
        if weight is not None:
            y *= weight.double()
    elif case["norm"] == "row":
        y /= (y.pow(2).sum((2, 3), keepdim=True) / (H * D) + _EPS).sqrt()
        if weight is not None:
            y *= weight.double().view(H, D)
    axes = _numbers(case["axes"])
    half, p = sum(axes) // 2, 0
    for axis, d in enumerate(axes):
        for j in range(d // 2):
            at = positions[:, axis].double() * 10000.0 ** (-2 * j / d)
            turn = torch.polar(torch.ones_like(at), at)[None, :, None]
            one, two = (2 * p, 2 * p + 1) if case["pairs"] == "adjacent" else (p, p + half)
            turned = torch.complex(y[..., one], y[..., two]) * turn
            y[..., one], y[..., two] = turned.real, turned.imag
            p += 1
    return y


def _exact_attention(q, k, v, causal, length=None, mask=None):
    Sq, H, D = q.shape
    out = torch.zeros(Sq, H, D, dtype=torch.float64, device=q.device)
    keys = k.shape[0] if length is None else length
    if keys == 0:
        return out
    for h in range(H):
        kd, vd = k[:keys, h * k.shape[1] // H].double(), v[:keys, h * k.shape[1] // H].double()
        kt = kd.t().contiguous()
        for r in range(0, Sq, 8192):
            s = torch.mm(q[r:r + 8192, h].double(), kt).div_(math.sqrt(D))
            if mask is not None:
                m = mask[h % mask.shape[0]].expand(Sq, -1)[r:r + 8192, :keys]
                s = s.masked_fill_(~m, -math.inf) if m.dtype == torch.bool else s.add_(m.double())
            if causal:
                hidden = torch.ones_like(s, dtype=torch.bool).triu_(1 + r + keys - Sq)
                s.masked_fill_(hidden, -math.inf)
            p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True)).nan_to_num_(0.0)  # (a row that sees nothing)
            out[r:r + 8192, h] = torch.mm(p, vd)
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "rope":
        return [_exact_rope(t[n], t[n + "_weight"], t["positions"], case) for n in ("q", "k")]
    if case["form"] == "packed":
        q_lens = _numbers(case["q_lens"])
        out, q0, k0 = [], 0, 0
        for nq, nk in zip(q_lens, _numbers(case["k_lens"]) or q_lens):
            out.append(_exact_attention(t["q"][q0:q0 + nq], t["k"][k0:k0 + nk], t["v"][k0:k0 + nk], case["causal"]))
            q0, k0 = q0 + nq, k0 + nk
        return torch.cat(out)
    lens = _numbers(case["lens"]) or [None] * case["B"]
    return torch.stack([_exact_attention(t["q"][b], t["k"][b], t["v"][b], case["causal"], lens[b],
                                         None if t["mask"] is None else t["mask"][b % t["mask"].shape[0]])
                        for b in range(case["B"])])
