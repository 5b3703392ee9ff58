"""Rotary positions of several axes, with the norm of queries and keys (no counterpart in the reference).

    table = rope_table(positions, (16, 56, 56))          # once for a picture's or a video's positions
    q, k = qk_norm_rope(q, k, table, q_weight=wq, k_weight=wk, norm="head")

A position has one coordinate for text, and two or three (time, height, width) for images and video. Each axis turns its
own part of a head: of the head's pairs of values the first axes[0] / 2 belong to the first axis, the next
axes[1] / 2 to the second. Pair j of an axis turns by the angle position * theta^(-2 j / axes[i]); with
ladder="shared" by position * theta^(-2 p / sum(axes)), p counting the pairs of all axes. Angles are fp64,
cosines and sines fp32.

A pair is values 2 p and 2 p + 1 of a head (pairs="adjacent") or p and P + p, P being the number of pairs
(pairs="halves"); values from 2 P on are not turned. Before it, norm="head" divides each head by
sqrt(mean(x^2) + eps) and multiplies by a weight (head_dim,); norm="row" does so with all heads of a token
together and a weight (heads * head_dim,). Everything is fp32 from the inputs to the results, which are
rounded once to their type: fp16, bf16 or fp32.

Tensors are (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), slices of a larger tensor (a layer's joint
output) included, with a head_dim of a multiple of 8 up to 256. Results are contiguous. Runs in
libfeatherops_amd.so on torch's current stream; there is no other compute path. Forward only: no gradients.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _lib

_lib.load_torch_ops()
_ops = torch.ops.feather_ops
_table = _ops.rope_table.default
_norm_rope = _ops.norm_rope.default
_qk_norm_rope = _ops.qk_norm_rope.default

_LADDERS = {"axis": False, "shared": True}
_NORMS = {None: 0, "head": 1, "row": 2}
_PAIRS = {"adjacent": False, "halves": True}


def _one_of(choices: dict, value, what: str):
    if value not in choices:
        raise ValueError(f"{what} must be one of {list(choices)}, got {value!r}")
    return choices[value]


def rope_table(positions: torch.Tensor, axes: Sequence[int], theta: float = 10000.0, *, ladder: str = "axis") -> torch.Tensor:
    """Cosines and sines (..., P, 2), fp32, for positions (..., len(axes)), whole or fp32 / fp64 numbers; axes holds
    how many of a head's values each axis turns (even, 256 at most together)."""
    return _table(positions, axes, theta, _one_of(_LADDERS, ladder, "ladder"))


def norm_rope(x: torch.Tensor, table: torch.Tensor | None = None, *, weight: torch.Tensor | None = None,
              norm: str | None = None, eps: float = 1e-6, pairs: str = "adjacent") -> torch.Tensor:
    """x normalised and turned; table (tokens, P, 2), or one for each sample, or None for the norm alone."""
    return _norm_rope(x, table, weight, _one_of(_NORMS, norm, "norm"), eps, _one_of(_PAIRS, pairs, "pairs"))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, norm: str | None = None, eps: float = 1e-6,
                 pairs: str = "adjacent") -> tuple[torch.Tensor, torch.Tensor]:
    """norm_rope of queries and keys of the same tokens in one launch; their numbers of heads may differ."""
    return _qk_norm_rope(q, k, table, q_weight, k_weight, _one_of(_NORMS, norm, "norm"), eps, _one_of(_PAIRS, pairs, "pairs"))
