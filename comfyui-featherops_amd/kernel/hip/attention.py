"""Attention on the matrix cores (no counterpart in the reference).

    o = attention(q, k, v)                                   # every token of a picture over every other
    o = attention(q, k, v, k_lengths=lengths)                # over padded prompts, or a cache filled up to a length
    o = packed_attention(q, k, v, offsets, causal=True)      # prompts of different lengths, one behind the other

    o[i] = sum_j p[i][j] * v[j],    p[i] = softmax over j of scale * q[i] . k[j] + mask[i][j]

over the keys that query i may see; a query that may see none gets zeros. q and the result are (batch, tokens, heads,
head_dim), k and v (batch, tokens, kv heads, head_dim), in fp16 or bf16, head_dim a multiple of 8 up to 256;
heads / kv heads consecutive query heads share a key head. Scores, maxima and sums are fp32; the weights p are
rounded to the tensors' type, as is the result. scale is 1 / sqrt(head_dim) by default, positive and 2^127 at most; q . k and
scale times it are to stay below 2^125 in magnitude.

Which keys a query sees:
  causal     query i of n sees the keys up to i + (keys - n): the last query sees all of them;
  k_lengths  (batch,) int32: a sample's keys are its first k_lengths ones. What lies behind them is not read;
  mask       broadcast against (batch, heads, q tokens, k tokens): bool (False: not seen), or values in fp32 or
             q's type that are added to the scores (-inf: not seen).
Keys that causality or a mask takes from a query have weight zero in its sum, as in any product with a zero: their
values must be finite for it to stay so.

Views are read in place if head_dim is contiguous and tokens and heads lie on 16-byte boundaries (a layer's joint output,
heads in front of tokens, a slice of a cache), others are copied first. A call has fewer than 2^24 workgroups (128 queries of a
head each, or 32 of a group of heads; some forms 2^23) and is refused beyond. Runs in libfeatherops_amd.so on
torch's current stream; there is no other compute path. Forward only: no gradients.
"""

from __future__ import annotations

import torch

from . import _lib

_lib.load_torch_ops()
_ops = torch.ops.feather_ops
_attention = _ops.attention.default
_packed = _ops.packed_attention.default


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: float | None = None,
              k_lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of samples of one size, from one query (a decoded token, a pooling query) to all tokens of a video."""
    return _attention(q, k, v, causal, scale, k_lengths, mask)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                     k_offsets: torch.Tensor | None = None, *, causal: bool = False, scale: float | None = None) -> torch.Tensor:
    """Attention of packed sequences: q (tokens, heads, head_dim), k and v (tokens, kv heads, head_dim); sequence s has
    the tokens from offsets[s] to offsets[s + 1] (int32, on the GPU, never falling; k_offsets by default q_offsets).
    A sequence may be empty on either side. Tokens outside every sequence get zeros."""
    return _packed(q, k, v, q_offsets, k_offsets, causal, scale)
