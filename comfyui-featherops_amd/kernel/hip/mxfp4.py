"""Linear algebra in microscaled 4-bit floating point (no counterpart in the reference).

MXFP4 holds 32 consecutive values of a row as 4-bit codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign)
under one power of two, 2^(floor(log2(largest magnitude)) - 2); include/featherops_amd.h has the
exact rules and the packed layout that the matrix instructions read. A block of 32 values with a
NaN or an infinity becomes NaN as a whole.

    w = quantize_mxfp4(weight)                   # or prepack_mxfp4(codes, scales) from a checkpoint
    y = mxfp4_mm(x, w, bias)                     # x in 16 bits is quantised in the call
    y = mxfp4_mm(quantize_mxfp4(x), w, bias)     # the same values; one quantised x for several weights

All of it runs in libfeatherops_amd.so on torch's current stream; there is no other compute path.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_lib.load_torch_ops()
_ops = torch.ops.feather_ops
_quantize = _ops.quantize_mxfp4.default
_dequantize = _ops.dequantize_mxfp4.default
_prepack = _ops.prepack_mxfp4.default
_unprepack = _ops.unprepack_mxfp4.default
_mm = _ops.mxfp4_mm.default
_mm_packed = _ops.mxfp4_mm_packed.default


class MXFP4Tensor(NamedTuple):
    """A tensor in MXFP4, blocks along its last dimension, in the packed layout."""

    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple

    @property
    def cols(self) -> int:
        return self.shape[-1]

    @property
    def rows(self) -> int:
        n = 1
        for d in self.shape[:-1]:
            n *= d
        return n


def quantize_mxfp4(x: torch.Tensor) -> MXFP4Tensor:
    """x (..., cols), fp16, bf16 or fp32, quantised along its last dimension; any number of columns
    (a last block shorter than 32 counts as continued by zeros)."""
    codes, scales = _quantize(x)
    return MXFP4Tensor(codes, scales, tuple(x.shape))


def dequantize_mxfp4(q: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that q stands for, each rounded once to dtype (fp16, bf16 or fp32)."""
    if len(q.shape) == 2:
        return _dequantize(q.codes, q.scales, *q.shape, dtype)
    return _dequantize(q.codes, q.scales, q.rows, q.cols, dtype).view(q.shape)


def prepack_mxfp4(codes: torch.Tensor, scales: torch.Tensor, cols: int | None = None) -> MXFP4Tensor:
    """A checkpoint's row-major codes (rows, blocks * 16), the earlier value of a pair in a byte's low
    half, and e8m0 scales (rows, blocks) in the packed layout. cols: the number of columns where it
    is not blocks * 32 (the codes beyond it must be zero)."""
    cols = codes.shape[-1] * 2 if cols is None else cols
    packed, packed_scales = _prepack(codes, scales, cols)
    return MXFP4Tensor(packed, packed_scales, (codes.shape[0], cols))


def unprepack_mxfp4(q: MXFP4Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The row-major codes and scales of q (prepack_mxfp4's arguments)."""
    return _unprepack(q.codes, q.scales, q.rows, q.cols)


def mxfp4_mm(a: torch.Tensor | MXFP4Tensor, w: MXFP4Tensor, bias: torch.Tensor | None = None,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """a (..., K) times the transpose of w (N, K), plus bias (N,): (..., N) in out_dtype (fp16 or bf16;
    by default that of a, bf16 for an MXFP4Tensor).

    a in fp16 or bf16 is held in MXFP4 on the way (quantize_mxfp4's values): inside the product for
    few rows, by a pass of its own otherwise. Products are exact, sums and the bias in fp32, and the
    result is rounded once."""
    N, K = w.shape
    if isinstance(a, MXFP4Tensor):
        if a.shape[-1] != K:
            raise RuntimeError(f"a has {a.shape[-1]} columns, w {K}")
        y = _mm_packed(a.codes, a.scales, a.rows, K, w.codes, w.scales, N, bias, out_dtype or torch.bfloat16)
        return y if len(a.shape) == 2 else y.view(*a.shape[:-1], N)
    if a.dim() < 1 or a.shape[-1] != K:
        raise RuntimeError(f"a must have w's {K} columns, got {tuple(a.shape)}")
    if a.dim() == 2:
        return _mm(a, w.codes, w.scales, N, bias, out_dtype or a.dtype)
    return _mm(a.reshape(-1, K), w.codes, w.scales, N, bias, out_dtype or a.dtype).view(*a.shape[:-1], N)
