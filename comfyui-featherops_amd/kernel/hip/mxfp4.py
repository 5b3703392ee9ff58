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

import math
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
    """A tensor in MXFP4, blocks along its last dimension, in the packed layout: `data` (uint8) holds the
    codes and, behind them, the scales."""

    data: torch.Tensor
    shape: tuple

    @property
    def cols(self) -> int:
        return self.shape[-1]

    @property
    def rows(self) -> int:
        return math.prod(self.shape[:-1])

    @property
    def codes(self) -> torch.Tensor:
        """(groups, steps, 4, 64, 16) view of the codes: include/featherops_amd.h."""
        groups, steps = (self.rows + 63) // 64, (self.cols + 127) // 128
        return self.data[:groups * steps * 4096].view(groups, steps, 4, 64, 16)

    @property
    def scales(self) -> torch.Tensor:
        """(groups, steps, 64, 4) view of the scales."""
        groups, steps = (self.rows + 63) // 64, (self.cols + 127) // 128
        return self.data[groups * steps * 4096:].view(groups, steps, 64, 4)


def quantize_mxfp4(x: torch.Tensor) -> MXFP4Tensor:
    """x (..., cols), fp16, bf16 or fp32, quantised along its last dimension; any number of columns
    (a last block shorter than 32 counts as continued by zeros)."""
    return MXFP4Tensor(_quantize(x), tuple(x.shape))


def dequantize_mxfp4(q: MXFP4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that q stands for, each rounded once to dtype (fp16, bf16 or fp32)."""
    return _dequantize(q.data, q.shape, dtype)


def prepack_mxfp4(codes: torch.Tensor, scales: torch.Tensor, cols: int | None = None) -> MXFP4Tensor:
    """A checkpoint's row-major codes (rows, blocks * 16), the earlier value of a pair in a byte's low
    half, and e8m0 scales (rows, blocks) in the packed layout. cols: the number of columns where it
    is not blocks * 32 (the codes beyond it must be zero)."""
    cols = codes.shape[-1] * 2 if cols is None else cols
    return MXFP4Tensor(_prepack(codes, scales, cols), (codes.shape[0], cols))


def unprepack_mxfp4(q: MXFP4Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The row-major codes and scales of q (prepack_mxfp4's arguments)."""
    return _unprepack(q.data, q.rows, q.cols)


def mxfp4_mm(a: torch.Tensor | MXFP4Tensor, w: MXFP4Tensor, bias: torch.Tensor | None = None,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """a (..., K) times the transpose of w (N, K), plus bias (N,): (..., N) in out_dtype (fp16 or bf16;
    by default that of a, bf16 for an MXFP4Tensor).

    a in fp16 or bf16 is held in MXFP4 on the way (quantize_mxfp4's values): inside the product for
    few rows, by a pass of its own otherwise. Products are exact, sums and the bias in fp32, and the
    result is rounded once."""
    N, K = w.shape
    if isinstance(a, MXFP4Tensor):
        return _mm_packed(a.data, a.shape, w.data, N, K, bias, out_dtype or torch.bfloat16)
    return _mm(a, w.data, N, K, bias, out_dtype)
