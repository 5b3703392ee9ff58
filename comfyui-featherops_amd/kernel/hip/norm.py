"""The norms around a transformer block, fused with its gate, residual and modulation (no counterpart
in the reference).

    y    = modulated_norm(x, scale=s, shift=t, kind="layer")                # before the first block
    x, y = gated_residual_norm(x, h, gate, scale=s, shift=t, kind="layer")  # behind a block, before the next

with norm(v) = v / sqrt(mean(v^2) + eps) ("rms") or (v - mean) / sqrt(variance + eps) ("layer") over the
last dimension, and

    h = norm(h) * post_weight                     (where post_weight is given)
    x = residual_scale * x + gate * h
    y = norm(x) * weight + bias;  y = y * (1 + scale) + shift

each factor or term left out where its argument is None. Everything is fp32 from the inputs to the two
results, which are rounded once: x to its own type, y to the block's (h's; for modulated_norm out_dtype,
by default x's). out_dtype="mxfp4" gives y as an MXFP4Tensor for mxfp4_mm instead, quantised from fp32.

x is fp32 or of the block's type. gate, scale and shift broadcast against x: (cols,), (batch, 1, cols) or
x's own shape, slices of a larger modulation tensor included. Vectors of the block's type are read as
they are; if any has another type (fp32 modulation beside bf16 weights), all are read as fp32 (those that
are not are cast first, on every call). scale and shift of which one is per sample and the other for all rows are
both written out row by row first: give both the same form. Up to 16384 columns. Runs in libfeatherops_amd.so on
torch's current stream; there is no other compute path.
"""

from __future__ import annotations

import torch

from . import _lib
from .mxfp4 import MXFP4Tensor

_lib.load_torch_ops()
_ops = torch.ops.feather_ops
_modulated = _ops.modulated_norm.default
_modulated_mxfp4 = _ops.modulated_norm_mxfp4.default
_gated = _ops.gated_residual_norm.default
_gated_mxfp4 = _ops.gated_residual_norm_mxfp4.default

_KINDS = {"rms": False, "layer": True}


def _is_layer(kind: str) -> bool:
    layer = _KINDS.get(kind)
    if layer is None:
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    return layer


def modulated_norm(x: torch.Tensor, *, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, kind: str = "rms",
                   eps: float = 1e-6, out_dtype: torch.dtype | str | None = None) -> torch.Tensor | MXFP4Tensor:
    """norm(x) * weight + bias, then * (1 + scale) + shift, in one pass over x."""
    if out_dtype == "mxfp4":
        return MXFP4Tensor(_modulated_mxfp4(x, weight, bias, scale, shift, _is_layer(kind), eps), tuple(x.shape))
    return _modulated(x, weight, bias, scale, shift, _is_layer(kind), eps, out_dtype)


def gated_residual_norm(x: torch.Tensor, h: torch.Tensor, gate: torch.Tensor | None = None, *,
                        post_weight: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                        shift: torch.Tensor | None = None, kind: str = "rms", eps: float = 1e-6,
                        residual_scale: float = 1.0, out_dtype: torch.dtype | str | None = None,
                        ) -> tuple[torch.Tensor, torch.Tensor | MXFP4Tensor]:
    """(x, y): the block's output h on the residual stream x, and the norm of the sum before it is
    rounded, in one pass over x and h."""
    if out_dtype == "mxfp4":
        stream, y = _gated_mxfp4(x, h, gate, post_weight, weight, bias, scale, shift, _is_layer(kind), eps, residual_scale)
        return stream, MXFP4Tensor(y, tuple(x.shape))
    return _gated(x, h, gate, post_weight, weight, bias, scale, shift, _is_layer(kind), eps, residual_scale, out_dtype)
