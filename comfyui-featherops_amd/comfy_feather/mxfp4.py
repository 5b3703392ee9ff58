"""Linear replacement with a 4-bit weight (no counterpart in the reference).

`mxfp4_ops(out_dtype, excluded_names)` returns an operations class for ComfyUI's `custom_operations`
hook, the 4-bit sibling of `feather_ops`. Its `Linear`:
  * at state-dict load quantizes the weight to packed MXFP4 on the GPU, or lays out one that the
    checkpoint holds in MXFP4 already (uint8 codes (N, blocks * 16) with uint8 `weight_scale` (N, blocks)),
    unless the layer is excluded or 1-wide. A `weight_scale` or `scale_weight` beside a weight in floating
    point (fp8 checkpoints, one scale or one per row) is multiplied in first;
  * in forward runs mxfp4_mm with the bias; activations in fp16 or bf16 (fp32 is cast to bf16), or an
    MXFP4Tensor that a norm left in 4 bits (kernel.hip.norm, out_dtype="mxfp4"), and applies basic LoRA
    patches as a separate pass over activations that are not in 4 bits;
  * converts the weight back for a merge (convert_weight) and takes the merged one (set_weight).

A quantized layer's `weight` parameter is its packed operand (uint8, codes and scales), so that whatever moves, sizes or
backs up parameters finds it; `mx_weight` is the same as an MXFP4Tensor, None for a layer that is not quantized. The
layer may lie in host memory: conversions run on the GPU and their results come back to where the weight is. A
state dict holds the row-major codes and scales, a copy of the weight's size for as long as the dict lives.

Inside ComfyUI it subclasses comfy.ops.manual_cast; without it the stand-in of `ops.py`.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from ..kernel.hip.mxfp4 import MXFP4Tensor, dequantize_mxfp4, mxfp4_mm, prepack_mxfp4, quantize_mxfp4, unprepack_mxfp4
from .lora import apply_lora_patches
from .ops import cast_bias_weight, manual_cast, run_every_op, uncast_bias_weight


def _on_gpu(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_cuda or t.is_meta else t.to("cuda")


def _scaled(weight: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The fp32 values that a checkpoint's weight and its scale (one, or one per row) stand for."""
    scale = scale.to(device=weight.device, dtype=torch.float32)
    if scale.numel() == 1:
        scale = scale.reshape(())
    elif weight.ndim != 2 or scale.shape != (weight.shape[0], 1):
        raise ValueError(f"weight scale must be one number or ({weight.shape[0]}, 1), got {tuple(scale.shape)}")
    return weight.to(torch.float32) * scale


def mxfp4_ops(out_dtype=torch.bfloat16, excluded_names=()):
    excluded_names = tuple(excluded_names)

    class MXFP4Ops(manual_cast):
        _excluded_names = excluded_names
        _out_dtype = out_dtype

        class Linear(manual_cast.Linear):
            def __init__(self, *args, **kwargs):
                super().__init__(*args, **kwargs)
                self.excluded_names = MXFP4Ops._excluded_names
                self.out_dtype = MXFP4Ops._out_dtype
                self.is_quantized = False

            @property
            def mx_weight(self) -> MXFP4Tensor | None:
                return MXFP4Tensor(self.weight, (self.out_features, self.in_features)) if self.is_quantized else None

            @mx_weight.setter
            def mx_weight(self, weight: MXFP4Tensor) -> None:
                self._hold(weight)

            def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs):
                weight = state_dict.pop(prefix + "weight", None)
                bias = state_dict.pop(prefix + "bias", None)
                scales = state_dict.pop(prefix + "weight_scale", None)
                if scales is None:
                    scales = state_dict.pop(prefix + "scale_weight", None)
                if weight is None:
                    missing_keys.append(prefix + "weight")
                elif scales is not None and weight.dtype == torch.uint8:
                    self._hold(prepack_mxfp4(_on_gpu(weight), _on_gpu(scales), self.in_features))
                elif (any(x in prefix for x in self.excluded_names) or weight.ndim == 1 or self.in_features == 1
                      or self.out_features == 1):
                    self.is_quantized = False
                    if scales is not None:  # (an 8-bit float cannot hold the product: the layer's type does)
                        weight = _scaled(weight, scales).to(weight.dtype if weight.element_size() > 1 else self.out_dtype)
                    self.weight = nn.Parameter(weight, requires_grad=False)
                else:
                    weight = _on_gpu(weight)
                    if scales is not None:
                        weight = _scaled(weight, scales)
                    elif weight.element_size() == 1 and weight.is_floating_point():  # (8-bit floats: bf16 holds all of their values)
                        weight = weight.to(torch.bfloat16)
                    self._hold(quantize_mxfp4(weight))
                if bias is not None:  # (beside a packed weight, which is on the GPU)
                    bias = nn.Parameter(bias.to(device=self.weight.device if self.is_quantized else None, dtype=self.out_dtype),
                                        requires_grad=False)
                self.bias = bias

            def _hold(self, weight: MXFP4Tensor) -> None:
                if weight.shape != (self.out_features, self.in_features):
                    raise ValueError(f"expected a ({self.out_features}, {self.in_features}) weight, got {weight.shape}")
                self.is_quantized = True
                self.weight = nn.Parameter(weight.data, requires_grad=False)

            def _operand(self, data: torch.Tensor) -> MXFP4Tensor:
                """A packed operand's bytes, wherever they lie, for the kernels."""
                return MXFP4Tensor(_on_gpu(data), (self.out_features, self.in_features))

            def _save_to_state_dict(self, destination, prefix, keep_vars):
                super()._save_to_state_dict(destination, prefix, keep_vars)
                if self.is_quantized:
                    codes = unprepack_mxfp4(self._operand(self.weight))
                    for name, t in zip(("weight", "weight_scale"), codes):
                        destination[prefix + name] = t.to(self.weight.device)

            def _apply(self, fn, recurse=True):
                def keep_bytes(t):  # the packed operand is moved between devices, never cast
                    moved = fn(t)
                    return moved if t.dtype != torch.uint8 or moved.dtype == torch.uint8 else t.to(moved.device)

                return super()._apply(keep_bytes, recurse)

            def convert_weight(self, weight=None, inplace=False, **kwargs):
                """The values, in the layer's output dtype, of `weight`: a packed operand as `weight` and `mx_weight`
                hold it and set_weight(return_weight=True) returns it; by default the layer's own."""
                if not self.is_quantized:
                    return self.weight if weight is None else weight
                if weight is None:
                    weight = self.weight
                if isinstance(weight, MXFP4Tensor):
                    if weight.shape != (self.out_features, self.in_features):
                        raise ValueError(f"expected a ({self.out_features}, {self.in_features}) weight, got {weight.shape}")
                    weight = weight.data
                if not isinstance(weight, torch.Tensor) or weight.dtype != torch.uint8 or weight.ndim != 1:
                    raise TypeError(f"expected a packed MXFP4 weight, got {getattr(weight, 'dtype', type(weight).__name__)}")
                return dequantize_mxfp4(self._operand(weight), self.out_dtype).to(weight.device)

            def set_weight(self, weight, inplace_update=False, seed=None, return_weight=False, **kwargs):
                if not self.is_quantized:
                    weight = weight.to(self.weight.dtype)
                    if return_weight:
                        return weight
                    self.weight = nn.Parameter(weight, requires_grad=False)
                    return None
                quantized = quantize_mxfp4(_on_gpu(weight))
                if return_weight:
                    return quantized
                assert inplace_update is False
                self._hold(quantized._replace(data=quantized.data.to(self.weight.device)))
                return None

            def forward(self, x: torch.Tensor | MXFP4Tensor) -> torch.Tensor:
                run_every_op()
                if not self.is_quantized:
                    weight, bias, offload_stream = cast_bias_weight(self, x, offloadable=True)
                    y = F.linear(x, weight, bias)
                    uncast_bias_weight(self, weight, bias, offload_stream)
                    return y
                if isinstance(x, MXFP4Tensor):
                    if self.weight_function:
                        raise NotImplementedError("LoRA patches need activations in 16 bits")
                    return self._product(x, x.data)
                dtype = x.dtype
                if dtype == torch.float32:
                    x = x.to(torch.bfloat16)
                y = self._product(x, x)
                if self.weight_function:
                    y = apply_lora_patches(x, y, self.weight_function)
                return y if y.dtype == dtype else y.to(dtype)

            def _product(self, x: torch.Tensor | MXFP4Tensor, data: torch.Tensor) -> torch.Tensor:
                # (not through Module's attribute lookup: 0.3 us of the host's time each, and it bounds small calls)
                weight, bias = self._parameters["weight"], self._parameters["bias"]
                shape = (self.out_features, self.in_features)
                device = data.device
                if weight.device == device and (bias is None or (bias.device == device and bias.dtype == self.out_dtype
                                                                 and not self.bias_function)):
                    return mxfp4_mm(x, MXFP4Tensor(weight, shape), bias, self.out_dtype)
                # an offloaded layer, or a patched bias: no patch is applied to the packed weight on its way
                saved_weight_function = self.weight_function
                self.weight_function = []
                try:
                    weight, bias, offload_stream = cast_bias_weight(self, data, dtype=torch.uint8,
                                                                    bias_dtype=self.out_dtype, offloadable=True)
                finally:
                    self.weight_function = saved_weight_function
                y = mxfp4_mm(x, MXFP4Tensor(weight, shape), bias, self.out_dtype)
                uncast_bias_weight(self, weight, bias, offload_stream)
                return y

    return MXFP4Ops
