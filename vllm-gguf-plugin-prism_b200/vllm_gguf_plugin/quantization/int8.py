# SPDX-License-Identifier: Apache-2.0
"""Layers of a GGUF file as 8-bit integers with one scale a weight row (no counterpart in the reference).

The block formats carry a scale for 32 values or fewer, so that their products either decode weights into 16-bit operands or rescale
every few steps.  These methods decode a layer once, when it is loaded, quantize its rows with ``ops.int8_quantize`` and multiply 8-bit
integers from then on (``ops.int8_mul_mat``, ``ops.int8_fused_moe``): a byte a weight, and the tensor cores' 8-bit rate for batches.
They take the place of ``GGUFLinearMethod`` / ``GGUFMoEMethod``, with the same loaders and signatures.  What is rounded is the weights'
row scale (instead of their blocks') and, as there, the activations, by the token instead of by 32 values."""
from __future__ import annotations

import torch
from torch.compiler import is_compiling

from .. import native, ops
from .fused_moe import GGUFMoEMethod
from .linear import GGUFLinearMethod, _weights_complete
from .utils import DEQUANT_TYPES, quant_sizes

_DECODED_VALUES = 1 << 26   # fp32 values that a layer's decoding holds at a time


def int8_rows(weight: torch.Tensor, weight_type: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of raw GGUF blocks ``uint8 [rows, bytes]`` (or of floats) -> ``(codes int8 [rows, K], scales float32 [rows])``."""
    if weight.is_floating_point():
        return ops.int8_quantize(weight)
    if int(weight_type) not in DEQUANT_TYPES:
        raise NotImplementedError(f"Unsupported GGUF quantization type: {int(weight_type)}")
    per, size = quant_sizes(weight_type)
    rows, k = weight.shape[0], weight.shape[1] // size * per
    codes = torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device=weight.device)[:, :k]
    scales = torch.empty((rows,), dtype=torch.float32, device=weight.device)
    step = max(1, _DECODED_VALUES // k)
    for r in range(0, rows, step):
        part = weight[r:r + step].contiguous()
        codes[r:r + step], scales[r:r + step] = ops.int8_quantize(ops.ggml_dequantize(part, weight_type, part.shape[0], k, torch.float32))
    return codes, scales


def _set(layer: torch.nn.Module, name: str, data: torch.Tensor) -> None:
    if name in layer._parameters:
        layer._parameters[name].data = data
    else:
        layer.register_parameter(name, torch.nn.Parameter(data, requires_grad=False))


class Int8LinearMethod(GGUFLinearMethod):
    """Linear method that loads like ``GGUFLinearMethod`` and multiplies 8-bit integers.  After loading a layer holds ``int8_weight [N, K]`` and
    ``int8_scales [N]``; the blocks are given back."""

    def process_weights_after_loading(self, layer: torch.nn.Module):
        super().process_weights_after_loading(layer)
        if layer.weight.numel() == 0:   # (no new weights since)
            return
        runs = self._runs(layer)
        parts = [int8_rows(layer.weight.data[start:start + rows, :width], t)
                 for t, start, rows, width in zip(runs[0::5], runs[1::5], runs[2::5], runs[3::5])]
        k = parts[0][0].shape[1]
        codes = torch.empty((sum(len(c) for c, _ in parts), (k + 15) // 16 * 16), dtype=torch.int8, device=layer.weight.device)[:, :k]
        start = 0
        for c, _ in parts:
            codes[start:start + len(c)] = c
            start += len(c)
        _set(layer, "int8_weight", codes)
        _set(layer, "int8_scales", torch.cat([s for _, s in parts]))
        layer.weight.data = torch.empty(0, dtype=torch.uint8, device=codes.device)
        _weights_complete(codes)

    def apply(self, layer: torch.nn.Module, x: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
        if self.layout is not None:
            x = self.layout.input_to_gguf(x)
        if bias is not None and bias.dtype != x.dtype:
            bias = bias.to(x.dtype)
        w, scales = layer.int8_weight, layer.int8_scales
        if not is_compiling():   # (loading has ended, so the product may start on the weights ahead of the stream)
            out = native.int8_mul_mat(w, scales, x, bias, True)
            if out is not None:
                return out
        return torch.ops._C_gguf.int8_mul_mat(w, scales, x, bias)


class Int8MoEMethod(GGUFMoEMethod):
    """MoE method that loads like ``GGUFMoEMethod`` and multiplies 8-bit integers.  After loading a layer holds ``w13_int8 [E, 2I, H]``,
    ``w13_scales [E, 2I]``, ``w2_int8 [E, H, I]`` and ``w2_scales [E, H]``; the blocks are given back."""

    @staticmethod
    def _load_weight(param, loaded_weight, weight_name=None, shard_id=None, expert_id=None, return_success=False):
        """As the blocks' loader, which puts zeros in place of what has not arrived; notes what has: (expert, or None for all; first row, rows)."""
        rows = loaded_weight.shape[-2]
        out = GGUFMoEMethod._load_weight(param, loaded_weight, weight_name, shard_id, expert_id, return_success)
        if shard_id in ("w1", "w3"):   # (of this tensor-parallel rank)
            rows = param.data.shape[1] // 2
        param.arrived = getattr(param, "arrived", []) + [(None if loaded_weight.dim() == 3 else int(expert_id), rows if shard_id == "w3" else 0, rows)]
        return out

    def process_weights_after_loading(self, layer: torch.nn.Module):
        """What has arrived since the last call becomes 8-bit integers; rows that have not keep those they have."""
        for name in ("w13", "w2"):
            param, kind = getattr(layer, name + "_weight"), getattr(layer, name + "_weight_type").weight_type
            if param.numel() == 0:
                continue
            experts, rows, width = param.shape
            per, size = quant_sizes(kind)
            had = layer._parameters.get(name + "_int8")
            if had is None or had.shape != (experts, rows, width // size * per):
                codes, scales = int8_rows(param.data.reshape(experts * rows, width), kind)
                _set(layer, name + "_int8", codes.unflatten(0, (experts, rows)))
                _set(layer, name + "_scales", scales.view(experts, rows))
            else:
                for expert, first, count in getattr(param, "arrived", None) or [(None, 0, rows)]:
                    part = slice(None) if expert is None else slice(expert, expert + 1)
                    blocks = param.data[part, first:first + count]
                    codes, scales = int8_rows(blocks.reshape(-1, width), kind)
                    had.data[part, first:first + count] = codes.unflatten(0, blocks.shape[:2])
                    getattr(layer, name + "_scales").data[part, first:first + count] = scales.view(blocks.shape[:2])
            param.data, param.arrived = torch.empty(0, dtype=torch.uint8, device=param.device), []

    def apply(self, layer, x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
              shared_experts=None, shared_experts_input: torch.Tensor | None = None) -> torch.Tensor:
        if getattr(layer, "apply_router_weight_on_input", False):
            raise NotImplementedError("Apply router weight on input is not supported for fused GGUF MoE method.")
        activation = getattr(layer, "activation", "silu")
        activation = getattr(activation, "value", activation)
        if activation not in ops.MOE_ACTIVATIONS:
            raise NotImplementedError(f"activation {activation!r}")
        return ops.int8_fused_moe(x, layer.w13_int8, layer.w13_scales, layer.w2_int8, layer.w2_scales, topk_weights, topk_ids, activation)
