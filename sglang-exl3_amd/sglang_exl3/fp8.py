"""Block-scaled FP8 linears beside the EXL3 ones.

An EXL3 checkpoint's other linears are often e4m3 with one fp32 scale for each
128 x 128 block (tensors ``weight`` and ``weight_scale_inv``); the reference hands
them to SGLang's FP8 method (src/sglang_exl3/exl3.py:1919-1967).
``FP8BlockLinearMethod`` runs them on the gfx950 kernels behind
``torch.ops.sglang_exl3.fp8_linear``.  ``EXL3Config.get_quant_method`` returns it
for the modules that the checkpoint stores so.

``apply`` takes 16-bit rows, which the product quantizes, or rows that are
quantized already, as the pair (q, scale) of ``fp8_norm_quant``,
``fp8_swiglu_quant`` or ``fp8_quant_rows``: a norm or an activation then writes half
the bytes, and layers that share an input share its quantization.
"""

from __future__ import annotations

import logging
from typing import Any, Optional, Tuple, Union

import torch
from torch.nn.parameter import Parameter

from .base import LinearMethodBase, set_weight_attrs

logger = logging.getLogger("sglang.exl3")

__all__ = ["BLOCK", "FP8BlockLinearMethod", "fp8_block_modules", "is_fp8_block_config"]

BLOCK = 128
_SHARDS = {"q": 0, "k": 1, "v": 2}
Rows = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def fp8_block_modules(tensor_storage: Any) -> set[str]:
    """Modules whose stored tensors are an e4m3 weight and its block scales."""
    out = set()
    for module, entry in dict(tensor_storage or {}).items():
        stored = dict(((entry or {}).get("stored_tensors") or {}))
        leaves = {str(name).rsplit(".", 1)[-1]: dict(meta or {}) for name, meta in stored.items()}
        dtype = str(leaves.get("weight", {}).get("dtype", "F8_E4M3")).upper()
        if {"weight", "weight_scale_inv"} <= set(leaves) and dtype in ("F8_E4M3", "FLOAT8_E4M3FN"):
            out.add(str(module))
    return out


def is_fp8_block_config(quantization: Any) -> bool:
    """Whether a checkpoint's ``non_routed_quantization`` is e4m3 in blocks of 128 x 128, rows quantized as they come."""
    q = quantization if isinstance(quantization, dict) else {}
    return (str(q.get("quant_method", "")).lower() == "fp8" and str(q.get("fmt", "e4m3")).lower() == "e4m3"
            and list(q.get("weight_block_size") or []) == [BLOCK, BLOCK]
            and str(q.get("activation_scheme", "dynamic")).lower() == "dynamic")


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


class FP8BlockLinearMethod(LinearMethodBase):
    """SGLang linear method for e4m3 weights with an fp32 scale for each 128 x 128 block."""

    def __init__(self, quant_config: Any = None) -> None:
        super().__init__()
        self.quant_config = quant_config

    # -------------------------------------------------------------- weights
    def create_weights(self, layer, input_size_per_partition: int, output_partition_sizes: list[int],
                       input_size: int, output_size: int, params_dtype: torch.dtype, **extra_weight_attrs) -> None:
        del input_size, output_size
        k, widths = int(input_size_per_partition), [int(v) for v in output_partition_sizes]
        if k % 16:
            raise ValueError(f"FP8 linear: the input width must be a multiple of 16, got {k}")
        if any(w % BLOCK for w in widths[:-1]):
            raise ValueError(f"FP8 linear: only the last of the output shards {widths} may end inside a block of {BLOCK}")
        n = sum(widths)
        extra = {key: v for key, v in extra_weight_attrs.items() if key != "weight_loader"}
        layer._fp8_widths = widths
        layer._fp8_out_dtype = params_dtype if params_dtype in (torch.float16, torch.bfloat16) else torch.bfloat16
        layer._fp8_loaded = set()
        for name, shape, dtype in (("weight", (n, k), torch.float8_e4m3fn),
                                   ("weight_scale_inv", (_blocks(n), _blocks(k)), torch.float32)):
            p = Parameter(torch.empty(shape, dtype=dtype), requires_grad=False)
            layer.register_parameter(name, p)
            set_weight_attrs(p, extra)
            p.weight_loader = self._load
            p._fp8_owner = layer
            p._fp8_unit = 1 if name == "weight" else BLOCK  # features of an index
            p._fp8_name = name

    @staticmethod
    def _part(src: torch.Tensor, dim: int, size: int, features: int, unit: int) -> torch.Tensor:
        """src, or this rank's part of it, with `size` indices along dim (`features` features)."""
        from .exl3 import _tp_rank_size

        have = int(src.shape[dim])
        if have == size:
            return src
        rank, ranks = _tp_rank_size()
        if ranks > 1 and have == size * ranks and (unit == 1 or features % BLOCK == 0):
            return src.narrow(dim, size * rank, size)
        raise ValueError(f"FP8 linear: a tensor of shape {tuple(src.shape)} does not give {size} indices along dimension "
                         f"{dim} to rank {rank} of {ranks} (parts of a weight are whole blocks of {BLOCK})")

    def _load(self, param, loaded_weight: torch.Tensor, shard_id=None) -> None:
        layer, unit = param._fp8_owner, param._fp8_unit
        src = loaded_weight.detach()
        if unit == 1 and src.dtype != torch.float8_e4m3fn:
            raise ValueError(f"FP8 linear: weight must be float8_e4m3fn, got {src.dtype}")
        widths = layer._fp8_widths
        shard = None if shard_id is None else _SHARDS.get(shard_id, shard_id)
        if shard is None and len(widths) > 1:
            first, rows, at = 0, sum(widths), range(len(widths))
        else:
            i = int(shard or 0)
            if not 0 <= i < len(widths):
                raise ValueError(f"FP8 linear: shard {shard_id!r} of a layer with {len(widths)} shards")
            first, rows, at = sum(widths[:i]), widths[i], (i,)
        whole = shard is None and len(widths) > 1  # several shards fused along the rows: no parts of it
        n = rows if unit == 1 else _blocks(rows)
        k = int(param.shape[1])
        if whole and int(src.shape[0]) != n:
            raise ValueError(f"FP8 linear: a tensor of shape {tuple(src.shape)} for {n} rows")
        src = self._part(src, 0, n, rows, unit)
        src = self._part(src, 1, k, int(layer.weight.shape[1]), unit)
        param.data[first // unit:first // unit + n].copy_(src)
        layer._fp8_loaded.update((param._fp8_name, i) for i in at)

    def process_weights_after_loading(self, layer) -> None:
        missing = {(name, i) for name in ("weight", "weight_scale_inv") for i in range(len(layer._fp8_widths))}
        missing -= layer._fp8_loaded
        if missing:
            raise RuntimeError(f"FP8 linear received no {sorted(missing)}; checkpoint/quantization mismatch?")

    # -------------------------------------------------------------- forward
    def apply(self, layer, x: Rows, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [..., k] in fp16, bf16 or fp32 (rounded to the layer's dtype first), or (q, scale); the result in
        the layer's dtype."""
        from .ops import register_custom_ops

        register_custom_ops()
        x, scale = x if isinstance(x, tuple) else (x, None)
        dtype = layer._fp8_out_dtype
        if x.dtype == torch.float32:
            x = x.to(dtype)
        y = torch.ops.sglang_exl3.fp8_linear(x, layer.weight, layer.weight_scale_inv, scale,
                                             None if bias is None else bias.to(dtype), dtype == torch.bfloat16)
        return y.view(*x.shape[:-1], y.shape[-1])
