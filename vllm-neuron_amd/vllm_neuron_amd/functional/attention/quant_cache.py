"""K/V cache of 8-bit codes with one scale per token and head.

The reference's FP8 caches have static scales, one per layer or head
(vllm_neuron/functional/attention/attention_decode.py:967-979), which must be
calibrated and clip what lies past them.  Here every row is scaled by its own
largest value as it is written, so int8 caches work too; the scales lie beside
the pool, ``[num_blocks, num_kv_heads, block_size]`` float32.
``cross_attention`` and ``shared_prefix_attention`` read such caches as they
lie; ``quant_kv_read`` gives the rows back to everything else.
"""
from __future__ import annotations

from typing import Tuple

import torch
from torch import Tensor

from ... import ops as K


def quant_kv_write(
    k: Tensor,          # [T, Hkv, d] bf16 / f16 / f32, any strides
    v: Tensor,          # [T, Hkv, d]
    slots: Tensor,      # [T] int32 / int64 slot = block * block_size + offset
    k_cache: Tensor,    # [nb, Hkv, bs, d] int8 or float8_e4m3fn
    v_cache: Tensor,
    k_scales: Tensor,   # [nb, Hkv, bs] float32
    v_scales: Tensor,
) -> None:
    """Quantises the rows of new tokens into their slots.

    ``scale = max|x| / Q`` and ``code = round(x * Q / max|x|)`` with Q = 127
    (int8, ties to even) or 448 (e4m3fn).  A row of zeros has scale 0; a row
    that holds a NaN or an infinity scale NaN, so that it reads back as NaN and
    touches nothing else.  Slots outside the pool (negative padding among them)
    are skipped; the others must differ from each other, as the tokens of a
    step do.
    """
    K.quant_kv_write(k, v, slots, k_cache, v_cache, k_scales, v_scales)


def quant_kv_read(
    k_cache: Tensor,
    v_cache: Tensor,
    k_scales: Tensor,
    v_scales: Tensor,
    slots: Tensor,      # [T] int32 / int64
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> Tuple[Tensor, Tensor]:
    """Rows of the given slots as ``(k, v) [T, Hkv, d]`` in ``dtype`` (bf16,
    f16 or f32): ``code * scale`` in float32, rounded once.  Slots outside the
    pool give zeros; a slot may occur several times."""
    return K.quant_kv_read(k_cache, v_cache, k_scales, v_scales, slots, dtype)
