"""Projections in 8-bit integers: one scale per token, one per output channel.

The reference leaves such products to its compiler's kernel library
(``quantization_type`` of vllm_neuron/functional/attention/qkv.py:672-730);
``qkv_proj`` reaches the two functions below with ``QuantizationType.ROW``.
"""
from __future__ import annotations

from typing import Optional, Tuple

from torch import Tensor

from ... import ops as K
from ...utils.common_types import NormType


def quant_rows(
    x: Tensor,                              # [..., K] bf16
    *,
    norm_type: NormType = NormType.NO_NORM,
    norm_weights: Optional[Tensor] = None,  # [K] bf16 / f32
    eps: float = 1e-6,
    hidden_actual: Optional[int] = None,
    mlp_prev: Optional[Tensor] = None,      # [..., K], added to x (bf16)
    attn_prev: Optional[Tensor] = None,
) -> Tuple[Tensor, Tensor]:
    """Rows as int8 codes ``[..., K]`` and float32 scales ``[...]``.

    ``scale = max|y| / 127`` and ``code = round(y * 127 / max|y|)`` (ties to
    even) of ``y = x (+ mlp_prev) (+ attn_prev)`` or its RMS norm, which is not
    rounded in between.  A row of zeros has scale 0; a row that holds a NaN or
    an infinity (or, in fp32, a product with ``norm_weights`` that is one) scale
    NaN and zero codes.  The rows of a weight ``[N, K]`` give
    what ``int8_linear`` takes.
    """
    if norm_type not in (NormType.NO_NORM, NormType.RMS_NORM, NormType.RMS_NORM_SKIP_GAMMA):
        raise NotImplementedError(f"quant_rows: {norm_type.name} is not supported")
    if norm_type != NormType.RMS_NORM and norm_weights is not None:
        raise ValueError(f"quant_rows: norm_weights with {norm_type.name}")
    return K.quant_rows(x, norm_type != NormType.NO_NORM, eps, norm_weights, add0=mlp_prev,
                        add1=attn_prev, dim_actual=hidden_actual or 0)


def int8_linear(
    x: Tensor,                      # [..., K] int8
    x_scales: Tensor,               # [...] float32
    w: Tensor,                      # [N, K] int8
    w_scales: Tensor,               # [N] float32
    *,
    bias: Optional[Tensor] = None,  # [N] bf16 / f32
    out: Optional[Tensor] = None,   # [..., N] bf16
) -> Tensor:
    """``x_scales * w_scales * (x @ w.T) + bias`` in bf16 ``[..., N]``: the sums
    exact in 32-bit integers, the rest in float32, rounded once.

    ``K`` is a multiple of 16 (below 131072), the rows of ``x`` and ``w`` are
    contiguous and 16-byte aligned, those of ``w`` less than 2^24 bytes apart.  A row
    with scale NaN gives NaN.
    """
    if x.dim() == 2:
        return K.int8_linear(x, x_scales, w, w_scales, bias, out)
    lead = x.shape[:-1]
    if x_scales.dim() != 1 and [n for n in x_scales.shape if n != 1] != [n for n in lead if n != 1]:
        raise ValueError(f"int8_linear: x_scales must be {tuple(lead)}, one per row of x, got "
                         f"{tuple(x_scales.shape)}")
    shape = (*lead, w.shape[0])
    if out is not None:
        if tuple(out.shape) != shape:
            raise ValueError(f"int8_linear: out must be {shape}, got {tuple(out.shape)}")
        flat = out.view(-1, shape[-1])
    else:
        flat = None
    y = K.int8_linear(x.reshape(-1, x.shape[-1]), x_scales.reshape(-1), w, w_scales, bias, flat)
    return y.view(shape) if out is None else out
