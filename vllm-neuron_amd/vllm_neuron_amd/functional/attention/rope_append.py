"""Rotary positions on one or several axes, applied where K and V are appended.

The reference expands cos and sin per token on its model side (for image and
video tokens from three position axes) and hands them to ``qkv_proj`` or
``attention_decode`` as tables, whose cache writes know bf16 and static FP8.
Here the angles are formed from the positions themselves, once per token, and
the rotated keys go to any cache of this package in the same pass.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from ... import ops as K


def _options(section_order: str, pairs: str) -> Tuple[bool, bool]:
    if section_order not in ("blocks", "cycle"):
        raise ValueError(f"section_order is 'blocks' or 'cycle', got {section_order!r}")
    if pairs not in ("half", "interleaved"):
        raise ValueError(f"pairs is 'half' or 'interleaved', got {pairs!r}")
    return section_order == "cycle", pairs == "interleaved"


def rope_kv_append(
    q: Tensor,                              # [T, Hq, d] bf16, rows 8-byte aligned, any strides
    k: Tensor,                              # [T, Hkv, d]
    v: Tensor,
    positions: Tensor,                      # [T] or [axes, T] int32 / int64
    inv_freq: Tensor,                       # [rot / 2] float32, rot <= d
    slots: Tensor,                          # [T] int32 / int64
    k_cache: Tensor,                        # [nb, Hkv, bs, d] bf16, float8_e4m3fn or int8
    v_cache: Tensor,
    *,
    sections: Optional[Sequence[int]] = None,
    section_order: str = "blocks",
    pairs: str = "half",
    rope_scale: float = 1.0,
    qk_norm: bool = False,
    q_gamma: Optional[Tensor] = None,       # [d] bf16 / f32
    k_gamma: Optional[Tensor] = None,
    eps: float = 1e-6,
    k_scales: Optional[Tensor] = None,      # [nb, Hkv, bs] float32, per token and head
    v_scales: Optional[Tensor] = None,
    k_dequant_scale: Optional[Tensor] = None,  # [Hkv], static scales of an fp8 cache
    v_dequant_scale: Optional[Tensor] = None,
    q_out: Optional[Tensor] = None,
    k_out: Optional[Tensor] = None,
) -> Tensor:
    """Rotates Q and K and writes K and V to their slots; returns the rotated Q
    ``[T, Hq, d]`` bf16 (in ``q_out`` where given, which may be ``q``).

    The first ``rot`` channels of a head are rotated; pair ``i`` is ``(i, i +
    rot / 2)`` (``pairs="half"``) or ``(2 i, 2 i + 1)`` (``"interleaved"``), its
    angle ``positions[axis(i)] * inv_freq[i]``, cos and sin times ``rope_scale``.
    ``sections`` says how many pairs each axis has, one axis after the other
    (``section_order="blocks"``); or, with ``"cycle"``, how many turns each axis
    takes: pair ``i`` is of axis ``i % axes`` where ``i < sections[i % axes] *
    axes``, else of axis 0.  Of ``n`` pairs no axis past the first can have more than
    every ``axes``-th so; a larger section is cut, and axis 0 has what is left
    (``[1, 1, 6]`` of 8 pairs is 0 1 2 0 0 2 0 0).  Angles are formed in 64 bits, so
    far positions rotate as near ones do.  With ``qk_norm`` the heads of Q and K are
    RMS-normalised first.  Q, and K in a bf16 cache, are rounded once.

    Caches: bf16; int8 or e4m3fn with per-token scales, as ``quant_kv_write``
    writes them (of the unrounded keys); e4m3fn of ``clamp(x / dequant_scale)``.
    Slots outside the pool (negative padding among them) are skipped; the others
    must differ from each other.  ``k_out`` (may be ``k``) takes the rotated
    keys as rows as well.  ``d`` and ``rot`` are multiples of 8, ``d`` up to 256.
    """
    cycle, interleaved = _options(section_order, pairs)
    if q_out is None:
        q_out = q.new_empty(q.shape, dtype=torch.bfloat16)
    K.rope_append(q, k, v, positions, inv_freq, slots, k_cache, v_cache, q_out, k_out,
                  sections=sections, cycle=cycle, interleaved=interleaved,
                  rope_scale=rope_scale, qk_norm=qk_norm, q_gamma=q_gamma, k_gamma=k_gamma,
                  eps=eps, k_scales=k_scales, v_scales=v_scales, k_dequant=k_dequant_scale,
                  v_dequant=v_dequant_scale)
    return q_out


def rope_rotate(
    q: Tensor,
    k: Tensor,
    positions: Tensor,
    inv_freq: Tensor,
    *,
    sections: Optional[Sequence[int]] = None,
    section_order: str = "blocks",
    pairs: str = "half",
    rope_scale: float = 1.0,
    qk_norm: bool = False,
    q_gamma: Optional[Tensor] = None,
    k_gamma: Optional[Tensor] = None,
    eps: float = 1e-6,
    q_out: Optional[Tensor] = None,
    k_out: Optional[Tensor] = None,
) -> Tuple[Tensor, Tensor]:
    """``rope_kv_append`` without a cache (image encoders): the rotated Q and K."""
    cycle, interleaved = _options(section_order, pairs)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=torch.bfloat16, device=k.device)
    K.rope_append(q, k, None, positions, inv_freq, None, None, None, q_out, k_out,
                  sections=sections, cycle=cycle, interleaved=interleaved,
                  rope_scale=rope_scale, qk_norm=qk_norm, q_gamma=q_gamma, k_gamma=k_gamma,
                  eps=eps)
    return q_out, k_out
