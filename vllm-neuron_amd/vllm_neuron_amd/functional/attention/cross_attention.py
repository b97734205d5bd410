"""Cross attention: decoder tokens over an encoder's states of another length.

No counterpart in the reference, which serves decoder-only models.  Its dense
``flash_attention`` takes one query and one key length for the whole batch and
its paged attention is causal; here every sequence has its own number of query
tokens and of keys, and every query sees every key of its sequence.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from ... import ops as K


def cross_attention(
    q: Tensor,                              # [T, Hq, d] bf16
    k: Tensor,                              # [nb, Hkv, bs, d] cache, or [B, Hkv, L, d]
    v: Tensor,
    key_lens: Tensor,                       # [B] int32
    *,
    block_table: Optional[Tensor] = None,   # [B, nblk] int32 (None: dense k, v)
    cu_seqlens_q: Optional[Tensor] = None,  # [B + 1] int32 (None: one token each)
    max_seqlen_q: Optional[int] = None,
    softmax_scale: Optional[float] = None,
    k_scales: Optional[Tensor] = None,      # [nb, Hkv, bs] float32, per token and head
    v_scales: Optional[Tensor] = None,
    k_dequant_scale: Optional[Tensor] = None,  # [Hkv], static scales of an fp8 cache
    v_dequant_scale: Optional[Tensor] = None,
    out: Optional[Tensor] = None,
    workspace: Optional[Tensor] = None,
) -> Tensor:
    """Returns ``[T, Hq, d]`` bf16.

    Sequence ``i`` has the query tokens ``cu_seqlens_q[i] : cu_seqlens_q[i+1]``
    of ``q`` (token ``i`` alone without ``cu_seqlens_q``, the decode step) and
    the keys ``0 : key_lens[i]`` of block table row ``i``, or of ``k[i]`` where
    ``k``/``v`` are dense.  Lengths are read on the device (a captured call
    follows them) and clamped to what the table or ``L`` holds;
    ``max_seqlen_q`` bounds the query tokens of a sequence (default: T), those
    past it are not computed.  A sequence without keys gives zeros.  Rows that
    nothing computes (past the maximum, or of no sequence) stay as they were in
    a given ``out`` and are zeros in the returned tensor otherwise; a
    ``cu_seqlens_q`` that decreases somewhere computes nothing at all.

    Caches: bf16; e4m3fn with static per-head scales; e4m3fn or int8 with the
    per-token scales of ``quant_kv_write``.  ``d`` is a multiple of 8 (8-bit
    caches: 16) up to 128; ``block_size`` with a table a multiple of 16.
    """
    return K.cross_attention(
        q, k, v, key_lens, block_table=block_table, cu_seqlens_q=cu_seqlens_q,
        max_seqlen_q=q.shape[0] if max_seqlen_q is None else max_seqlen_q,
        softmax_scale=q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale,
        k_scales=k_scales, v_scales=v_scales, k_dequant=k_dequant_scale,
        v_dequant=v_dequant_scale, out=out, workspace=workspace)
