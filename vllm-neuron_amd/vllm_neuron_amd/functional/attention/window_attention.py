"""Attention with a sliding window and a few first tokens that stay visible.

The reference's windows forget every token behind them
(vllm_neuron/functional/attention/attention_segmented_cte.py:122-246,
attention_decode_mask.py:94-236); its sinks are logits, not tokens.  Here the
first tokens of a sequence stay in view however far the window has moved, over
the paged cache and for prompts and single tokens alike, so that a sequence of
any length keeps the blocks of its first tokens and of its window alone.

Keys are taken as they were stored.  Rotated ones keep the positions that they
were rotated by, so the distance of a query from the first tokens grows with the
sequence; positions counted inside the cache are not offered.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from ... import ops as K


def window_attention(
    q: Tensor,                              # [T, Hq, d] bf16
    k_cache: Tensor,                        # [nb, Hkv, bs, d]
    v_cache: Tensor,
    block_table: Tensor,                    # [B, nblk] int32
    seq_lens: Tensor,                       # [B] int32
    *,
    window: int,
    first_tokens: int = 0,
    cu_seqlens_q: Optional[Tensor] = None,  # [B + 1] int32 (None: one token each)
    max_seqlen_q: Optional[int] = None,
    softmax_scale: Optional[float] = None,
    sink: Optional[Tensor] = None,          # [Hq] logits in the denominator
    k_scales: Optional[Tensor] = None,      # [nb, Hkv, bs] float32, per token and head
    v_scales: Optional[Tensor] = None,
    k_dequant_scale: Optional[Tensor] = None,  # [Hkv], static scales of an fp8 cache
    v_dequant_scale: Optional[Tensor] = None,
    out: Optional[Tensor] = None,
    workspace: Optional[Tensor] = None,
) -> Tensor:
    """Returns ``[T, Hq, d]`` bf16.

    Sequence ``i`` has the query tokens ``cu_seqlens_q[i] : cu_seqlens_q[i+1]``
    of ``q`` (token ``i`` alone without ``cu_seqlens_q``, the decode step), the
    last of its ``seq_lens[i]`` tokens; their keys are in the cache already.  The
    query at position ``p`` sees key ``t <= p`` where ``t < first_tokens`` or ``t >
    p - window``.  Blocks that hold no such key may be freed: their table
    entries are never used.

    Lengths are read on the device (a captured call follows them) and clamped to
    what the table holds; ``max_seqlen_q`` bounds the query tokens of a sequence
    (default: T, at the cost of a workgroup for every row tile that a sequence of
    T tokens would have), those past it are not computed; ``cu_seqlens_q`` must not
    decrease.  A query without keys gives zeros.  Rows that nothing computes stay
    as they were in a given ``out`` and are zeros in the returned tensor
    otherwise.  A NaN or infinity in a value row reaches the queries that see it,
    and may reach others of the same sequence and call.

    Where ``min(max_seqlen_q, T)`` times the heads of a kv head is at most 32,
    probabilities meet V as two bf16 numbers each (2^-16 of them is lost), else as
    one (2^-8).  The bound decides for the whole call: a single token beside a long
    prompt is computed as the prompt is, and faster in a call of its own.

    Caches: bf16; e4m3fn with static per-head scales; e4m3fn or int8 with the
    per-token scales of ``quant_kv_write`` and ``rope_kv_append``.  ``d`` is a
    multiple of 8 (8-bit caches: 16) up to 128, ``block_size`` of 16.
    """
    return K.window_attention(
        q, k_cache, v_cache, block_table, seq_lens, window=window, first_tokens=first_tokens,
        cu_seqlens_q=cu_seqlens_q,
        max_seqlen_q=q.shape[0] if max_seqlen_q is None else max_seqlen_q,
        softmax_scale=q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale,
        sink=sink, k_scales=k_scales, v_scales=v_scales, k_dequant=k_dequant_scale,
        v_dequant=v_dequant_scale, out=out, workspace=workspace)
