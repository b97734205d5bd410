"""Decode attention of a batch that shares a long prefix.

The reference's decode (vllm_neuron/functional/attention/attention_decode.py:
910-1161) walks every row's whole context; rows behind one system prompt or
document read its keys once per row.  Here the prefix is one span for the whole
batch, read once and multiplied with all rows' queries, each row's own keys are
a second span, and both are joined by one softmax.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from ... import ops as K


def shared_prefix_attention(
    q: Tensor,              # [B, S, Hq, d] bf16
    k_cache: Tensor,        # [nb, Hkv, bs, d] bf16, e4m3fn or int8
    v_cache: Tensor,
    prefix_table: Tensor,   # [nblk_p] int32: blocks of the shared prefix
    prefix_len: Tensor,     # int32, one element on the device
    block_table: Tensor,    # [B, nblk] int32: each row's own blocks
    seq_lens: Tensor,       # [B] int32: each row's own tokens, the S new ones included
    *,
    softmax_scale: Optional[float] = None,
    sink: Optional[Tensor] = None,          # [Hq]
    k_scales: Optional[Tensor] = None,      # [nb, Hkv, bs] float32, per token and head
    v_scales: Optional[Tensor] = None,
    k_dequant_scale: Optional[Tensor] = None,  # [Hkv], static scales of an fp8 cache
    v_dequant_scale: Optional[Tensor] = None,
    out: Optional[Tensor] = None,
    workspace: Optional[Tensor] = None,
) -> Tensor:
    """Returns ``[B, S, Hq, d]`` bf16.

    Every row sees the keys ``0 : prefix_len`` of ``prefix_table``; token ``s``
    of row ``b`` also sees its own keys ``0 : seq_lens[b] - S + 1 + s`` of
    ``block_table[b]``.  The new tokens' K/V are in the cache already
    (``quant_kv_write``, or the cache write of ``qkv_proj``), as the last S of
    the row's own keys.  The sink logit joins the denominator.  A row without
    any key gives zeros.  Lengths are read on the device (a captured call
    follows them) and clamped to what the tables hold.

    Caches as for ``cross_attention``; at most 64 new tokens per row, and fewer
    than 2^26 (token, head) rows in a call.
    """
    return K.shared_prefix_attention(
        q, k_cache, v_cache, prefix_table, prefix_len, block_table, seq_lens,
        softmax_scale=q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale,
        sink=sink, k_scales=k_scales, v_scales=v_scales, k_dequant=k_dequant_scale,
        v_dequant=v_dequant_scale, out=out, workspace=workspace)
