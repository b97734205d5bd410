"""Attention functionals (vllm_neuron/functional/__init__.py:7-14)."""
from .attention.attention_cte import flash_attention
from .attention.attention_decode import attention_decode, scatter_packed_k
from .attention.attention_decode_mask import gen_attention_decode_mask
from .attention.attention_segmented_cte import segmented_attention
from .attention.cross_attention import cross_attention
from .attention.int8_linear import int8_linear, quant_rows
from .attention.mixed_batch import mixed_batch_attention
from .attention.qkv import qkv_proj
from .attention.quant_cache import quant_kv_read, quant_kv_write
from .attention.rope_append import rope_kv_append, rope_rotate
from .attention.shared_prefix import shared_prefix_attention
from .attention.swa_fused import swa_fused_attention
from .attention.window_attention import window_attention

__all__ = [
    "flash_attention",
    "attention_decode",
    "gen_attention_decode_mask",
    "segmented_attention",
    "scatter_packed_k",
    "mixed_batch_attention",
    "qkv_proj",
    "swa_fused_attention",
    "quant_kv_write",
    "quant_kv_read",
    "cross_attention",
    "shared_prefix_attention",
    "quant_rows",
    "int8_linear",
    "rope_kv_append",
    "rope_rotate",
    "window_attention",
]
