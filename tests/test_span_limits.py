"""Sizes that a launch of the span-attention entry points cannot hold are
refused before anything reaches the device."""
import ctypes

import pytest

from vllm_neuron_amd import _native as N

FAKE = 0x10000  # never dereferenced


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _prefix(batch, s, heads):
    a = N.SharedPrefixArgs()
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "seq_lens", "prefix_table",
              "prefix_len", "workspace"):
        setattr(a, f, FAKE)
    a.q_stride = a.out_stride = _i64(s * heads * 8, heads * 8, 8, 1)
    a.batch, a.s_active = batch, s
    a.num_q_heads, a.num_kv_heads, a.head_dim = heads, 8, 8
    a.cache_dtype, a.num_blocks, a.block_size = N.DTYPE_BF16, 10, 16
    a.prefix_blocks, a.blocks_per_seq, a.prefix_stride = 4, 4, 1
    a.k_cache_stride = a.v_cache_stride = _i64(1024, 128, 8, 1)
    a.bt_stride = _i64(4, 1)
    a.softmax_scale = 0.125
    return a


def test_rows_of_a_shared_prefix_call():
    """The join has up to 64 threads per (token, head) along one axis of its
    grid, which holds 2^32: calls from 2^26 rows on are refused, smaller ones
    get as far as the (missing) workspace."""
    L = N.lib()
    call = lambda *a: N.check(L.mia_shared_prefix_attention(ctypes.byref(_prefix(*a)), None), "prefix")
    for args in ((32768, 64, 64), (1 << 20, 1, 64), (1 << 23, 1, 8)):
        with pytest.raises(ValueError, match="2\\^26"):
            call(*args)
        assert L.mia_shared_prefix_workspace_bytes(ctypes.byref(_prefix(*args))) == 0
    with pytest.raises(ValueError, match="workspace"):
        call((1 << 20) - 1, 1, 64)
