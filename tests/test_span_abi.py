"""Refusals of the quantised-cache and span-attention entry points on the CPU:
every call fails validation before anything reaches the device."""
import ctypes

import pytest

from vllm_neuron_amd import _native as N

FAKE = 0x10000  # never dereferenced


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _quant(**over):
    a = N.QuantKvArgs()
    for f in ("k", "v", "slots", "k_cache", "v_cache", "k_scales", "v_scales"):
        setattr(a, f, FAKE)
    a.row_dtype, a.code_dtype, a.slot_dtype = N.DTYPE_BF16, N.DTYPE_I8, N.DTYPE_I64
    a.k_stride = a.v_stride = _i64(512, 64, 1)
    a.k_cache_stride = a.v_cache_stride = _i64(8192, 1024, 64, 1)
    a.k_scale_stride = a.v_scale_stride = _i64(128, 16, 1)
    a.num_tokens, a.num_blocks, a.block_size, a.num_kv_heads, a.head_dim = 4, 10, 16, 8, 64
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _cross(**over):
    a = N.CrossArgs()
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "key_lens", "cu_seqlens_q"):
        setattr(a, f, FAKE)
    a.q_stride = a.out_stride = _i64(2048, 64, 1)
    a.num_tokens, a.num_seqs, a.max_seqlen_q = 12, 3, 5
    a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 8, 64
    a.cache_dtype, a.num_blocks, a.block_size, a.blocks_per_seq = N.DTYPE_BF16, 10, 16, 4
    a.k_cache_stride = a.v_cache_stride = _i64(8192, 1024, 64, 1)
    a.bt_stride = _i64(4, 1)
    a.softmax_scale = 0.125
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _prefix(**over):
    a = N.SharedPrefixArgs()
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "seq_lens", "prefix_table", "prefix_len"):
        setattr(a, f, FAKE)
    a.q_stride = a.out_stride = _i64(2048, 2048, 64, 1)
    a.batch, a.s_active = 3, 1
    a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 8, 64
    a.cache_dtype, a.num_blocks, a.block_size = N.DTYPE_BF16, 10, 16
    a.prefix_blocks, a.blocks_per_seq, a.prefix_stride = 4, 4, 1
    a.k_cache_stride = a.v_cache_stride = _i64(8192, 1024, 64, 1)
    a.bt_stride = _i64(4, 1)
    a.softmax_scale = 0.125
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,err,text", [
    (dict(k=None), ValueError, "null"),
    (dict(num_tokens=-1), ValueError, "num_tokens"),
    (dict(num_tokens=1 << 30), ValueError, "2\\^31"),
    (dict(row_dtype=N.DTYPE_I32), NotImplementedError, "row dtype"),
    (dict(code_dtype=N.DTYPE_BF16), NotImplementedError, "cache dtype"),
    (dict(slot_dtype=N.DTYPE_F32), ValueError, "slot dtype"),
    (dict(head_dim=520), NotImplementedError, "512"),
    (dict(block_size=0), ValueError, "geometry"),
])
def test_quant_refusals(over, err, text):
    L = N.lib()
    for fn in (L.mia_quant_kv_write, L.mia_quant_kv_read):
        with pytest.raises(err, match=text):
            N.check(fn(ctypes.byref(_quant(**over)), None), "quant")


SHARED = [
    (dict(num_q_heads=30), ValueError, "GQA"),
    (dict(num_kv_heads=0), ValueError, "GQA"),
    (dict(head_dim=60), NotImplementedError, "head_dim"),
    (dict(head_dim=136), NotImplementedError, "head_dim"),
    (dict(cache_dtype=N.DTYPE_F16), NotImplementedError, "cache dtype"),
    (dict(cache_dtype=N.DTYPE_I8), ValueError, "int8"),
    (dict(cache_dtype=N.DTYPE_FP8_E4M3FN, head_dim=72), NotImplementedError, "head_dim"),
    (dict(k_scales=FAKE, v_scales=FAKE), ValueError, "bf16 cache"),
    (dict(cache_dtype=N.DTYPE_I8, k_scales=FAKE), ValueError, "go together"),
    (dict(block_size=24), NotImplementedError, "block_size"),
    (dict(block_size=1 << 28), ValueError, "2\\^30"),
    (dict(blocks_per_seq=0), ValueError, "empty"),
    (dict(k_cache=FAKE + 8), ValueError, "16-byte"),
    (dict(k_cache_stride=_i64(8192, 1024, 60, 1)), ValueError, "16-byte"),
    (dict(v_cache_stride=_i64(8192, 1024, 64, 2)), ValueError, "contiguous"),
    (dict(v_cache_stride=_i64(8192, 1024, 1 << 27, 1)), ValueError, "token stride"),
    (dict(q=FAKE + 2), ValueError, "q rows"),
    (dict(out=FAKE + 2), ValueError, "out rows"),
    (dict(workspace=None), ValueError, "workspace"),
    (dict(workspace=FAKE + 8, workspace_bytes=1 << 40), ValueError, "workspace"),
    (dict(workspace=FAKE, workspace_bytes=100), ValueError, "workspace"),
]


@pytest.mark.parametrize("over,err,text", SHARED + [
    (dict(key_lens=None), ValueError, "null"),
    (dict(max_seqlen_q=0), ValueError, "max_seqlen_q"),
    (dict(block_table=None), ValueError, "dense"),
    (dict(num_seqs=-1), ValueError, "shape"),
    (dict(num_tokens=1 << 28), ValueError, "2\\^30"),
    (dict(num_tokens=1 << 24, blocks_per_seq=1 << 16), ValueError, "key tiles"),
])
def test_cross_refusals(over, err, text):
    L = N.lib()
    with pytest.raises(err, match=text):
        N.check(L.mia_cross_attention(ctypes.byref(_cross(**over)), None), "cross")


@pytest.mark.parametrize("over,err,text", SHARED + [
    (dict(seq_lens=None), ValueError, "null"),
    (dict(s_active=0), ValueError, "shape"),
    (dict(s_active=65), NotImplementedError, "64"),
    (dict(prefix_blocks=0), ValueError, "prefix"),
    (dict(batch=1 << 20, blocks_per_seq=1 << 16), ValueError, "key tiles"),
])
def test_prefix_refusals(over, err, text):
    L = N.lib()
    with pytest.raises(err, match=text):
        N.check(L.mia_shared_prefix_attention(ctypes.byref(_prefix(**over)), None), "prefix")


def test_workspace_sizes():
    """The size grows with the call's rows and is 0 for what is refused or
    has nothing to compute."""
    L = N.lib()
    cross = lambda **o: L.mia_cross_workspace_bytes(ctypes.byref(_cross(**o)))
    prefix = lambda **o: L.mia_shared_prefix_workspace_bytes(ctypes.byref(_prefix(**o)))
    assert 0 < cross(max_seqlen_q=1) < cross(max_seqlen_q=12)
    assert cross(head_dim=60) == 0 and cross(num_seqs=0) == 0
    assert 0 < prefix(batch=1) < prefix(batch=300)
    assert prefix(s_active=65) == 0 and prefix(batch=0) == 0
    N.check(L.mia_cross_attention(ctypes.byref(_cross(num_tokens=0)), None), "cross")
    N.check(L.mia_shared_prefix_attention(ctypes.byref(_prefix(batch=0)), None), "prefix")
    N.check(L.mia_quant_kv_write(ctypes.byref(_quant(num_tokens=0)), None), "quant")
