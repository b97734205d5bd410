"""Refusals of the rotation and windowed-attention entry points on the CPU:
every call fails validation before anything reaches the device."""
import ctypes

import pytest
import torch

from vllm_neuron_amd import _native as N
from vllm_neuron_amd.functional import rope_kv_append, rope_rotate, window_attention

FAKE = 0x10000  # never dereferenced


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _rope(**over):
    a = N.RopeAppendArgs()
    for f in ("q", "k", "v", "q_out", "positions", "inv_freq", "slots", "k_cache", "v_cache"):
        setattr(a, f, FAKE)
    a.q_stride = a.q_out_stride = a.k_stride = a.v_stride = _i64(2048, 64)
    a.num_tokens, a.num_q_heads, a.num_kv_heads, a.head_dim, a.rot_dim = 4, 32, 8, 64, 64
    a.pos_stride, a.pos_dtype, a.axes = _i64(4, 1), N.DTYPE_I64, 1
    a.section = (ctypes.c_int32 * 4)(32, 0, 0, 0)
    a.slot_dtype, a.cache_dtype = N.DTYPE_I64, N.DTYPE_BF16
    a.k_cache_stride = a.v_cache_stride = _i64(8192, 1024, 64, 1)
    a.num_blocks, a.block_size, a.rope_scale = 10, 16, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _window(**over):
    a = N.WindowArgs()
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "seq_lens", "cu_seqlens_q"):
        setattr(a, f, FAKE)
    a.q_stride = a.out_stride = _i64(2048, 64, 1)
    a.num_tokens, a.num_seqs, a.max_seqlen_q = 12, 3, 5
    a.num_q_heads, a.num_kv_heads, a.head_dim = 32, 8, 64
    a.cache_dtype, a.num_blocks, a.block_size, a.blocks_per_seq = N.DTYPE_BF16, 10, 16, 4
    a.k_cache_stride = a.v_cache_stride = _i64(8192, 1024, 64, 1)
    a.bt_stride = _i64(4, 1)
    a.window, a.first_tokens, a.softmax_scale = 64, 4, 0.125
    for k, v in over.items():
        setattr(a, k, v)
    return a


SEC = lambda *v: (ctypes.c_int32 * 4)(*v)


@pytest.mark.parametrize("over,err,text", [
    (dict(q=None), ValueError, "null"),
    (dict(inv_freq=None), ValueError, "null"),
    (dict(v_cache=None), ValueError, "null"),
    (dict(num_tokens=-1), ValueError, "num_tokens"),
    (dict(num_tokens=1 << 24), ValueError, "2\\^24"),
    (dict(num_kv_heads=0), ValueError, "head counts"),
    (dict(head_dim=60), NotImplementedError, "head_dim"),
    (dict(head_dim=264), NotImplementedError, "head_dim"),
    (dict(rot_dim=36), NotImplementedError, "multiple of 8"),
    (dict(rot_dim=72), ValueError, "more rotated"),
    (dict(pos_dtype=N.DTYPE_F32), ValueError, "positions"),
    (dict(axes=0), NotImplementedError, "axes"),
    (dict(axes=5), NotImplementedError, "axes"),
    (dict(axes=2, section=SEC(40, -8, 0, 0)), ValueError, "negative"),
    (dict(section=SEC(31, 0, 0, 0)), ValueError, "sections"),
    (dict(q=FAKE + 4), ValueError, "8-byte"),
    (dict(k_stride=_i64(2048, 66)), ValueError, "8-byte"),
    (dict(slots=None), ValueError, "without a cache"),
    (dict(slots=None, v=None), ValueError, "without a cache"),
    (dict(slot_dtype=N.DTYPE_F32), ValueError, "slot dtype"),
    (dict(cache_dtype=N.DTYPE_F16), NotImplementedError, "cache dtype"),
    (dict(cache_dtype=N.DTYPE_I8), ValueError, "int8"),
    (dict(k_scales=FAKE), ValueError, "go together"),
    (dict(k_scales=FAKE, v_scales=FAKE), ValueError, "bf16 cache"),
    (dict(k_dequant=FAKE, v_dequant=FAKE), ValueError, "static scales"),
    (dict(cache_dtype=N.DTYPE_FP8_E4M3FN, k_dequant=FAKE, v_dequant=FAKE, k_scales=FAKE, v_scales=FAKE), ValueError,
     "static scales"),
    (dict(block_size=0), ValueError, "empty"),
    (dict(k_cache=FAKE + 4), ValueError, "4 elements"),
    (dict(v_cache_stride=_i64(8192, 1024, 64, 2)), ValueError, "contiguous"),
    (dict(v_cache_stride=_i64(8192, 1024, 66, 1)), ValueError, "4 elements"),
])
def test_rope_refusals(over, err, text):
    with pytest.raises(err, match=text):
        N.check(N.lib().mia_rope_append(ctypes.byref(_rope(**over)), None), "rope")


@pytest.mark.parametrize("over,err,text", [
    (dict(seq_lens=None), ValueError, "null"),
    (dict(block_table=None), ValueError, "null"),
    (dict(num_seqs=-1), ValueError, "shape"),
    (dict(max_seqlen_q=0), ValueError, "max_seqlen_q"),
    (dict(cu_seqlens_q=None, num_seqs=13), ValueError, "fewer tokens"),
    (dict(window=0), ValueError, "window"),
    (dict(window=(1 << 30) + 1), ValueError, "window"),
    (dict(first_tokens=-1), ValueError, "first_tokens"),
    (dict(num_q_heads=30), ValueError, "GQA"),
    (dict(head_dim=60), NotImplementedError, "head_dim"),
    (dict(cache_dtype=N.DTYPE_I8), ValueError, "int8"),
    (dict(block_size=24), NotImplementedError, "block_size"),
    (dict(k_cache=FAKE + 8), ValueError, "16-byte"),
    (dict(q=FAKE + 2), ValueError, "q rows"),
    (dict(num_tokens=1 << 20, num_seqs=1 << 12, max_seqlen_q=1 << 20), ValueError, "2\\^23"),
    (dict(num_seqs=1, num_tokens=1, max_seqlen_q=1, num_q_heads=4, num_kv_heads=1, blocks_per_seq=1000,
          window=1 << 20), ValueError, "workspace"),
])
def test_window_refusals(over, err, text):
    with pytest.raises(err, match=text):
        N.check(N.lib().mia_window_attention(ctypes.byref(_window(**over)), None), "window")


def test_workspace_and_empty_calls():
    L = N.lib()
    size = lambda **o: L.mia_window_workspace_bytes(ctypes.byref(_window(**o)))
    one = dict(num_seqs=1, num_tokens=1, max_seqlen_q=1, blocks_per_seq=1000, window=1 << 20)
    assert size(**one) > 0
    assert size(num_seqs=1, num_tokens=1, max_seqlen_q=1) == 0         # a table of few tiles
    assert size(**{**one, "num_seqs": 500, "num_tokens": 500}) == 0    # rows enough for the device
    assert size(head_dim=60) == 0 and size(num_tokens=0) == 0
    # partials of many short sequences beside a long one stay bounded
    assert size(num_seqs=128, num_tokens=1 << 12, max_seqlen_q=1 << 12, num_q_heads=4, num_kv_heads=1,
                blocks_per_seq=1000, window=1 << 20) <= 129 << 20
    N.check(L.mia_window_attention(ctypes.byref(_window(num_tokens=0)), None), "window")
    N.check(L.mia_window_attention(ctypes.byref(_window(num_seqs=0)), None), "window")
    N.check(L.mia_rope_append(ctypes.byref(_rope(num_tokens=0)), None), "rope")


def test_no_cpu_path():
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    pos, inv = torch.arange(2), torch.ones(32)
    cache = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        rope_kv_append(q, k, k, pos, inv, pos, cache, cache)
    with pytest.raises(RuntimeError):
        rope_rotate(q, k, pos, inv)
    with pytest.raises(ValueError, match="section_order"):
        rope_rotate(q, k, pos, inv, section_order="x")
    with pytest.raises(ValueError, match="pairs"):
        rope_rotate(q, k, pos, inv, pairs="x")
    with pytest.raises(RuntimeError):
        window_attention(q, cache, cache, pos[:, None].int(), pos.int(), window=4)


def test_shapes_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="cuda")
        q, k = e(5, 4, 64), e(5, 2, 64)
        pos, K = e(3, 5, dt=torch.int64), e(8, 2, 16, 64)
        out = rope_kv_append(q, k, k, pos, e(32, dt=torch.float32), pos[0], K, K, sections=[12, 10, 10])
        assert out.shape == q.shape
        assert rope_rotate(q, k, pos, e(32, dt=torch.float32), sections=[12, 10, 10])[1].shape == k.shape
        got = window_attention(q, K, K, e(5, 4, dt=torch.int32), e(5, dt=torch.int32), window=9, first_tokens=1)
        assert got.shape == q.shape and got.dtype == torch.bfloat16
