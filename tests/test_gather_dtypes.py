"""The block-table gather copies elements of 1, 2 or 4 bytes by the cache's
dtype: any other dtype (int8 codes among them) is refused before anything
reaches the device, where a wrong element size would read and write past the
tensors."""
import ctypes

import pytest
import torch

from vllm_neuron_amd import _native as N


def _args(dtype, out_dim=0):
    a = N.GatherArgs()
    a.cache = a.block_table = a.out = 0x10000  # never dereferenced
    a.cache_dtype = dtype
    a.cache_stride = (ctypes.c_int64 * 5)(4096, 4096, 128, 1, 0)
    a.bt_stride = (ctypes.c_int64 * 3)(4, 0, 1)
    a.batch, a.num_kv_heads, a.blocks_per_seq, a.block_size, a.head_dim = 1, 1, 4, 32, 128
    a.num_blocks, a.out_dim = 8, out_dim
    return a


@pytest.mark.parametrize("dtype", [N.DTYPE_I8, N.DTYPE_I32, N.DTYPE_I64, N.DTYPE_U32, 99, -1])
@pytest.mark.parametrize("out_dim", [0, 128, 136])
def test_other_dtypes_are_refused(dtype, out_dim):
    with pytest.raises(NotImplementedError, match="gather"):
        N.check(N.lib().mia_gather_kv(ctypes.byref(_args(dtype, out_dim)), None), "gather_kv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int8, torch.int32, torch.int64])
def test_other_tensors_are_refused(gpu, dtype):
    from vllm_neuron_amd import ops

    cache = torch.zeros(3, 2, 16, 64, dtype=dtype, device=gpu)
    table = torch.zeros(1, 2, dtype=torch.int32, device=gpu)
    with pytest.raises(NotImplementedError):
        ops.gather_kv(cache, table)
