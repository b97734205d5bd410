"""Quantised cache: calls of more rows than one axis of a launch grid holds
(2^32 threads along x, 64 lanes to a row of any d off the vector form)."""
import pytest
import torch

from span_ref import quantise
from vllm_neuron_amd.functional import quant_kv_read, quant_kv_write

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_grid_axis(gpu):
    """2^26 + 512 rows in one call equal the same rows in four."""
    T, h, d, bs = (1 << 23) + 64, 8, 7, 64
    nb = T // bs
    g = torch.Generator(device=gpu).manual_seed(1)
    k = torch.randn(T, h, d, generator=g, device=gpu, dtype=torch.bfloat16)
    v = k.flip(0)
    slots = torch.arange(T, dtype=torch.int32, device=gpu).flip(0)
    mk = lambda: ([torch.zeros(nb, h, bs, d, dtype=torch.int8, device=gpu) for _ in "kv"]
                  + [torch.full((nb, h, bs), -2.0, device=gpu) for _ in "kv"])
    one, four = mk(), mk()
    quant_kv_write(k, v, slots, *one)
    step = T // 4
    for i in range(0, T, step):
        quant_kv_write(k[i:i + step], v[i:i + step], slots[i:i + step], *four)
    for a, b in zip(one, four):
        assert torch.equal(a, b)
    for at in (0, T // 2, T - 3):
        want, want_s = quantise(k[at:at + 3], torch.int8)
        for t in range(3):
            s = int(slots[at + t])
            assert torch.equal(one[0][s // bs, :, s % bs].cpu().double(), want[t])
            assert torch.equal(one[2][s // bs, :, s % bs].cpu().double(), want_s[t])
    rk, rv = quant_kv_read(*one, slots)
    for i in range(0, T, step):
        a, b = quant_kv_read(*one, slots[i:i + step])
        assert torch.equal(rk[i:i + step], a) and torch.equal(rv[i:i + step], b)
