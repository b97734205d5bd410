"""Window attention: any bound of the query tokens is a bound, and tables too
wide for their count's 32 bits are refused."""
import pytest
import torch

from vllm_neuron_amd.functional import window_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _call(gpu, **over):
    g = torch.Generator().manual_seed(1)
    q, K, V = (torch.randn(s, generator=g).to(BF).to(gpu) for s in ((7, 4, 64), (6, 2, 16, 64), (6, 2, 16, 64)))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    kw = dict(block_table=i32(1, 2, 3, 4).view(2, 2), seq_lens=i32(20, 30), window=9, first_tokens=2,
              cu_seqlens_q=i32(0, 3, 7))
    kw.update(over)
    return window_attention(q, K, V, **kw)


@pytest.mark.parametrize("most", [7, 1 << 20, (1 << 31) - 1, 1 << 31, 1 << 40])
def test_a_bound_past_32_bits_is_no_bound(gpu, most):
    assert torch.equal(_call(gpu, max_seqlen_q=most), _call(gpu))


def test_sizes_past_32_bits_are_refused(gpu):
    wide = torch.ones(2, 1, dtype=torch.int32, device=gpu).expand(2, 1 << 31)
    with pytest.raises(ValueError):
        _call(gpu, block_table=wide)
    for most in (0, -1, -(1 << 31) - 1):
        with pytest.raises(ValueError):
            _call(gpu, max_seqlen_q=most)
