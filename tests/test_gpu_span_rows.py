"""Rows that no key reaches: sequences without keys beside ordinary ones."""
import random

import pytest
import torch

from span_ref import attend, check
from vllm_neuron_amd.functional import cross_attention

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(shape, generator=_gen(seed)).to(BF)


def _i32(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _dense(gpu, hq, hkv, d, L, lens, new, seed=0):
    """Dense keys, out given (7 beforehand, two rows more than the sequences
    have, a column range of a wider tensor): every sequence against float64."""
    B, T = len(lens), sum(new)
    q, k, v = _randn(seed, T + 2, hq, d), _randn(seed + 1, B, hkv, L, d), _randn(seed + 2, B, hkv, L, d)
    cu = [sum(new[:i]) for i in range(B + 1)]
    wide = torch.full((T + 2, hq, d + 8), 7.0, dtype=BF, device=gpu)
    out = wide[..., :d]
    cross_attention(q.to(gpu), k.to(gpu), v.to(gpu), _i32(gpu, *lens), cu_seqlens_q=_i32(gpu, *cu),
                    max_seqlen_q=max(new), out=out)
    assert (out[T:] == 7.0).all() and (wide[..., d:] == 7.0).all()
    got = out.cpu()
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        n = lens[i]
        if n == 0:
            assert (got[a:b] == 0).all(), i
            continue
        o, bound = attend(q[a:b], k[i, :, :n].transpose(0, 1).double(), v[i, :, :n].transpose(0, 1).double(),
                          d ** -0.5)
        check(got[a:b], o, bound, f"sequence {i}")


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (3, 1, 8), (5, 5, 72), (10, 2, 80)])
def test_long_prompt_without_keys(gpu, hq, hkv, d):
    """A text-only prompt beside prompts with keys, longer than the launch has
    workgroups."""
    _dense(gpu, hq, hkv, d, 40, [0, 40, 0, 7, 0], [2048, 16, 1, 3, 0])


def test_many_sequences_without_keys(gpu):
    r = random.Random(3)
    new = [r.choice([0, 1, 2, 5]) for _ in range(700)]
    _dense(gpu, 2, 1, 16, 9, [r.choice([0, 0, r.randint(1, 9)]) for _ in new], new)


def _median(f, n=15):
    f()
    torch.cuda.synchronize()
    t = []
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        t.append(a.elapsed_time(b))
    return sorted(t)[n // 2]


def test_a_prompt_without_keys_costs_no_more_than_one_with_keys(gpu):
    """No workgroup alone clears a sequence's rows (as it did: 20 times the
    time of the same prompt with one key)."""
    q, k = _randn(1, 2048 + 16, 32, 128).to(gpu), _randn(2, 2, 8, 400, 128).to(gpu)
    out, cu = torch.empty_like(q), _i32(gpu, 0, 2048, 2064)
    call = lambda lens: lambda: cross_attention(q, k, k, lens, cu_seqlens_q=cu, max_seqlen_q=2048, out=out)
    none, one = _median(call(_i32(gpu, 0, 400))), _median(call(_i32(gpu, 1, 400)))
    assert none <= 4 * one, (none, one)
