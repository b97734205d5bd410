"""Rows that no key reaches (sequences without keys beside ordinary ones) and
rows that nothing computes."""
import random

import pytest
import torch

from span_ref import attend, check
from vllm_neuron_amd.functional import (
    cross_attention,
    quant_kv_read,
    quant_kv_write,
    shared_prefix_attention,
)

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


def _into_used_memory(q, *args, **kw):
    """A call without ``out`` whose output takes memory that held sevens."""
    used = torch.full(q.shape, 7.0, dtype=BF, device=q.device)
    del used
    return cross_attention(q, *args, **kw)


def _computed(cu, most, T):
    """Tokens that the call computes, by sequence."""
    if any(b < a for a, b in zip(cu, cu[1:])):
        return []
    clip = lambda x: min(max(x, 0), T)
    return [(clip(a), min(clip(b), clip(a) + most)) for a, b in zip(cu, cu[1:])]


@pytest.mark.parametrize("cu,most", [
    ([0, 4, 9, 9, 12], 12),          # rows behind the last sequence
    ([3, 4, 9, 9, 20], 20),          # and before the first
    ([0, 6, 9, 15, 20], 4),          # past the maximum
    ([-5, 6, 9, 15, 99], 4),
    ([20, 20, 20, 20, 20], 3),       # sequences without tokens
    ([0, 9, 5, 15, 20], 20),         # a list that decreases
])
def test_rows_of_an_allocated_output(gpu, cu, most):
    """Rows that nothing computes are zeros there, and stay in a given one."""
    T, B, hq, hkv, d, L = 20, 4, 6, 2, 80, 33
    q, k, v = _randn(1, T, hq, d), _randn(2, B, hkv, L, d), _randn(3, B, hkv, L, d)
    lens = [33, 7, 5, 0]
    args = (q.to(gpu), k.to(gpu), v.to(gpu), _i32(gpu, *lens))
    kw = dict(cu_seqlens_q=_i32(gpu, *cu), max_seqlen_q=most)
    got = _into_used_memory(*args, **kw)
    kept = cross_attention(*args, out=torch.full((T, hq, d), 7.0, dtype=BF, device=gpu), **kw)
    rest = torch.ones(T, dtype=torch.bool)
    for i, (a, b) in enumerate(_computed(cu, most, T)):
        rest[a:b] = False
        n = lens[i]
        o, bound = attend(q[a:b], k[i, :, :n].transpose(0, 1).double(), v[i, :, :n].transpose(0, 1).double(),
                          d ** -0.5)
        check(got[a:b], o, bound, f"sequence {i}")
        assert torch.equal(got[a:b], kept[a:b])
    assert (got.cpu()[rest] == 0).all() and (kept.cpu()[rest] == 7.0).all()


def test_more_tokens_than_sequences(gpu):
    """One token each without a list of first tokens; no sequence at all; one
    row tile form and the other, and more rows than workgroups."""
    hq, hkv, d, L = 4, 2, 64, 20
    q = _randn(1, 3000, hq, d).to(gpu)
    k = _randn(2, 5, hkv, L, d).to(gpu)
    got = _into_used_memory(q, k, k, _i32(gpu, 20, 3, 0, 9, 20))
    assert (got[5:] == 0).all() and (got[2] == 0).all() and (got[[0, 1, 3, 4]] != 0).any(-1).all()
    none = _into_used_memory(q, k, k, _i32(gpu))
    assert (none == 0).all()
    tall = _into_used_memory(q, k, k, _i32(gpu, 20, 3, 0, 9, 20), cu_seqlens_q=_i32(gpu, 0, 40, 41, 90, 91, 130))
    assert (tall[130:] == 0).all() and (tall[41:90] == 0).all() and (tall[:41] != 0).any(-1).all()


def test_many_sequences_past_the_maximum(gpu):
    """Several sequences to a thread of the plan, each with rows left over."""
    r = random.Random(7)
    cu = [2]
    for _ in range(600):
        cu.append(cu[-1] + r.choice([0, 1, 2, 5]))
    T, most = cu[-1] + 3, 2
    q, k = _randn(1, T, 2, 16), _randn(2, 600, 1, 9, 16)
    lens = [r.choice([0, 4, 9]) for _ in range(600)]
    got = _into_used_memory(q.to(gpu), k.to(gpu), k.to(gpu), _i32(gpu, *lens), cu_seqlens_q=_i32(gpu, *cu),
                            max_seqlen_q=most).cpu()
    rest = torch.ones(T, dtype=torch.bool)
    for i, (a, b) in enumerate(_computed(cu, most, T)):
        if lens[i]:
            rest[a:b] = False
            kk = k[i, :, :lens[i]].transpose(0, 1).double()
            check(got[a:b], *attend(q[a:b], kk, kk, 0.25), f"sequence {i}")
    assert (got[rest] == 0).all()


def test_padded_batch_in_a_graph(gpu):
    """A captured call without ``out``: replays clear what earlier ones wrote."""
    T, B, hq, hkv, d, L = 64, 3, 4, 2, 64, 50
    q, k = _randn(1, T, hq, d).to(gpu), _randn(2, B, hkv, L, d).to(gpu)
    lens, cu = _i32(gpu, 50, 50, 50), _i32(gpu, 0, 20, 40, 64)
    call = lambda: cross_attention(q, k, k, lens, cu_seqlens_q=cu, max_seqlen_q=24)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for ends in ([20, 40, 64], [1, 2, 3], [5, 5, 9], [30, 40, 64], [9, 3, 4], [0, 0, 64]):
        cu.copy_(torch.tensor([0] + ends, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        done = _computed([0] + ends, 24, T)
        rest = torch.ones(T, dtype=torch.bool)
        for a, b in done:
            rest[a:b] = False
        assert (out.cpu()[rest] == 0).all() and (out.cpu()[~rest] != 0).any(-1).all()


def test_compiled_call_clears_its_rows(gpu):
    q, k = _randn(1, 10, 4, 64).to(gpu), _randn(2, 2, 2, 20, 64).to(gpu)
    lens, cu = _i32(gpu, 20, 20), _i32(gpu, 2, 3, 7)
    step = torch.compile(lambda q: cross_attention(q, k, k, lens, cu_seqlens_q=cu) + 1, fullgraph=True,
                         backend="aot_eager")
    want = cross_attention(q, k, k, lens, cu_seqlens_q=cu) + 1
    got = step(q)
    assert torch.equal(want, got)
    assert (got[:2] == 1).all() and (got[7:] == 1).all()


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("S", [1, 4])
def test_decode_of_a_quantised_cache(gpu, code, S):
    """An ordinary decode step: no prefix, and a prefix table of one entry that
    is never read (out of the pool here)."""
    B, hq, hkv, d, bs, nb = 5, 8, 2, 128, 16, 40
    kc, vc = (torch.zeros(nb, hkv, bs, d, dtype=code, device=gpu) for _ in "kv")
    ks, vs = (torch.zeros(nb, hkv, bs, device=gpu) for _ in "kv")
    lens = [100, 4, 17, 64, 33]
    t = torch.randperm(nb, generator=_gen(1))[:B * 7].view(B, 7).to(torch.int32)
    slots = torch.cat([t[b].long().repeat_interleave(bs)[:n] * bs + torch.arange(n) % bs for b, n in enumerate(lens)])
    quant_kv_write(_randn(2, len(slots), hkv, d).to(gpu), _randn(3, len(slots), hkv, d).to(gpu), slots.to(gpu),
                   kc, vc, ks, vs)
    q = _randn(4, B, S, hq, d)
    out = shared_prefix_attention(q.to(gpu), kc, vc, _i32(gpu, 1 << 30), _i32(gpu, 0), t.to(gpu), _i32(gpu, *lens),
                                  k_scales=ks, v_scales=vs)
    k, v = (x.cpu().double() for x in quant_kv_read(kc, vc, ks, vs, slots.to(gpu), dtype=torch.float32))
    at = 0
    for b, n in enumerate(lens):
        for s in range(S):
            e = n - S + 1 + s
            check(out[b, s:s + 1], *attend(q[b, s:s + 1], k[at:at + e], v[at:at + e], d ** -0.5), f"row {b}, token {s}")
        at += n
