"""The operators of an 8-bit attention layer together, as a serving step runs
them: row-quantised projection, rotation by several axes with the append to an
int8 cache, windowed attention with visible first tokens, output projection;
prompts and decode steps of the same sequences, eager and captured."""
import math

import pytest
import torch

from rope_ref import rms, rotate
from vllm_neuron_amd.functional import (int8_linear, qkv_proj, quant_kv_read, quant_rows, rope_kv_append,
                                        window_attention)
from vllm_neuron_amd.utils.common_types import NormType, QuantizationType

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HQ, HKV, D, H, BS = 8, 2, 64, 512, 16
FUSED = (HQ + 2 * HKV) * D


class Layer:
    def __init__(self, gpu, window, first, cache=torch.int8, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = torch.randn(FUSED, H, generator=g) * H ** -0.5
        wo = torch.randn(H, HQ * D, generator=g) * (HQ * D) ** -0.5
        self.w, self.ws = quant_rows(w.to(BF).to(gpu))  # laid out once
        self.wo, self.wos = quant_rows(wo.to(BF).to(gpu))
        self.gamma = (1 + 0.1 * torch.randn(H, generator=g)).to(BF).to(gpu)
        self.inv = torch.tensor([10000.0 ** (-2.0 * i / D) for i in range(D // 2)], device=gpu)
        self.sections, self.window, self.first = [12, 10, 10], window, first
        nb = 64
        pool = lambda: torch.zeros((nb, HKV, BS, D), dtype=cache, device=gpu)
        self.K, self.V = pool(), pool()
        self.ks = self.vs = None
        if cache != BF:
            self.ks, self.vs = torch.zeros((nb, HKV, BS), device=gpu), torch.zeros((nb, HKV, BS), device=gpu)

    def step(self, x, positions, slots, table, lens, cu, most):
        """[T, H] hidden states -> [T, H], the cache extended."""
        T = x.shape[0]
        qkv = qkv_proj(x.view(1, T, H), self.w.t(), norm_type=NormType.RMS_NORM, norm_weights=self.gamma,
                       quantization_type=QuantizationType.ROW, qkv_w_scale=self.ws).view(T, -1, D)
        q = rope_kv_append(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], positions, self.inv, slots, self.K,
                           self.V, sections=self.sections, qk_norm=True, k_scales=self.ks, v_scales=self.vs)
        o = window_attention(q, self.K, self.V, table, lens, window=self.window, first_tokens=self.first,
                             cu_seqlens_q=cu, max_seqlen_q=most, k_scales=self.ks, v_scales=self.vs)
        c, s = quant_rows(o.view(T, HQ * D))
        return int8_linear(c, s, self.wo, self.wos)

    def reference(self, x, positions):
        """float64, one sequence of all its tokens, unquantised activations and
        cache."""
        w, wo = self.w.double().cpu() * self.ws.double().cpu()[:, None], self.wo.double().cpu() * self.wos.double().cpu()[:, None]
        qkv = (rms(x, self.gamma, 1e-6) @ w.t()).view(x.shape[0], -1, D)
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
        q, k = (rotate(rms(t, None, 1e-6), positions, self.inv, self.sections, "blocks", "half")[0] for t in (q, k))
        n = x.shape[0]
        t, p = torch.arange(n)[None], torch.arange(n)[:, None]
        seen = (t <= p) & ((t < self.first) | (t > p - self.window))
        k, v = k.repeat_interleave(HQ // HKV, 1), v.repeat_interleave(HQ // HKV, 1)
        s = torch.einsum("mhd,nhd->hmn", q, k) / math.sqrt(D)
        o = torch.einsum("hmn,nhd->mhd", torch.softmax(s.masked_fill(~seen, -math.inf), -1), v)
        return o.reshape(n, -1) @ wo.t()


def _sequences(gpu, lens, seed):
    """Hidden states, three-axis positions and a block table of each sequence."""
    g = torch.Generator().manual_seed(seed)
    xs = [torch.randn(n, H, generator=g).to(BF).to(gpu) for n in lens]
    pos = [torch.stack([torch.arange(n), torch.arange(n) // 7, torch.arange(n) % 7]) for n in lens]
    per = [(n + BS - 1) // BS for n in lens]
    ids = torch.randperm(63, generator=g)[:sum(per)] + 1
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = ids[at:at + n].int()
        at += n
    return xs, pos, table


def _slots(table, i, start, stop):
    t = torch.arange(start, stop)
    return table[i, t // BS].long() * BS + t % BS


@pytest.mark.parametrize("cache", [torch.int8, torch.float8_e4m3fn, BF])
@pytest.mark.parametrize("window,first", [(40, 4), (1000, 0), (16, 20)])
def test_prompts_then_single_tokens(gpu, cache, window, first):
    """Ragged prompts in one call, then decode steps of all sequences: what the
    layer gives at every token against the unquantised float64 layer.  The error
    is that of 8-bit activations and cache: each quantisation is off by a
    uniform half step of 1/127 of the row's maximum (about 4 times its root mean
    square over 512 channels), 0.0091 of the row's norm; two projections, the
    keys (through the scores, whose spread about 1 makes it a relative error of
    the same size) and the values: 0.0091 * 2 = 0.018 together where independent,
    and e4m3fn caches 2^-4 / sqrt(3) = 0.036 for keys and values each: 0.055."""
    lens, steps = [70, 1, 133], 3
    layer = Layer(gpu, window, first, cache)
    total = [n + steps for n in lens]
    xs, pos, table = _sequences(gpu, total, 1)
    refs = [layer.reference(x, p) for x, p in zip(xs, pos)]
    dev = lambda t: t.to(gpu)
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    got = [torch.zeros(n, H, dtype=torch.float64) for n in total]
    y = layer.step(torch.cat([x[:n] for x, n in zip(xs, lens)]),
                   dev(torch.cat([p[:, :n] for p, n in zip(pos, lens)], 1)),
                   dev(torch.cat([_slots(table, i, 0, n) for i, n in enumerate(lens)])), dev(table),
                   torch.tensor(lens, dtype=torch.int32, device=gpu), torch.tensor(cu, dtype=torch.int32, device=gpu),
                   max(lens))
    for i, n in enumerate(lens):
        got[i][:n] = y[cu[i]:cu[i + 1]].double().cpu()
    for k in range(steps):
        now = [n + k for n in lens]
        y = layer.step(torch.stack([x[n] for x, n in zip(xs, now)]),
                       dev(torch.stack([p[:, n] for p, n in zip(pos, now)], 1)),
                       dev(torch.cat([_slots(table, i, n, n + 1) for i, n in enumerate(now)])), dev(table),
                       torch.tensor([n + 1 for n in now], dtype=torch.int32, device=gpu), None, 1)
        for i, n in enumerate(now):
            got[i][n] = y[i].double().cpu()
    limit = 0.08 if cache == torch.float8_e4m3fn else 0.04
    for g, r in zip(got, refs):
        rel = (g - r).norm(dim=1) / r.norm(dim=1)
        assert rel.max() < limit, rel.max()


def test_a_captured_decode_step_follows_its_tensors(gpu):
    layer = Layer(gpu, 24, 3)
    lens = [30, 45]
    xs, pos, table = _sequences(gpu, [n + 5 for n in lens], 2)
    tab = table.to(gpu)
    for i, n in enumerate(lens):
        layer.step(xs[i][:n], pos[i][:, :n].to(gpu), _slots(table, i, 0, n).to(gpu), tab[i:i + 1],
                   torch.tensor([n], dtype=torch.int32, device=gpu), torch.tensor([0, n], dtype=torch.int32, device=gpu), n)
    kept = [t.clone() for t in (layer.K, layer.V, layer.ks, layer.vs)]
    put = lambda saved: [a.copy_(b) for a, b in zip((layer.K, layer.V, layer.ks, layer.vs), saved)]
    x, p = torch.zeros(2, H, dtype=BF, device=gpu), torch.zeros(3, 2, dtype=torch.int64, device=gpu)
    s, n = torch.zeros(2, dtype=torch.int64, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)

    def fill(k):
        x.copy_(torch.stack([xs[i][m + k] for i, m in enumerate(lens)]))
        p.copy_(torch.stack([pos[i][:, m + k] for i, m in enumerate(lens)], 1))
        s.copy_(torch.cat([_slots(table, i, m + k, m + k + 1) for i, m in enumerate(lens)]))
        n.copy_(torch.tensor([m + k + 1 for m in lens], dtype=torch.int32))

    want = []
    for k in range(5):
        fill(k)
        want.append(layer.step(x, p, s, tab, n, None, 1).clone())
    after = [t.clone() for t in (layer.K, layer.V, layer.ks, layer.vs)]
    put(kept)
    fill(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step(x, p, s, tab, n, None, 1)
    put(kept)
    for k in range(5):
        fill(k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[k]), k
    assert all(torch.equal(a, b) for a, b in zip(after, (layer.K, layer.V, layer.ks, layer.vs)))
    # the whole step under torch.compile
    put(kept)
    fill(0)
    compiled = torch.compile(lambda *a: layer.step(*a, None, 1), fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(x, p, s, tab, n), want[0])


def test_blocks_behind_the_window_may_be_freed(gpu):
    """A long decode keeps the blocks of its first tokens and of its window: the
    entries of the others are -1 and their blocks hold something else."""
    layer = Layer(gpu, 32, 5)
    xs, pos, table = _sequences(gpu, [200], 3)
    tab = table.to(gpu)
    args = lambda a, b: (xs[0][a:b], pos[0][:, a:b].to(gpu), _slots(table, 0, a, b).to(gpu))
    layer.step(*args(0, 199), tab, torch.tensor([199], dtype=torch.int32, device=gpu),
               torch.tensor([0, 199], dtype=torch.int32, device=gpu), 199)
    last = lambda t: layer.step(*args(199, 200), t, torch.tensor([200], dtype=torch.int32, device=gpu), None, 1)
    want = last(tab)
    freed = tab.clone()
    for j in range(1, (200 - 32) // BS):
        layer.ks[table[0, j]] = math.nan
        layer.vs[table[0, j]] = math.nan
        freed[0, j] = -1
    assert torch.equal(last(freed), want)
    k, _ = quant_kv_read(layer.K, layer.V, layer.ks, layer.vs, _slots(table, 0, 195, 200).to(gpu))
    assert torch.isfinite(k).all()
