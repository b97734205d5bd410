"""Shared-prefix attention and the paged decode over [prefix | own] tables
compute the same attention: both within the bound of the float64 statement,
which neither a zero output nor one over fewer keys meets.

The decode multiplies the unscaled bf16 rows and scales the scores in fp32,
rounds probabilities to bf16 for its second product and keeps sums and partials
in fp32: the same roundings as the span kernels', so the same bound."""
import pytest
import torch

from span_ref import attend, check
from test_gpu_span_attention import Pool, _gen, _randn, _tables

P, LENS = 256, [33, 1, 64, 100]
SHAPES = [(8, 2, 128, 32, False), (16, 2, 64, 16, True), (4, 4, 128, 64, True)]


class Case:
    def __init__(self, hq, hkv, d, bs, sink, dev):
        self.tp, nb = _tables([P], bs, 1, 0, spare=0)
        self.t, nb = _tables(LENS, bs, nb, 1, spare=0)
        self.pool = Pool("bf16", nb, hkv, bs, d, 2, dev)
        self.joined = torch.cat([self.tp.expand(len(LENS), -1), self.t], 1)
        self.q = _randn(_gen(3), len(LENS), 1, hq, d)
        self.sink = torch.randn(hq, generator=_gen(4)) if sink else None
        self.scale = d ** -0.5

    def rows(self, b):
        return self.pool.rows(self.joined[b], P + LENS[b])

    def exact(self, b, keep=None, heads=None):
        k, v = self.rows(b)
        if keep is not None:
            k, v = k[keep], v[keep]
        if heads is not None:
            k, v = k[:, heads], v[:, heads]
        return attend(self.q[b], k, v, self.scale, self.sink)


@pytest.mark.parametrize("shape", SHAPES)
def test_the_bound_tells_other_attentions_apart(shape):
    """Zeros, the first 64 keys, the prefix or the own keys alone and another
    head's keys all lie past the bound."""
    c = Case(*shape, "cpu")
    for b, n in enumerate(LENS):
        o, bound = c.exact(b)
        past = lambda x: ((x - o).abs() > bound).any(-1).all()  # in every row and head
        assert not ((o - o).abs() > bound).any()
        assert past(torch.zeros_like(o))
        assert past(c.exact(b, slice(0, 64))[0])
        assert past(c.exact(b, slice(P, None))[0])
        if n > 1:
            assert past(c.exact(b, slice(0, P))[0])
        assert past(c.exact(b, heads=list(range(1, c.pool.k.shape[1])) + [0])[0])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_prefix_and_decode_within_one_bound(gpu, shape):
    from vllm_neuron_amd.functional import shared_prefix_attention
    from vllm_neuron_amd.functional.attention.attention_decode import paged_decode_core

    c = Case(*shape, gpu)
    bs, B = shape[3], len(LENS)
    c.pool.up()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    sink = None if c.sink is None else c.sink.to(gpu)
    got = shared_prefix_attention(c.q.to(gpu), c.pool.gk, c.pool.gv, c.tp[0].to(gpu), i32(P), c.t.to(gpu),
                                  i32(*LENS), sink=sink)
    at = torch.tensor([n - 1 for n in LENS])
    blk = c.t.gather(1, (at // bs).view(-1, 1)).view(-1).long()
    new = lambda x: x[blk.to(gpu), :, (at % bs).to(gpu)].unsqueeze(1)
    dec = paged_decode_core(c.q.to(gpu), new(c.pool.gk), new(c.pool.gv), c.pool.gk, c.pool.gv, c.joined.to(gpu),
                            block_len=bs, S_ctx=c.joined.shape[1] * bs,
                            pos_ids=(at + P).float().view(B, 1).to(gpu), sink=sink, softmax_scale=c.scale)
    for b in range(B):
        o, bound = c.exact(b)
        check(got[b], o, bound, f"prefix, row {b}")
        check(dec[b], o, bound, f"decode, row {b}")
