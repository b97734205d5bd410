"""Cross attention and shared-prefix attention on the GPU against float64, with
elementwise bounds; masks, ragged and empty lengths, caches, strides, graphs."""
import math
import random

import pytest
import torch

from span_ref import attend, check, pool_rows, quantise
from vllm_neuron_amd.functional import (
    cross_attention,
    quant_kv_read,
    quant_kv_write,
    shared_prefix_attention,
)

pytestmark = pytest.mark.gpu
I8, FP8, BF = torch.int8, torch.float8_e4m3fn, torch.bfloat16
CACHES = ["bf16", "fp8", "fp8_token", "int8"]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g).to(BF)


class Pool:
    """K/V cache of a kind; block 0 and every slot the tests do not own hold
    what a reused pool may hold: NaN and infinities."""

    def __init__(self, kind, nb, hkv, bs, d, seed, dev):
        g = _gen(seed)
        k, v = _randn(g, nb, hkv, bs, d), _randn(g, nb, hkv, bs, d)
        k[..., 3::16] *= 4
        self.kind, self.dev, self.kw, self.factors = kind, dev, {}, (None, None)
        self.scales = (None, None)
        if kind == "bf16":
            self.k, self.v = k, v
        elif kind == "fp8":
            self.k, self.v = (x.float().mul(8).clamp(-448, 448).to(FP8) for x in (k, v))
            self.factors = tuple(torch.rand(hkv, generator=g) * 0.2 + 0.05 for _ in "kv")
            self.kw = dict(k_dequant_scale=self.factors[0].to(dev),
                           v_dequant_scale=self.factors[1].to(dev))
        else:
            code = I8 if kind == "int8" else FP8
            (kc, ks), (vc, vs) = quantise(k, code), quantise(v, code)
            self.k, self.v = kc.float().to(code), vc.float().to(code)
            self.scales = (ks.float(), vs.float())
        self.nb, self.bs = nb, bs

    def poison(self, owned):
        """NaN / Inf in every (block, offset) outside ``owned``."""
        free = torch.ones(self.nb * self.bs, dtype=torch.bool)
        free[[b * self.bs + o for b, o in owned]] = False
        at = free.nonzero()[:, 0]
        b, o = at // self.bs, at % self.bs
        for x, sign in ((self.k, 1), (self.v, -1)):
            if x.dtype == BF:
                x[b, :, o] = math.nan
                x[b[::2], :, o[::2]] = sign * math.inf
            elif x.dtype == FP8:
                x.view(torch.uint8)[b, :, o] = 0x7F
        for s in self.scales:
            if s is not None:
                s[b, :, o] = math.nan

    def up(self):
        self.gk, self.gv = self.k.to(self.dev), self.v.to(self.dev)
        if self.scales[0] is not None:
            self.kw = dict(k_scales=self.scales[0].to(self.dev), v_scales=self.scales[1].to(self.dev))
        return self

    def rows(self, blocks, n):
        return (pool_rows(self.k, self.scales[0], blocks, n, self.factors[0]),
                pool_rows(self.v, self.scales[1], blocks, n, self.factors[1]))


def _tables(lens, bs, first, seed, spare=1):
    per = [(n + bs - 1) // bs for n in lens]
    perm = (torch.randperm(max(1, sum(per)), generator=_gen(seed)) + first).to(torch.int32)
    t = torch.full((len(lens), max(per + [0]) + spare), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, first + sum(per)


def _owned(tables, lens, bs):
    return [(int(t[k // bs]), k % bs) for t, n in zip(tables, lens) for k in range(n)]


# ---------------------------------------------------------------------------
# cross attention
# ---------------------------------------------------------------------------
def _cross(gpu, kind, hq, hkv, d, bs, lens, new, seed=0, scale=None):
    t, nb = _tables(lens, bs, 1, seed)
    pool = Pool(kind, nb + 1, hkv, bs, d, seed + 1, gpu)
    pool.poison(_owned(t, lens, bs))
    pool.up()
    T = len(lens) if new is None else sum(new)
    q = _randn(_gen(seed + 2), T + 2, hq, d)       # two rows of no sequence
    out = torch.full((T + 2, hq, d), 7.0, dtype=BF, device=gpu)
    kw = dict(pool.kw)
    if new is not None:
        cu = [sum(new[:i]) for i in range(len(new) + 1)]
        kw.update(cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device=gpu),
                  max_seqlen_q=max(new))
    got = cross_attention(q.to(gpu), pool.gk, pool.gv,
                          torch.tensor(lens, dtype=torch.int32, device=gpu),
                          block_table=t.to(gpu), out=out, softmax_scale=scale, **kw)
    assert got is out and (out[T:] == 7.0).all()
    at = 0
    for i, n in enumerate(lens):
        m = 1 if new is None else new[i]
        k, v = pool.rows(t[i], n)
        o, bound = attend(q[at:at + m], k, v, d ** -0.5 if scale is None else scale)
        check(out[at:at + m], o, bound, f"sequence {i}: {m} x {n}")
        at += m
    return out


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (8, 2, 128), (16, 2, 64), (10, 2, 80)])
def test_cross_single_token(gpu, kind, hq, hkv, d):
    _cross(gpu, kind, hq, hkv, d, 16, [1, 0, 63, 64, 65, 17, 500, 129], None)


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("hq,hkv,d,bs", [(4, 4, 64, 16), (8, 2, 128, 32), (6, 2, 80, 48), (3, 1, 16, 64),
                                         (7, 7, 112, 16)])
def test_cross_ragged(gpu, kind, hq, hkv, d, bs):
    _cross(gpu, kind, hq, hkv, d, bs, [70, 0, 1, 300, 128, 16], [1, 3, 130, 33, 0, 64])


@pytest.mark.parametrize("d", [8, 24, 72, 104])
def test_cross_odd_dims(gpu, d):
    _cross(gpu, "bf16", 6, 3, d, 32, [33, 200, 1], [40, 5, 9])


def test_cross_wide_groups(gpu):
    _cross(gpu, "bf16", 71, 1, 64, 16, [100, 33], [3, 2])
    _cross(gpu, "int8", 64, 2, 128, 16, [700], None)


def test_cross_scales(gpu):
    """Zero, negative and large softmax scales."""
    for s in (0.0, -0.2, 1.0):
        _cross(gpu, "bf16", 4, 2, 64, 16, [90, 5], [9, 3], scale=s)


def test_cross_long(gpu):
    """One row over a long context: many pieces are joined."""
    _cross(gpu, "bf16", 8, 8, 64, 64, [50001], None)
    _cross(gpu, "int8", 8, 2, 128, 64, [8191, 40], [5, 2])


def test_cross_many_sequences(gpu):
    r = random.Random(5)
    lens = [r.randint(0, 40) for _ in range(700)]
    _cross(gpu, "bf16", 2, 1, 64, 16, lens, None)


@pytest.mark.parametrize("L", [1, 50, 129])
def test_cross_dense(gpu, L):
    """Encoder states as the projection leaves them: [B, L, Hkv, d] seen head
    first, K and V ranges of one tensor, any L."""
    B, hq, hkv, d = 3, 8, 4, 64
    g = _gen(3)
    kv = _randn(g, B, L, 2 * hkv, d)
    lens = [L, max(0, L - 7), 0]
    for i, n in enumerate(lens):
        kv[i, n:] = math.nan
    q = _randn(g, B * 2, hq, d)
    kvd = kv.to(gpu)
    out = cross_attention(q.to(gpu), kvd[:, :, :hkv].transpose(1, 2), kvd[:, :, hkv:].transpose(1, 2),
                          torch.tensor(lens, dtype=torch.int32, device=gpu),
                          cu_seqlens_q=torch.tensor([0, 1, 5, 6], dtype=torch.int32, device=gpu),
                          max_seqlen_q=4)
    for i, (a, b) in enumerate([(0, 1), (1, 5), (5, 6)]):
        o, bound = attend(q[a:b], kv[i, :lens[i], :hkv].double(), kv[i, :lens[i], hkv:].double(), d ** -0.5)
        check(out[a:b], o, bound, f"sequence {i}")


def test_cross_visible_nan(gpu):
    """A NaN in a key that is seen reaches its sequence's rows of that kv head
    and no other; lengths past the table are clamped to it."""
    B, hq, hkv, d, L = 3, 4, 2, 64, 70
    g = _gen(8)
    k, v = _randn(g, B, hkv, L, d), _randn(g, B, hkv, L, d)
    q = _randn(g, B, hq, d)
    bad = v.clone()
    bad[1, 0, 69] = math.nan
    lens = torch.tensor([200, 200, -4], dtype=torch.int32, device=gpu)
    out = cross_attention(q.to(gpu), k.to(gpu), bad.to(gpu), lens).cpu()
    assert torch.isnan(out[1, :2]).all()
    for i, heads in ((0, slice(0, 4)), (1, slice(2, 4))):
        o, bound = attend(q[i:i + 1], k[i].transpose(0, 1).double(), v[i].transpose(0, 1).double(), d ** -0.5)
        check(out[i:i + 1, heads], o[:, heads], bound[:, heads])
    assert (out[2] == 0).all()


def test_cross_strides(gpu):
    """q as a range of a projection, out as a range of a wider tensor, the
    table as a strided view."""
    B, hq, hkv, d, bs = 4, 4, 2, 64, 16
    lens = [30, 100, 1, 64]
    t, nb = _tables(lens, bs, 0, 1)
    pool = Pool("bf16", nb, hkv, bs, d, 2, gpu).up()
    proj = _randn(_gen(4), B, (hq + 2) * d).to(gpu)
    q = proj[:, d:(hq + 1) * d].view(B, hq, d)
    wide = torch.zeros(B, hq, 2 * d, dtype=BF, device=gpu)
    tt = torch.stack([t, torch.full_like(t, 9999)], -1).to(gpu)[..., 0]
    cross_attention(q, pool.gk, pool.gv, torch.tensor(lens, dtype=torch.int32, device=gpu), block_table=tt,
                    out=wide[..., :d])
    assert (wide[..., d:] == 0).all()
    for i, n in enumerate(lens):
        o, bound = attend(q[i:i + 1].cpu(), *pool.rows(t[i], n), d ** -0.5)
        check(wide[i:i + 1, :, :d], o, bound)


def test_cross_bad_table_stays_in_bounds(gpu):
    """Entries outside the pool read its first or last block (never outside)."""
    hkv, bs, d = 2, 16, 64
    pool = Pool("bf16", 3, hkv, bs, d, 2, gpu).up()
    q = _randn(_gen(4), 2, 4, d)
    t = torch.tensor([[-1, 1 << 30], [2, -7]], dtype=torch.int32)
    out = cross_attention(q.to(gpu), pool.gk, pool.gv, torch.tensor([32, 32], dtype=torch.int32, device=gpu),
                          block_table=t.to(gpu))
    for i, row in enumerate([[0, 2], [2, 0]]):
        o, bound = attend(q[i:i + 1], *pool.rows(row, 32), d ** -0.5)
        check(out[i:i + 1], o, bound)


def test_cross_large_offsets(gpu):
    """Blocks past 2^31 elements of the pool."""
    hkv, bs, d, nb = 8, 128, 128, 17000          # 2.2e9 elements per cache
    k = torch.empty(nb, hkv, bs, d, dtype=BF, device=gpu)
    v = torch.empty(nb, hkv, bs, d, dtype=BF, device=gpu)
    blocks = [nb - 1, 3, nb - 2]
    g = _gen(6)
    small = Pool("bf16", 3, hkv, bs, d, 5, gpu)
    for i, b in enumerate(blocks):
        k[b], v[b] = small.k[i].to(gpu), small.v[i].to(gpu)
    q = _randn(g, 1, 16, d)
    out = cross_attention(q.to(gpu), k, v, torch.tensor([350], dtype=torch.int32, device=gpu),
                          block_table=torch.tensor([blocks], dtype=torch.int32, device=gpu))
    o, bound = attend(q, *small.rows([0, 1, 2], 350), d ** -0.5)
    check(out, o, bound)


def test_cross_deterministic(gpu):
    a = _cross(gpu, "fp8_token", 8, 2, 128, 16, [333, 1000, 5], [17, 60, 1])
    b = _cross(gpu, "fp8_token", 8, 2, 128, 16, [333, 1000, 5], [17, 60, 1])
    assert torch.equal(a, b)


def test_cross_graph(gpu):
    """A captured call follows its lengths; replays equal eager calls."""
    B, hq, hkv, d, L = 6, 8, 4, 64, 400
    g = _gen(1)
    q, k, v = _randn(g, B, hq, d).to(gpu), _randn(g, B, hkv, L, d).to(gpu), _randn(g, B, hkv, L, d).to(gpu)
    lens = torch.tensor([400, 3, 77, 0, 256, 65], dtype=torch.int32, device=gpu)
    cross_attention(q, k, v, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cross_attention(q, k, v, lens)
    for s in range(4):
        q.copy_(_randn(_gen(s + 9), B, hq, d))
        lens.copy_(torch.randint(0, L + 1, (B,), generator=_gen(s), dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cross_attention(q, k, v, lens))


def test_cross_side_stream_and_compile(gpu):
    B, hq, hkv, d, L = 4, 8, 4, 64, 100
    g = _gen(1)
    q, k, v = _randn(g, B, hq, d).to(gpu), _randn(g, B, hkv, L, d).to(gpu), _randn(g, B, hkv, L, d).to(gpu)
    lens = torch.tensor([100, 3, 77, 0], dtype=torch.int32, device=gpu)
    want = cross_attention(q, k, v, lens)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = cross_attention(q, k, v, lens)
    torch.cuda.synchronize()
    assert torch.equal(want, got)
    step = torch.compile(lambda q, l: cross_attention(q, k, v, l) * 2, fullgraph=True, backend="aot_eager")
    assert torch.equal(step(q, lens), want * 2)


# ---------------------------------------------------------------------------
# shared prefix
# ---------------------------------------------------------------------------
def _prefix(gpu, kind, hq, hkv, d, bs, P, lens, S=1, sink=False, seed=0, spare=1):
    tp, nb = _tables([P], bs, 1, seed, spare)
    t, nb = _tables(lens, bs, nb, seed + 1, spare)
    pool = Pool(kind, nb + 1, hkv, bs, d, seed + 2, gpu)
    pool.poison(_owned(tp, [P], bs) + _owned(t, lens, bs))
    pool.up()
    B = len(lens)
    q = _randn(_gen(seed + 3), B, S, hq, d)
    sk = torch.randn(hq, generator=_gen(seed + 4)) if sink else None
    out = shared_prefix_attention(
        q.to(gpu), pool.gk, pool.gv, tp[0].to(gpu), torch.tensor([P], dtype=torch.int32, device=gpu),
        t.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu),
        sink=None if sk is None else sk.to(gpu), **pool.kw)
    kp, vp = pool.rows(tp[0], P)
    for b, n in enumerate(lens):
        k, v = pool.rows(t[b], n)
        for s in range(S):
            e = max(0, n - S + 1 + s)
            o, bound = attend(q[b, s:s + 1], torch.cat([kp, k[:e]]), torch.cat([vp, v[:e]]), d ** -0.5, sk)
            check(out[b, s:s + 1], o, bound, f"row {b}, token {s}: {P} + {e}")
    return out


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("hq,hkv,d,bs", [(8, 2, 128, 32), (16, 2, 64, 16), (10, 2, 80, 48)])
@pytest.mark.parametrize("S,sink", [(1, False), (1, True), (3, False)])
def test_prefix(gpu, kind, hq, hkv, d, bs, S, sink):
    _prefix(gpu, kind, hq, hkv, d, bs, 333, [5, 3, 64, 65, 130, 100], S, sink)


@pytest.mark.parametrize("P", [0, 1, 63, 64, 65, 2000])
@pytest.mark.parametrize("S", [1, 2])
def test_prefix_lengths(gpu, P, S):
    _prefix(gpu, "bf16", 8, 2, 64, 16, P, [2, 1, 0, 63, 64, 66], S, sink=P == 0)


def test_prefix_short_own(gpu):
    """More new tokens than own keys: the first tokens see the prefix alone."""
    _prefix(gpu, "int8", 8, 2, 128, 16, 100, [0, 1, 4, 7, 8, 9], S=8)
    _prefix(gpu, "bf16", 4, 2, 64, 16, 0, [0, 3, 5], S=5)


def test_prefix_one_row_and_many(gpu):
    _prefix(gpu, "bf16", 4, 4, 128, 16, 700, [9])
    _prefix(gpu, "fp8_token", 8, 1, 64, 16, 150, [1 + i % 37 for i in range(300)])


def test_prefix_large_batch_of_tokens(gpu):
    """More than one row tile per kv head, ragged at its end."""
    _prefix(gpu, "bf16", 8, 1, 64, 16, 200, [70, 16, 33, 40, 17], S=16)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_prefix_nan_in_later_tokens(gpu, kind):
    """A NaN in a new token's key or value stays with the rows that see it."""
    hq, hkv, d, bs, P, S = 4, 2, 64, 16, 40, 4
    lens = [20, 9]
    tp, nb = _tables([P], bs, 1, 0)
    t, nb = _tables(lens, bs, nb, 1)
    pool = Pool(kind, nb, hkv, bs, d, 2, gpu).up()
    q = _randn(_gen(3), 2, S, hq, d)
    call = lambda: shared_prefix_attention(
        q.to(gpu), pool.gk, pool.gv, tp[0].to(gpu), torch.tensor([P], dtype=torch.int32, device=gpu), t.to(gpu),
        torch.tensor(lens, dtype=torch.int32, device=gpu), **pool.kw)
    want = call()
    at = int(t[0, 18 // bs]), 18 % bs       # token s = 2 of row 0
    if kind == "bf16":
        pool.gv[at[0], :, at[1]] = math.nan
        pool.gk[at[0], :, at[1]] = math.inf
    else:
        pool.kw["v_scales"][at[0], :, at[1]] = math.nan
    got = call()
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, :2], want[0, :2])
    assert torch.isnan(got[0, 2:]).all()


def test_prefix_padded_rows(gpu):
    """Padding rows (length 0, table -1) give the prefix's attention and do
    not disturb the others."""
    a = _prefix(gpu, "bf16", 8, 2, 64, 16, 90, [30, 0, 17, 0, 0], 1)
    b = _prefix(gpu, "bf16", 8, 2, 64, 16, 90, [30, 0, 17], 1)
    assert not torch.isnan(a).any() and b.shape[0] == 3


def test_prefix_graph(gpu):
    hq, hkv, d, bs, B = 8, 2, 64, 16, 5
    tp, nb = _tables([512], bs, 1, 0)
    t, nb = _tables([96] * B, bs, nb, 1)
    pool = Pool("bf16", nb, hkv, bs, d, 2, gpu).up()
    q = _randn(_gen(3), B, 1, hq, d).to(gpu)
    P = torch.tensor([512], dtype=torch.int32, device=gpu)
    lens = torch.tensor([96, 1, 5, 64, 65], dtype=torch.int32, device=gpu)
    tp, t = tp[0].to(gpu), t.to(gpu)
    call = lambda: shared_prefix_attention(q, pool.gk, pool.gv, tp, P, t, lens)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for s in range(4):
        q.copy_(_randn(_gen(s + 9), B, 1, hq, d))
        lens.copy_(torch.randint(0, 97, (B,), generator=_gen(s), dtype=torch.int32))
        P.fill_([512, 0, 77, 300][s])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_prefix_random_shapes(gpu):
    r = random.Random(11)
    for i in range(25):
        hkv = r.choice([1, 2, 3, 8])
        G = r.choice([1, 2, 5, 8])
        kind = r.choice(CACHES)
        d = r.choice([16, 48, 64, 80, 128])
        S = r.choice([1, 1, 2, 4])
        B = r.randint(1, 20)
        _prefix(gpu, kind, hkv * G, hkv, d, r.choice([16, 32, 64, 80]), r.choice([0, 5, r.randint(1, 900)]),
                [r.randint(0, r.choice([3, 70, 300])) for _ in range(B)], S, r.random() < 0.3, seed=i * 10)


def test_cross_random_shapes(gpu):
    r = random.Random(12)
    for i in range(25):
        hkv = r.choice([1, 2, 3, 8])
        G = r.choice([1, 2, 5, 8])
        B = r.randint(1, 9)
        new = None if r.random() < 0.4 else [r.randint(0, r.choice([3, 40, 200])) for _ in range(B)]
        if new is not None and not sum(new):
            new[0] = 1
        _cross(gpu, r.choice(CACHES), hkv * G, hkv, r.choice([16, 48, 64, 80, 128]), r.choice([16, 32, 64, 80]),
               [r.randint(0, r.choice([3, 70, 900])) for _ in range(B)], new, seed=i * 10)


def test_prefix_many_new_tokens(gpu):
    """Up to 64 new tokens a row: the last 63 keys are seen by some rows only."""
    _prefix(gpu, "bf16", 2, 1, 64, 16, 50, [64, 100, 10, 200], S=64)
    _prefix(gpu, "int8", 4, 2, 128, 16, 0, [40, 33], S=33)


def test_lengths_of_any_int32(gpu):
    """The ends of int32 as lengths: nothing, or all that the tables hold."""
    hq, hkv, d, bs = 4, 2, 64, 16
    pool = Pool("bf16", 12, hkv, bs, d, 2, gpu).up()
    lo, hi = -2 ** 31, 2 ** 31 - 1
    q = _randn(_gen(4), 2, 3, hq, d)
    t = torch.tensor([[1, 2], [3, 4]], dtype=torch.int32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    out = shared_prefix_attention(q.to(gpu), pool.gk, pool.gv, i32(5, 6, 7), i32(hi), t.to(gpu), i32(lo, hi))
    kp, vp = pool.rows([5, 6, 7], 48)
    k, v = pool.rows([3, 4], 32)
    for s in range(3):
        o, bound = attend(q[0, s:s + 1], kp, vp, d ** -0.5)
        check(out[0, s:s + 1], o, bound)
        o, bound = attend(q[1, s:s + 1], torch.cat([kp, k]), torch.cat([vp, v]), d ** -0.5)
        check(out[1, s:s + 1], o, bound)
    out = shared_prefix_attention(q.to(gpu), pool.gk, pool.gv, i32(5, 6, 7), i32(lo), t.to(gpu), i32(lo, 2))
    assert (out[0] == 0).all() and (out[1, 0] == 0).all()
    out = cross_attention(q[:, 0].to(gpu), pool.gk, pool.gv, i32(lo, hi), block_table=t.to(gpu))
    o, bound = attend(q[1:2, 0], k, v, d ** -0.5)
    assert (out[0] == 0).all()
    check(out[1:], o, bound)


def test_axes_of_one_entry_have_any_stride(gpu):
    """Strides that no address uses are not asked to be aligned."""
    hkv, bs, d, n = 1, 16, 64, 40
    big = _randn(_gen(3), 8, 3 * d + 1).to(gpu)
    q = big[2:3, :2 * d].as_strided((1, 2, d), (3 * d + 1, d, 1), 0)  # one token, odd row stride
    pool = Pool("bf16", 4, hkv, bs, d, 2, gpu).up()
    k, v = (x.as_strided(x.shape, (x.stride(0), 3, d, 1)) for x in (pool.gk, pool.gv))
    t = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    out = cross_attention(q, k, v, lens, block_table=t.to(gpu))
    o, bound = attend(q.cpu(), *pool.rows(t[0], n), d ** -0.5)
    check(out, o, bound)


def test_query_tokens_past_the_maximum(gpu):
    """max_seqlen_q bounds what is computed; the rest of out stays."""
    hq, hkv, d, L = 4, 2, 64, 33
    g = _gen(5)
    q, k, v = _randn(g, 10, hq, d), _randn(g, 2, hkv, L, d), _randn(g, 2, hkv, L, d)
    out = torch.full((10, hq, d), 5.0, dtype=BF, device=gpu)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    cross_attention(q.to(gpu), k.to(gpu), v.to(gpu), i32(L, L), cu_seqlens_q=i32(0, 6, 8), max_seqlen_q=4, out=out)
    for i, (a, b) in enumerate([(0, 4), (6, 8)]):
        o, bound = attend(q[a:b], k[i].transpose(0, 1).double(), v[i].transpose(0, 1).double(), d ** -0.5)
        check(out[a:b], o, bound)
    assert (out[4:6] == 5.0).all() and (out[8:] == 5.0).all()


@pytest.mark.parametrize("new_max", [2, 64])
def test_decreasing_first_tokens_compute_nothing(gpu, new_max):
    """Sequences would share tokens: the rows stay as they were, captured pieces
    of an earlier call in the workspace included; a rising list is computed."""
    B, hq, hkv, d, L = 6, 8, 2, 64, 900
    g = _gen(5)
    q = _randn(g, B * new_max, hq, d).to(gpu)
    k, v = (_randn(g, B, hkv, L, d).to(gpu) for _ in range(2))
    lens = torch.tensor([L, 0, 17, L, 300, L], dtype=torch.int32, device=gpu)
    rising = torch.arange(B + 1, dtype=torch.int32, device=gpu) * new_max
    want = cross_attention(q, k, v, lens, cu_seqlens_q=rising, max_seqlen_q=new_max)
    ws = torch.empty(1 << 28, dtype=torch.uint8, device=gpu)
    got = cross_attention(q, k, v, lens, cu_seqlens_q=rising, max_seqlen_q=new_max, workspace=ws)
    assert torch.equal(got, want)
    falling = rising.clone()
    falling[3] = 0
    out = torch.full_like(q, 7.0)
    cross_attention(q, k, v, lens, cu_seqlens_q=falling, max_seqlen_q=new_max, out=out,
                    workspace=ws)
    assert (out == 7.0).all()


def test_two_streams_and_a_given_workspace(gpu):
    """Calls at once on two streams; a given workspace is used and gives the
    same bits, one too small is not."""
    hq, hkv, d, bs, B = 8, 2, 64, 16, 6
    tp, nb = _tables([300], bs, 1, 0)
    t, nb = _tables([96] * B, bs, nb, 1)
    pool = Pool("bf16", nb, hkv, bs, d, 2, gpu).up()
    q = _randn(_gen(3), B, 1, hq, d).to(gpu)
    args = (pool.gk, pool.gv, tp[0].to(gpu), torch.tensor([300], dtype=torch.int32, device=gpu), t.to(gpu),
            torch.tensor([96, 1, 5, 64, 65, 33], dtype=torch.int32, device=gpu))
    want = shared_prefix_attention(q, *args)
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=gpu)
    assert torch.equal(want, shared_prefix_attention(q, *args, workspace=ws))
    assert (ws != 255).any()
    assert torch.equal(want, shared_prefix_attention(q, *args, workspace=ws[:100]))
    with pytest.raises(ValueError):
        shared_prefix_attention(q, *args, workspace=ws[::2])
    with pytest.raises(ValueError):
        shared_prefix_attention(q, *args, workspace=ws[1:])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(shared_prefix_attention(q, *args))
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in outs)


def test_prefix_compiles(gpu):
    hq, hkv, d, bs, B = 8, 2, 64, 16, 3
    tp, nb = _tables([50], bs, 1, 0)
    t, nb = _tables([20] * B, bs, nb, 1)
    pool = Pool("int8", nb, hkv, bs, d, 2, gpu).up()
    q = _randn(_gen(3), B, 1, hq, d).to(gpu)
    P = torch.tensor([50], dtype=torch.int32, device=gpu)
    lens = torch.tensor([20, 3, 7], dtype=torch.int32, device=gpu)
    tp, t = tp[0].to(gpu), t.to(gpu)
    slots = torch.tensor([7, 8, 9], device=gpu)
    rows = _randn(_gen(4), B, hkv, d).to(gpu)
    kv = (pool.gk, pool.gv, pool.kw["k_scales"], pool.kw["v_scales"])

    def step(q, rows):
        quant_kv_write(rows, rows, slots, *kv)
        return shared_prefix_attention(q, pool.gk, pool.gv, tp, P, t, lens, **pool.kw) + 1

    want = step(q, rows)
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, rows)
    assert torch.equal(want, got)


# ---------------------------------------------------------------------------
# the operators together, and against the framework's decode
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("code", [I8, FP8])
def test_run_of_the_operators(gpu, code):
    """A step as a serving loop runs it: an encoder's K/V and a prompt's are
    quantised into the cache, then two decode steps write their token and
    attend to the shared prefix with their own keys, and cross-attend to the
    encoder; every output against float64 over what the cache reads back."""
    hq, hkv, d, bs, B, P, E = 8, 2, 128, 16, 4, 70, 45
    g = _gen(21)
    nb = 60
    kc, vc = (torch.zeros(nb, hkv, bs, d, dtype=code, device=gpu) for _ in "kv")
    ks, vs = (torch.zeros(nb, hkv, bs, device=gpu) for _ in "kv")
    tp, n1 = _tables([P], bs, 0, 1)
    t, n2 = _tables([bs] * B, bs, n1, 2)
    te, _ = _tables([E] * B, bs, n2, 3)
    slot = lambda row, pos: (row[pos // bs].long() * bs + pos % bs)
    write = lambda rows, slots: quant_kv_write(rows[0].to(gpu), rows[1].to(gpu), slots.to(gpu), kc, vc, ks, vs)
    pos = torch.arange(P)
    write((_randn(g, P, hkv, d), _randn(g, P, hkv, d)), slot(tp[0], pos))
    for b in range(B):
        write((_randn(g, E, hkv, d), _randn(g, E, hkv, d)), slot(te[b], torch.arange(E)))
    read = lambda slots: tuple(x.cpu().double() for x in
                               quant_kv_read(kc, vc, ks, vs, slots.to(gpu), dtype=torch.float32))
    kw = dict(k_scales=ks, v_scales=vs)
    for step in range(2):
        write((_randn(g, B, hkv, d), _randn(g, B, hkv, d)), slot(t.t(), torch.tensor(step)))
        q = _randn(g, B, 1, hq, d)
        out = shared_prefix_attention(
            q.to(gpu), kc, vc, tp[0].to(gpu), torch.tensor([P], dtype=torch.int32, device=gpu), t.to(gpu),
            torch.full((B,), step + 1, dtype=torch.int32, device=gpu), **kw)
        kp, vp = read(slot(tp[0], pos))
        x = out[:, 0]
        cross = cross_attention(x, kc, vc, torch.full((B,), E, dtype=torch.int32, device=gpu),
                                block_table=te.to(gpu), **kw)
        for b in range(B):
            k, v = read(slot(t[b], torch.arange(step + 1)))
            o, bound = attend(q[b], torch.cat([kp, k]), torch.cat([vp, v]), d ** -0.5)
            check(out[b], o, bound, f"step {step}, row {b}")
            o, bound = attend(x[b:b + 1].cpu(), *read(slot(te[b], torch.arange(E))), d ** -0.5)
            check(cross[b:b + 1], o, bound, f"cross, step {step}, row {b}")


def test_prefix_equals_decode_over_joined_tables(gpu):
    """The decode path over [prefix | own] tables gives the same attention
    (its own error bound added: it rounds q after scaling it too)."""
    from vllm_neuron_amd.functional.attention.attention_decode import paged_decode_core

    hq, hkv, d, bs, P, B = 8, 2, 128, 32, 256, 4
    lens = [33, 1, 64, 100]
    tp, nb = _tables([P], bs, 1, 0, spare=0)
    t, nb = _tables(lens, bs, nb, 1, spare=0)
    pool = Pool("bf16", nb, hkv, bs, d, 2, gpu).up()
    q = _randn(_gen(3), B, 1, hq, d).to(gpu)
    out = shared_prefix_attention(q, pool.gk, pool.gv, tp[0].to(gpu),
                                  torch.tensor([P], dtype=torch.int32, device=gpu), t.to(gpu),
                                  torch.tensor(lens, dtype=torch.int32, device=gpu))
    joined = torch.cat([tp.expand(B, -1), t], 1)
    at = torch.tensor([n - 1 for n in lens])
    blk = t.gather(1, (at // bs).view(-1, 1)).view(-1).long()
    new = lambda c: c[blk.to(gpu), :, (at % bs).to(gpu)].view(B, 1, hkv, d)
    want = paged_decode_core(q, new(pool.gk), new(pool.gv), pool.gk, pool.gv, joined.to(gpu), block_len=bs,
                             S_ctx=joined.shape[1] * bs,
                             pos_ids=(at + P).float().view(B, 1).to(gpu), softmax_scale=d ** -0.5)
    for b, n in enumerate(lens):
        k, v = pool.rows(joined[b], P + n)
        o, bound = attend(q[b].cpu(), k, v, d ** -0.5)
        check(out[b], o, bound)
        # scores of at most 40 / 128^0.5 x 2^-8 off per rounded q: |ds| <= U sum|q k| scale
        ds = 2.0 ** -8 * (q[b].cpu().double().abs().amax() * k.abs().sum(-1).amax() * d ** -0.5)
        assert ((want[b].double().cpu() - o).abs() <= bound + 2 * ds * v.abs().amax()).all()


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals(gpu):
    hq, hkv, d, bs = 4, 2, 64, 16
    k = torch.zeros(4, hkv, bs, d, dtype=BF, device=gpu)
    q = torch.zeros(2, hq, d, dtype=BF, device=gpu)
    lens = torch.zeros(2, dtype=torch.int32, device=gpu)
    t = torch.zeros(2, 2, dtype=torch.int32, device=gpu)
    sc = torch.zeros(4, hkv, bs, device=gpu)
    i8 = torch.zeros(4, hkv, bs, d, dtype=I8, device=gpu)
    f8 = i8.view(FP8)
    fac = torch.ones(hkv, device=gpu)
    for err, args, kw in [
        (RuntimeError, (q.cpu(), k, k, lens), {}),
        (NotImplementedError, (q.float(), k, k, lens), {}),
        (ValueError, (q[..., :32], k, k, lens), {}),
        (ValueError, (q[:, :3], k, k, lens), {}),
        (ValueError, (q[:1], k, k, lens), {}),
        (ValueError, (q, k, k[:, :1], lens), {}),
        (ValueError, (q, k, k, lens.long()), {}),
        (ValueError, (q, k, k, lens), dict(block_table=t.long())),
        (ValueError, (q, k, k, lens), dict(block_table=t[:1])),
        (ValueError, (q, k, k, lens), dict(k_scales=sc, v_scales=sc)),
        (ValueError, (q, i8, i8, lens), {}),
        (ValueError, (q, i8, i8, lens), dict(k_scales=sc)),
        (ValueError, (q, i8, i8, lens), dict(k_scales=sc[:2], v_scales=sc[:2])),
        (ValueError, (q, f8, f8, lens), dict(k_scales=sc, v_scales=sc, k_dequant_scale=fac, v_dequant_scale=fac)),
        (ValueError, (q, k, k, lens), dict(k_dequant_scale=fac, v_dequant_scale=fac)),
        (ValueError, (q, k, k, lens), dict(out=torch.zeros(2, hq, d, device=gpu))),
        (ValueError, (q, k, k, lens), dict(cu_seqlens_q=lens)),
        (NotImplementedError, (q, k.half(), k.half(), lens), {}),
    ]:
        with pytest.raises(err):
            cross_attention(*args, **kw)
    qq = q.view(2, 1, hq, d)
    P = torch.zeros(1, dtype=torch.int32, device=gpu)
    for err, args in [
        (ValueError, (q, k, k, t[0], P, t, lens)),
        (ValueError, (qq, k, k, t, P, t, lens)),
        (ValueError, (qq, k, k, t[0], P.long(), t, lens)),
        (ValueError, (qq, k, k, t[0], lens, t, lens)),
        (ValueError, (qq, k, k, t[0], P, t[:1], lens)),
        (ValueError, (qq, k, k, t[0], P, t, lens[:1])),
    ]:
        with pytest.raises(err):
            shared_prefix_attention(*args)
    with pytest.raises(ValueError):
        shared_prefix_attention(qq, k, k, t[0], P, t, lens, sink=torch.zeros(3, device=gpu))
    # nothing to compute
    assert cross_attention(q[:0], k, k, lens[:0]).shape == (0, hq, d)
    assert shared_prefix_attention(qq[:0], k, k, t[0], P, t[:0], lens[:0]).shape == (0, 1, hq, d)
