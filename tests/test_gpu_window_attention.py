"""Attention with a sliding window and visible first tokens on the GPU, against
the float64 formula: single tokens and prompts, every cache, windows and first
tokens at tile borders, freed blocks, empty rows, pieces, strides, graphs."""
import math

import pytest
import torch

from span_ref import check, quantise
from vllm_neuron_amd import _native as N
from vllm_neuron_amd.functional import window_attention
from window_ref import reference

pytestmark = pytest.mark.gpu
BF, FP8 = torch.bfloat16, torch.float8_e4m3fn


class Call:
    """A cache with tables in random order, blocks that no query sees freed
    (their entries -1) and, where asked, full of NaN; queries of each sequence."""

    def __init__(self, gpu, new, lens, Hq=4, Hkv=2, d=64, bs=16, window=64, first=4, cache="bf16", sink=False, seed=0,
                 poison=True, cap=None):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.window, self.first = new, lens, window, first
        nblk = max(1, cap or max((n + bs - 1) // bs for n in lens))
        table = torch.full((len(lens), nblk), -1, dtype=torch.int32)
        live = [[j for j in range((min(n, nblk * bs) + bs - 1) // bs)
                 if j * bs < first or (j + 1) * bs > n - m - window + 1] for m, n in zip(new, lens)]
        nb = 2 + sum(len(r) for r in live)
        ids, at = torch.randperm(nb - 2, generator=g).int() + 1, 0
        for i, r in enumerate(live):
            for j in r:
                table[i, j] = ids[at]
                at += 1
        shape = (nb, Hkv, bs, d)
        k = torch.randn(shape, generator=g)
        k[..., 3::16] *= 3.0
        v = torch.randn(shape, generator=g)
        self.ks = self.vs = self.kd = self.vd = None
        if cache == "bf16":
            K, V = k.to(BF), v.to(BF)
        elif cache == "fp8s":
            self.kd, self.vd = torch.rand(Hkv, generator=g) + 0.5, torch.rand(Hkv, generator=g) + 0.5
            K, V = (k / self.kd.view(1, -1, 1, 1)).to(FP8), (v / self.vd.view(1, -1, 1, 1)).to(FP8)
        else:
            code = torch.int8 if cache == "int8" else FP8
            k = k * (torch.rand(shape[:3], generator=g)[..., None] + 0.5)
            v = v * (torch.rand(shape[:3], generator=g)[..., None] * 3 + 0.2)
            (kc, ks), (vc, vs) = quantise(k.to(BF), code), quantise(v.to(BF), code)
            K, V, self.ks, self.vs = kc.float().to(code), vc.float().to(code), ks.float(), vs.float()
        if poison:
            # everything that no query sees: the block entries of -1 read, and
            # the keys behind the last and before the window
            seen = torch.zeros(nb, bs, dtype=torch.bool)
            for i, (m, n) in enumerate(zip(new, lens)):
                n = min(n, nblk * bs)
                for t in range(n):
                    if (t < first or t > n - m - window) and table[i, t // bs] >= 0 and m > 0:
                        seen[table[i, t // bs], t % bs] = True
            dead = (~seen)[:, None, :].expand(nb, Hkv, bs)
            if cache == "bf16":
                K[dead], V[dead] = math.nan, math.nan
            elif cache in ("fp8", "fp8s"):
                for x in (K, V):
                    b = x.view(torch.uint8)
                    b[dead] = 0x7f
            if self.ks is not None:
                self.ks[dead], self.vs[dead] = math.nan, math.inf
        self.K, self.V = K.to(gpu), V.to(gpu)
        self.q = torch.randn(sum(new), Hq, d, generator=g).to(BF).to(gpu)
        self.table = table.to(gpu)
        self.cu = [sum(new[:i]) for i in range(len(new) + 1)]
        self.sink = torch.randn(Hq, generator=g) if sink else None
        self.scale = d ** -0.5
        self.gpu = gpu

    def run(self, **over):
        dev = lambda t: None if t is None else t.to(self.gpu)
        kw = dict(window=self.window, first_tokens=self.first, max_seqlen_q=max(1, max(self.new)),
                  cu_seqlens_q=torch.tensor(self.cu, dtype=torch.int32, device=self.gpu), sink=dev(self.sink),
                  k_scales=dev(self.ks), v_scales=dev(self.vs), k_dequant_scale=dev(self.kd), v_dequant_scale=dev(self.vd))
        kw.update(over)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.gpu)
        return window_attention(self.q, self.K, self.V, self.table, lens, **kw)

    def check(self, got=None, what="", **over):
        ref, bound = reference(self.q, self.K, self.V, self.table, self.lens, self.cu, self.scale, self.window,
                               self.first, self.sink, self.ks, self.vs, self.kd, self.vd)
        got = self.run(**over) if got is None else got
        check(got, ref, bound, what)
        return got


CACHES = ["bf16", "fp8s", "fp8", "int8"]


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("Hq,Hkv,d,bs", [(4, 2, 64, 16), (8, 1, 128, 32), (64, 8, 64, 32), (6, 6, 96, 16), (32, 1, 16, 64),
                                         (3, 1, 80, 16), (40, 2, 128, 48)])
@pytest.mark.parametrize("window,first", [(1, 0), (16, 4), (64, 64), (100, 1), (4096, 4), (33, 100)])
def test_single_tokens(gpu, cache, Hq, Hkv, d, bs, window, first):
    lens = [1, 2, 16, 31, 32, 33, 64, 65, 130, 400, 700]
    Call(gpu, [1] * len(lens), lens, Hq, Hkv, d, bs, window, first, cache, sink=Hq == 64).check()


@pytest.mark.parametrize("cache", ["bf16", "int8"])
@pytest.mark.parametrize("new", [2, 3, 5, 8, 16, 31])
@pytest.mark.parametrize("G", [1, 2, 4])
def test_a_few_tokens_each(gpu, cache, new, G):
    lens = [new, new + 1, 40 + new, 64, 65, 300]
    Call(gpu, [new] * len(lens), lens, 2 * G, 2, 64, 16, 24, 6, cache).check()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("Hq,Hkv,d,bs", [(4, 2, 64, 16), (8, 2, 128, 32), (16, 2, 64, 32), (3, 3, 80, 16), (5, 1, 32, 64),
                                         (12, 2, 112, 16)])
@pytest.mark.parametrize("window,first", [(1, 0), (17, 3), (64, 64), (128, 4), (1000, 0), (200, 130)])
def test_prompts(gpu, cache, Hq, Hkv, d, bs, window, first):
    new = [1, 63, 64, 65, 130, 300, 40]
    ctx = [0, 0, 5, 200, 64, 77, 500]
    Call(gpu, new, [a + b for a, b in zip(new, ctx)], Hq, Hkv, d, bs, window, first, cache, sink=Hq == 16).check()


@pytest.mark.parametrize("first", [0, 1, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 250])
@pytest.mark.parametrize("window", [31, 32, 33, 63, 64, 65])
def test_first_tokens_meet_the_window_at_every_border(gpu, window, first):
    Call(gpu, [1, 1, 1, 1, 1, 1], [96, 97, 127, 128, 129, 190], 4, 1, 64, 16, window, first).check()
    Call(gpu, [190, 70], [190, 200], 4, 1, 64, 16, window, first).check()


@pytest.mark.parametrize("cache", ["bf16", "int8"])
@pytest.mark.parametrize("new", [1, 4, 70])
def test_rows_without_keys(gpu, cache, new):
    """Sequences of no tokens, shorter than their queries, or emptier than
    nothing: rows that see no key are zeros, sink or not."""
    for sink in (False, True):
        c = Call(gpu, [new] * 5, [0, -3, max(1, new // 2), new, new + 40], 4, 2, 64, 16, 20, 3, cache, sink=sink)
        got = c.check()
        assert (got[:new * 2] == 0).all()


@pytest.mark.parametrize("batch,Hkv,new,lens,window", [(1, 1, 1, 9000, 8192), (2, 2, 1, 5000, 4096), (1, 1, 2, 3001, 2500),
                                                       (1, 1, 100, 4000, 3500), (2, 1, 200, 2600, 2200),
                                                       (3, 1, 1, 700, 100000)])
@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_keys_cut_into_pieces(gpu, cache, batch, Hkv, new, lens, window):
    """Few rows over many keys: the pieces' results are joined."""
    c = Call(gpu, [new] * batch, [lens - 7 * i for i in range(batch)], 4 * Hkv, Hkv, 128, 32, window, 4, cache, sink=True)
    c.check()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("Hq,Hkv,d", [(4, 1, 64), (20, 1, 128), (2, 1, 96)])
def test_more_sequences_than_compute_units(gpu, cache, Hq, Hkv, d):
    lens = [1 + 37 * i % 310 for i in range(300)]
    Call(gpu, [1] * len(lens), lens, Hq, Hkv, d, 16, 170, 5, cache).check()


@pytest.mark.parametrize("cache", ["bf16", "int8", "fp8s"])
@pytest.mark.parametrize("Hq,d,window", [(4, 64, 500), (4, 64, 1200), (4, 64, 1290), (24, 64, 2500), (8, 128, 560),
                                         (8, 128, 660), (30, 128, 1500)])
def test_long_windows_of_one_token(gpu, cache, Hq, d, window):
    """Keys that one workgroup takes whole and keys that are cut."""
    Call(gpu, [1, 1], [window + 300, window - 100], Hq, 1, d, 32, window, 4, cache, sink=True).check()


def test_many_prompts_without_a_bound(gpu):
    """max_seqlen_q is all tokens where it is not given: most workgroups have no
    rows."""
    new = [1 + 7 * i % 41 for i in range(300)]
    c = Call(gpu, new, [n + 11 * i % 50 for i, n in enumerate(new)], 64, 8, 64, 16, 20, 3)
    c.check(max_seqlen_q=None)


def test_token_per_sequence_without_a_list(gpu):
    c = Call(gpu, [1] * 6, [1, 5, 64, 80, 200, 0], 8, 2, 64, 16, 48, 2)
    a = c.run()
    b = c.run(cu_seqlens_q=None, max_seqlen_q=None)
    assert torch.equal(a, b)
    c.check(b)


def test_lengths_past_the_table_and_wide_windows(gpu):
    c = Call(gpu, [3, 1], [500, 64], 4, 2, 64, 16, 1 << 30, 1 << 30, cap=4)
    c.check()


def test_longest_allowed_and_rows_of_no_sequence(gpu):
    """Tokens past max_seqlen_q, before the first and behind the last sequence:
    zeros in a new output, as they were in a given one."""
    for new, most in (([5, 90, 3], 64), ([2, 3, 1], 2)):
        c = Call(gpu, new, [n + 20 for n in new], 4, 2, 64, 16, 30, 2)
        T = sum(new) + 9
        q = torch.randn(T, 4, 64, device=gpu).to(BF)
        q[4:4 + sum(new)] = c.q
        cu = torch.tensor([4 + x for x in c.cu], dtype=torch.int32, device=gpu)
        dev = dict(window=30, first_tokens=2, cu_seqlens_q=cu, max_seqlen_q=most)
        lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
        ref, bound = reference(c.q, c.K, c.V, c.table, c.lens, c.cu, c.scale, 30, 2)
        mine = torch.zeros(T, dtype=torch.bool)
        for i, n in enumerate(new):
            mine[4 + c.cu[i]:4 + c.cu[i] + min(n, most)] = True
        for out in (None, torch.full((T, 4, 64), 7.0, dtype=BF, device=gpu)):
            got = window_attention(q, c.K, c.V, c.table, lens, out=out, **dev)
            keep = mine[4:4 + sum(new)]
            check(got.cpu()[mine], ref[keep], bound[keep])
            assert (got.cpu()[~mine] == (0.0 if out is None else 7.0)).all()
    # without a list: one token per sequence, the rows behind them
    c = Call(gpu, [1] * 3, [10, 20, 30], 4, 2, 64, 16, 30, 2)
    q = torch.cat([c.q, c.q])
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    got = window_attention(q, c.K, c.V, c.table, lens, window=30, first_tokens=2)
    c.check(got[:3])
    assert (got[3:] == 0).all()


def test_strides(gpu):
    c = Call(gpu, [1, 70, 4], [50, 170, 30], 6, 2, 64, 16, 40, 5, poison=False)
    want = c.check()
    wide = torch.zeros(c.q.shape[0], 10, 80, dtype=BF, device=gpu)
    wide[:, 2:8, 8:72] = c.q
    c.q = wide[:, 2:8, 8:72]
    turned = torch.zeros(c.K.shape[0] * 2, 16, 2, 72, dtype=BF, device=gpu)  # token-major, padded rows
    for name in ("K", "V"):
        t = turned.clone()
        t.transpose(1, 2)[::2, :, :, :64] = getattr(c, name)
        setattr(c, name, t.transpose(1, 2)[::2, :, :, :64])
    table = torch.full((2 * c.table.shape[1], 3), -1, dtype=torch.int32, device=gpu)
    table[::2] = c.table.t()
    c.table = table[::2].t()
    out = torch.zeros(6, c.q.shape[0], 64, dtype=BF, device=gpu)
    got = c.run(out=out.transpose(0, 1))
    assert torch.equal(got, want) and got.data_ptr() == out.data_ptr()


@pytest.mark.parametrize("cache", ["bf16", "int8"])
@pytest.mark.parametrize("d", [16, 64, 80, 96, 128])
def test_outputs_that_start_at_eight_bytes(gpu, d, cache):
    c = Call(gpu, [1, 70, 130], [50, 170, 131], 6, 2, d, 16, 40, 5, cache, poison=False)
    want = c.check()
    room = torch.full((c.q.shape[0], 6, d + 12), 3.0, dtype=BF, device=gpu)
    out = room[..., 4:4 + d]
    c.run(out=out)
    assert torch.equal(out, want) and (room[..., :4] == 3.0).all() and (room[..., 4 + d:] == 3.0).all()


def test_scales_and_signs(gpu):
    c = Call(gpu, [1, 90], [70, 130], 4, 2, 64, 16, 50, 3, "fp8s")
    for s in (-0.3, 0.0, 2.0):
        c.scale = s
        c.check(softmax_scale=s)
    c.kd[0] = -c.kd[0]
    c.scale = 0.2
    c.check(softmax_scale=0.2)


def test_large_scores_and_sinks(gpu):
    c = Call(gpu, [1, 80], [90, 120], 4, 2, 64, 16, 50, 3, sink=True, poison=False)
    c.q *= 8
    c.sink = torch.tensor([100.0, -100.0, 0.0, 3.0])
    c.check()


@pytest.mark.parametrize("new", [1, 75])
def test_special_values_in_seen_rows(gpu, new):
    """A NaN in a value row reaches the queries that see it; other sequences stay
    as they are.  An infinity in an unseen row reaches nothing."""
    c = Call(gpu, [new, new], [100, 100], 4, 2, 64, 16, 30, 2, poison=False)
    want = c.run()
    c.V[c.table[0, 6], 0, 3] = math.nan  # key 99, the last, head 0
    got = c.run()
    assert torch.isnan(got[new - 1, :2]).all()
    assert torch.equal(got[new:], want[new:]) and torch.equal(got[:, 2:], want[:, 2:])
    if new == 1:
        c = Call(gpu, [1], [100], 4, 2, 64, 16, 30, 2, poison=False)
        want = c.run()
        for x, val in ((c.K, math.inf), (c.V, -math.inf)):
            x[c.table[0, 0], :, 2:] = val      # keys 2 .. 15: past the first, before the window
            x[c.table[0, 4], :, :6] = math.nan  # keys 64 .. 69; the window begins at 70
            x[c.table[0, 6], :, 4:] = val      # behind the last
        assert torch.equal(c.run(), want)


def test_workspace_streams_graphs_and_compiled_steps(gpu):
    c = Call(gpu, [1, 1], [4000, 3900], 4, 1, 128, 32, 3000, 4, poison=False)
    want = c.check()
    a = N.WindowArgs()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=gpu)
    ws.fill_(0xff)
    assert torch.equal(c.run(workspace=ws), want)
    assert torch.equal(c.run(workspace=ws[:256]), want)  # too small: replaced
    with pytest.raises(ValueError, match="contiguous"):
        c.run(workspace=ws[::2])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    step = lambda q, lens: window_attention(q, c.K, c.V, c.table, lens, window=3000, first_tokens=4)
    graph, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    q2 = c.q.flip(0).contiguous()
    with torch.cuda.graph(graph):
        out = step(c.q, lens)
    with torch.cuda.graph(g2):
        out2 = step(q2, lens)
    for i in range(3):
        lens -= 5 * i
        graph.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(c.q, lens)) and torch.equal(out2, step(q2, lens))
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(c.q, lens), step(c.q, lens))
    del a


def test_repeated_calls_give_the_same_bits(gpu):
    for new, lens, W in (([1, 1], [5000, 4000], 4096), ([300], [2000], 1500)):
        c = Call(gpu, new, lens, 8, 2, 64, 16, W, 8, poison=False)
        want = c.run()
        assert all(torch.equal(c.run(), want) for _ in range(3))


def test_empty_calls(gpu):
    c = Call(gpu, [1], [10], poison=False)
    e = c.q[:0]
    z = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert c.run(cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=gpu)).eq(0).all()
    got = window_attention(e, c.K, c.V, c.table, torch.tensor([10], dtype=torch.int32, device=gpu), window=3,
                           cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=gpu))
    assert got.shape == e.shape
    got = window_attention(c.q, c.K, c.V, c.table[:0], z[:0], window=3, cu_seqlens_q=z)
    assert (got == 0).all()


def test_refusals(gpu):
    c = Call(gpu, [1, 2], [10, 20], poison=False)
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    cu = torch.tensor(c.cu, dtype=torch.int32, device=gpu)
    ok = dict(q=c.q, k_cache=c.K, v_cache=c.V, block_table=c.table, seq_lens=lens, window=8, cu_seqlens_q=cu)
    for over, err in [(dict(window=0), ValueError), (dict(window=(1 << 30) + 1), ValueError),
                      (dict(first_tokens=-1), ValueError), (dict(q=c.q.float()), NotImplementedError),
                      (dict(q=c.q[:, :3]), ValueError), (dict(q=c.q[0]), ValueError),
                      (dict(v_cache=c.V[:1]), ValueError), (dict(block_table=c.table[:1]), ValueError),
                      (dict(block_table=c.table.long()), ValueError), (dict(seq_lens=lens.long()), ValueError),
                      (dict(cu_seqlens_q=cu[:2]), ValueError), (dict(max_seqlen_q=0), ValueError),
                      (dict(k_cache=c.K.to(torch.int8), v_cache=c.V.to(torch.int8)), ValueError),
                      (dict(k_cache=c.K.half(), v_cache=c.V.half()), NotImplementedError),
                      (dict(k_cache=c.K[:, :, :8], v_cache=c.V[:, :, :8]), NotImplementedError),
                      (dict(sink=torch.zeros(3, device=gpu)), ValueError), (dict(out=c.q[:1]), ValueError),
                      (dict(seq_lens=lens.cpu()), RuntimeError),
                      (dict(cu_seqlens_q=None, seq_lens=lens.repeat(2), block_table=c.table.repeat(2, 1)), ValueError)]:
        with pytest.raises(err):
            window_attention(**{**ok, **over})
    window_attention(**ok)
