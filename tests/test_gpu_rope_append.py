"""Rotation by several position axes with the cache append on the GPU, against
the float64 formula: axes, sections, pairs, norms, caches, slots, strides."""
import math

import pytest
import torch

from rope_ref import fp32_error, rms, rotate
from span_ref import TOP, quantise
from vllm_neuron_amd.functional import quant_kv_read, quant_kv_write, rope_kv_append, rope_rotate

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _inv(rot, theta=500000.0):
    return torch.tensor([theta ** (-2.0 * i / rot) for i in range(rot // 2)])


def _rows(T, hq, hkv, d, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, hq + 2 * hkv, d, generator=g)
    return (x * torch.exp2(torch.randint(-3, 4, (T, hq + 2 * hkv, 1), generator=g))).to(BF)


def _split(x, hq, hkv):
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def _close(got, ref, mag, what):
    """One rounding to bf16 (2^-8 of the value) behind the fp32 error."""
    err = (got.double().cpu() - ref).abs()
    bound = 2.0 ** -8 * ref.abs() + 1.01 * fp32_error(mag)
    assert not torch.isnan(got.float()).any(), what
    assert (err <= bound).all(), (what, (err - bound).max().item())


def _codes_close(code, scale, ref, mag, dtype, what):
    """Codes of fp32 values: the nearest code of the quotient, off by half a
    step and what the fp32 error of the value and of the row's maximum moves the
    quotient (each at most fp32_error of the row's largest magnitude, relative
    to the maximum)."""
    top = TOP[dtype]
    amax = ref.abs().amax(-1, keepdim=True)
    e = fp32_error(mag).amax(-1, keepdim=True)
    q = ref * top / amax
    code, scale = code.double().cpu(), scale.double().cpu()
    moved = 2.0 * top * e / amax
    half = 0.5 if dtype == torch.int8 else torch.clamp(2.0 ** -4 * q.abs(), min=2.0 ** -10)
    assert ((code - q).abs() <= half + 1.1 * moved).all(), what
    assert ((scale - amax[..., 0] / top).abs() <= e[..., 0] / top + 2.0 ** -23 * amax[..., 0] / top).all(), what


SECTIONS = {1: lambda h: [h], 2: lambda h: [h - h // 3, h // 3], 3: lambda h: [h - 2 * (h // 3), h // 3, h // 3],
            4: lambda h: [h - 3 * (h // 4), h // 4, 0, 2 * (h // 4)]}


@pytest.mark.parametrize("T,hq,hkv,d,rot", [(1, 1, 1, 64, 64), (3, 4, 2, 64, 32), (7, 5, 1, 80, 80), (5, 32, 8, 128, 128),
                                            (33, 6, 3, 128, 64), (4, 3, 1, 8, 8), (9, 2, 2, 96, 40), (6, 4, 4, 256, 256),
                                            (2, 3, 3, 200, 16), (600, 8, 2, 64, 64), (513, 48, 8, 128, 128)])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("order,pairs", [("blocks", "half"), ("cycle", "half"), ("blocks", "interleaved"),
                                         ("cycle", "interleaved")])
def test_rotation_and_bf16_cache(gpu, T, hq, hkv, d, rot, axes, order, pairs):
    x = _rows(T, hq, hkv, d, T + d)
    g = torch.Generator().manual_seed(axes)
    pos = torch.randint(0, 200000, (axes, T), generator=g)
    inv, sec = _inv(rot), SECTIONS[axes](rot // 2)
    bs, nb = 16, T // 16 + 2
    slots = torch.randperm(nb * bs, generator=g)[:T]
    pool = lambda: torch.full((nb, hkv, bs, d), 5.0, dtype=BF, device=gpu)
    K, V = pool(), pool()
    q, k, v = _split(x.to(gpu), hq, hkv)
    out = rope_kv_append(q, k, v, pos.to(gpu), inv.to(gpu), slots.to(gpu), K, V, sections=sec, section_order=order,
                         pairs=pairs)
    qr, kr, vr = _split(x, hq, hkv)
    _close(out, *rotate(qr, pos, inv, sec, order, pairs), "q")
    rows = lambda p: p[slots.to(gpu) // bs, :, slots.to(gpu) % bs]
    _close(rows(K), *rotate(kr, pos, inv, sec, order, pairs), "k")
    assert torch.equal(rows(V).cpu(), vr)
    # channels past the rotated ones as they were, other slots untouched
    assert torch.equal(out[..., rot:].cpu(), qr[..., rot:]) and torch.equal(rows(K)[..., rot:].cpu(), kr[..., rot:])
    left = torch.ones(nb * bs, dtype=torch.bool)
    left[slots] = False
    for p in (K, V):
        assert (p.transpose(1, 2).reshape(nb * bs, -1).cpu()[left] == 5.0).all()
    # without a cache, in place
    q2, k2 = rope_rotate(q, k, pos.to(gpu), inv.to(gpu), sections=sec, section_order=order, pairs=pairs)
    assert torch.equal(q2, out) and torch.equal(k2, rows(K))


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("T,hq,hkv,d,rot", [(1, 2, 1, 64, 64), (5, 32, 8, 128, 128), (17, 3, 2, 80, 40), (3, 2, 2, 256, 128)])
def test_quantised_caches(gpu, code, norm, T, hq, hkv, d, rot):
    x = _rows(T, hq, hkv, d, 1)
    pos, inv = torch.randint(0, 1 << 20, (3, T), generator=torch.Generator().manual_seed(2)), _inv(rot)
    sec, bs = SECTIONS[3](rot // 2), 8
    nb = T // bs + 2
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(3))[:T]
    pool = lambda: torch.zeros((nb, hkv, bs, d), dtype=torch.uint8, device=gpu).view(code)
    scale = lambda: torch.full((nb, hkv, bs), -3.0, device=gpu)
    K, V, ks, vs = pool(), pool(), scale(), scale()
    qg, kg = (1 + 0.1 * torch.randn(2, d, generator=torch.Generator().manual_seed(4))) if norm else (None, None)
    dev = lambda t: None if t is None else t.to(gpu)
    q, k, v = _split(x.to(gpu), hq, hkv)
    out = rope_kv_append(q, k, v, pos.to(gpu), inv.to(gpu), slots.to(gpu), K, V, sections=sec, qk_norm=norm,
                         q_gamma=dev(qg), k_gamma=dev(kg), eps=1e-5, k_scales=ks, v_scales=vs)
    qr, kr, vr = _split(x, hq, hkv)
    n = lambda t, g: rms(t, g, 1e-5) if norm else t
    _close(out, *rotate(n(qr, qg), pos, inv, sec, "blocks", "half"), "q")
    rows = lambda p: p.view(torch.uint8)[slots.to(gpu) // bs, :, slots.to(gpu) % bs].view(code).float()
    sc = lambda p: p[slots.to(gpu) // bs, :, slots.to(gpu) % bs]
    _codes_close(rows(K), sc(ks), *rotate(n(kr, kg), pos, inv, sec, "blocks", "half"), code, "k")
    want, want_s = quantise(vr, code)
    assert torch.equal(rows(V).double().cpu(), want) and torch.equal(sc(vs).double().cpu(), want_s)
    # what quant_kv_write writes of the same V, and reads back
    K2, V2, k2, v2 = pool(), pool(), scale(), scale()
    quant_kv_write(k, v, slots.to(gpu), K2, V2, k2, v2)
    assert torch.equal(V2.view(torch.uint8), V.view(torch.uint8)) and torch.equal(v2, vs)
    assert not torch.isnan(quant_kv_read(K, V, ks, vs, slots.to(gpu))[0]).any()


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("d", [8, 24, 40, 72, 80, 104, 120, 136, 200, 248])
def test_normalised_heads_narrower_than_their_lanes(gpu, code, d):
    """Lanes past the head dim hold zeros, whatever their registers held: they
    enter the row's maximum.  Behind kernels that leave NaN in registers."""
    T, hkv, bs = 300, 3, 16
    x = _rows(T, 1, hkv, d, d)
    pos, inv, slots = torch.arange(T), _inv(d), torch.arange(T)
    g = 1 + 0.1 * torch.randn(d, generator=torch.Generator().manual_seed(4))
    k, v = x[:, 1:1 + hkv], x[:, 1 + hkv:]
    K = torch.zeros((20, hkv, bs, d), dtype=torch.uint8, device=gpu).view(code)
    V, ks = K.clone(), torch.zeros((20, hkv, bs), device=gpu)
    vs = ks.clone()
    junk = torch.full((256, 1 << 14), math.nan, device=gpu)
    for _ in range(3):
        junk = torch.tanh(junk) * junk
        rope_kv_append(x[:, :1].to(gpu), k.to(gpu), v.to(gpu), pos.to(gpu), inv.to(gpu), slots.to(gpu), K, V, qk_norm=True,
                       q_gamma=g.to(gpu), k_gamma=g.to(gpu), eps=1e-5, k_scales=ks, v_scales=vs)
        at = slots.to(gpu)
        rows = K.view(torch.uint8)[at // bs, :, at % bs].view(code).float()
        _codes_close(rows, ks[at // bs, :, at % bs], *rotate(rms(k, g, 1e-5), pos, inv, None, "blocks", "half"), code, "k")


@pytest.mark.parametrize("factors", [False, True])
def test_static_fp8_cache(gpu, factors):
    T, hq, hkv, d, bs = 9, 4, 2, 64, 16
    x = _rows(T, hq, hkv, d, 1)
    pos, inv = torch.arange(T) * 1000, _inv(d)
    K = torch.zeros((2, hkv, bs, d), dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    V = K.clone()
    kd, vd = torch.tensor([0.01, 0.7]), torch.tensor([0.02, 0.5])
    kw = dict(k_dequant_scale=kd.to(gpu), v_dequant_scale=vd.to(gpu)) if factors else {}
    q, k, v = _split(x.to(gpu), hq, hkv)
    slots = torch.arange(T) + 3
    rope_kv_append(q, k, v, pos.to(gpu), inv.to(gpu), slots.to(gpu), K, V, **kw)
    _, kr, vr = _split(x, hq, hkv)
    ref, mag = rotate(kr, pos, inv, None, "blocks", "half")
    one = torch.ones(hkv)
    for pool, r, m, f in ((K, ref, mag, kd if factors else one), (V, vr.double(), vr.double().abs(), vd if factors else one)):
        y = (r / f.double()[:, None]).clamp(-448, 448)
        got = pool.float().cpu().double()[slots // bs, :, slots % bs]
        # half a step of the code, or 2^-10 below the least normal code
        bound = torch.clamp(2.0 ** -4 * y.abs(), min=2.0 ** -10) + 1.1 * fp32_error(m) / f.double()[:, None]
        assert ((got - y).abs() <= bound).all()


@pytest.mark.parametrize("gamma", [None, torch.float32, BF, torch.float16])
def test_head_norms(gpu, gamma):
    T, hq, hkv, d = 6, 4, 2, 128
    x = _rows(T, hq, hkv, d, 5)
    x[2, 1] = 0
    pos, inv = torch.arange(T) * 77, _inv(d)
    g = None if gamma is None else (1 + 0.3 * torch.randn(2, d, generator=torch.Generator().manual_seed(6))).to(gamma)
    kw = {} if g is None else dict(q_gamma=g[0].to(gpu), k_gamma=g[1].to(gpu))
    q, k, _ = _split(x.to(gpu), hq, hkv)
    for scale in (1.0, 1.3):
        qo, ko = rope_rotate(q, k, pos.to(gpu), inv.to(gpu), qk_norm=True, eps=1e-6, rope_scale=scale, **kw)
        qr, kr, _ = _split(x, hq, hkv)
        for got, r, w in ((qo, qr, None if g is None else g[0]), (ko, kr, None if g is None else g[1])):
            _close(got, *rotate(rms(r, w, 1e-6), pos, inv, None, "blocks", "half", scale), scale)
    # one gamma of two types: as both in fp32
    if g is not None and gamma != torch.float32:
        a = rope_rotate(q, k, pos.to(gpu), inv.to(gpu), qk_norm=True, q_gamma=kw["q_gamma"], k_gamma=kw["k_gamma"].float())
        b = rope_rotate(q, k, pos.to(gpu), inv.to(gpu), qk_norm=True, q_gamma=kw["q_gamma"].float(), k_gamma=kw["k_gamma"].float())
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_far_and_negative_positions(gpu):
    T, d = 8, 64
    x = _rows(T, 2, 1, d, 7)
    pos = torch.tensor([0, 1, -1, -12345, 1 << 24, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31])
    q, k, _ = _split(x.to(gpu), 2, 1)
    inv = _inv(d, 10000.0)
    for p in (pos, pos.int()):
        qo, ko = rope_rotate(q, k, p.to(gpu), inv.to(gpu))
        _close(qo, *rotate(x[:, :2], pos, inv, None, "blocks", "half"), "q")
        _close(ko, *rotate(x[:, 2:3], pos, inv, None, "blocks", "half"), "k")
    assert torch.equal(qo[0], q[0])  # position 0: nothing moves


def test_sentinel_slots_special_values_and_in_place(gpu):
    T, hq, hkv, d, bs = 6, 2, 2, 64, 16
    x = _rows(T, hq, hkv, d, 8)
    x[1, hq], x[2, hq + hkv, 3] = math.nan, math.inf
    slots = torch.tensor([0, 5, 17, -1, 32, 1 << 40])
    pos, inv = torch.arange(T), _inv(d)
    K = torch.full((2, hkv, bs, d), 9, dtype=torch.int8, device=gpu)
    V, ks = K.clone(), torch.full((2, hkv, bs), -1.0, device=gpu)
    vs = ks.clone()
    xg = x.to(gpu)
    q, k, v = _split(xg, hq, hkv)
    want_q, want_k = rope_rotate(q, k, pos.to(gpu), inv.to(gpu))
    got = rope_kv_append(q, k, v, pos.to(gpu), inv.to(gpu), slots.to(gpu), K, V, k_scales=ks, v_scales=vs, q_out=q, k_out=k)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want_q)
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(want_k))
    # a bad row: zero codes and scale NaN, its neighbours whole
    assert (K[0, 0, 5] == 0).all() and math.isnan(ks[0, 0, 5].item()) and not math.isnan(ks[0, 1, 5].item())
    assert (V[1, 0, 1] == 0).all() and math.isnan(vs[1, 0, 1].item()) and not math.isnan(vs[1, 1, 1].item())
    written = torch.zeros(2, bs, dtype=torch.bool)
    written[0, 0] = written[0, 5] = written[1, 1] = True
    assert (K.transpose(1, 2).cpu()[~written] == 9).all() and (ks.transpose(1, 2).cpu()[~written] == -1).all()
    # int32 slots
    K2, V2, k2, v2 = torch.full_like(K, 9), torch.full_like(K, 9), torch.full_like(ks, -1), torch.full_like(ks, -1)
    q, k, v = _split(x.to(gpu), hq, hkv)
    rope_kv_append(q, k, v, pos.int().to(gpu), inv.to(gpu), slots.clamp(max=1000).int().to(gpu), K2, V2, k_scales=k2,
                   v_scales=v2)
    assert torch.equal(K2, K) and torch.equal(V2, V)


def test_strided_rows_tables_and_pools(gpu):
    T, hq, hkv, d, bs = 12, 3, 2, 64, 16
    x = _rows(T, hq, hkv, d, 9).to(gpu)
    wide = torch.zeros(T, hq + 2 * hkv, d + 8, dtype=BF, device=gpu)
    wide[..., :d] = x
    pos = torch.randint(0, 5000, (T, 2), generator=torch.Generator().manual_seed(1)).to(gpu)
    inv, sec = _inv(d).to(gpu), [20, 12]
    slots = torch.arange(2 * T, device=gpu)[::2]
    both = torch.zeros((2, 4, hkv, bs, d), dtype=BF, device=gpu)
    rope_kv_append(*_split(x, hq, hkv), pos.t(), inv, slots, both[0], both[1], sections=sec)
    turned = torch.zeros((4, bs, hkv, d + 16), dtype=BF, device=gpu)  # token-major pool, padded rows
    K, V = turned.transpose(1, 2)[..., :d], torch.zeros_like(turned).transpose(1, 2)[..., :d]
    out = torch.zeros(hq, T, d, dtype=BF, device=gpu)
    rope_kv_append(*_split(wide[..., :d], hq, hkv), pos.t().contiguous(), inv, slots.contiguous(), K, V, sections=sec,
                   q_out=out.transpose(0, 1))
    assert torch.equal(K, both[0]) and torch.equal(V, both[1])
    assert torch.equal(out.transpose(0, 1), rope_rotate(*_split(x, hq, hkv)[:2], pos.t(), inv, sections=sec)[0])
    assert (turned[..., d:] == 0).all()


def test_empty_call(gpu):
    e = torch.empty(0, 2, 64, dtype=BF, device=gpu)
    K = torch.zeros((1, 2, 16, 64), dtype=BF, device=gpu)
    none = torch.empty(0, dtype=torch.int64, device=gpu)
    assert rope_kv_append(e, e, e, none, _inv(64).to(gpu), none, K, K.clone()).shape == (0, 2, 64)


def test_other_streams_graphs_and_compiled_steps(gpu):
    T, hq, hkv, d, bs = 5, 4, 2, 64, 16
    x, inv = _rows(T, hq, hkv, d, 10).to(gpu), _inv(d).to(gpu)
    pos, slots = torch.arange(T, device=gpu) + 100, torch.arange(T, device=gpu) + 2
    pool = lambda: torch.zeros((2, hkv, bs, d), dtype=torch.int8, device=gpu)
    sc = lambda: torch.zeros((2, hkv, bs), device=gpu)

    def step(x, pos, slots, K, V, ks, vs):
        return rope_kv_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pos, inv, slots, K, V, k_scales=ks,
                              v_scales=vs)

    ref = (pool(), pool(), sc(), sc())
    want = step(x, pos, slots, *ref)
    other = (pool(), pool(), sc(), sc())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x, pos, slots, *other)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(ref, other))
    kept = (pool(), pool(), sc(), sc())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, pos, slots, *kept)
    for i in range(3):
        pos += 17
        slots += 3
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(x, pos, slots, *ref))
        b = slots // bs
        assert torch.equal(kept[0][b, :, slots % bs], ref[0][b, :, slots % bs])
    fresh, eager = (pool(), pool(), sc(), sc()), (pool(), pool(), sc(), sc())
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(x, pos, slots, *fresh), step(x, pos, slots, *eager))
    assert all(torch.equal(a, b) for a, b in zip(fresh, eager))


def test_refusals(gpu):
    T, hq, hkv, d, bs = 4, 4, 2, 64, 16
    x, inv = _rows(T, hq, hkv, d, 11).to(gpu), _inv(d).to(gpu)
    q, k, v = _split(x, hq, hkv)
    pos, slots = torch.arange(T, device=gpu), torch.arange(T, device=gpu)
    K = torch.zeros((2, hkv, bs, d), dtype=BF, device=gpu)
    K8, sc = K.to(torch.int8), torch.zeros((2, hkv, bs), device=gpu)
    ok = dict(q=q, k=k, v=v, positions=pos, inv_freq=inv, slots=slots, k_cache=K, v_cache=K.clone())
    for over, err in [(dict(q=q.float()), NotImplementedError), (dict(k=k[:3]), ValueError), (dict(v=v[:, :1]), ValueError),
                      (dict(positions=pos[:3]), ValueError), (dict(positions=pos.float()), ValueError),
                      (dict(positions=pos.expand(2, T)), ValueError), (dict(sections=[30]), ValueError),
                      (dict(positions=pos.expand(2, T), sections=[40, -8]), ValueError),
                      (dict(positions=pos.expand(5, T), sections=[8, 8, 8, 4, 4]), NotImplementedError),
                      (dict(inv_freq=inv.double()), ValueError), (dict(inv_freq=inv[:14]), NotImplementedError),
                      (dict(inv_freq=_inv(128).to(gpu)), ValueError),
                      (dict(slots=slots[:3]), ValueError), (dict(slots=slots.float()), ValueError),
                      (dict(k_cache=K[:, :1]), ValueError), (dict(k_cache=K[..., :32], v_cache=K[..., :32]), ValueError),
                      (dict(k_cache=K8), ValueError), (dict(k_cache=K8, v_cache=K8.clone()), ValueError),
                      (dict(k_cache=K.half(), v_cache=K.half()), NotImplementedError),
                      (dict(k_scales=sc, v_scales=sc.clone()), ValueError), (dict(k_scales=sc), ValueError),
                      (dict(k_dequant_scale=sc[0, :, 0], v_dequant_scale=sc[0, :, 0]), ValueError),
                      (dict(q_gamma=inv), ValueError), (dict(section_order="rows"), ValueError),
                      (dict(pairs="adjacent"), ValueError), (dict(q_out=q[:3]), ValueError),
                      (dict(q=x[:, :hq, 1:41], k=k[..., 1:41], v=v[..., 1:41], inv_freq=inv[:8],
                            k_cache=K[..., :40], v_cache=K[..., :40]), ValueError),
                      (dict(slots=slots.cpu()), RuntimeError)]:
        with pytest.raises(err):
            rope_kv_append(**{**ok, **over})
    rope_kv_append(**ok)
