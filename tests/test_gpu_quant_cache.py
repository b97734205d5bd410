"""Quantised K/V cache on the GPU: codes and scales bit for bit against the
float64 definition, rows read back, sentinels, strides, special values."""
import math

import pytest
import torch

from span_ref import TOP, quantise
from vllm_neuron_amd.functional import quant_kv_read, quant_kv_write

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]


def _pool(nb, hkv, bs, d, code, dev):
    mk = lambda: torch.full((nb, hkv, bs, d), 3, dtype=torch.uint8, device=dev).view(code)
    sc = lambda: torch.full((nb, hkv, bs), -2.0, device=dev)
    return mk(), mk(), sc(), sc()


def _rows(T, h, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, h, d, generator=g) * torch.exp2(torch.randint(-8, 9, (T, h, 1), generator=g))
    return x.to(dtype)


def _check_written(rows, pool, scales, slots, code):
    bs = pool.shape[2]
    want, want_s = quantise(rows, code)
    got = pool.float().cpu().double()
    sc = scales.cpu()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pool.shape[0] * bs:
            assert torch.equal(got[s // bs, :, s % bs], want[t]), (t, s)
            assert torch.equal(sc[s // bs, :, s % bs].double(), want_s[t]), (t, s)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,h,d,bs", [(1, 1, 64, 16), (5, 8, 64, 16), (33, 3, 128, 32), (7, 2, 80, 16),
                                      (9, 2, 7, 5), (3, 1, 1, 1), (6, 2, 200, 8), (4, 2, 512, 16),
                                      (300, 4, 128, 64)])
def test_write_and_read(gpu, code, dtype, T, h, d, bs):
    nb = (T + bs - 1) // bs + 3
    k, v = _rows(T, h, d, dtype, 1), _rows(T, h, d, dtype, 2)
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(3))[:T]
    if T > 2:
        slots[1], slots[2] = -1, nb * bs  # sentinels
    kc, vc, ks, vs = _pool(nb, h, bs, d, code, gpu)
    before = kc.view(torch.uint8).clone()
    quant_kv_write(k.to(gpu), v.to(gpu), slots.to(gpu), kc, vc, ks, vs)
    _check_written(k, kc, ks, slots, code)
    _check_written(v, vc, vs, slots, code)
    # everything else as it was
    mask = torch.ones(nb * bs, dtype=torch.bool)
    mask[[s for s in slots.tolist() if 0 <= s < nb * bs]] = False
    flat = lambda t: t.transpose(1, 2).reshape(nb * bs, -1).cpu()[mask]
    assert torch.equal(flat(kc.view(torch.uint8)), flat(before))
    assert (ks.transpose(1, 2).reshape(nb * bs, h).cpu()[mask] == -2.0).all()
    for out in (torch.bfloat16, torch.float16, torch.float32):
        rk, rv = quant_kv_read(kc, vc, ks, vs, slots.to(gpu), dtype=out)
        for got, pool, sc in ((rk, kc, ks), (rv, vc, vs)):
            for t, s in enumerate(slots.tolist()):
                if 0 <= s < nb * bs:
                    want = (pool[s // bs, :, s % bs].float() * sc[s // bs, :, s % bs, None]).to(out)
                else:
                    want = torch.zeros_like(got[t])
                assert torch.equal(got[t], want), (out, t)


@pytest.mark.parametrize("code", CODES)
def test_fp32_rows(gpu, code):
    """fp32 sources: the code of the quotient or, within 2^-20 of a border, of
    its neighbour (product, quotient and remainder round at 2^-24 each)."""
    T, h, d, bs = 64, 2, 128, 16
    k = _rows(T, h, d, torch.float32, 5)
    kc, vc, ks, vs = _pool(T // bs, h, bs, d, code, gpu)
    quant_kv_write(k.to(gpu), k.to(gpu), torch.arange(T, device=gpu), kc, vc, ks, vs)
    got = kc.float().cpu().double().transpose(1, 2).reshape(T, h, d)
    r = k.double()
    amax = r.abs().amax(-1, keepdim=True)
    y = r * TOP[code] / amax
    want, _ = quantise(k, code)
    same = got == want
    step = torch.ones_like(y) if code == torch.int8 else torch.exp2(
        torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    # elsewhere: the quotient lies on the border between the two codes
    assert ((y - (got + want) / 2).abs()[~same] <= 2.0 ** -20 * y.abs()[~same]).all()
    assert ((got - want).abs() <= step * 1.0000001).all()
    assert torch.equal(ks.cpu().transpose(1, 2).reshape(T, h), (amax.float() / TOP[code])[..., 0])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_special_rows(gpu, code, dtype):
    """Zeros, non-finite values, the ends of the exponent range, ties."""
    d, bs = 64, 16
    fi = torch.finfo(dtype)
    x = torch.randn(9, 1, d, generator=torch.Generator().manual_seed(7)).to(dtype)
    x[0] = 0
    x[1, 0, 5] = math.nan
    x[2, 0, 6] = math.inf
    x[3, 0, 7] = -math.inf
    x[4, 0, ::3] = fi.max
    x[4, 0, 1] = fi.min
    x[5] = 0
    x[5, 0, 3] = fi.tiny
    x[6] = 0
    x[6, 0, 3] = -0.0
    x[7] = torch.arange(d).to(dtype)            # amax 63
    x[8] = torch.linspace(-127, 127, d).round().to(dtype) * 0.5  # ties of x * Q / amax
    x[8, 0, 0] = 127.0
    kc, vc, ks, vs = _pool(1, 1, bs, d, code, gpu)
    quant_kv_write(x.to(gpu), x.to(gpu), torch.arange(9, device=gpu), kc, vc, ks, vs)
    want, want_s = quantise(x, code)
    got = kc.float().cpu().double()[0, 0, :9]
    sc = ks.cpu()[0, 0, :9].double()
    assert torch.isnan(sc[1:4]).all() and (got[1:4] == 0).all()
    keep = [0, 4, 5, 6, 7, 8]
    assert torch.equal(got[keep], want[keep, 0])
    assert torch.equal(sc[keep], want_s[keep, 0])
    rk, _ = quant_kv_read(kc, vc, ks, vs, torch.arange(9, device=gpu), dtype=torch.float32)
    assert torch.isnan(rk[1:4]).all()
    assert torch.isfinite(rk[keep]).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("shift", [0, 1])
def test_views(gpu, code, shift):
    """K and V as ranges of one projection, caches stacked [2, ...], scales as
    views, int32 slots; shift = 1: rows and cache off the vector alignment."""
    T, h, d, bs, nb = 21, 2, 64, 16, 4
    qkv = _rows(T, 1, 6 * d + shift, torch.bfloat16, 9)[:, 0].to(gpu)
    k = qkv[:, shift + d:shift + 3 * d].view(T, h, d)
    v = qkv[:, shift + 3 * d:shift + 5 * d].view(T, h, d)
    both = torch.zeros(2, nb, h, bs, d + shift, dtype=torch.uint8, device=gpu).view(code)[..., shift:]
    sc = torch.zeros(2, nb, bs, h, device=gpu).transpose(2, 3)
    slots = torch.randperm(nb * bs)[:T].to(torch.int32)
    quant_kv_write(k, v, slots.to(gpu), both[0], both[1], sc[0], sc[1])
    _check_written(k.cpu(), both[0], sc[0], slots, code)
    _check_written(v.cpu(), both[1], sc[1], slots, code)
    wide = torch.cat([slots, slots[:3]]).to(gpu)  # read: a slot may come twice
    rk, rv = quant_kv_read(both[0], both[1], sc[0], sc[1], wide)
    assert torch.equal(rk[T:], rk[:3]) and torch.equal(rv[T:], rv[:3])


def test_large_pool(gpu):
    """Slots past 2^31 bytes of the pool."""
    nb, h, bs, d = 9000, 16, 128, 128  # 2.36 GB per cache
    kc = torch.empty(nb, h, bs, d, dtype=torch.int8, device=gpu)
    ks = torch.empty(nb, h, bs, device=gpu)
    k = _rows(3, h, d, torch.bfloat16, 11)
    slots = torch.tensor([nb * bs - 1, 17, (nb - 1) * bs])
    quant_kv_write(k.to(gpu), k.to(gpu), slots.to(gpu), kc, kc, ks, ks)
    want, want_s = quantise(k, torch.int8)
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(kc[s // bs, :, s % bs].cpu().double(), want[t])
        assert torch.equal(ks[s // bs, :, s % bs].cpu().double(), want_s[t])


def test_empty_and_refusals(gpu):
    kc, vc, ks, vs = _pool(2, 2, 16, 64, torch.int8, gpu)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    slots = torch.zeros(3, dtype=torch.int64, device=gpu)
    quant_kv_write(rows[:0], rows[:0], slots[:0], kc, vc, ks, vs)
    assert quant_kv_read(kc, vc, ks, vs, slots[:0])[0].shape == (0, 2, 64)
    bad = [
        (ValueError, (rows, rows, slots[:2], kc, vc, ks, vs)),
        (ValueError, (rows[:, :1], rows[:, :1], slots, kc, vc, ks, vs)),
        (ValueError, (rows, rows[..., :32], slots, kc, vc, ks, vs)),
        (ValueError, (rows, rows.float(), slots, kc, vc, ks, vs)),
        (ValueError, (rows, rows, slots, kc, vc, ks[:1], vs)),
        (ValueError, (rows, rows, slots, kc, vc, ks.half(), vs)),
        (ValueError, (rows, rows, slots.float(), kc, vc, ks, vs)),
        (NotImplementedError, (rows, rows, slots, kc.to(torch.bfloat16), vc.to(torch.bfloat16), ks, vs)),
        (NotImplementedError, (rows.double(), rows.double(), slots, kc, vc, ks, vs)),
        (RuntimeError, (rows.cpu(), rows, slots, kc, vc, ks, vs)),
    ]
    for err, args in bad:
        with pytest.raises(err):
            quant_kv_write(*args)


def test_graph_replay(gpu):
    T, h, d, bs, nb = 40, 4, 128, 16, 8
    k, v = (_rows(T, h, d, torch.bfloat16, s).to(gpu) for s in (1, 2))
    slots = torch.randperm(nb * bs)[:T].to(gpu)
    kc, vc, ks, vs = _pool(nb, h, bs, d, torch.int8, gpu)
    quant_kv_write(k, v, slots, kc, vc, ks, vs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        quant_kv_write(k, v, slots, kc, vc, ks, vs)
        rk, rv = quant_kv_read(kc, vc, ks, vs, slots)
    for seed in (5, 6, 7):
        k.copy_(_rows(T, h, d, torch.bfloat16, seed))
        slots.copy_(torch.randperm(nb * bs)[:T])
        g.replay()
        torch.cuda.synchronize()
        _check_written(k.cpu(), kc, ks, slots.cpu(), torch.int8)
        e = _pool(nb, h, bs, d, torch.int8, gpu)
        quant_kv_write(k, v, slots, *e)
        a, b = quant_kv_read(*e, slots)
        assert torch.equal(a, rk) and torch.equal(b, rv)
