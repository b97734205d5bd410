"""float64 statements of the quantised cache and of attention over key spans,
and the error bound of the bf16 kernels (plain torch, test infrastructure)."""
import math

import torch

U = 2.0 ** -8          # half a bf16 step, relative
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def quantise(x, dtype):
    """(codes as float64 values, scales float64) of rows x [..., d]."""
    r = x.double().cpu()
    amax = r.abs().amax(-1, keepdim=True)
    scale = amax.float() / TOP[dtype]
    # code Q must read back finite
    over = torch.isinf(scale * TOP[dtype]) & torch.isfinite(amax.float())
    scale = torch.where(over, torch.nextafter(scale, torch.zeros_like(scale)), scale).double()
    bad = ~torch.isfinite(amax)
    y = torch.where((amax > 0) & ~bad, r * TOP[dtype] / amax, torch.zeros_like(r))
    if dtype == torch.int8:
        code = torch.round(y)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        code = torch.round(y / step) * step
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    return code, scale[..., 0]


def pool_rows(pool, scales, blocks, n, factor=None):
    """float64 [n, Hkv, d] (CPU) of the first n tokens of a row of block ids."""
    bs = pool.shape[2]
    t = torch.arange(n)
    b = torch.as_tensor([int(i) for i in blocks])[t // bs] if n else t
    raw = pool.float().cpu()[b, :, t % bs].double()
    if scales is not None:
        raw = raw * scales.cpu().double()[b, :, t % bs][..., None]
    if factor is not None:
        raw = raw * factor.cpu().double().view(1, -1, 1)
    return raw


def attend(q, k, v, scale, sink=None):
    """softmax over all keys: q [m, Hq, d], k/v [n, Hkv, d] float64 ->
    (out [m, Hq, d], bound [m, Hq, d]).

    The bound: probabilities rounded to bf16 are off by at most U each, so the
    weighted sum by U sum(p |v|) / sum(p); the output's rounding adds U |out|;
    fp32 products, sums, exponentials and joins stay below 2^-12 of sum(p |v|)
    / sum(p) at the tests' sizes (at most 2^13 terms of a sum in fp32 chains
    of 2^6, scores below 2^7, so exponents are off by 2^-24 2^7 2^3 at most)."""
    m, Hq, d = q.shape
    G = Hq // k.shape[1]
    if k.shape[0] == 0:
        return torch.zeros(m, Hq, d, dtype=torch.float64), torch.zeros(m, Hq, d)
    kk = k.repeat_interleave(G, 1)
    vv = v.repeat_interleave(G, 1)
    s = torch.einsum("mhd,nhd->mhn", q.double(), kk) * scale
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.double().view(1, Hq, 1))
    p = torch.exp(s - top)
    den = p.sum(-1, keepdim=True)
    if sink is not None:
        den = den + torch.exp(sink.double().view(1, Hq, 1) - top)
    o = torch.einsum("mhn,nhd->mhd", p, vv) / den
    a = torch.einsum("mhn,nhd->mhd", p, vv.abs()) / den
    return o, U * a + U * o.abs() + 2.0 ** -12 * a


def check(got, ref, bound, what=""):
    err = (got.double().cpu() - ref).abs() - bound - 1e-30
    worst = err.max().item() if err.numel() else 0.0
    assert not torch.isnan(got.float()).any(), f"{what}: NaN"
    assert worst <= 0, f"{what}: past the bound by {worst}"
