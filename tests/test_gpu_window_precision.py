"""Window attention of few rows carries its probabilities in two bf16 parts: its
outputs are off by their own rounding and 2^-12 of sum(p |v|) / sum(p).

Keys of two kinds: of score 0 (the largest, probability 1) and of score log(b),
their values 1 and -1 / b times one number, so that the weighted sum nearly vanishes:
the output's own rounding is small, and what the probabilities' rounding does to b is
seen whole.  One bf16 part may be off by 2^-8 of b, that is 2^-9 of sum(p |v|) /
sum(p); two by 2^-16 of b.  The rest of the bound is float32's: scores of two
products (2^-23 of at most 4), exponentials (2^-22), and sums of at most 2^9 terms
in chains of 2^7 at most, 2^-17: together below 2^-15."""
import pytest
import torch

from span_ref import U, quantise
from vllm_neuron_amd.functional import window_attention
from window_ref import attend

BF, FP8 = torch.bfloat16, torch.float8_e4m3fn
CACHES = ["bf16", "fp8s", "fp8", "int8"]


def _case(cache, d, Hkv, n, seed):
    """K and V of one sequence [n, Hkv, d] (codes and scales of the cache) and
    their values in float64; q [Hkv * G, d] is one everywhere at channels 0, 1."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.zeros(n, Hkv, d), torch.zeros(n, Hkv, d)
    small = torch.arange(n) % 2 == 1
    s = -0.05 - 3.0 * torch.rand(Hkv, generator=g)
    if cache in ("bf16", "fp8s"):
        k[small, :, 0] = s.to(BF).float()
        k[small, :, 1] = s - s.to(BF).float()
    else:
        k[small, :, 0] = s
    kq, ks = _quant(k, cache)
    b = torch.exp((kq * ks[..., None])[1, :, :2].sum(-1))            # [Hkv], the probabilities
    size = 0.5 + torch.rand(Hkv, d, generator=g)
    v[~small] = size
    v[small] = -size / b.float()[:, None]
    vq, vs = _quant(v, cache)
    return kq, ks, vq, vs


def _quant(x, cache):
    """Codes and scales [n, Hkv] in float64."""
    if cache == "bf16":
        return x.to(BF).double(), torch.ones(x.shape[:2], dtype=torch.float64)
    if cache == "fp8s":
        return x.to(FP8).double(), torch.ones(x.shape[:2], dtype=torch.float64)
    return quantise(x.to(BF), torch.int8 if cache == "int8" else FP8)


def _reference(kq, ks, vq, vs, Hq, parts):
    """(out, bound) with probabilities whole, or rounded to one bf16 part."""
    k, v = kq * ks[..., None], vq * vs[..., None]
    n, Hkv, d = k.shape
    q = torch.zeros(1, Hq, d)
    q[..., :2] = 1.0
    o, _ = attend(q, k, v, 1.0, torch.tensor([n - 1]), n, 0)
    a, _ = attend(q, k, v.abs(), 1.0, torch.tensor([n - 1]), n, 0)
    if parts == 1:
        p = torch.exp(k[..., :2].sum(-1))                            # [n, Hkv]; the largest is 1
        scale = vs if (vs != 1).any() else torch.ones_like(vs)
        w = (p * scale).to(torch.float32).to(BF).double()
        o = (torch.einsum("nh,nhd->hd", w, vq) / p.sum(0)[:, None]).repeat_interleave(Hq // Hkv, 0)[None]
    return o, U * o.abs() + 2.0 ** -12 * a


SHAPES = [(1, 64, 2, 100), (4, 128, 3, 257), (8, 64, 2, 512), (3, 96, 2, 40)]  # heads per kv head, d, kv heads, keys


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("G,d,Hkv,n", SHAPES)
def test_the_bound_tells_one_part_from_two(cache, G, d, Hkv, n):
    past = 0
    for seed in range(12):
        case = _case(cache, d, Hkv, n, seed)
        ref, bound = _reference(*case, G * Hkv, 2)
        one, _ = _reference(*case, G * Hkv, 1)
        past += ((one - ref).abs() > bound).any().item()
    assert past >= 3


@pytest.mark.gpu
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("G,d,Hkv,n", SHAPES)
def test_outputs_of_few_rows(gpu, cache, G, d, Hkv, n):
    bs, seqs, Hq = 16, 12, G * Hkv
    nblk = (n + bs - 1) // bs
    code = {"bf16": BF, "int8": torch.int8}.get(cache, FP8)
    pool = lambda: torch.zeros(seqs, nblk * bs, Hkv, d)
    K, V, ks, vs = pool(), pool(), torch.ones(seqs, nblk * bs, Hkv), torch.ones(seqs, nblk * bs, Hkv)
    ref, bound = torch.zeros(seqs, Hq, d).double(), torch.zeros(seqs, Hq, d).double()
    for i in range(seqs):
        case = _case(cache, d, Hkv, n, i)
        for t, x in zip((K, ks, V, vs), case):
            t[i, :n] = x.float()
        ref[i], bound[i] = (x[0] for x in _reference(*case, Hq, 2))
    blocks = lambda t: t.view(seqs * nblk, bs, Hkv, -1).transpose(1, 2).contiguous()
    kw = {} if cache in ("bf16", "fp8s") else dict(k_scales=blocks(ks)[..., 0].contiguous().to(gpu),
                                                   v_scales=blocks(vs)[..., 0].contiguous().to(gpu))
    table = torch.arange(seqs * nblk, dtype=torch.int32, device=gpu).view(seqs, nblk)
    q = torch.zeros(seqs, Hq, d, dtype=BF, device=gpu)
    q[..., :2] = 1.0
    got = window_attention(q, blocks(K).to(code).to(gpu), blocks(V).to(code).to(gpu), table,
                           torch.full((seqs,), n, dtype=torch.int32, device=gpu), window=n, softmax_scale=1.0, **kw)
    err = (got.double().cpu() - ref).abs()
    assert (err <= bound).all(), ((err - bound).max().item(), (err / bound).max().item())
