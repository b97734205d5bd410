"""Performance cases of an attention layer with 8-bit projections, rotated keys
of several position axes and a bounded view of the cache: what each case stands
for, its inputs, one pass in plain torch or through the public entry points, the
work a pass cannot do without, and its float64 statement.

Kinds
  linear  rows quantised to int8 with one scale per token (after an RMS norm
          where the layer has one), times int8 weights with one scale per
          output channel (``quant_rows``, ``int8_linear``)
  rope    Q and K rotated by positions on one or several axes, K and V appended
          to a paged cache in the same pass (``rope_kv_append``)
  window  attention over a paged cache with a sliding window and a few first
          tokens that stay visible, single tokens and ragged prompts
          (``window_attention``)

Conventions: hidden states, Q, K, V ~ N(0, 1) with a few channels of larger
values, as projections have them; rows of a quantised cache differ in
magnitude.  Physical blocks are a random permutation; table entries of blocks
that no query sees are -1, as they are once such blocks are freed.  Lengths
belong to the case, every value to the seed.
"""
import math
import os
import random
import sys

import torch

own = False

BF = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
FP8 = torch.float8_e4m3fn
I8 = torch.int8
I32 = torch.int32
DEV = "cuda:0"
CODES = {"int8": (I8, 127.0), "fp8": (FP8, 448.0)}

# Head geometries of the repository's workload table and its dense cases.
SHAPES = {
    "llama3_1b": dict(heads=32, kv=8, d=64, bs=16, sink=False),
    "llama3_8b": dict(heads=32, kv=8, d=128, bs=32, sink=False),
    "gptoss": dict(heads=64, kv=8, d=64, bs=32, sink=True),
    "long_48q": dict(heads=48, kv=8, d=128, bs=64, sink=False),
    "mha_d80": dict(heads=16, kv=16, d=80, bs=16, sink=False),
}


def listed():
    return [
        # The smallest product: the output projection of a small model's decode
        # step; two launches and the host's time count.
        dict(name="linear_step_b4", kind="linear", tokens=4, k=2048, n=2048, norm=False, bias=False),
        # A full decode batch of an 8B layer, norm to projection.
        dict(name="linear_step_b64", kind="linear", tokens=64, k=4096, n=6144, norm=True, bias=False),
        # A ragged chunk over widths that are no powers of two, with a bias.
        dict(name="linear_chunk", kind="linear", tokens=517, k=2880, n=5120, norm=True, bias=True),
        # The largest product: a long prompt of a wide layer.
        dict(name="linear_prompt", kind="linear", tokens=8191, k=8192, n=10240, norm=True, bias=False),
        # A decode step far into its contexts, keys to an int8 cache.
        dict(name="rope_step_int8", kind="rope", shape="llama3_8b", tokens=8, axes=1, rot=128, split="blocks",
             pairs="half", norm=False, far=131000, cache="int8"),
        # An image's tokens with positions in time, height and width, Q and K
        # normalised per head.
        dict(name="rope_image", kind="rope", shape="long_48q", tokens=2047, axes=3, rot=128, split="cycle",
             pairs="half", norm=True, far=4096, cache="bf16"),
        # A whole long prompt.
        dict(name="rope_prompt", kind="rope", shape="llama3_8b", tokens=16383, axes=3, rot=128, split="blocks",
             pairs="half", norm=False, far=32768, cache="bf16"),
        # A few requests of a small model in long conversations.
        dict(name="window_step_b4", kind="window", shape="llama3_1b", batch=4, new_lo=1, new_hi=1, ctx_lo=100,
             ctx_hi=9001, window=1024, first=4, cache="bf16"),
        # A full batch of an 8B layer, wide window.
        dict(name="window_step_b64", kind="window", shape="llama3_8b", batch=64, new_lo=1, new_hi=1, ctx_lo=1000,
             ctx_hi=30000, window=4096, first=4, cache="bf16"),
        # Many streams with a short window and sinks, int8 cache.
        dict(name="window_step_int8", kind="window", shape="gptoss", batch=128, new_lo=1, new_hi=1, ctx_lo=1,
             ctx_hi=5000, window=512, first=16, cache="int8"),
        # Ragged chunks of a batch behind earlier tokens.
        dict(name="window_ragged", kind="window", shape="gptoss", batch=6, new_lo=1, new_hi=700, ctx_lo=0,
             ctx_hi=1500, window=128, first=4, cache="bf16"),
        # The largest: a long prompt of one sequence.
        dict(name="window_prompt", kind="window", shape="llama3_8b", batch=1, new_lo=8191, new_hi=8191, ctx_lo=0,
             ctx_hi=0, window=2048, first=64, cache="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "rope", "window", "window"])
    if kind == "linear":
        k = 16 * _log_int(rng, 16, 512)
        n = _log_int(rng, 200, 10000)
        return dict(kind=kind, tokens=_log_int(rng, 1, 8000), k=k, n=n, norm=rng.random() < 0.5,
                    bias=rng.random() < 0.3)
    if kind == "rope":
        shape = rng.choice(sorted(SHAPES))
        d = SHAPES[shape]["d"]
        return dict(kind=kind, shape=shape, tokens=_log_int(rng, 1, 16384), axes=rng.choice([1, 2, 3, 3]),
                    rot=rng.choice([d, d, d // 2]), split=rng.choice(["blocks", "cycle"]),
                    pairs=rng.choice(["half", "half", "interleaved"]), norm=rng.random() < 0.5,
                    far=_log_int(rng, 100, 1000000), cache=rng.choice(["bf16", "bf16", "int8", "fp8"]))
    shape = rng.choice(sorted(SHAPES))
    s = SHAPES[shape]
    window, first = _log_int(rng, 16, 4096), rng.choice([0, 1, 4, 16, 64])
    cache = rng.choice(["bf16", "bf16", "int8", "fp8"])
    if rng.random() < 0.5:
        new = rng.choice([1, 1, 1, 2, 4])
        return dict(kind=kind, shape=shape, batch=_log_int(rng, 1, 48 // new), new_lo=new, new_hi=new,
                    ctx_lo=_log_int(rng, 1, 200), ctx_hi=_log_int(rng, 201, 30000), window=window, first=first,
                    cache=cache)
    batch = rng.randint(1, 6)
    # at most half of the largest case's operations
    most = int(1.3e11 / (4.0 * batch * (window + first) * s["heads"] * s["d"]))
    return dict(kind=kind, shape=shape, batch=batch, new_lo=1, new_hi=_log_int(rng, 2, max(4, min(4096 // batch, most))),
                ctx_lo=0, ctx_hi=_log_int(rng, 1, 5000), window=window, first=first, cache=cache)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(n, lo, hi, salt=0):
    """Lengths of a case: spread over [lo, hi], the longest among them, the
    same for every seed."""
    r = random.Random("%d %d %d %d" % (n, lo, hi, salt))
    lens = [r.randint(min(lo, hi), hi) for _ in range(n)]
    lens[r.randrange(n)] = hi
    return lens


def _window_lens(case):
    """New tokens and lengths (earlier tokens and the new ones) of a window
    case's sequences."""
    new = _lens(case["batch"], case["new_lo"], case["new_hi"], 1)
    ctx = _lens(case["batch"], case["ctx_lo"], case["ctx_hi"])
    return new, [c + n for c, n in zip(ctx, new)]


class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape, dtype=BF):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=self.g, device=DEV) * (hi - lo) + lo

    def integers(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device=DEV)

    def spiky(self, *shape):
        """[..., d] with one channel in sixteen four times as large."""
        x = self.normal(*shape)
        x[..., 5::16] *= 4.0
        return x

    def blocks(self, n, first):
        return torch.randperm(max(1, n), generator=self.g, device=DEV).to(I32)[:n] + first


def _codes(x, cache, amax=None):
    """fp32 x [..., d] as codes and scales of its rows: scale = max|x| / Q,
    code = round(x Q / max|x|)."""
    dtype, top = CODES[cache]
    amax = x.abs().amax(-1, keepdim=True)
    y = torch.where(amax > 0, x * top / amax, torch.zeros_like(x))
    return y.round().to(I8) if dtype is I8 else y.to(FP8), (amax / top).squeeze(-1)


def _linear_inputs(case, gen):
    M, K, N = case["tokens"], case["k"], case["n"]
    x = gen.spiky(M, K)
    x.mul_(gen.uniform(M, 1, lo=0.25, hi=4.0).to(BF))
    w, ws = _codes(gen.normal(N, K, dtype=F32) * (K ** -0.5), "int8")
    return dict(x=x, w=w, ws=ws, gamma=1.0 + 0.1 * gen.normal(K, dtype=F32) if case["norm"] else None,
                bias=gen.normal(N) if case["bias"] else None)


def _sections(case):
    """Channel pairs of each axis: the first axis a quarter of them (time), the
    others the rest in equal parts."""
    half, axes = case["rot"] // 2, case["axes"]
    if axes == 1:
        return [half]
    rest = half - half // (axes + 1)
    parts = [rest // (axes - 1)] * (axes - 1)
    return [half - sum(parts)] + parts


def _axis_of_pair(case):
    """Axis of each channel pair: contiguous blocks of pairs ("blocks"), or the
    axes in turn while their parts last, the rest of the first axis at the end
    ("cycle")."""
    sec, half = _sections(case), case["rot"] // 2
    if case["split"] == "blocks":
        return [a for a, n in enumerate(sec) for _ in range(n)]
    out = [0] * half
    for a in range(1, len(sec)):
        for i in range(a, min(sec[a] * len(sec), half), len(sec)):
            out[i] = a
    return out


def _rope_inputs(case, gen):
    s = SHAPES[case["shape"]]
    T, kv, d, bs = case["tokens"], s["kv"], s["d"], s["bs"]
    nb = 1 + (T + bs - 1) // bs
    table = gen.blocks(nb - 1, 1).long()
    t = torch.arange(T, device=DEV)
    # Q, K and V are column ranges of one projection output
    rows = gen.spiky(T, s["heads"] + 2 * kv, d)
    rows.mul_(gen.uniform(T, s["heads"] + 2 * kv, 1, lo=0.25, hi=4.0).to(BF))
    quant = case["cache"] in CODES
    pool = lambda: torch.zeros((nb, kv, bs, d), dtype=CODES[case["cache"]][0] if quant else BF, device=DEV)
    scale = lambda: torch.zeros((nb, kv, bs), device=DEV) if quant else None
    inv = torch.tensor([500000.0 ** (-2.0 * i / case["rot"]) for i in range(case["rot"] // 2)], device=DEV)
    positions = gen.integers(case["far"], case["axes"], T)
    return dict(q=rows[:, :s["heads"]], k=rows[:, s["heads"]:s["heads"] + kv], v=rows[:, s["heads"] + kv:],
                positions=positions, inv=inv, slots=table[t // bs] * bs + t % bs, K=pool(), V=pool(), ks=scale(),
                vs=scale(), axis=torch.tensor(_axis_of_pair(case), device=DEV),
                qn=1.0 + 0.1 * gen.normal(d, dtype=F32) if case["norm"] else None,
                kn=1.0 + 0.1 * gen.normal(d, dtype=F32) if case["norm"] else None)


def _window_inputs(case, gen):
    s = SHAPES[case["shape"]]
    kv, d, bs = s["kv"], s["d"], s["bs"]
    new, lens = _window_lens(case)
    # blocks that a query sees
    seen = [[j for j in range((n + bs - 1) // bs) if j * bs < case["first"] or (j + 1) * bs > n - m - case["window"] + 1]
            for m, n in zip(new, lens)]
    ids = gen.blocks(sum(len(r) for r in seen), 1)
    table = torch.full((len(lens), max((n + bs - 1) // bs for n in lens)), -1, dtype=I32)
    at, host = 0, ids.cpu()
    for i, r in enumerate(seen):
        table[i, torch.tensor(r, dtype=torch.long)] = host[at:at + len(r)]
        at += len(r)
    shape = (1 + at, kv, bs, d)
    k, v = gen.spiky(*shape), gen.normal(*shape)
    x = dict(K=k, V=v, ks=None, vs=None)
    if case["cache"] in CODES:
        # rows of unlike magnitude: what one scale per row is for
        k = k.float() * gen.uniform(*shape[:3], 1, lo=0.5, hi=2.0)
        v = v.float() * gen.uniform(*shape[:3], 1, lo=0.25, hi=4.0)
        (kc, ks), (vc, vs) = _codes(k, case["cache"]), _codes(v, case["cache"])
        x = dict(K=kc, V=vc, ks=ks, vs=vs)
    at = [sum(new[:i]) for i in range(len(new) + 1)]
    x.update(q=gen.normal(sum(new), s["heads"], d), table=table.to(DEV), lens=torch.tensor(lens, dtype=I32, device=DEV),
             cu=torch.tensor(at, dtype=I32, device=DEV), most=max(new),
             sink=gen.uniform(s["heads"], lo=-1.0, hi=1.0) if s["sink"] else None)
    return x


def _inputs(case, seed):
    return {"linear": _linear_inputs, "rope": _rope_inputs, "window": _window_inputs}[case["kind"]](case, _Gen(seed))


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if case["kind"] == "rope":
        x["sections"] = _sections(case)
    return x


# ---------------------------------------------------------------------------
# one pass, plain form
# ---------------------------------------------------------------------------
EPS = 1e-6


def _rms(x, gamma):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma


def _plain_linear(x):
    rows = x["x"].float()
    if x["gamma"] is not None:
        rows = _rms(rows, x["gamma"])
    code, scale = _codes(rows, "int8")
    y = torch.matmul(code.float(), x["w"].float().t()) * scale[:, None] * x["ws"]
    if x["bias"] is not None:
        y = y + x["bias"].float()
    return y.to(BF), scale


def _rotated(x, cos, sin, rot, pairs):
    """fp32 x [T, H, d] with its first ``rot`` channels rotated by [T, 1, rot / 2]."""
    head, tail = x[..., :rot], x[..., rot:]
    if pairs == "half":
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, tail], -1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), tail], -1)


def _plain_rope(x):
    case = x["case"]
    # angles of far positions need more than 32 bits
    angle = x["positions"].double()[x["axis"]].t() * x["inv"].double()
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    q, k, v = x["q"].float(), x["k"].float(), x["v"].float()
    if case["norm"]:
        q, k = _rms(q, x["qn"]), _rms(k, x["kn"])
    q = _rotated(q, cos, sin, case["rot"], case["pairs"]).to(BF)
    k = _rotated(k, cos, sin, case["rot"], case["pairs"])
    bs = x["K"].shape[2]
    b, o = x["slots"] // bs, x["slots"] % bs
    if case["cache"] == "bf16":
        x["K"][b, :, o] = k.to(BF)
        x["V"][b, :, o] = x["v"]
        return q, x["K"], x["V"]
    (kc, ks), (vc, vs) = _codes(k, case["cache"]), _codes(v, case["cache"])
    # the pools as bytes: indexed stores of 8-bit floats are not there for every type
    x["K"].view(torch.uint8)[b, :, o] = kc.view(torch.uint8)
    x["V"].view(torch.uint8)[b, :, o] = vc.view(torch.uint8)
    x["ks"][b, :, o], x["vs"][b, :, o] = ks, vs
    back = lambda pool, sc: (pool.view(torch.uint8)[b, :, o].view(pool.dtype).float() * sc[b, :, o].unsqueeze(-1)).to(BF)
    return q, back(x["K"], x["ks"]), back(x["V"], x["vs"])


def _plain_window(x):
    case = x["case"]
    W, F, S, B = case["window"], case["first"], x["most"], case["batch"]
    kv, bs, d = x["K"].shape[1:]
    Hq = x["q"].shape[1]
    lens, cu = x["lens"].long(), x["cu"].long()
    new = cu[1:] - cu[:-1]
    # the keys that a sequence's queries may see: the first ones, and from the
    # window of its first query on (as many as the longest sequence needs)
    first = torch.arange(F, device=DEV).expand(B, F)
    start = (lens - new - W + 1).clamp(min=F)
    pos = torch.cat([first, start[:, None] + torch.arange(W + S - 1, device=DEV)], 1)
    there = pos < lens[:, None]
    at = torch.where(there, pos, torch.zeros_like(pos))
    blk, off = torch.gather(x["table"].long(), 1, at // bs).clamp(min=0), at % bs

    def rows(pool, scale):
        r = pool.view(torch.uint8)[blk, :, off].view(pool.dtype) if scale is not None else pool[blk, :, off]
        r = r.float() if scale is None else r.float() * scale[blk, :, off].unsqueeze(-1)
        return r.permute(0, 2, 1, 3)  # [B, kv, keys, d]

    K, V = rows(x["K"], x["ks"]), rows(x["V"], x["vs"])
    # query tokens padded to the longest sequence
    tok = torch.arange(S, device=DEV)
    live = tok < new[:, None]
    index = torch.where(live, cu[:-1, None] + tok, torch.zeros_like(cu[:-1, None] + tok))
    q = (x["q"].float() * d ** -0.5)[index].view(B, S, kv, Hq // kv, d).permute(0, 2, 1, 3, 4).reshape(B, kv, -1, d)
    s = torch.matmul(q, K.transpose(2, 3)).view(B, kv, S, Hq // kv, -1)
    p = (lens - new)[:, None, None] + tok[:, None]
    seen = there[:, None] & (pos[:, None] <= p) & ((pos[:, None] < F) | (pos[:, None] > p - W))
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    sink = None
    if x["sink"] is not None:
        sink = x["sink"].view(1, kv, 1, Hq // kv, 1)
        m = torch.maximum(m, sink)
    # (a padded query may see nothing)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(s - m)
    den = e.sum(-1, keepdim=True)
    if sink is not None:
        den = den + torch.exp(sink - m)
    o = torch.matmul(e.view(B, kv, -1, e.shape[-1]), V).view(B, kv, S, Hq // kv, d)
    o = torch.where(den > 0, o / den, torch.zeros_like(o))
    return o.permute(0, 2, 1, 3, 4).reshape(B, S, Hq, d)[live].to(BF)


# ---------------------------------------------------------------------------
# one pass, the framework's operators
# ---------------------------------------------------------------------------
_entry = None


def _framework():
    global _entry
    if _entry is None:
        pkg = os.path.join(os.getcwd(), "vllm-neuron_amd")
        if pkg not in sys.path:
            sys.path.append(pkg)
        from vllm_neuron_amd import functional
        from vllm_neuron_amd.utils.common_types import NormType

        _entry = functional, NormType
    return _entry


def _own_pass(x):
    (F, NormType), case = _framework(), x["case"]
    if case["kind"] == "linear":
        norm = NormType.RMS_NORM if case["norm"] else NormType.NO_NORM
        code, scale = F.quant_rows(x["x"], norm_type=norm, norm_weights=x["gamma"], eps=EPS)
        return F.int8_linear(code, scale, x["w"], x["ws"], bias=x["bias"]), scale
    if case["kind"] == "rope":
        q = F.rope_kv_append(x["q"], x["k"], x["v"], x["positions"], x["inv"], x["slots"], x["K"], x["V"],
                             k_scales=x["ks"], v_scales=x["vs"], sections=x["sections"],
                             section_order=case["split"], pairs=case["pairs"], q_gamma=x["qn"], k_gamma=x["kn"],
                             qk_norm=case["norm"], eps=EPS)
        if case["cache"] == "bf16":
            return q, x["K"], x["V"]
        return (q, *F.quant_kv_read(x["K"], x["V"], x["ks"], x["vs"], x["slots"]))
    return F.window_attention(x["q"], x["K"], x["V"], x["table"], x["lens"], window=case["window"],
                              first_tokens=case["first"], cu_seqlens_q=x["cu"], max_seqlen_q=x["most"], sink=x["sink"],
                              k_scales=x["ks"], v_scales=x["vs"])


def run(state):
    if own:
        return _own_pass(state)
    return {"linear": _plain_linear, "rope": _plain_rope, "window": _plain_window}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    if case["kind"] == "linear":
        M, K, N = case["tokens"], case["k"], case["n"]
        # rows in, weights and their scales, rows out and the row scales
        return {"bytes": 2 * M * K + N * K + 4 * N + 2 * M * N + 4 * M, "flops": 2 * M * K * N}
    s = SHAPES[case["shape"]]
    kv, d, heads = s["kv"], s["d"], s["heads"]
    # bytes of one K or V row of one head: codes and their scale, or bf16
    row = d + 4 if case["cache"] in CODES else 2 * d
    if case["kind"] == "rope":
        T = case["tokens"]
        back = 2 * kv * (row + 2 * d) if case["cache"] in CODES else 0
        return {"bytes": T * ((2 * heads + 2 * kv) * 2 * d + 2 * kv * row + back + 8 * case["axes"] + 8),
                "flops": T * (6 * (heads + kv) * (case["rot"] // 2) + (4 * (heads + kv) * d if case["norm"] else 0))}
    new, lens = _window_lens(case)
    W, F = case["window"], case["first"]
    keys = pairs = 0
    for m, n in zip(new, lens):
        lo = max(0, n - m - W + 1)  # first key of the first query's window
        keys += n - lo + min(F, lo)
        for p in range(n - m, n):
            low = max(0, p - W + 1)
            pairs += p + 1 - low + min(F, low)
    return {"bytes": 2 * keys * kv * row + 2 * 2 * sum(new) * heads * d, "flops": 4 * pairs * heads * d}


# ---------------------------------------------------------------------------
# float64 statement
# ---------------------------------------------------------------------------
def _exact_codes(r, cache):
    """Values and float32 scales of the float64 rows r, as the quantisation is
    defined: the nearest code of r Q / max|r|."""
    top = CODES[cache][1]
    amax = r.abs().amax(-1, keepdim=True)
    y = torch.where(amax > 0, r * top / amax, torch.zeros_like(r))
    if cache == "int8":
        return torch.round(y), amax / top
    # the nearest multiple of the step of y's binade (ties to even): 3 bits
    # after the leading one, 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, amax / top


def _exact_norm(r, gamma):
    return r / torch.sqrt(r.square().mean(-1, keepdim=True) + EPS) * gamma.to(F64)


def _exact_linear(case, x):
    r = x["x"].to(F64)
    if case["norm"]:
        r = _exact_norm(r, x["gamma"])
    code, scale = _exact_codes(r, "int8")
    y = code @ x["w"].to(F64).t().contiguous()
    y = y * scale * x["ws"].to(F64)
    return y if x["bias"] is None else y + x["bias"].to(F64), scale[:, 0]


def _exact_rope(case, x):
    rot, axis = case["rot"], _axis_of_pair(case)

    def rotate(r):
        out = r.clone()
        for i in range(rot // 2):
            angle = x["positions"][axis[i]].to(F64) * x["inv"][i].to(F64)
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            a, b = (i, i + rot // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
            out[..., a] = r[..., a] * c - r[..., b] * s
            out[..., b] = r[..., b] * c + r[..., a] * s
        return out

    q, k, v = (x[n].to(F64) for n in "qkv")
    if case["norm"]:
        q, k = _exact_norm(q, x["qn"]), _exact_norm(k, x["kn"])
    q, k = rotate(q), rotate(k)
    if case["cache"] in CODES:
        return (q, *(c * s for c, s in (_exact_codes(k, case["cache"]), _exact_codes(v, case["cache"]))))
    bs = x["K"].shape[2]
    out = [q]
    for r in (k, v):
        pool = torch.zeros(x["K"].shape, dtype=F64, device=DEV)
        pool[x["slots"] // bs, :, x["slots"] % bs] = r
        out.append(pool)
    return tuple(out)


def _exact_window(case, x):
    new, lens = _window_lens(case)
    W, F = case["window"], case["first"]
    Hq, d = x["q"].shape[1:]
    kv, bs = x["K"].shape[1:3]
    out, at = torch.zeros(x["q"].shape, dtype=F64, device=DEV), 0
    for i, (m, n) in enumerate(zip(new, lens)):
        low = max(0, n - m - W + 1)
        t = torch.tensor([j for j in range(n) if j < F or j >= low], device=DEV)
        blk = x["table"][i][torch.div(t, bs, rounding_mode="floor")].long()
        pair = []
        for pool, sc in ((x["K"], x["ks"]), (x["V"], x["vs"])):
            r = pool[blk, :, t % bs] if sc is None else pool.view(torch.uint8)[blk, :, t % bs].view(pool.dtype)
            r = r.to(F32).to(F64)
            pair.append(r if sc is None else r * sc[blk, :, t % bs].to(F64)[..., None])
        p = n - m + torch.arange(m, device=DEV)[:, None]
        hidden = (t > p) | ((t >= F) & (t <= p - W))
        for h in range(Hq):
            g = h // (Hq // kv)
            s = x["q"][at:at + m, h].to(F64) @ pair[0][:, g].t().contiguous() / math.sqrt(d)
            s = s.masked_fill(hidden, -math.inf)
            if x["sink"] is not None:
                s = torch.cat([s, x["sink"][h].to(F64).expand(m, 1)], 1)
            out[at:at + m, h] = torch.softmax(s, 1)[:, :t.numel()] @ pair[1][:, g].contiguous()
        at += m
    return out


def exact(case, seed):
    return {"linear": _exact_linear, "rope": _exact_rope, "window": _exact_window}[case["kind"]](case, _inputs(case, seed))
