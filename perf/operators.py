"""Performance cases of the quantised K/V cache and of attention over keys of
another length: what each case stands for, its inputs, one pass in plain torch
or through the public entry points, the work a pass cannot do without, and its
float64 statement.

Kinds
  cache   K/V rows quantised into a paged cache with one scale per token and
          head, and read back (``quant_kv_write``, ``quant_kv_read``)
  prefix  decode attention of a batch that shares a long prefix
          (``shared_prefix_attention``)
  cross   attention of ragged queries over the keys of an encoder, of another
          length (``cross_attention``)

Conventions: Q, K, V ~ N(0, 1), K with a few channels of larger values, as
projections have them; rows of a quantised cache differ in magnitude.  Physical
blocks are a random permutation, table tails are -1.  Lengths belong to the
case, every value to the seed.
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
DEV = "cuda:0"

# Head geometries of the repository's workload table and its dense cases.
SHAPES = {
    "llama3_1b": dict(heads=32, kv=8, d=64, bs=16, sink=False),
    "llama3_8b": dict(heads=32, kv=8, d=128, bs=32, sink=False),
    "gptoss": dict(heads=64, kv=8, d=64, bs=32, sink=True),
    "long_48q": dict(heads=48, kv=8, d=128, bs=64, sink=False),
    "mha_d64": dict(heads=16, kv=16, d=64, bs=16, sink=False),
    "mha_d80": dict(heads=16, kv=16, d=80, bs=16, sink=False),
}


def listed():
    return [
        # The smallest call: the new tokens of a decode step go to an int8
        # cache; launches and host time count.
        dict(name="cache_step_int8", kind="cache", shape="llama3_1b", tokens=4, cache="int8"),
        # A prefill chunk written to an FP8 cache with dynamic scales.
        dict(name="cache_chunk_fp8", kind="cache", shape="llama3_8b", tokens=2048, cache="fp8"),
        # A whole long prompt, odd length.
        dict(name="cache_prompt_int8", kind="cache", shape="llama3_8b", tokens=16383, cache="int8"),
        # A small model answering a few requests under one system prompt.
        dict(name="prefix_1b_b4", kind="prefix", shape="llama3_1b", batch=4, new=1, prefix=1001, lo=1, hi=200,
             cache="bf16"),
        # A full batch of an 8B model's layer behind a long common document.
        dict(name="prefix_8b_b64", kind="prefix", shape="llama3_8b", batch=64, new=1, prefix=8192, lo=64, hi=1024,
             cache="bf16"),
        # d = 64, group 8, sinks: many samples of one prompt.
        dict(name="prefix_gptoss_b128", kind="prefix", shape="gptoss", batch=128, new=1, prefix=4133, lo=16, hi=700,
             cache="bf16"),
        # Four drafted tokens a row are checked behind a very long prefix in
        # an int8 cache.
        dict(name="prefix_draft_int8", kind="prefix", shape="long_48q", batch=16, new=4, prefix=32768, lo=16, hi=2048,
             cache="int8"),
        # One decoder token per sequence over encoder states of ragged length,
        # as the encoder's projection leaves them.
        dict(name="cross_step_b32", kind="cross", shape="mha_d64", batch=32, new_lo=0, new_hi=0, lo=100, hi=1500,
             cache="dense"),
        # The same over image keys in a paged FP8 cache, grouped heads.
        dict(name="cross_step_fp8", kind="cross", shape="llama3_8b", batch=8, new_lo=0, new_hi=0, lo=1601, hi=6404,
             cache="fp8"),
        # Decoder prompts of ragged length over ragged encoder states.
        dict(name="cross_prompt_b8", kind="cross", shape="mha_d64", batch=8, new_lo=1, new_hi=448, lo=200, hi=1500,
             cache="dense"),
        # A head dim between the usual ones.
        dict(name="cross_prompt_d80", kind="cross", shape="mha_d80", batch=3, new_lo=300, new_hi=900, lo=900, hi=2500,
             cache="bf16"),
        # The largest: a long text prompt over the keys of an image.
        dict(name="cross_image", kind="cross", shape="llama3_8b", batch=1, new_lo=2048, new_hi=2048, lo=6404, hi=6404,
             cache="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "prefix", "prefix", "cross", "cross"])
    if kind == "cache":
        return dict(kind=kind, shape=rng.choice(sorted(SHAPES)), tokens=_log_int(rng, 1, 16384),
                    cache=rng.choice(["int8", "fp8"]))
    if kind == "prefix":
        shape = rng.choice(["llama3_1b", "llama3_8b", "gptoss", "long_48q"])
        s = SHAPES[shape]
        new = rng.choice([1, 1, 1, 2, 3, 5, 8])
        batch = max(1, _log_int(rng, 1, 128) // new)
        # at most a quarter of the largest case's operations
        most = int(5.0e10 / (4.0 * batch * new * s["heads"] * s["d"]))
        hi = _log_int(rng, 8, 2048)
        return dict(kind=kind, shape=shape, batch=batch, new=new, prefix=_log_int(rng, 100, min(32768, max(200, most))),
                    lo=max(1, hi // 16), hi=hi, cache=rng.choice(["bf16", "bf16", "int8", "fp8"]))
    shape = rng.choice(["llama3_1b", "llama3_8b", "mha_d64", "mha_d80"])
    cache = rng.choice(["dense", "bf16", "int8", "fp8"])
    hi = _log_int(rng, 64, 6404)
    if rng.random() < 0.5:
        return dict(kind=kind, shape=shape, batch=_log_int(rng, 1, 64), new_lo=0, new_hi=0, lo=hi // 8, hi=hi,
                    cache=cache)
    batch = rng.randint(1, 8)
    most = int(1.0e11 / (4.0 * batch * hi * SHAPES[shape]["heads"] * SHAPES[shape]["d"]))
    new = _log_int(rng, 2, max(4, min(2048, most)))
    return dict(kind=kind, shape=shape, batch=batch, new_lo=1, new_hi=new, lo=hi // 4, hi=hi, cache=cache)


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


def _key_lens(case):
    return _lens(case["batch"], case["lo"], case["hi"])


def _query_lens(case):
    """Query tokens per sequence of a cross case (None: one each)."""
    return _lens(case["batch"], case["new_lo"], case["new_hi"], 1) if case["new_hi"] else None


class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape, dtype=BF):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=self.g, device=DEV) * (hi - lo) + lo

    def keys(self, *shape):
        """Keys [..., d]: one channel in sixteen four times as large."""
        x = self.normal(*shape)
        x[..., 5::16] *= 4.0
        return x

    def tables(self, lens, bs, first):
        """-1 padded int32 tables of rows of ``lens`` tokens over a random
        permutation of the blocks from ``first`` on, and the block count."""
        per = [(n + bs - 1) // bs for n in lens]
        perm = torch.randperm(max(1, sum(per)), generator=self.g, device=DEV).to(torch.int32) + first
        t = torch.full((len(lens), max(1, max(per))), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(per):
            t[i, :n] = perm[at:at + n]
            at += n
        return t, first + sum(per)


CODES = {"int8": (I8, 127.0), "fp8": (FP8, 448.0)}


def _codes(x, cache):
    """Codes and scales of the rows x [..., d] (in chunks of the first axis).
    x and the row's maximum are finite and far from the ends of the exponent
    range, so that both products and the quotient are exact or correctly
    rounded in 32 bits, and no quotient of such rows falls near a border
    between two codes without lying on it."""
    dtype, top = CODES[cache]
    code = torch.empty(x.shape, dtype=dtype, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=F32, device=x.device)
    step = max(1, (1 << 26) // max(1, x[0].numel()))
    for i in range(0, x.shape[0], step):
        c = x[i:i + step].float()
        amax = c.abs().amax(-1, keepdim=True)
        scale[i:i + step] = (amax / top).squeeze(-1)
        y = torch.where(amax > 0, c * top / amax, torch.zeros_like(c))
        code[i:i + step] = y.round().to(I8) if dtype is I8 else y.to(FP8)
    return code, scale


def _pool(gen, case, shape):
    """K and V of a cache of the case's kind and their scales (None: bf16)."""
    k, v = gen.keys(*shape), gen.normal(*shape)
    if case["cache"] not in CODES:
        return dict(K=k, V=v, ks=None, vs=None)
    # rows of unlike magnitude: what one scale per row is for
    k.mul_(gen.uniform(*shape[:-1], 1, lo=0.5, hi=2.0).to(BF))
    v.mul_(gen.uniform(*shape[:-1], 1, lo=0.25, hi=4.0).to(BF))
    (kc, ks), (vc, vs) = _codes(k, case["cache"]), _codes(v, case["cache"])
    return dict(K=kc, V=vc, ks=ks, vs=vs)


def _cache_inputs(case, s, gen):
    T, kv, d, bs = case["tokens"], s["kv"], s["d"], s["bs"]
    t, nb = gen.tables([T], bs, 1)
    p = torch.arange(T, device=DEV)
    dtype = CODES[case["cache"]][0]
    # K and V are column ranges of one projection output
    kv_rows = gen.normal(T, 2 * kv, d)
    kv_rows[:, :kv, 5::16] *= 4.0
    kv_rows.mul_(gen.uniform(T, 2 * kv, 1, lo=0.25, hi=4.0).to(BF))
    zeros = lambda *shape, dt: torch.zeros(shape, dtype=dt, device=DEV)
    return dict(k=kv_rows[:, :kv], v=kv_rows[:, kv:], slots=t[0, p // bs].long() * bs + p % bs,
                K=zeros(nb, kv, bs, d, dt=dtype), V=zeros(nb, kv, bs, d, dt=dtype), ks=zeros(nb, kv, bs, dt=F32),
                vs=zeros(nb, kv, bs, dt=F32))


def _prefix_inputs(case, s, gen):
    bs, lens = s["bs"], _key_lens(case)
    tp, nb = gen.tables([case["prefix"]], bs, 1)
    # a row holds its new tokens at least
    t, nb = gen.tables([max(n, case["new"]) for n in lens], bs, nb)
    x = _pool(gen, case, (nb, s["kv"], bs, s["d"]))
    x.update(q=gen.normal(case["batch"], case["new"], s["heads"], s["d"]), prefix_table=tp[0],
             prefix_len=torch.tensor([case["prefix"]], dtype=torch.int32, device=DEV), table=t,
             lens=torch.tensor([max(n, case["new"]) for n in lens], dtype=torch.int32, device=DEV),
             sink=gen.uniform(s["heads"], lo=-1.0, hi=1.0) if s["sink"] else None)
    return x


def _cross_inputs(case, s, gen):
    lens, new = _key_lens(case), _query_lens(case)
    if case["cache"] == "dense":
        # [B, L, kv, d] as the projection leaves them, seen head first
        k = gen.keys(case["batch"], max(1, max(lens)), s["kv"], s["d"]).transpose(1, 2)
        v = gen.normal(case["batch"], max(1, max(lens)), s["kv"], s["d"]).transpose(1, 2)
        x = dict(K=k, V=v, ks=None, vs=None, table=None)
    else:
        t, nb = gen.tables(lens, s["bs"], 1)
        x = _pool(gen, case, (nb, s["kv"], s["bs"], s["d"]))
        x.update(table=t)
    rows = case["batch"] if new is None else sum(new)
    cu = None
    if new is not None:
        cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    x.update(q=gen.normal(rows, s["heads"], s["d"]), cu=cu, most=0 if new is None else max(new),
             lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    return x


def _inputs(case, seed):
    make = {"cache": _cache_inputs, "prefix": _prefix_inputs, "cross": _cross_inputs}[case["kind"]]
    return make(case, SHAPES[case["shape"]], _Gen(seed))


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    # host-side lengths: the plain form's loops run over them
    if case["kind"] == "prefix":
        x["host_lens"] = [max(n, case["new"]) for n in _key_lens(case)]
    elif case["kind"] == "cross":
        x["host_lens"] = _key_lens(case)
        x["host_new"] = _query_lens(case) or [1] * case["batch"]
    return x


# ---------------------------------------------------------------------------
# one pass, plain form
# ---------------------------------------------------------------------------
def _gathered(pool, scale, table, n):
    """fp32 rows [kv, n, d] of the first n tokens of a block table row."""
    nblk = (n + pool.shape[2] - 1) // pool.shape[2]
    ids = table[:nblk].long()
    x = pool[ids].float()
    if scale is not None:
        x = x * scale[ids].unsqueeze(-1)
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def _softmax_parts(s):
    """Row maxima, exponentials and their sums of scores s [..., keys]."""
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m)
    return m, e, e.sum(-1, keepdim=True)


def _plain_cache(x):
    for rows, pool, scales in ((x["k"], x["K"], x["ks"]), (x["v"], x["V"], x["vs"])):
        code, scale = _codes(rows, x["case"]["cache"])
        bs = pool.shape[2]
        b, o = x["slots"] // bs, x["slots"] % bs
        # the pool as bytes: indexed stores of 8-bit floats are not there for every type
        pool.view(torch.uint8)[b, :, o] = code.view(torch.uint8)
        scales[b, :, o] = scale
    out = []
    for pool, scales in ((x["K"], x["ks"]), (x["V"], x["vs"])):
        bs = pool.shape[2]
        b, o = x["slots"] // bs, x["slots"] % bs
        code = pool.view(torch.uint8)[b, :, o].view(pool.dtype)
        out.append((code.float() * scales[b, :, o].unsqueeze(-1)).to(BF))
    return out[0], out[1], x["ks"], x["vs"]


def _plain_prefix(x):
    B, S, Hq, d = x["q"].shape
    kv = x["K"].shape[1]
    G = Hq // kv
    q = (x["q"].float() * d ** -0.5).view(B, S, kv, G, d)
    # the prefix once, for all rows
    kp = _gathered(x["K"], x["ks"], x["prefix_table"], x["case"]["prefix"])
    vp = _gathered(x["V"], x["vs"], x["prefix_table"], x["case"]["prefix"])
    rows = q.permute(2, 0, 1, 3, 4).reshape(kv, B * S * G, d)
    m, e, l = _softmax_parts(torch.matmul(rows, kp.transpose(1, 2)))
    back = lambda t: t.view(kv, B, S, G, -1).permute(1, 2, 0, 3, 4)
    mp, lp, op = back(m), back(l), back(torch.matmul(e, vp))
    out = torch.empty((B, S, Hq, d), dtype=F32, device=DEV)
    for b, n in enumerate(x["host_lens"]):
        k = _gathered(x["K"], x["ks"], x["table"][b], n)
        v = _gathered(x["V"], x["vs"], x["table"][b], n)
        s = torch.matmul(q[b].permute(1, 0, 2, 3).reshape(kv, S * G, d), k.transpose(1, 2)).view(kv, S, G, n)
        seen = torch.arange(n, device=DEV) <= (n - S + torch.arange(S, device=DEV)).view(S, 1, 1)
        m, e, l = _softmax_parts(s.masked_fill(~seen, -math.inf))
        o = torch.matmul(e.view(kv, S * G, n), v).view(kv, S, G, d)
        m, l, o = (t.transpose(0, 1) for t in (m, l, o))
        top = torch.maximum(m, mp[b])
        if x["sink"] is not None:
            top = torch.maximum(top, x["sink"].view(1, kv, G, 1))
        a, c = torch.exp(m - top), torch.exp(mp[b] - top)
        den = l * a + lp[b] * c
        if x["sink"] is not None:
            den = den + torch.exp(x["sink"].view(1, kv, G, 1) - top)
        out[b] = ((o * a + op[b] * c) / den).reshape(S, Hq, d)
    return out.to(BF)


def _plain_cross(x):
    T, Hq, d = x["q"].shape
    kv = x["K"].shape[1]
    G = Hq // kv
    out = torch.empty((T, Hq, d), dtype=F32, device=DEV)
    at = 0
    for b, (n, m) in enumerate(zip(x["host_lens"], x["host_new"])):
        if x["table"] is None:
            k, v = x["K"][b, :, :n].float(), x["V"][b, :, :n].float()
        else:
            k = _gathered(x["K"], x["ks"], x["table"][b], n)
            v = _gathered(x["V"], x["vs"], x["table"][b], n)
        q = (x["q"][at:at + m].float() * d ** -0.5).view(m, kv, G, d).transpose(0, 1).reshape(kv, m * G, d)
        _, e, l = _softmax_parts(torch.matmul(q, k.transpose(1, 2)))
        o = torch.matmul(e, v) / l
        # no key at all: zeros
        out[at:at + m] = o.view(kv, m, G, d).transpose(0, 1).reshape(m, Hq, d) if n else 0.0
        at += m
    return out.to(BF)


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

        _entry = functional
    return _entry


def _own_pass(x):
    F, kind = _framework(), x["case"]["kind"]
    if kind == "cache":
        F.quant_kv_write(x["k"], x["v"], x["slots"], x["K"], x["V"], x["ks"], x["vs"])
        k, v = F.quant_kv_read(x["K"], x["V"], x["ks"], x["vs"], x["slots"])
        return k, v, x["ks"], x["vs"]
    if kind == "prefix":
        return F.shared_prefix_attention(x["q"], x["K"], x["V"], x["prefix_table"], x["prefix_len"], x["table"],
                                         x["lens"], sink=x["sink"], k_scales=x["ks"], v_scales=x["vs"])
    return F.cross_attention(x["q"], x["K"], x["V"], x["lens"], block_table=x["table"], cu_seqlens_q=x["cu"],
                             max_seqlen_q=x["most"] or None, k_scales=x["ks"], v_scales=x["vs"])


def run(state):
    if own:
        return _own_pass(state)
    return {"cache": _plain_cache, "prefix": _plain_prefix, "cross": _plain_cross}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    s = SHAPES[case["shape"]]
    kv, d, heads = s["kv"], s["d"], s["heads"]
    # bytes of one K or V row of one head: codes and their scale, or bf16
    row = d + 4 if case["cache"] in CODES else 2 * d
    if case["kind"] == "cache":
        rows = 2 * case["tokens"] * kv
        # written: bf16 in, codes and scale out; read back: the reverse
        return {"bytes": rows * 2 * (2 * d + row) + 2 * 8 * case["tokens"], "flops": rows * d * 6}
    if case["kind"] == "prefix":
        P, S, G = case["prefix"], case["new"], heads // kv
        lens = [max(n, S) for n in _key_lens(case)]
        keys = P + sum(lens)
        seen = sum(S * (P + n) - S * (S - 1) // 2 for n in lens)
        return {"bytes": 2 * keys * kv * row + 2 * 2 * case["batch"] * S * heads * d, "flops": 4 * seen * heads * d}
    lens, new = _key_lens(case), _query_lens(case) or [1] * case["batch"]
    pairs = sum(n * m for n, m in zip(lens, new))
    return {"bytes": 2 * sum(lens) * kv * row + 2 * 2 * sum(new) * heads * d, "flops": 4 * pairs * heads * d}


# ---------------------------------------------------------------------------
# float64 statement
# ---------------------------------------------------------------------------
def _exact_rows(pool, scale, n, block):
    """float64 [n, kv, d]: token t of the sequence is pool row
    (block(t // bs), :, t % bs)."""
    bs = pool.shape[2]
    t = torch.arange(n, device=DEV)
    b = block(torch.div(t, bs, rounding_mode="floor"))
    flat = pool.view(torch.uint8)[b, :, t % bs].view(pool.dtype) if scale is not None else pool[b, :, t % bs]
    x = flat.to(F32).to(F64)
    return x if scale is None else x * scale[b, :, t % bs].to(F64)[..., None]


def _exact_attend(q, k, v, seen, sink):
    """softmax(q k^T / sqrt(d)) v of queries [m, heads, d] over [n, kv, d],
    one kv head and query token block at a time; seen [m, n] or None."""
    m, heads, d = q.shape
    G = heads // k.shape[1]
    out = torch.zeros((m, heads, d), dtype=F64, device=DEV)
    for h in range(heads):
        kh, vh = k[:, h // G].contiguous(), v[:, h // G].contiguous()
        s = q[:, h].to(F64) @ kh.t().contiguous() / math.sqrt(d)
        if seen is not None:
            s = s.masked_fill(~seen, -math.inf)
        if sink is not None:
            s = torch.cat([s, sink[h].to(F64).expand(m, 1)], 1)
        if s.shape[1]:
            p = torch.softmax(s, 1)
            out[:, h] = p[:, :k.shape[0]] @ vh
    return out


def exact(case, seed):
    x, s = _inputs(case, seed), SHAPES[case["shape"]]
    if case["kind"] == "cache":
        top = CODES[case["cache"]][1]
        outs, scales = [], []
        for rows in (x["k"], x["v"]):
            r = rows.to(F64)
            amax = r.abs().amax(-1, keepdim=True)
            scale = (amax.to(F32) / top).to(F64)
            y = torch.where(amax > 0, r * top / amax, torch.zeros_like(r))
            if case["cache"] == "int8":
                code = torch.round(y)
            else:
                # nearest multiple of the step of y's binade (ties to even):
                # 3 bits after the leading one, 2^-9 below 2^-6
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                code = torch.round(y / step) * step
            outs.append(code * scale)
            pool = torch.zeros(x["ks"].shape, dtype=F64, device=DEV)
            bs = s["bs"]
            pool[x["slots"] // bs, :, x["slots"] % bs] = scale[..., 0]
            scales.append(pool)
        return outs[0], outs[1], scales[0], scales[1]
    if case["kind"] == "prefix":
        B, S, Hq, d = x["q"].shape
        P = case["prefix"]
        out = torch.empty((B, S, Hq, d), dtype=F64, device=DEV)
        if 4.0 * B * S * Hq * d * P > 2.0e12:
            return None
        kp = _exact_rows(x["K"], x["ks"], P, lambda j: x["prefix_table"][j].long())
        vp = _exact_rows(x["V"], x["vs"], P, lambda j: x["prefix_table"][j].long())
        for b, n in enumerate(x["lens"].tolist()):
            own_block = lambda j: x["table"][b][j].long()
            k = torch.cat([kp, _exact_rows(x["K"], x["ks"], n, own_block)])
            v = torch.cat([vp, _exact_rows(x["V"], x["vs"], n, own_block)])
            at = torch.arange(P + n, device=DEV)
            seen = at[None, :] < (P + n - S + 1 + torch.arange(S, device=DEV))[:, None]
            out[b] = _exact_attend(x["q"][b], k, v, seen, x["sink"])
        return out
    out, at = [], 0
    new = _query_lens(case) or [1] * case["batch"]
    for b, (n, m) in enumerate(zip(x["lens"].tolist(), new)):
        block = (lambda j: torch.full_like(j, b)) if x["table"] is None else (lambda j: x["table"][b][j].long())
        k, v = _exact_rows(x["K"], x["ks"], n, block), _exact_rows(x["V"], x["vs"], n, block)
        out.append(_exact_attend(x["q"][at:at + m], k, v, None, None))
        at += m
    return torch.cat(out)
