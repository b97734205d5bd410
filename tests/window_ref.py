"""float64 statement of attention with a sliding window and visible first
tokens, and the error bound of the bf16 kernels (test infrastructure)."""
import torch

from span_ref import U, pool_rows


def attend(q, k, v, scale, pos, window, first, sink=None):
    """q [m, Hq, d] at positions pos [m] over k/v [n, Hkv, d] float64 ->
    (out, bound); the bound as for attention over all keys: probabilities and
    the output round at U of themselves, the rest below 2^-12 of
    sum(p |v|) / sum(p)."""
    m, Hq, d = q.shape
    n = k.shape[0]
    if n == 0 or m == 0:
        return torch.zeros(m, Hq, d, dtype=torch.float64), torch.zeros(m, Hq, d, dtype=torch.float64)
    t, p = torch.arange(n)[None], pos[:, None]
    seen = (t <= p) & ((t < first) | (t > p - window))
    kk, vv = k.repeat_interleave(Hq // k.shape[1], 1), v.repeat_interleave(Hq // v.shape[1], 1)
    # rows that no query sees hold anything at all
    used = seen.any(0)
    kk, vv = kk[used], vv[used]
    seen = seen[:, used]
    if not used.any():
        return torch.zeros(m, Hq, d, dtype=torch.float64), torch.zeros(m, Hq, d, dtype=torch.float64)
    s = torch.einsum("mhd,nhd->hmn", q.double(), kk) * scale
    s = s.masked_fill(~seen[None], -torch.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    if sink is not None:
        top = torch.maximum(top, sink.double().view(Hq, 1, 1))
    e = torch.exp(s - top)
    den = e.sum(-1, keepdim=True)
    if sink is not None:
        den = den + torch.exp(sink.double().view(Hq, 1, 1) - top)
    den = den.clamp(min=1e-300)
    o = (torch.einsum("hmn,nhd->hmd", e, vv) / den).transpose(0, 1)
    a = (torch.einsum("hmn,nhd->hmd", e, vv.abs()) / den).transpose(0, 1)
    return o, U * a + U * o.abs() + 2.0 ** -12 * a


def reference(q, K, V, table, lens, cu, scale, window, first, sink=None, ks=None, vs=None, kd=None, vd=None):
    """(out, bound) [T, Hq, d] of all sequences; rows of none are zeros."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    cap = table.shape[1] * K.shape[2]
    q = q.cpu()
    for i, n in enumerate(lens):
        n = min(max(n, 0), cap)
        m = cu[i + 1] - cu[i]
        blocks = table[i].cpu().clamp(0, K.shape[0] - 1).tolist()
        k, v = pool_rows(K, ks, blocks, n, kd), pool_rows(V, vs, blocks, n, vd)
        o, b = attend(q[cu[i]:cu[i + 1]], k, v, scale, n - m + torch.arange(m), window, first,
                      None if sink is None else sink.cpu())
        out[cu[i]:cu[i + 1]], bound[cu[i]:cu[i + 1]] = o, b
    return out, bound
