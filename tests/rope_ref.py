"""float64 statement of the rotation by several position axes (plain torch on
the CPU, test infrastructure)."""
import torch


def axes_of(sections, rot, order):
    """Axis of each channel pair."""
    n = len(sections)
    if order == "blocks":
        return [a for a in range(n) for _ in range(sections[a])]
    return [i % n if i < sections[i % n] * n else 0 for i in range(rot // 2)]


def rms(x, gamma, eps):
    r = x.double().cpu()
    y = r / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    return y if gamma is None else y * gamma.double().cpu()


def rotate(x, positions, inv_freq, sections, order, pairs, scale=1.0):
    """x [T, H, d] -> (float64 rotated rows, sum of the magnitudes that enter
    each channel)."""
    x, pos = x.double().cpu(), positions.cpu()
    pos = pos[None] if pos.dim() == 1 else pos
    rot = 2 * inv_freq.numel()
    axis = torch.tensor(axes_of(sections or [rot // 2], rot, order))
    ang = pos.double()[axis].t() * inv_freq.double().cpu()          # [T, rot / 2]
    c, s = torch.cos(ang)[:, None] * scale, torch.sin(ang)[:, None] * scale
    i = torch.arange(rot // 2)
    a, b = (i, i + rot // 2) if pairs == "half" else (2 * i, 2 * i + 1)
    out, mag = x.clone(), x.abs()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    both = (x[..., a].abs() + x[..., b].abs()) * abs(scale)
    mag[..., a] = both
    mag[..., b] = both
    return out, mag


def fp32_error(mag):
    """Of a rotated channel before its last rounding.  A turn is reduced in 64
    bits to half a turn held to 2^-25, 2^-22.3 in radians; sine and cosine are
    off by 2 ulp of at most 1, 2^-23, and the products with the scale, the head's
    norm (fp32 sums of up to 256 squares, a root, a quotient and gamma: 2^-20 in
    all) and the rotation's own round at 2^-24 each: below 2^-19 of the
    magnitudes that enter."""
    return 2.0 ** -19 * mag
