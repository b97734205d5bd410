"""int8 projections at the ends of their ranges on the GPU: normalised rows of
zeros and of values whose squares leave float32, scales of leading axes, rows far
apart, vectors of another device, sizes past 32 bits."""
import pytest
import torch

from vllm_neuron_amd import ops
from vllm_neuron_amd.functional import int8_linear, quant_rows
from vllm_neuron_amd.utils.common_types import NormType

pytestmark = pytest.mark.gpu
BF, RMS = torch.bfloat16, NormType.RMS_NORM
DIMS = [64, 70, 520, 2048, 2880, 8192, 12288]  # a wave, any width, two, a workgroup ...


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_normalised_rows_of_zeros(gpu, dim, eps):
    x = torch.randn(5, dim, generator=torch.Generator().manual_seed(dim)).to(BF)
    x[1] = x[4] = 0
    g = torch.ones(dim, device=gpu)
    zero = torch.zeros(dim, device=gpu)
    for codes, scales in (quant_rows(x.to(gpu), norm_type=RMS, norm_weights=g, eps=eps),
                          ops.quant_rows(x.to(gpu), True, eps),
                          quant_rows(x.to(gpu), norm_type=RMS, norm_weights=zero, eps=eps)):
        assert (codes[[1, 4]] == 0).all() and (scales[[1, 4]] == 0).all()
        assert not torch.isnan(scales).any()
    assert (codes == 0).all() and (scales == 0).all()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("adds", [False, True])
def test_normalised_rows_whose_squares_leave_float32(gpu, dim, eps, adds):
    """The definition in float64, whatever the row's size.  Scales as for
    ordinary rows: fp32 but for the sum; a code may be the neighbour where the
    quotient lies within 2^-20 of a border.  The powers of two keep the values at
    bf16's steps, so that sums and products with gamma round as ordinary ones do."""
    gen = torch.Generator().manual_seed(dim)
    size = torch.tensor([0, 60, 63, 64, 70, 120, -55, -60, -63, -75, -100, 0, 126])
    x = (torch.rand(len(size), dim, generator=gen) - 0.5).double() * torch.exp2(size.double())[:, None]
    x = x.to(BF)
    x[11] = 0
    x[11, dim // 2] = 2.0 ** 100  # one value alone
    gamma = torch.exp2(torch.randint(-1, 1, (dim,), generator=gen).float())
    more = {}
    if adds:
        a, b = x / 4, x.flip(1) / 4
        more, (x, base) = dict(mlp_prev=a.to(gpu), attn_prev=b.to(gpu)), ((x / 2 + a) + b, x / 2)
    else:
        base = x
    codes, scales = quant_rows(base.to(gpu), norm_type=RMS, norm_weights=gamma.to(gpu), eps=eps, **more)
    r = x.double()
    y = r / torch.sqrt(r.square().mean(-1, keepdim=True) + eps) * gamma.double()
    amax = y.abs().amax(-1, keepdim=True)
    q = y * 127.0 / amax
    assert ((codes.cpu().double() - q).abs() <= 0.5 + q.abs() * 2.0 ** -20).all()
    want = amax[:, 0] / 127.0
    assert ((scales.cpu().double() - want).abs() <= want * 2.0 ** -20).all(), scales.cpu().double() / want


def test_scales_of_leading_axes(gpu):
    x = torch.randint(-127, 128, (2, 3, 64), device=gpu, dtype=torch.int32).to(torch.int8)
    w, ws = x.view(6, 64)[:5].contiguous(), torch.ones(5, device=gpu)
    xs = torch.rand(2, 3, device=gpu)
    want = int8_linear(x.view(6, 64), xs.view(6), w, ws)
    assert torch.equal(int8_linear(x, xs, w, ws).view(6, 5), want)
    assert torch.equal(int8_linear(x[0, 0], xs[0, 0], w, ws), want[0])
    for same in (xs.view(6), xs[..., None], xs[None]):
        assert torch.equal(int8_linear(x, same, w, ws).view(6, 5), want)
    for bad in (xs.t(), xs.view(3, 2), xs.view(1, 6), xs[:1]):
        with pytest.raises(ValueError, match="x_scales"):
            int8_linear(x, bad, w, ws)


@pytest.mark.parametrize("m", [1, 3, 40])
def test_rows_far_apart(gpu, m):
    """The last token of each sequence: rows 2^24 bytes apart and more."""
    k, n = 256, 48
    g = torch.Generator().manual_seed(m)
    codes = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int32).to(torch.int8).to(gpu)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8).to(gpu)
    xs, ws = torch.rand(m, generator=g).to(gpu), torch.rand(n, generator=g).to(gpu)
    pool = torch.zeros(m, (1 << 24) // k + 1, k, dtype=torch.int8, device=gpu)
    pool[:, -1] = codes
    x = pool[:, -1]
    assert x.stride(0) > 1 << 24
    assert torch.equal(int8_linear(x, xs, w, ws), int8_linear(codes, xs, w, ws))
    if m == 1:  # one channel: the stride of its axis is never used
        one = pool[:, -1]
        assert torch.equal(int8_linear(codes, xs, one, ws[:1]), int8_linear(codes, xs, one.contiguous(), ws[:1]))


def test_vectors_of_another_device_are_refused(gpu):
    x = torch.ones(4, 64, dtype=BF, device=gpu)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        quant_rows(x, norm_type=RMS, norm_weights=torch.ones(64))


def test_sizes_past_32_bits_are_refused(gpu):
    x, one = torch.zeros(1, 16, dtype=torch.int8, device=gpu), torch.ones(1, device=gpu)
    out, many = torch.zeros(1, 1, dtype=BF, device=gpu), torch.empty(1 << 31, device=gpu)
    with pytest.raises(ValueError):
        ops.int8_linear(x.expand(1 << 31, 16), many, x, one, out=out.expand(1 << 31, 1))
    with pytest.raises(ValueError):
        ops.int8_linear(x, one, x.expand(1 << 31, 16), many, out=out.expand(1, 1 << 31))
    with pytest.raises(ValueError):
        quant_rows(torch.empty(0, 1 << 31, dtype=BF, device=gpu))
