"""int8 projections on the GPU: codes bit for bit and scales against the float64
definition, products against exact integer sums; norms, residual adds, strides,
special values, ``qkv_proj`` with row-wise weights, streams and graphs."""
import math

import pytest
import torch

from span_ref import quantise
from vllm_neuron_amd import ops
from vllm_neuron_amd.functional import int8_linear, qkv_proj, quant_rows
from vllm_neuron_amd.utils.common_types import NormType, QuantizationType

pytestmark = pytest.mark.gpu
RMS = NormType.RMS_NORM


def _x(rows, dim, seed, spread=8):
    g = torch.Generator().manual_seed(seed)
    s = torch.exp2(torch.randint(-spread, spread + 1, (rows, 1), generator=g).float())
    return (torch.randn(rows, dim, generator=g) * s).to(torch.bfloat16)


def _w(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8),
            torch.rand(n, generator=g) * 0.02 + 1e-4)


def _norm64(x, gamma, eps, n=None):
    r = x.double()
    y = r / torch.sqrt(r.square().sum(-1, keepdim=True) / (n or r.shape[-1]) + eps)
    return y if gamma is None else y * gamma.double()


def _check_codes(codes, scales, y):
    """Codes of fp32 rows y (float64 here): the nearest integer of the quotient,
    or its neighbour where the quotient lies within 2^-20 of a border: products
    with gamma, the quotient and its remainder round at 2^-24 each.  The scale
    is off by the norm's fp32 sums (2^-20 at most at these widths)."""
    amax = y.abs().amax(-1, keepdim=True)
    q = torch.where(amax > 0, y * 127.0 / amax, torch.zeros_like(y))
    got = codes.cpu().double()
    assert ((got - q).abs() <= 0.5 + q.abs() * 2.0 ** -20).all()
    want = amax[:, 0] / 127.0
    assert ((scales.cpu().double() - want).abs() <= want * 2.0 ** -20).all()


def _check_product(y, codes, xs, w, ws, bias=None):
    """The integer sum is exact; its conversion, the products with the scales
    and the bias round at 2^-24 of their values, the result at 2^-8 of itself."""
    acc = codes.cpu().double() @ w.cpu().double().t()
    prod = acc * xs.cpu().double()[:, None] * ws.cpu().double()
    ref = prod if bias is None else prod + bias.cpu().double()
    bound = 2.0 ** -8 * ref.abs() + 2.0 ** -21 * (prod.abs() + ref.abs()) + 1e-38
    err = (y.cpu().double() - ref).abs()
    assert not torch.isnan(y).any()
    assert (err <= bound).all(), (err - bound).max().item()


@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (2, 8), (5, 64), (4, 512), (7, 520), (9, 1024), (2, 1030),
                                      (3, 2048), (2, 2880), (5, 4096), (3, 8192), (2, 8200), (2, 16384),
                                      (1, 16400), (517, 96)])
def test_codes_and_scales_bit_for_bit(gpu, rows, dim):
    x = _x(rows, dim, rows + dim)
    if rows > 1:
        x[1] = 0
    codes, scales = quant_rows(x.to(gpu))
    want, want_s = quantise(x, torch.int8)
    assert torch.equal(codes.cpu().double(), want)
    assert torch.equal(scales.cpu().double(), want_s)


@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 7), (4, 512), (3, 1000), (2, 2880), (5, 4096), (2, 8192), (2, 12288),
                                      (1, 20000)])
@pytest.mark.parametrize("weights", [None, torch.float32, torch.bfloat16, torch.float16])
def test_normalised_rows(gpu, rows, dim, weights):
    x = _x(rows, dim, 3)
    g = None if weights is None else (1.0 + 0.2 * torch.randn(dim, generator=torch.Generator().manual_seed(4))).to(weights)
    kind = RMS if weights is not None else NormType.RMS_NORM_SKIP_GAMMA
    codes, scales = quant_rows(x.to(gpu), norm_type=kind, norm_weights=None if g is None else g.to(gpu), eps=1e-5)
    _check_codes(codes, scales, _norm64(x, g, 1e-5))


@pytest.mark.parametrize("dim", [64, 70, 4096])
def test_residual_adds_round_as_bf16_additions(gpu, dim):
    a, b, c = (_x(5, dim, s, 2) for s in (1, 2, 3))
    codes, scales = quant_rows(a.to(gpu), mlp_prev=b.to(gpu), attn_prev=c.to(gpu))
    want, want_s = quantise((a + b) + c, torch.int8)
    assert torch.equal(codes.cpu().double(), want) and torch.equal(scales.cpu().double(), want_s)
    codes, scales = quant_rows(a.to(gpu), attn_prev=c.to(gpu), norm_type=RMS, eps=1e-6)
    _check_codes(codes, scales, _norm64(a + c, None, 1e-6))
    # the mean over the channels that are there
    x = _x(4, dim, 6)
    x[:, dim // 2:] = 0
    codes, scales = quant_rows(x.to(gpu), norm_type=RMS, eps=1e-6, hidden_actual=dim // 2)
    _check_codes(codes, scales, _norm64(x, None, 1e-6, dim // 2))


def test_rows_of_special_values(gpu):
    x = _x(8, 256, 5)
    x[1, 3], x[2, 200], x[3, 0] = math.inf, -math.inf, math.nan
    x[4], x[5] = 0, torch.finfo(torch.bfloat16).max
    x[6] = 2.0 ** -133  # below the least normal number
    codes, scales = quant_rows(x.to(gpu))
    want, want_s = quantise(x, torch.int8)
    assert torch.equal(codes.cpu().double(), want)
    assert torch.equal(torch.isnan(scales.cpu()), torch.isnan(want_s))
    ok = ~torch.isnan(want_s)
    assert torch.equal(scales.cpu().double()[ok], want_s[ok])
    # such a row gives NaN and touches no other
    w, ws = _w(48, 256, 6)
    y = int8_linear(codes, scales, w.to(gpu), ws.to(gpu))
    assert torch.isnan(y[1:4]).all() and not torch.isnan(y[0]).any() and not torch.isnan(y[4:]).any()
    assert (y[4] == 0).all()


def test_rows_of_any_stride(gpu):
    wide = _x(6, 512, 7).to(gpu)
    for x in (wide[:, 64:192], wide[::2], wide[:, 3:100], wide.t()[:96], wide.view(2, 3, 512)):
        codes, scales = quant_rows(x)
        c2, s2 = quant_rows(x.contiguous())
        assert codes.shape == x.shape and scales.shape == x.shape[:-1]
        assert torch.equal(codes, c2) and torch.equal(scales, s2)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 200, 256, 300])
@pytest.mark.parametrize("n,k", [(1, 16), (7, 48), (16, 64), (33, 128), (100, 144), (256, 512), (270, 1040),
                                 (515, 2880)])
def test_products(gpu, m, n, k):
    x, (w, ws) = _x(m, k, m + n), _w(n, k, k)
    codes, xs = quant_rows(x.to(gpu))
    y = int8_linear(codes, xs, w.to(gpu), ws.to(gpu))
    _check_product(y, codes, xs, w, ws)


@pytest.mark.parametrize("m,n,k", [(4, 2048, 2048), (64, 6144, 4096), (517, 5120, 2880), (1500, 4100, 1024),
                                   (2048, 6144, 528), (3000, 10240, 272)])
def test_products_of_layer_sizes(gpu, m, n, k):
    x, (w, ws) = _x(m, k, 1, 2), _w(n, k, 2)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3))
    for b in (None, bias, bias.to(torch.bfloat16), bias.to(torch.float16)):
        codes, xs = quant_rows(x.to(gpu))
        y = int8_linear(codes, xs, w.to(gpu), ws.to(gpu), bias=None if b is None else b.to(gpu))
        # exact in float32 pieces: |sum| < 2^24 over 1024 channels
        acc = torch.zeros(m, n, dtype=torch.float64, device=gpu)
        for i in range(0, k, 1024):
            acc += (codes[:, i:i + 1024].float() @ w.to(gpu)[:, i:i + 1024].float().t()).double()
        prod = acc * xs.double()[:, None] * ws.to(gpu).double()
        ref = prod if b is None else prod + b.to(gpu).double()
        err = (y.double() - ref).abs()
        assert (err <= 2.0 ** -8 * ref.abs() + 2.0 ** -21 * (prod.abs() + ref.abs())).all()


@pytest.mark.parametrize("m", [3, 100])
def test_largest_sums(gpu, m):
    """Every code at an end of its range, k at the limit."""
    k = 131056
    x = torch.full((m, k), 127, dtype=torch.int8, device=gpu)
    w = torch.full((20, k), 127, dtype=torch.int8, device=gpu)
    w[1] = -127
    one = torch.ones(m, device=gpu)
    y = int8_linear(x, one, w, torch.ones(20, device=gpu))
    want = torch.tensor([127.0 * 127 * k]).to(torch.bfloat16).item()
    assert (y[:, 0] == want).all() and (y[:, 1] == -want).all()
    # (-128 is a code that a weight may have)
    y = int8_linear(torch.full_like(x, -128), one, torch.full_like(w, 127), torch.ones(20, device=gpu))
    assert (y == torch.tensor([-128.0 * 127 * k]).to(torch.bfloat16).item()).all()
    y = int8_linear(torch.full_like(x, -128), one, torch.full_like(w, -128), torch.ones(20, device=gpu))
    assert (y == torch.tensor([128.0 * 128 * k]).to(torch.bfloat16).item()).all()


@pytest.mark.parametrize("m", [5, 90])
def test_strided_operands_and_outputs(gpu, m):
    k, n = 192, 130
    big = torch.randint(-127, 128, (m, 512), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).to(torch.int8)
    x = big.to(gpu)[:, 32:32 + k]
    w, ws = _w(n, 640, 2)
    wv = w.to(gpu)[:, 256:256 + k]
    xs = torch.rand(m, generator=torch.Generator().manual_seed(2)).to(gpu)
    out = torch.full((m, 200), 7.0, dtype=torch.bfloat16, device=gpu)
    y = int8_linear(x, xs, wv, ws.to(gpu), out=out[:, 40:40 + n])
    assert y.data_ptr() == out[:, 40:].data_ptr()
    _check_product(y, x, xs, wv, ws)
    assert (out[:, :40] == 7).all() and (out[:, 40 + n:] == 7).all()
    # leading axes
    x3 = x.contiguous()[:m // 5 * 5].view(5, -1, k)
    y3 = int8_linear(x3, xs[:m // 5 * 5].view(5, -1), wv, ws.to(gpu))
    assert torch.equal(y3.view(-1, n), y[:m // 5 * 5])
    assert int8_linear(x[:0], xs[:0], wv, ws.to(gpu)).shape == (0, n)
    assert int8_linear(x, xs, wv[:0], ws[:0].to(gpu)).shape == (m, 0)


def test_refusals_on_the_device(gpu):
    x, (w, ws) = torch.zeros(4, 64, dtype=torch.int8, device=gpu), _w(32, 64, 1)
    w, ws, xs = w.to(gpu), ws.to(gpu), torch.ones(4, device=gpu)
    for bad, err in [((x.float(), xs, w, ws), ValueError), ((x, xs[:3], w, ws), ValueError),
                     ((x, xs.double(), w, ws), ValueError), ((x, xs, w[:, :48], ws), ValueError),
                     ((x, xs, w, ws[:5]), ValueError), ((x, xs, w.t()[:32, :].t(), ws), ValueError),
                     ((x[:, :40], xs, w[:, :40], ws), NotImplementedError),
                     ((x[:, 8:56], xs, w[:, 8:56], ws), ValueError),
                     ((x, xs.cpu(), w, ws), RuntimeError)]:
        with pytest.raises(err):
            int8_linear(*bad)
    with pytest.raises(ValueError, match="out must"):
        int8_linear(x, xs, w, ws, out=torch.empty(4, 31, dtype=torch.bfloat16, device=gpu))
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, xs, w, ws, bias=torch.zeros(31, device=gpu))
    h = torch.zeros(4, 64, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(NotImplementedError):
        quant_rows(h.float())
    with pytest.raises(ValueError):
        quant_rows(h, mlp_prev=h[:3])
    with pytest.raises(ValueError):
        quant_rows(h, norm_type=RMS, norm_weights=torch.ones(63, device=gpu))
    with pytest.raises(ValueError):
        quant_rows(h, norm_type=RMS, hidden_actual=65)


@pytest.mark.parametrize("norm", [NormType.NO_NORM, RMS, NormType.RMS_NORM_SKIP_GAMMA, NormType.LAYER_NORM])
@pytest.mark.parametrize("T", [3, 130])
def test_qkv_proj_with_row_quantised_weights(gpu, norm, T):
    """``qkv_proj`` computes what the two functions do, then its epilogue."""
    Hq, Hkv, d, H = 8, 2, 64, 512
    fused = (Hq + 2 * Hkv) * d
    x = _x(T, H, 1, 1).view(1, T, H).to(gpu)
    r1, r2 = _x(T, H, 2, 1).view(1, T, H).to(gpu), _x(T, H, 3, 1).view(1, T, H).to(gpu)
    w, ws = _w(fused, H, 4)
    w, ws = w.to(gpu), ws.to(gpu)
    gamma = (1 + 0.1 * torch.randn(1, H, device=gpu)).to(torch.bfloat16)
    bias = torch.randn(1, fused, device=gpu).to(torch.bfloat16)
    ang = torch.rand(1, T, d // 2, device=gpu) * 6.0
    cos, sin = torch.cat([ang.cos()] * 2, -1), torch.cat([ang.sin()] * 2, -1)
    kw = dict(norm_type=norm, eps=1e-6, mlp_prev=r1, attn_prev=r2, bias=bias, num_q_heads=Hq, num_kv_heads=Hkv,
              cos_cache=cos, sin_cache=sin)
    if norm in (RMS, NormType.LAYER_NORM):
        kw["norm_weights"] = gamma
    got = qkv_proj(x, w.t(), quantization_type=QuantizationType.ROW, qkv_w_scale=ws.view(1, -1), **kw)
    if norm == NormType.LAYER_NORM:
        y = ops.row_norm(x, ops.NORM_LAYER, 1e-6, gamma.view(-1), None, add0=r1, add1=r2)
        c, s = quant_rows(y)
    else:
        c, s = quant_rows(x, norm_type=norm, norm_weights=gamma if norm == RMS else None, eps=1e-6, mlp_prev=r1,
                          attn_prev=r2)
    y = int8_linear(c, s, w, ws, bias=bias.view(-1))
    _check_product(y[0], c[0], s[0], w, ws, bias.view(-1))
    heads = y.view(T, Hq + 2 * Hkv, d).clone()
    ops.qkv_epilogue(y.view(T, fused), Hq, Hkv, d, rope_mode=ops.ROPE_HALF, cos=cos[0], sin=sin[0], cos_hi_off=d // 2,
                     sin_hi_off=0, q_out=heads[:, :Hq], k_out=heads[:, Hq:Hq + Hkv], v_out=heads[:, Hq + Hkv:])
    assert torch.equal(got.view(T, -1, d), heads)


def test_calls_on_other_streams_and_in_graphs(gpu):
    m, n, k = 70, 320, 1024
    x, (w, ws) = _x(m, k, 1, 2).to(gpu), _w(n, k, 2)
    w, ws, g = w.to(gpu), ws.to(gpu), torch.ones(k, device=gpu)
    step = lambda t: int8_linear(*quant_rows(t, norm_type=RMS, norm_weights=g), w, ws)
    want = step(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = step(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(3):
        fresh = _x(m, k, 10 + i, 2).to(gpu)
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(fresh))
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    assert torch.equal(compiled(x), want)


@pytest.mark.parametrize("rows,dim", [((1 << 24) + 3, 7), ((1 << 25) + 5, 8)])
@pytest.mark.parametrize("norm", [NormType.NO_NORM, RMS])
def test_more_rows_than_a_grid_holds(gpu, rows, dim, norm):
    x = torch.randint(-1000, 1000, (rows, dim), device=gpu, dtype=torch.int16).to(torch.bfloat16)
    g = torch.ones(dim, device=gpu) if norm == RMS else None
    code, scale = quant_rows(x, norm_type=norm, norm_weights=g)
    for i in range(0, rows, 1 << 22):
        c, s = quant_rows(x[i:i + (1 << 22)], norm_type=norm, norm_weights=g)
        assert torch.equal(code[i:i + (1 << 22)], c) and torch.equal(scale[i:i + (1 << 22)], s)


def _exact_product(gpu, m, n, k):
    g = torch.Generator(device=gpu).manual_seed(m)
    x = torch.randint(-127, 128, (m, k), generator=g, device=gpu, dtype=torch.int32).to(torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device=gpu, dtype=torch.int32).to(torch.int8)
    xs = torch.rand(m, generator=g, device=gpu) + 0.1
    ws = torch.rand(n, generator=g, device=gpu) * 0.01
    y = int8_linear(x, xs, w, ws)
    acc = torch.zeros(m, n, dtype=torch.float64, device=gpu)
    for i in range(0, k, 1024):  # exact in float32: 1024 products of at most 127 * 127 are below 2^24
        acc += (x[:, i:i + 1024].float() @ w[:, i:i + 1024].float().t()).double()
    ref = acc * xs.double()[:, None] * ws.double()
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -21 * ref.abs()).all()


@pytest.mark.parametrize("m,n,k", [(1, 700, 4096), (16, 5000, 1040), (30, 9000, 272), (40, 2500, 4112), (64, 6144, 144),
                                   (100, 17000, 80), (150, 4100, 2064), (260, 3000, 3088), (600, 2050, 400),
                                   (513, 520, 8208), (1300, 5200, 656), (4100, 2570, 336), (5000, 7000, 64),
                                   (2049, 8193, 16)])
def test_products_whatever_form_is_taken(gpu, m, n, k):
    """Sizes across the forms' ranges, with ragged last tiles in every axis."""
    _exact_product(gpu, m, n, k)


@pytest.mark.parametrize("k", [16, 112, 128, 144, 240, 256, 272, 384, 400, 512, 528, 640, 656, 768, 784, 1024, 1040, 1264,
                               1280, 1296, 1536, 1552])
@pytest.mark.parametrize("m,n", [(129, 12000), (129, 4100), (70, 9000), (300, 12000), (400, 10200), (500, 10200), (5, 4100)])
def test_few_tiles_of_k(gpu, m, n, k):
    """Fewer tiles along k than a ring holds, as many, and more, whole and not."""
    _exact_product(gpu, m, n, k)
