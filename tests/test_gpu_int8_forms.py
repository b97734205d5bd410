"""Every form of the int8 product at every kind of k, whatever sizes the cost model
gives it: whole last tiles and cut ones, fewer tiles than its ring has stages, as
many, more and many more; ragged rows and columns; nothing read past k counts and
nothing outside the output is written."""
import ctypes

import pytest
import torch

from vllm_neuron_amd import _native as N

BF = torch.bfloat16
FORMS = 10       # mia_int8_linear_forms(), checked below
FEW = FORMS - 1  # the form of at most 16 rows
KS = [16, 48, 64, 80, 112, 128, 144, 192, 208, 240, 256, 272, 320, 384, 400, 448, 512, 528, 576, 640, 656, 704, 768, 784, 896,
      1024, 1040, 1280, 1296, 1536, 1552, 2048, 2880, 4096, 5136]


def _choice(m, n, k):
    a = N.Int8LinearArgs()
    for f in ("x", "w", "x_scales", "w_scales", "out"):
        setattr(a, f, 0x10000)  # never dereferenced
    a.rows, a.n, a.k, a.x_stride, a.w_stride, a.out_stride = m, n, k, k, k, n
    return N.lib().mia_int8_linear_choice(ctypes.byref(a))


def test_every_form_is_taken_by_some_size():
    assert N.lib().mia_int8_linear_forms() == FORMS
    rows = (1, 4, 16, 17, 33, 64, 100, 129, 160, 200, 300, 333, 517, 560, 600, 850, 1500, 2048, 4096, 8191)
    taken = {_choice(m, n, k) for m in rows for n in (512, 2048, 4096, 5120, 6144, 8192, 10240)
             for k in (256, 1024, 2048, 2880, 4096, 8192, 14336)}
    assert taken == set(range(FORMS))
    assert all(_choice(m, 4096, 4096) != FEW for m in rows if m > 16)
    assert _choice(0, 64, 64) == _choice(64, 0, 64) == _choice(64, 64, 24) == -1


@pytest.mark.parametrize("form,rows,text", [(-1, 4, "no such form"), (FORMS, 4, "no such form"), (FEW, 17, "more rows")])
def test_refusals(form, rows, text):
    a = N.Int8LinearArgs()
    for f in ("x", "w", "x_scales", "w_scales", "out"):
        setattr(a, f, 0x10000)
    a.rows, a.n, a.k, a.x_stride, a.w_stride, a.out_stride = rows, 64, 64, 64, 64, 64
    with pytest.raises(ValueError, match=text):
        N.check(N.lib().mia_int8_linear_form(ctypes.byref(a), form, None), "int8_linear")
    # more tiles than a grid's threads hold
    a.rows, a.n, a.out_stride = 4, 1 << 27, 1 << 27
    with pytest.raises(ValueError, match="grid"):
        N.check(N.lib().mia_int8_linear_form(ctypes.byref(a), FEW, None), "int8_linear")
    assert _choice(4, 1 << 27, 64) != FEW


def _product(form, x, xs, w, ws, bias, out):
    a = N.Int8LinearArgs()
    a.x, a.x_stride, a.x_scales = x.data_ptr(), x.stride(0), xs.data_ptr()
    a.w, a.w_stride, a.w_scales = w.data_ptr(), w.stride(0), ws.data_ptr()
    a.bias, a.bias_bf16 = (0, 0) if bias is None else (bias.data_ptr(), bias.dtype == BF)
    a.out, a.out_stride = out.data_ptr(), out.stride(0)
    a.rows, a.n, a.k = x.shape[0], w.shape[0], x.shape[1]
    N.launch(lambda p, s: N.lib().mia_int8_linear_form(p, form, s), a, x.device, "int8_linear")


def _check(gpu, form, m, n, k, bias=None):
    g = torch.Generator(device=gpu).manual_seed(m + n + k)
    codes = lambda r: torch.randint(-127, 128, (r, k + 32), generator=g, device=gpu, dtype=torch.int32).to(torch.int8)[:, :k]
    x, w = codes(m), codes(n)
    xs, ws = torch.rand(m, generator=g, device=gpu) + 0.1, torch.rand(n, generator=g, device=gpu) * 0.01
    b = None if bias is None else torch.randn(n, generator=g, device=gpu).to(bias)
    room = torch.full((m + 2, n + 16), 7.0, dtype=BF, device=gpu)
    y = room[1:m + 1, 8:8 + n]
    _product(form, x, xs, w, ws, b, y)
    # (exact in float64)
    prod = x.double() @ w.double().t() * xs.double()[:, None] * ws.double()
    ref = prod if b is None else prod + b.double()
    # the sum's conversion, two products and the bias at 2^-24 each, the output's rounding
    err = (y.double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + 2.0 ** -21 * (prod.abs() + ref.abs())).all(), (m, n, k, err.max().item())
    assert (room[0] == 7).all() and (room[-1] == 7).all() and (room[:, :8] == 7).all() and (room[:, 8 + n:] == 7).all()
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("k", KS)
@pytest.mark.parametrize("form", range(FORMS))
def test_every_form_at_every_k(gpu, form, k):
    sizes = [(1, 1), (13, 531), (16, 64)] if form == FEW else [(1, 1), (300, 531), (257, 264)]
    for m, n in sizes:
        _check(gpu, form, m, n, k)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2500, 1100, 320), (2310, 3300, 336), (33, 9000, 1024), (65, 8200, 2096)])
@pytest.mark.parametrize("form", range(FORMS))
def test_many_tiles(gpu, form, m, n, k):
    """More row tiles than a group of them, more tiles than compute units."""
    _check(gpu, form, min(m, 16) if form == FEW else m, n, k, (None, torch.float32, BF)[form % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(11, 70, 272), (9, 260, 4096)])
def test_all_forms_give_the_same_bits(gpu, m, n, k):
    want = _check(gpu, 0, m, n, k)
    for form in range(1, FORMS):
        assert torch.equal(_check(gpu, form, m, n, k), want)
