"""Refusals of the int8 projection entry points on the CPU: every call fails
validation before anything reaches the device."""
import ctypes

import pytest
import torch

from vllm_neuron_amd import _native as N
from vllm_neuron_amd import ops
from vllm_neuron_amd.functional import int8_linear, qkv_proj, quant_rows
from vllm_neuron_amd.utils.common_types import NormType, QuantizationType

FAKE = 0x10000  # never dereferenced


def _rows(**over):
    a = N.QuantRowsArgs()
    a.x = a.codes = a.scales = FAKE
    a.x_stride = a.codes_stride = a.dim = 256
    a.rows = 4
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _linear(**over):
    a = N.Int8LinearArgs()
    for f in ("x", "w", "x_scales", "w_scales", "out"):
        setattr(a, f, FAKE)
    a.rows, a.n, a.k = 4, 64, 256
    a.x_stride = a.w_stride = 256
    a.out_stride = 64
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,err,text", [
    (dict(x=None), ValueError, "null"),
    (dict(scales=None), ValueError, "null"),
    (dict(rows=-1), ValueError, "shape"),
    (dict(dim=0), ValueError, "shape"),
    (dict(rows=1 << 31), ValueError, "2\\^31"),
    (dict(norm=2), NotImplementedError, "norm"),
    (dict(dim_actual=257), ValueError, "dim_actual"),
])
def test_quant_rows_refusals(over, err, text):
    with pytest.raises(err, match=text):
        N.check(N.lib().mia_quant_rows(ctypes.byref(_rows(**over)), None), "quant_rows")


@pytest.mark.parametrize("over,err,text", [
    (dict(w=None), ValueError, "null"),
    (dict(out=None), ValueError, "null"),
    (dict(rows=-1), ValueError, "shape"),
    (dict(k=0), ValueError, "shape"),
    (dict(k=24), NotImplementedError, "multiple of 16"),
    (dict(k=131072, x_stride=131072, w_stride=131072), NotImplementedError, "131072"),
    (dict(x=FAKE + 8), ValueError, "16-byte"),
    (dict(w=FAKE + 4), ValueError, "16-byte"),
    (dict(x_stride=264), ValueError, "16-byte"),
    (dict(w_stride=264), ValueError, "16-byte"),
    (dict(x_stride=1 << 24), ValueError, "stride"),
    (dict(w_stride=-256), ValueError, "stride"),
    (dict(rows=1 << 20, n=1 << 20), ValueError, "2\\^34"),
])
def test_int8_linear_refusals(over, err, text):
    with pytest.raises(err, match=text):
        N.check(N.lib().mia_int8_linear(ctypes.byref(_linear(**over)), None), "int8_linear")


def test_empty_calls_reach_no_device():
    N.check(N.lib().mia_quant_rows(ctypes.byref(_rows(rows=0)), None), "quant_rows")
    N.check(N.lib().mia_int8_linear(ctypes.byref(_linear(rows=0)), None), "int8_linear")
    N.check(N.lib().mia_int8_linear(ctypes.byref(_linear(n=0)), None), "int8_linear")


def test_functional_refusals():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="LAYER_NORM"):
        quant_rows(x, norm_type=NormType.LAYER_NORM)
    with pytest.raises(ValueError, match="norm_weights"):
        quant_rows(x, norm_weights=torch.ones(64))
    # a CPU tensor never falls back to a CPU path
    with pytest.raises(RuntimeError):
        quant_rows(x)
    c, s = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(RuntimeError):
        int8_linear(c, s, c, s)


def test_qkv_proj_row_quantisation_asks_for_its_layout():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    w, s = torch.zeros(128, 64, dtype=torch.int8), torch.ones(128)
    row = QuantizationType.ROW
    with pytest.raises(ValueError, match="int8 weights and qkv_w_scale"):
        qkv_proj(x, w.t(), quantization_type=row)
    with pytest.raises(ValueError, match="int8 weights and qkv_w_scale"):
        qkv_proj(x, w.t().to(torch.bfloat16), quantization_type=row, qkv_w_scale=s)
    with pytest.raises(ValueError, match="transposed view"):
        qkv_proj(x, w.t().contiguous(), quantization_type=row, qkv_w_scale=s)
    with pytest.raises(NotImplementedError, match="static input"):
        qkv_proj(x, w.t(), quantization_type=row, qkv_w_scale=s, qkv_in_scale=s)
    with pytest.raises(RuntimeError):
        qkv_proj(x, w.t(), quantization_type=row, qkv_w_scale=s)


def test_schemas_and_shapes_without_a_device():
    assert "mia::int8_linear" in str(torch.ops.mia.int8_linear.default._schema)
    sch = str(torch.ops.mia.int8_linear.default._schema)
    assert "!) out" in sch and "quant_rows" in ops.OPS
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 5, 64, dtype=torch.bfloat16, device="cuda")
        c, s = quant_rows(x)
        assert c.shape == (3, 5, 64) and c.dtype == torch.int8
        assert s.shape == (3, 5) and s.dtype == torch.float32
        w = torch.empty(48, 64, dtype=torch.int8, device="cuda")
        y = int8_linear(c, s, w, torch.empty(48, device="cuda"))
        assert y.shape == (3, 5, 48) and y.dtype == torch.bfloat16
