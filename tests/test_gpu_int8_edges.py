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
