"""Which axis each channel pair turns by, section by section: counted from the
rotation itself, one axis at a time, against lists written out by hand."""
import pytest
import torch

from vllm_neuron_amd.functional import rope_rotate

CASES = [
    # order, sections, axes of the pairs
    ("blocks", [2, 3, 3], "00111222"),
    ("blocks", [0, 5, 0, 3], "11111333"),
    ("cycle", [4, 2, 2], "01201200"),
    ("cycle", [4, 4], "01010101"),
    ("cycle", [6, 2], "01010000"),
    # sections that hold more pairs than fall to their axis: the rest is axis 0's
    ("cycle", [2, 6], "01010101"),
    ("cycle", [1, 1, 6], "01200200"),
    ("cycle", [0, 0, 0, 8], "00030003"),
    ("cycle", [1, 2, 0, 5], "01030103"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("order,sections,axes", CASES)
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
def test_axis_of_every_pair(gpu, order, sections, axes, pairs):
    d, n = 16, len(sections)
    # token a turns a quarter on axis a alone: (1, 0) becomes (0, 1)
    pos = torch.eye(n, dtype=torch.int64, device=gpu)
    inv = torch.full((8,), torch.pi / 2, device=gpu)
    x = torch.zeros(n, 1, d, dtype=torch.bfloat16, device=gpu)
    first = slice(0, 8) if pairs == "half" else slice(0, d, 2)
    x[..., first] = 1.0
    q, k = rope_rotate(x, x, pos, inv, sections=sections, section_order=order, pairs=pairs)
    turned = (q[:, 0, first].abs() < 0.5).cpu()  # [axis, pair]
    assert "".join(str(turned[:, i].nonzero().item()) for i in range(8)) == axes
    assert torch.equal(q, k)
