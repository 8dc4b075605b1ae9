"""Layers of experts on the GPU: what a token's result depends on."""
import pytest
import torch

from test_lm_more_gpu import BF16, F32, Layer, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m, experts, top, kernel", [(40, 8, 2, "w4_experts_16x128"), (60, 4, 2, "w4_experts_32x128"), (100, 4, 2, "w4_experts_64x128"), (300, 13, 3, "w4_experts_64x128"),
                                                     (1500, 4, 2, "w4_experts_128x256")])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_rows_of_the_tiles_do_not_depend_on_others(m, experts, top, kernel, group):
    """Other tokens that choose other experts leave a token's result as it is, bit by bit, wherever its rows then lie."""
    g = gen(m + group)
    layer = Layer(g, BF16, experts, 1056, 2080, 300, top, group)
    assert layer.plan.kernel(m) == kernel
    x, s = randn(g, BF16, m, 1056), randn(g, F32, m, experts)
    first = layer.plan(x, s)
    stay = torch.rand(m, device="cuda", generator=g) < 0.3
    for expert in (0, experts - 1):
        other = torch.where(stay[:, None], s, randn(g, F32, m, experts))
        other[~stay, expert] += 4
        assert torch.equal(layer.plan(x, other)[stay], first[stay])
