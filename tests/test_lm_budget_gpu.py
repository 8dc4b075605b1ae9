"""The cache held to a budget on the GPU: weights where scores are not finite."""
import math

import pytest
import torch

from test_lm_more_gpu import BF16, Sequences, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new, group, dim", [(1, 1, 64), (1, 8, 128), (3, 2, 128), (3, 8, 64), (40, 2, 64), (70, 2, 128)])
@pytest.mark.parametrize("other", [math.nan, math.inf])
def test_weigh_scores_of_either_infinity(new, group, dim, other):
    """A score of NaN or +infinity makes the weights of all that its row sees NaN, those with a score of -infinity too; without one these get nothing."""
    g = gen(new + group)
    s = Sequences(g, BF16, [300], 1, dim, 16, False)
    q = randn(g, BF16, new, group, dim)
    q[..., 0] = q[..., 0].abs() + 1
    place = lambda t: (int(s.blocks[0, t // 16]), 0, t % 16, 0)  # noqa: E731
    s.cache.k[place(20)] = s.cache.k[place(150)] = -math.inf  # scores of -infinity
    before = s.of(s.weights, 0)[0].clone()
    weigh = lambda: s.of(s.cache.weigh(q, s.ints([0, new]), s.ints([300]), s.ints(s.blocks), new, s.weights, out=torch.zeros_like(s.weights)), 0)[0]  # noqa: E731
    got = weigh()
    assert torch.isfinite(got).all() and torch.equal(got[[20, 150]], before[[20, 150]])
    s.cache.k[place(77)] = other
    assert torch.isnan(weigh()).all()
