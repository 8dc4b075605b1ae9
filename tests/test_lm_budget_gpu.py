"""The cache held to a budget on the GPU: weights where scores are not finite, scores kept by pages."""
import math

import numpy as np
import pytest
import torch

from nart_amd import hipq
from test_lm_more_gpu import BF16, Sequences, gen, randn, whole

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


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens, counts, heads, group, dim, page", [([700, 1, 90, 300], [1, 1, 0, 1], 2, 8, 64, 48), ([5000, 31], [3, 13], 3, 1, 128, 64), ([64, 65, 300], [2, 2, 1], 2, 12, 256, 32),
                                                                   ([33, 16, 15], [1, 1, 1], 4, 7, 128, 16)])
@pytest.mark.parametrize("tree", [False, True])
def test_weigh_with_wide_tables(lens, counts, heads, group, dim, page, int8, tree):
    """Scores that lie as the cache's tokens do, where a table has room for more than the cache holds: the same weights, and no others touched."""
    g = gen(sum(lens))
    s = Sequences(g, BF16, lens, heads, dim, page, int8)
    q, starts = randn(g, BF16, sum(counts), heads * group, dim), s.ints([0] + list(np.cumsum(counts)))
    mask = whole(g, 0, 2 ** 62, torch.int64, sum(counts)) if tree else None
    table = s.ints(s.blocks)
    table[0, (lens[0] - 1) // page // 2] = -1
    wide = torch.cat((table, torch.full((len(lens), 10 * table.shape[1]), 1 << 30, dtype=torch.int32, device="cuda")), 1)
    run = lambda cache, weights: cache.weigh(q, starts, s.ints(lens), wide, max(counts), weights, mask=mask, out=torch.full_like(weights, 7.0))  # noqa: E731
    asked, bytes_like = [], hipq._bytes_like
    hipq._bytes_like = lambda t, count: asked.append(count) or bytes_like(t, count).fill_(255)  # NaN
    try:
        got = run(s.cache, s.weights)
    finally:
        hipq._bytes_like = bytes_like
    # in a cache of more pages they lie sequence by sequence
    more_pages = lambda p: None if p is None else torch.cat((p, p.new_zeros((11 * s.pages, *p.shape[1:]))))  # noqa: E731
    large = run(hipq.KvCache(*(more_pages(p) for p in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale))), more_pages(s.weights))
    assert torch.equal(got, large[:s.pages]) and (large[s.pages:] == 7).all()
    assert torch.isfinite(got).all() and (got != 7).sum() >= sum(n for n, c in zip(lens, counts) if c) * heads - heads * page
    rows = max(counts) * group
    assert len(asked) == 1 and rows * s.pages * heads * page * 4 <= asked[0] <= rows * heads * (s.pages * page * 4 + len(lens) * 256 * 8) + 256
