"""The cache held to a budget on the GPU: weights where scores are not finite, scores kept by pages, long sequences whose tokens several work-groups choose from,
blocks that are not there."""
import math

import numpy as np
import pytest
import torch

import lm_more_reference as more
from nart_amd import hipq
from test_lm_more_gpu import BF16, F16, F32, Sequences, check_evicted, check_weighed, gen, randn, same, whole

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


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens, counts, heads, group, dim", [([1500, 700], [700, 513], 2, 4, 128), ([2100], [300], 1, 3, 256), ([900, 40], [260, 40], 1, 8, 64)])
def test_weigh_a_prompt(lens, counts, heads, group, dim, int8):
    """Some hundred new tokens, which pass through LDS in several rounds."""
    g = gen(sum(counts))
    check_weighed(g, Sequences(g, BF16, lens, heads, dim, 48, int8), BF16, counts, group)


# ---- eviction: long sequences, whose tokens several work-groups choose from ------------------------------------------------------
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("what", ["equal", "few values", "zeros", "not finite", "either sign", "close", "one heavy part"])
def test_evict_ties_of_several_parts(what, in_place):
    """Equal weights at the border on both sides of the parts' ends, beside a sequence within the budget."""
    g = gen(10)
    s = Sequences(g, F16, [40000, 16400, 77], 2, 64, 32, False, spare=3 * 282)
    w = s.weights
    if what == "equal":
        w.fill_(0.25)
    elif what == "few values":
        w.copy_(whole(g, 0, 3, torch.int32, *w.shape).float())
    elif what == "zeros":
        w.copy_(torch.where(torch.rand(w.shape, device="cuda", generator=g) < 0.97, 0.0, w))
        w[::2] *= -1
    elif what == "not finite":
        u = torch.rand(w.shape, device="cuda", generator=g)
        w.copy_(torch.where(u < 0.5, math.nan, torch.where(u < 0.9, -math.inf, torch.where(u < 0.95, math.inf, w))))
    elif what == "either sign":
        w.copy_(randn(g, F32, *w.shape))
    elif what == "close":
        w.copy_(1 + whole(g, 0, 3000, torch.int32, *w.shape).float() * 2.0 ** -23)
    else:
        w.zero_()
        w[torch.from_numpy(s.blocks[0, 2 * 256 + 3:3 * 256 + 3]).cuda()] = 1.0  # the third part's, nearly
    check_evicted(s, 9000, 20, 5, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens, budget, recent, first", [([40000, 300, 17000], 9000, 8600, 400), ([40000], 9000, 0, 9000), ([20000, 16385], 16384, 0, 0), ([40000, 8192, 8193], 20000, 8500, 9000),
                                                         ([33000, 24576], 24575, 1, 0), ([17000], 1, 0, 0)])
def test_evict_forced_tokens_of_several_parts(lens, budget, recent, first, in_place):
    """First and last tokens that fill the budget, or whole parts."""
    g = gen(sum(lens))
    s = Sequences(g, BF16, lens, 2, 64, 32, True, spare=len(lens) * (-(-budget // 32) + 1))
    check_evicted(s, budget, recent, first, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens, budget", [([300, 200, 33], 64), ([17000, 90], 5000)])
def test_evict_blocks_outside(lens, budget, int8, in_place):
    """Tokens whose block or whose new one is not there are not moved, all others are, and nothing else changes."""
    g = gen(budget)
    page, heads, need = 16, 2, -(-budget // 16)
    s = Sequences(g, BF16, lens, heads, 64, page, int8, spare=len(lens) * need)
    blocks = s.blocks.copy()
    to = blocks if in_place else np.random.default_rng(2).permutation(s.rest)[:len(lens) * need].reshape(len(lens), need)
    blocks[0, 2], blocks[0, lens[0] // page - 1], blocks[1, 1], blocks[1, lens[1] // page] = -1, s.pages, -2 ** 31, 2 ** 31 - 1
    if not in_place:
        to[0, 1], to[1, 3] = s.pages + 5, -1
    before = {name: p.clone() for name, p in (("k", s.cache.k), ("v", s.cache.v), ("ks", s.cache.k_scale), ("vs", s.cache.v_scale), ("w", s.weights)) if p is not None}
    ranked = []
    for b, n in enumerate(lens):
        t = np.arange(n)
        there = (blocks[b, t // page] >= 0) & (blocks[b, t // page] < s.pages)
        at = torch.from_numpy(np.where(there, blocks[b, t // page], 0)).cuda()
        w = before["w"][at, :, torch.from_numpy(t % page).cuda()].t()
        ranked.append(torch.where(torch.from_numpy(there).cuda(), w, math.nan))
    want = more.evict(ranked, lens, budget, 7, 3)
    expected = {name: p.clone() for name, p in before.items()}
    for b, n in enumerate(lens):
        for h in range(heads):
            t, j = want[b][h], np.arange(min(n, budget))
            source, target = blocks[b, t // page], to[b, j // page]
            ok = (source >= 0) & (source < s.pages) & (target >= 0) & (target < s.pages)
            index = lambda x: torch.from_numpy(np.ascontiguousarray(x[ok])).long().cuda()  # noqa: E731
            for name, p in before.items():
                expected[name][index(target), h, index(j % page)] = p[index(source), h, index(t % page)]
    table = s.ints(blocks)
    left, kept = s.cache.evict(s.weights, s.ints(lens), table, budget, recent=7, first=3, to=None if in_place else s.ints(to))
    assert left.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        assert np.array_equal(kept[b, :, :min(n, budget)].cpu().numpy(), want[b]) and (kept[b, :, min(n, budget):] == -1).all()
    for name, p in (("k", s.cache.k), ("v", s.cache.v), ("ks", s.cache.k_scale), ("vs", s.cache.v_scale), ("w", s.weights)):
        assert p is None or same(p, expected[name]), name
