"""The operators of language models on the GPU against lm_bounds.py: what roundings leave, and no more."""
import math

import numpy as np
import pytest
import torch

import lm_bounds
from nart_amd import hipq
from lm_reference import pack_rows
from test_lm_gpu import fill_cache, gen, randn, tokens_of, trees, weights

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def index(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts_of(counts):
    return np.concatenate(([0], np.cumsum(counts))).tolist()


# ---- products with 4-bit weights ----------------------------------------------------------------------------------------
KERNELS = [(16, 200, 1056, "w4_stream_16"), (3, 20500, 1056, "w4_tile_16x128"), (24, 9000, 2080, "w4_tile_32x128"), (33, 300, 2112, "w4_tile_32x128"), (60, 16400, 160, "w4_tile_64x128"),
           (100, 400, 4128, "w4_tile_64x128"), (90, 16400, 160, "w4_tile_128x128"), (200, 300, 2112, "w4_tile_128x128"), (140, 8200, 1056, "w4_tile_128x256")]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group, zeros", [(128, False), (128, True), (64, False), (64, True), (32, False), (32, True)])
@pytest.mark.parametrize("m, n, k, kernel", KERNELS)
def test_linear_spread(m, n, k, kernel, group, zeros, dtype):
    """Every kernel rounds once: weights that were rounded, or sums in 16 bits, would not keep to this."""
    g = gen(m + group)
    q, scales, z, b = weights(g, dtype, n, k, group, zeros=zeros)
    x = randn(g, dtype, m, k)
    plan = hipq.LinearW4(pack_rows(q), scales, group, zeros=z, bias=b)
    assert plan.kernel(m) == kernel
    lm_bounds.check_linear_spread(plan(x), x, q, scales, group, z, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group, zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("m, n, k, kernel", KERNELS)
def test_linear_large_x_at_zero_points(m, n, k, kernel, group, zeros, dtype):
    """Some x of 10^3 to 10^4 meet codes that are their zero points, which they do nothing to but in the roundings: those of sums of 63 |x|."""
    g = gen(m + group)
    q, scales, z, b = weights(g, dtype, n, k, group, zeros=zeros)
    x = randn(g, dtype, m, k)
    at = torch.randperm(k, device="cuda", generator=g)[:k // 40 + 1]
    x[:, at] = (x[:, at] * 3000).to(dtype)
    q[:, at] = 8 if z is None else z[:, at // group]
    got = hipq.LinearW4(pack_rows(q), scales, group, zeros=z, bias=b)(x)
    lm_bounds.check_linear_spread(got, x, q, scales, group, z, b)
    want, off = lm_bounds.linear_spread(x, q, scales, group, z, b)
    half = torch.finfo(dtype).eps / 2
    assert ((got.double() - want).abs() <= half * want.abs() + 8 * off + torch.finfo(dtype).smallest_normal).all()  # 8: of some million normal ones


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("group, zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("m, n, k, kernel", KERNELS)
def test_linear_rows_that_are_not_finite(m, n, k, kernel, group, zeros, act):
    """A row with an infinity, with two of either sign, or with NaN: NaN throughout; the other rows get what they got."""
    g = gen(m + group)
    q, scales, z, b = weights(g, BF16, n if act is None else n // 2 * 2, k, group, zeros=zeros)
    plan, x = hipq.LinearW4(pack_rows(q), scales, group, zeros=z, bias=b, activation=act), randn(g, BF16, m, k)
    want, bad = plan(x), x.clone()
    bad[0, 5], bad[m // 2, k - 1], bad[m - 1, 7], bad[m - 1, k // 2] = math.inf, math.nan, -math.inf, math.inf
    got = plan(bad)
    rows = [0, m // 2, m - 1]
    others = [r for r in range(m) if r not in rows]
    assert torch.isnan(got[rows]).all() and torch.equal(got[others], want[others])


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype, group", [(BF16, 128), (F16, 64), (BF16, 32)])
@pytest.mark.parametrize("m, n, k", [(16, 330, 160), (20, 100, 512), (7, 10300, 1056), (60, 8200, 160), (100, 200, 2112), (140, 4200, 160)])
def test_linear_gated_spread(m, n, k, dtype, group, act):
    g = gen(m)
    q, scales, z, b = weights(g, dtype, 2 * n, k, group)
    x = randn(g, dtype, m, k)
    lm_bounds.check_linear_spread(hipq.LinearW4(pack_rows(q), scales, group, zeros=z, bias=b, activation=act)(x), x, q, scales, group, z, b, act)


# ---- attention over the cache ---------------------------------------------------------------------------------------------
def check(cache, blocks, q, counts, lens, mask=None, scale=None):
    heads, dim = cache.k.shape[1], cache.k.shape[-1]
    starts = starts_of(counts)
    got = cache.attend(q, index(starts), index(lens), blocks, max(counts), mask=mask, scale=scale)
    k, v = ([tokens_of(p, blocks[b], n) for b, n in enumerate(lens)] for p in (cache.k, cache.v))
    ks, vs = ([tokens_of(p[..., None], blocks[b], n)[..., 0] for b, n in enumerate(lens)] if p is not None else None for p in (cache.k_scale, cache.v_scale))
    lm_bounds.check_attend_spread(got, *lm_bounds.attend_spread(q, k, v, starts, lens, mask, dim ** -0.5 if scale is None else scale, q.shape[1] // heads, ks, vs))
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dim, hq, hkv, counts, lens, tree", [
    (64, 6, 2, [1] * 5, [2000, 700, 33, 129, 1024], False), (128, 8, 2, [1] * 3, [9000, 257, 5000], False), (256, 4, 1, [1] * 3, [600, 4000, 31], False),
    (64, 4, 1, [40, 3, 1], [300, 1000, 77], False), (128, 16, 4, [16, 9, 30], [2500, 40, 1111], True), (256, 6, 2, [5, 20], [800, 300], True),
    (128, 32, 8, [34, 20, 64, 5], [1000, 1900, 600, 1024], True), (128, 16, 8, [300, 129], [300, 4000], False)])
def test_attend_spread(dim, hq, hkv, counts, lens, tree, int8, dtype):
    """All kernels: single tokens, chains, trees, prompts, many rows; scores that are close together and, with a larger scale, far apart."""
    g, rng = gen(sum(lens)), np.random.default_rng(sum(lens))
    cache, blocks = fill_cache(g, dtype, len(lens), hkv, 48, dim, max(lens), int8)
    q, mask = randn(g, dtype, sum(counts), hq, dim), trees(rng, counts) if tree else None
    for scale in (None, 2.0):
        check(cache, blocks, q, counts, lens, mask, scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
def test_attend_spread_long(int8, dtype):
    """Many parts and their joins: a lost tile of 32 tokens would be 4 % of the result, ten times what is allowed."""
    g = gen(80)
    lens = [20000, 19999, 131072]
    cache, blocks = fill_cache(g, dtype, 3, 1, 64, 128, max(lens), int8)
    for counts in ([1, 1, 1], [1, 2, 9]):
        check(cache, blocks, randn(g, dtype, sum(counts), 4, 128), counts, lens)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n, rows, heads", [(20000, 1, 1), (3001, 1, 1), (4500, 40, 8)])
def test_attend_every_token_is_found(n, rows, heads, int8):
    """One token's score is far above the others', at places over the whole sequence: its value is the result."""
    g = gen(n)
    cache, blocks = fill_cache(g, F16, 1, heads, 64, 128, n, int8, spare=0)
    q = torch.full((rows, 4 * heads, 128), 1.0, dtype=F16, device="cuda")
    cache.k.fill_(0)
    if int8:
        cache.k_scale.fill_(0.25)
    old = n - rows
    where = sorted({t for t in list(range(0, old, max(1, old // 70))) + [31, 32, 127, 128, 255, 256, old // 2 // 128 * 128, old - 33, old - 32, old - 1] if 0 <= t < old})
    for t in where:
        page, at = blocks[0, t // 64].long(), t % 64
        cache.k[page, :, at] = 100
        got = cache.attend(q, index([0, rows]), index([n]), blocks, rows)
        v = cache.v[page, :, at].double() * (cache.v_scale[page, :, at, None].double() if int8 else 1)
        want = v.repeat_interleave(4, 0)[None].expand(rows, -1, -1)
        assert ((got.double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -24).all(), t  # two roundings: the weight's, the result's
        cache.k[page, :, at] = 0


def cache_with_scores(g, dtype, heads, dim, scores, int8, page=64):
    """One sequence whose token t has score scores[t] for queries of ones and a scale of 1 / dim; values are positive."""
    n = len(scores)
    cache, blocks = fill_cache(g, dtype, 1, heads, page, dim, n, int8, spare=0)
    at = torch.arange(n, device="cuda")
    pages, places = blocks[0].long()[at // page], at % page
    if int8:
        cache.k.fill_(1)
        cache.k_scale[pages, :, places] = scores.float()[:, None].cuda()
        cache.v.copy_(torch.randint(1, 128, cache.v.shape, dtype=torch.int8, device="cuda", generator=g))
    else:
        cache.k[pages, :, places] = scores.to(dtype)[:, None, None].cuda()
        cache.v.copy_((torch.randn(cache.v.shape, device="cuda", generator=g) + 1).to(dtype))
    return cache, blocks, pages, places


# rows: single tokens, a chain, many rows (each kernel), whose queries are ones
ROWS = [(1, 1, 4, 64), (1, 1, 4, 128), (9, 1, 4, 256), (40, 8, 32, 128)]
FRONT = [3, 35, 67, 99]  # a token for each wave of a work-group that takes tiles of 32 in turn


def check_alike(cache, blocks, rows, hq, dim, n, dtype):
    """Queries of ones: one sequence alone, divided among as many work-groups as there can be, and as many sequences over the same pages as make
    every work-group go over all of one."""
    heads = cache.k.shape[1]
    for sequences in (1, 512 // heads):
        q = torch.ones((sequences * rows, hq, dim), dtype=dtype, device="cuda")
        got = cache.attend(q, index(list(range(0, sequences * rows + 1, rows))), index([n] * sequences), blocks.expand(sequences, -1).contiguous(), rows, scale=1 / dim)
        assert (got.view(sequences, rows, hq, dim) == got[:rows]).all()
        k, v, ks, vs = (None if p is None else [tokens_of(p, blocks[0], n)] for p in (cache.k, cache.v, *(None if t is None else t[..., None] for t in (cache.k_scale, cache.v_scale))))
        ks, vs = (None if t is None else [t[0][..., 0]] for t in (ks, vs))
        lm_bounds.check_attend_spread(got[:rows], *lm_bounds.attend_spread(q[:rows], k, v, [0, rows], [n], None, 1 / dim, hq // heads, ks, vs), rows=1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, heads, hq, dim", ROWS)
@pytest.mark.parametrize("n, gap, ratio", [(8192, 9, 4096), (32768, 12, 256), (32768, 11, 16), (8192, 9, 1e-4)])
def test_attend_codes_of_many_sizes(n, gap, ratio, rows, heads, hq, dim, dtype):
    """An int8 cache with some scores far above the others and some value scales many times the others' (or 10^-4 of them)."""
    g = gen(n + dim)
    scores = torch.from_numpy(np.random.default_rng(n).standard_normal(n) * 0.5)
    scores[FRONT] = gap
    cache, blocks, pages, places = cache_with_scores(g, dtype, heads, dim, scores, True)
    for shift in (2, n // 2):
        at = torch.tensor(FRONT) + shift
        before = cache.v_scale[pages[at], :, places[at]].clone()
        cache.v_scale[pages[at], :, places[at]] *= ratio
        check_alike(cache, blocks, rows, hq, dim, n, dtype)
        cache.v_scale[pages[at], :, places[at]] = before


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("rows, heads, hq, dim", ROWS)
@pytest.mark.parametrize("gap", [15, 17])
def test_attend_long_tail(gap, rows, heads, hq, dim, int8, dtype):
    """Many tokens behind some whose scores are 15 or 17 above theirs: together they are some hundredths or thousandths of the result."""
    g, n = gen(gap), 131072 if heads == 1 else 32768
    scores = torch.zeros(n)
    scores[FRONT] = gap
    cache, blocks, pages, places = cache_with_scores(g, dtype, heads, dim, scores, int8)
    cache.v[pages[FRONT], :, places[FRONT]] = -1
    check_alike(cache, blocks, rows, hq, dim, n, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, heads, hq, dim", [(1, 1, 4, 64), (5, 2, 6, 128), (40, 8, 32, 128), (12, 1, 2, 256)])
def test_attend_value_scales_over_four_decades(rows, heads, hq, dim, dtype):
    """Scales from 10^-3 to 10 of single tokens, and of tokens that follow each other by size, up and down, beside scores that fall and rise."""
    g = gen(rows + dim)
    n = 3000
    cache, blocks = fill_cache(g, dtype, 1, heads, 64, dim, n, True, spare=0)
    at = torch.arange(n, device="cuda")
    pages, places = blocks[0].long()[at // 64], at % 64
    q = randn(g, dtype, rows, hq, dim)
    by_size = 10.0 ** (at.double() / n * 4 - 3)
    for scales in (10.0 ** (torch.rand(n, device="cuda", generator=g).double() * 4 - 3), by_size, by_size.flip(0)):
        cache.v_scale[pages, :, places] = scales.float()[:, None]
        check(cache, blocks, q, [rows], [n])
    cache.k.fill_(1)
    for scores in (at.double() / n * 9, 9 - at.double() / n * 9):  # the scores undo the scales, and the other way round
        cache.k_scale[pages, :, places] = scores.float()[:, None]
        check_alike(cache, blocks, rows, hq, dim, n, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows, heads, hq, n", [(3, 1, 4, 1000), (40, 8, 32, 9000), (17, 2, 2, 100)])
@pytest.mark.parametrize("tree", [False, True])
def test_attend_scales_of_tokens_that_are_not_seen(rows, heads, hq, n, tree, dtype):
    """A drafted token's value scale of 2^12 to 2^100 times the others', or infinite: rows that do not see it get what they got."""
    g = gen(rows)
    cache, blocks = fill_cache(g, dtype, 1, heads, 64, 128, n, True, spare=0)
    q = randn(g, dtype, rows, hq, 128)
    words = [1 | 1 << i for i in range(rows)] if tree else None  # the first token, and branches of one
    mask = torch.tensor(words, dtype=torch.int64, device="cuda") if tree else None
    call = lambda: cache.attend(q, index([0, rows]), index([n]), blocks, rows, mask=mask)  # noqa: E731
    want = call()
    new = rows - 1 if not tree else 1
    at = n - rows + new
    page, place = blocks[0, at // 64].long(), at % 64
    others = [r for r in range(rows) if r != new]
    for factor in (2.0 ** 12, 2.0 ** 40, 2.0 ** 100, math.inf, math.nan):
        before = cache.v_scale[page, :, place].clone()
        cache.v_scale[page, :, place] *= factor
        assert torch.equal(call()[others], want[others]), factor
        cache.v_scale[page, :, place] = before
