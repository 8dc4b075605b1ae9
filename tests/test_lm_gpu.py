"""The operators of language models on the GPU, against their formulas in 64 bits (lm_reference.py)."""
import math

import numpy as np
import pytest
import torch

import lm_reference as ref
from nart_amd import hipq

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, dtype, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


# ---- products with 4-bit weights ------------------------------------------------------------------------------------
def weights(g, dtype, rows, k, group, zeros=True, bias=True):
    groups = -(-k // group)
    q = torch.randint(0, 16, (rows, k), dtype=torch.uint8, device="cuda", generator=g)
    scales = (torch.rand((rows, groups), device="cuda", generator=g) * 0.02 + 0.002).to(dtype)
    z = torch.randint(0, 16, (rows, groups), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    return q, scales, z, randn(g, dtype, rows) if bias else None


def check_linear(x, w, group, act=None, y=None):
    q, scales, z, b = w
    plan = hipq.LinearW4(ref.pack_rows(q), scales, group, zeros=z, bias=b, activation=act)
    got = plan(x, y)
    want, off = ref.linear(x, q, scales, group, z, b, act)
    ok, far = ref.within(got, want, off)
    assert ok, "%s: %g too far" % (plan.kernel(x.shape[0]), far)
    return plan, got


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 193, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_rows(m, dtype):
    g = gen(m)
    check_linear(randn(g, dtype, m, 288), weights(g, dtype, 200, 288, 128), 128)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n, k", [(1, 32), (16, 64), (17, 96), (31, 160), (130, 1024), (257, 4128)])
@pytest.mark.parametrize("m", [3, 40, 200])
def test_linear_shapes(m, n, k, group):
    g = gen(n + k)
    dtype = BF16 if n % 2 else F16
    check_linear(randn(g, dtype, m, k), weights(g, dtype, n, k, group, zeros=n != 17, bias=n != 31), group)


@pytest.mark.parametrize("dtype, group, zeros", [(BF16, 128, False), (F16, 128, True), (BF16, 64, True), (F16, 64, False), (BF16, 32, True), (F16, 32, False)])
@pytest.mark.parametrize("m, n, k, kernel", [(3, 20500, 1056, "w4_tile_16x128"), (9, 16500, 2144, "w4_tile_16x128"), (24, 9000, 2080, "w4_tile_32x128"), (33, 300, 2112, "w4_tile_32x128"),
                                             (60, 16400, 96, "w4_tile_64x128"), (100, 400, 2112, "w4_tile_64x128"), (90, 16400, 160, "w4_tile_128x128"),
                                             (200, 300, 2112, "w4_tile_128x128"), (150, 8200, 160, "w4_tile_128x256"), (140, 8200, 1056, "w4_tile_128x256")])
def test_linear_kernels(m, n, k, kernel, dtype, group, zeros):
    """Every kernel, with and without work-groups that share the reduction, and reductions that end inside a block."""
    g = gen(m + group)
    plan, _ = check_linear(randn(g, dtype, m, k), weights(g, dtype, n, k, group, zeros=zeros), group)
    assert plan.kernel(m) == kernel


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m, n, k, group", [(1, 100, 256, 128), (16, 33, 160, 32), (20, 100, 512, 64), (70, 16, 128, 128), (210, 200, 384, 64), (7, 10300, 1056, 128), (140, 4200, 160, 32), (50, 9000, 96, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_gated(dtype, m, n, k, group, act):
    g = gen(m)
    check_linear(randn(g, dtype, m, k), weights(g, dtype, 2 * n, k, group), group, act)


@pytest.mark.parametrize("m", [1, 5, 24, 90, 260])
def test_linear_rows_with_gaps(m):
    """Rows of x and y inside wider ones: what lies between y's rows, and behind the last one, stays."""
    g = gen(m)
    x, y = randn(g, BF16, m, 400), torch.full((m + 2, 77), 7.0, dtype=BF16, device="cuda")
    check_linear(x[:, 16:16 + 320], weights(g, BF16, 70, 320, 64), 64, y=y[1:m + 1, 3:73])
    assert (y[0] == 7).all() and (y[m + 1] == 7).all() and (y[:, :3] == 7).all() and (y[:, 73:] == 7).all()


@pytest.mark.parametrize("m", [1, 24, 90, 260])
def test_linear_extremes(m):
    """Every code at one end, zero points at the other; a row of zeros, a row of large numbers; infinities stay in their rows."""
    g = gen(m)
    q = torch.zeros((48, 256), dtype=torch.uint8, device="cuda")
    q[::2] = 15
    z = torch.full((48, 2), 15, dtype=torch.uint8, device="cuda")
    z[::2] = 0
    x = randn(g, BF16, m, 256)
    x[0] = 0
    w = (q, torch.ones((48, 2), dtype=BF16, device="cuda"), z, None)
    plan, y = check_linear(x, w, 128)
    assert (y[0] == 0).all()
    if m > 1:
        bad = x.clone()
        bad[1, 5] = math.inf
        bad[m - 1, 200] = math.nan
        again = plan(bad)
        assert not torch.isfinite(again[1]).any() and torch.isnan(again[m - 1]).all()
        same = [i for i in range(m) if i not in (1, m - 1)]
        assert torch.equal(again[same], y[same])


def test_linear_more_dimensions_and_no_rows():
    g = gen(1)
    w = weights(g, BF16, 40, 64, 32)
    plan = hipq.LinearW4(ref.pack_rows(w[0]), w[1], 32, zeros=w[2], bias=w[3])
    x = randn(g, BF16, 2, 3, 64)
    assert torch.equal(plan(x).view(6, 40), plan(x.view(6, 64)))
    assert plan(x[:0, 0]).shape == (0, 40)


def test_linear_same_result_every_time():
    g = gen(2)
    w = weights(g, BF16, 600, 4096, 128)
    plan = hipq.LinearW4(ref.pack_rows(w[0]), w[1], 128, zeros=w[2], bias=w[3])
    for m in (1, 30, 130, 400):
        x = randn(g, BF16, m, 4096)
        first = plan(x)
        assert all(torch.equal(first, plan(x)) for _ in range(5))


# ---- the cache ----------------------------------------------------------------------------------------------------------
def new_cache(dtype, pages, heads, page, dim, int8, fill=0):
    place = torch.int8 if int8 else dtype
    k, v = (torch.full((pages, heads, page, dim), fill, dtype=place, device="cuda") for _ in range(2))
    scales = [torch.full((pages, heads, page), float(fill), device="cuda") for _ in range(2)] if int8 else [None, None]
    return hipq.KvCache(k, v, *scales)


def check_placed(pool, scales, slots, want, off, fill, exact=False):
    pages, heads, page, dim = pool.shape
    flat = pool.transpose(1, 2).reshape(pages * page, heads, dim)
    there = slots >= 0
    at = slots[there].long()
    got = flat[at]
    if scales is None:
        assert ref.within(got, want[there], off[there])[0]
    else:
        s = scales.transpose(1, 2).reshape(pages * page, heads)[at].double()
        most = want[there].abs().amax(-1)
        assert ((s - most / 127).abs() <= ref.STEP32 * most / 127 + off[there].amax(-1) / 127 + 1e-45).all()
        # half a step of rounding, what the value was off, and what that makes of the scale (at most 127 times)
        slack = s[..., None] * (0.5 + 2.0 ** -14) + off[there] + off[there].amax(-1, keepdim=True)
        assert ((got.double() * s[..., None] - want[there]).abs() <= slack).all()
        assert (got.abs() <= 127).all()
    left = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    left[at] = False
    assert (flat[left] == fill).all()
    if scales is not None:
        assert (scales.transpose(1, 2).reshape(pages * page, heads)[left] == fill).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tokens, hq, hkv, dim, page, rot, interleaved, norm", [
    (1, 1, 1, 64, 16, 64, False, False), (3, 8, 2, 128, 32, 128, False, True), (7, 5, 5, 128, 48, 64, True, True), (33, 4, 1, 256, 16, 256, True, False),
    (20, 12, 4, 64, 64, 48, False, True), (5, 3, 1, 256, 16, 16, False, False), (300, 32, 8, 128, 64, 128, False, True), (1500, 7, 7, 64, 32, 32, True, False),
    (6, 4, 2, 128, 16, 0, False, True)])
def test_append(tokens, hq, hkv, dim, page, rot, interleaved, norm, int8, dtype):
    g = gen(tokens)
    pages = -(-tokens // page) + 3
    cache = new_cache(dtype, pages, hkv, page, dim, int8, fill=3)
    qkv = randn(g, dtype, tokens, hq + 2 * hkv, dim)  # one tensor, as a projection leaves them
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    far = 5000
    positions = torch.randint(0, far, (tokens,), device="cuda", generator=g).to(torch.int32)
    positions[0] = far - 1
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens].to(torch.int32)
    if tokens > 2:
        slots[1] = -1  # a padded row
    table = hipq.rotation_table(far, rot) if rot else None
    wq, wk = ((torch.rand(dim, device="cuda", generator=g) + 0.5).to(dtype) for _ in range(2)) if norm else (None, None)
    out = torch.full((tokens, hq, dim), 5.0, dtype=dtype, device="cuda")
    got = cache.append(q, k, v, positions, slots, table, out=out, q_norm=wq, k_norm=wk, eps=1e-5, interleaved=interleaved)
    cos, sin = (table[positions.long()] if rot else torch.zeros((tokens, 0), device="cuda")).chunk(2, -1) if rot else (torch.zeros((tokens, 0), device="cuda"),) * 2
    there = slots >= 0
    want, off = ref.rotate(q, wq, 1e-5, cos, sin, interleaved)
    ok, far_off = ref.within(got[there], want[there], off[there])
    assert ok, far_off
    assert (got[~there] == 5).all()
    want, off = ref.rotate(k, wk, 1e-5, cos, sin, interleaved)
    check_placed(cache.k, cache.k_scale, slots, want, off, 3)
    check_placed(cache.v, cache.v_scale, slots, v.double(), torch.zeros_like(want), 3)


def test_append_in_place_and_out_of_range():
    """q may be written over; slots and positions outside leave everything as it is."""
    g = gen(5)
    cache, table = new_cache(BF16, 2, 2, 16, 128, False), hipq.rotation_table(10, 128)
    q, k, v = randn(g, BF16, 6, 4, 128), randn(g, BF16, 6, 2, 128), randn(g, BF16, 6, 2, 128)
    before = q.clone()
    positions = torch.tensor([0, 9, 10, -1, 3, 3], dtype=torch.int32, device="cuda")
    slots = torch.tensor([31, 0, 1, 2, 32, -7], dtype=torch.int32, device="cuda")
    cache.append(q, k, v, positions, slots, table, out=q)
    want, off = ref.rotate(before, None, 0, table[positions.clamp(0, 9).long()][:, :64], table[positions.clamp(0, 9).long()][:, 64:], False)
    assert ref.within(q[:2], want[:2], off[:2])[0] and torch.equal(q[2:], before[2:])
    rest = cache.v.transpose(1, 2).reshape(32, 2, 128)
    assert torch.equal(rest[31], v[0]) and torch.equal(rest[0], v[1]) and (rest[1:31] == 0).all()


def test_append_int8_zero_and_tiny_heads():
    cache = new_cache(F16, 1, 1, 16, 64, True, fill=9)
    k = torch.zeros((3, 1, 64), dtype=F16, device="cuda")
    k[1, 0, 3] = 6e-8  # the smallest float16
    k[2] = 60000.0
    index = torch.arange(3, dtype=torch.int32, device="cuda")
    cache.append(k, k, -k, index, index, None)
    codes, scales = cache.k[0, 0, :3], cache.k_scale[0, 0, :3]
    assert (codes[0] == 0).all() and scales[0] == 0
    assert codes[1, 3] == 127 and codes[1].abs().sum() == 127
    assert (codes[2] == 127).all() and (cache.v[0, 0, 2] == -127).all()
    assert (scales[2].double() * 127 - 60000.0).abs() < 60000 * 2 ** -23


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_append_int8_codes_are_the_rounded_quotients(dtype, dim):
    """Bit by bit: code = value / scale in float32, rounded to nearest even, for heads of all magnitudes (in float16 some of 2^14 times a
    normal number hold infinities: their codes are not defined)."""
    g = gen(dim)
    n = 3000
    size = torch.exp2(torch.randint(-20, 15, (n, 1, 1), device="cuda", generator=g).double())
    k, v = ((torch.randn((n, 1, dim), device="cuda", generator=g, dtype=torch.float64) * size).to(dtype) for _ in range(2))
    k[5], k[6, 0, 1:] = 0, 0
    cache = new_cache(dtype, -(-n // 16), 1, 16, dim, True)
    index = torch.arange(n, dtype=torch.int32, device="cuda")
    cache.append(k.new_empty((n, 0, dim)), k, v, index, index, None)
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        x, s = x.float().cpu()[:, 0], scales.flatten()[:n].cpu()[:, None]
        assert torch.equal(s, x.abs().amax(-1, keepdim=True) / 127)
        want, finite = torch.where(s > 0, torch.round(x / s), 0.0), torch.isfinite(s[:, 0])
        assert torch.equal(codes.reshape(-1, dim)[:n].cpu().float()[finite], want[finite]) and finite.sum() > 0.9 * n


def fill_cache(g, dtype, b, heads, page, dim, longest, int8, spare=3):
    """A cache whose pages are in a random order, and its blocks."""
    per = -(-longest // page)
    pages = b * per + spare
    if int8:
        k, v = (torch.randint(-127, 128, (pages, heads, page, dim), dtype=torch.int8, device="cuda", generator=g) for _ in range(2))
        ks, vs = (torch.rand((pages, heads, page), device="cuda", generator=g) * 0.02 + 0.001 for _ in range(2))
    else:
        k, v, ks, vs = randn(g, dtype, pages, heads, page, dim), randn(g, dtype, pages, heads, page, dim), None, None
    blocks = torch.randperm(pages, device="cuda", generator=g)[:b * per].view(b, per).to(torch.int32)
    return hipq.KvCache(k, v, ks, vs), blocks


def tokens_of(pool, blocks, n):
    """[heads, n, ...] of one sequence."""
    x = pool[blocks.long()]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def check_attend(g, cache, blocks, counts, lens, hq, dtype, mask=None, scale=None, most=None, longest=None, spare_rows=2):
    heads, dim = cache.k.shape[1], cache.k.shape[-1]
    total = sum(counts)
    starts = np.concatenate(([0], np.cumsum(counts))).tolist()
    q = randn(g, dtype, total + spare_rows, hq, dim)
    out = torch.full_like(q, 11.0)
    if mask is not None:
        mask = torch.cat((mask, torch.zeros(spare_rows, dtype=torch.int64, device="cuda")))
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = cache.attend(q, index(starts), index(lens), blocks, most or max(counts), mask=mask, scale=scale, out=out, longest=longest)
    k, v = ([tokens_of(p, blocks[b], n) for b, n in enumerate(lens)] for p in (cache.k, cache.v))
    ks, vs = ([tokens_of(p[..., None], blocks[b], n)[..., 0] for b, n in enumerate(lens)] if p is not None else None for p in (cache.k_scale, cache.v_scale))
    want, off = ref.attend(q, k, v, starts, lens, mask, dim ** -0.5 if scale is None else scale, hq // heads, ks, vs)
    ok, far = ref.within(got[:total], want[:total], off[:total])
    assert ok, far
    assert (got[total:] == 11).all()
    return q, got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq, hkv", [(1, 1), (8, 2), (20, 4), (24, 1)])
def test_attend_one_token(hq, hkv, dim, int8, dtype):
    g = gen(dim + hq)
    lens = [1, 15, 16, 17, 33, 129, 700]
    cache, blocks = fill_cache(g, dtype, len(lens), hkv, 16, dim, max(lens), int8)
    check_attend(g, cache, blocks, [1] * len(lens), lens, hq, dtype)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("dtype, dim, hq, hkv", [(BF16, 128, 4, 2), (F16, 64, 6, 1), (BF16, 256, 2, 1)])
def test_attend_chain(dtype, dim, hq, hkv, page, int8):
    """Chains of new tokens, ragged: none, one, all of a sequence, more than a work-group's rows."""
    g = gen(page)
    counts, lens = [3, 0, 1, 40, 17, 64], [90, 50, 1, 40, 300, 1000]
    cache, blocks = fill_cache(g, dtype, len(lens), hkv, page, dim, max(lens), int8)
    check_attend(g, cache, blocks, counts, lens, hq, dtype)


@pytest.mark.parametrize("new", [130, 300])
def test_attend_prompt(new):
    """A chain of any length: a prompt in one piece, and the second piece of one."""
    g = gen(new)
    cache, blocks = fill_cache(g, BF16, 2, 2, 32, 128, 500, False)
    check_attend(g, cache, blocks, [new, new - 100], [new, 450], 4, BF16)


def trees(rng, counts):
    words = []
    for c in counts:
        own = []
        for i in range(c):
            own.append((1 << i) | (own[rng.integers(max(0, i - 4), i)] if i else 0))
        words += own
    return torch.from_numpy(np.array(words, np.uint64).view(np.int64)).cuda()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype, dim, hq, hkv", [(BF16, 128, 8, 2), (F16, 64, 3, 3), (F16, 128, 32, 4)])
def test_attend_tree(dtype, dim, hq, hkv, int8):
    g, rng = gen(hq), np.random.default_rng(hq)
    counts, lens = [1, 5, 64, 16, 33], [1, 5, 2000, 100, 40]
    cache, blocks = fill_cache(g, dtype, len(lens), hkv, 48, dim, max(lens), int8)
    check_attend(g, cache, blocks, counts, lens, hq, dtype, mask=trees(rng, counts))


@pytest.mark.parametrize("int8", [False, True])
def test_attend_rows_that_see_nothing(int8):
    """A mask without a bit on a sequence of new tokens alone, a sequence of no tokens: zeros.  A bit of its own only."""
    g = gen(3)
    counts, lens = [4, 2, 64], [4, 60, 64]
    mask = torch.zeros(70, dtype=torch.int64, device="cuda")
    mask[1], mask[3] = 2, 5
    mask[6 + 63] = -(1 << 63)  # the last bit
    cache, blocks = fill_cache(g, BF16, 3, 2, 16, 128, 64, int8)
    q, got = check_attend(g, cache, blocks, counts, lens, 4, BF16, mask=mask)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (got[6:6 + 63] == 0).all() and got[6 + 63].abs().max() > 0
    empty = cache.attend(q[:2], torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), blocks[:2], 1,
                         out=torch.ones_like(q[:2]))
    assert (empty == 0).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("mask", [False, True])
def test_attend_nothing_from_behind_the_end(int8, mask):
    """Behind a sequence's end its last page holds infinities and NaN, and its blocks entries that are no pages: none of it shows."""
    g, rng = gen(7), np.random.default_rng(7)
    counts, lens = [5, 1, 9], [37, 16, 100]
    cache, blocks = fill_cache(g, F16, 3, 2, 16, 64, 400, int8)
    words = trees(rng, counts) if mask else None
    q, want = check_attend(g, cache, blocks, counts, lens, 4, F16, mask=words)
    bad = [math.nan, math.inf, -math.inf]
    for b, n in enumerate(lens):
        page = int(blocks[b, n // 16])
        if int8:
            cache.k_scale[page, :, n % 16:], cache.v_scale[page, :, n % 16:] = bad[b], math.nan
        else:
            cache.k[page, :, n % 16:], cache.v[page, :, n % 16:] = bad[b], bad[2 - b]
        blocks[b, n // 16 + 1:] = [-1, 1 << 30, -(1 << 31)][b]
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = np.concatenate(([0], np.cumsum(counts))).tolist()
    words = None if words is None else torch.cat((words, words[:2]))
    got = cache.attend(q, index(starts), index(lens), blocks, 9, mask=words)
    assert torch.equal(got[:15], want[:15])


def test_attend_values_that_are_not_finite():
    """An infinity in a drafted token's value reaches the rows that see that token and no other."""
    g = gen(8)
    cache, blocks = fill_cache(g, BF16, 1, 1, 16, 128, 64, False)
    mask = torch.tensor([1, 3, 5], dtype=torch.int64, device="cuda")  # two branches behind the first token
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, BF16, 3, 2, 128)
    args = (q, index([0, 3]), index([50]), blocks, 3)
    want = cache.attend(*args, mask=mask)
    at = 48  # the second of the new tokens 47, 48, 49
    cache.v[blocks[0, at // 16].long(), 0, at % 16, 7] = math.inf
    got = cache.attend(*args, mask=mask)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert not torch.isfinite(got[1, :, 7]).any()
    keep = [i for i in range(128) if i != 7]
    assert torch.equal(got[1][:, keep], want[1][:, keep])


def test_attend_pages_that_are_not_there():
    """A block outside the cache inside a sequence holds no tokens."""
    g = gen(9)
    cache, blocks = fill_cache(g, BF16, 1, 2, 16, 64, 96, False)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, BF16, 1, 2, 64)
    holes = blocks.clone()
    holes[0, 2], holes[0, 4] = -1, cache.k.shape[0]
    packed = blocks[:, [0, 1, 3, 5]]
    a = cache.attend(q, index([0, 1]), index([96]), holes, 1)
    b = cache.attend(q, index([0, 1]), index([64]), packed.contiguous(), 1)
    assert (a.double() - b.double()).abs().max() <= 2 ** -7 * b.abs().max()


# many rows of heads of 128 over sequences that may be long: 128 rows of a work-group
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tree", [False, True])
def test_attend_many_rows(dtype, int8, tree):
    g, rng = gen(50), np.random.default_rng(50)
    counts, lens = [34, 0, 1, 20, 64, 33, 17, 5], [1000, 50, 1, 20, 600, 33, 97, 1024]
    cache, blocks = fill_cache(g, dtype, 8, 8, 48, 128, 1024, int8)
    check_attend(g, cache, blocks, counts, lens, 32, dtype, mask=trees(rng, counts) if tree else None)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts, lens, hq", [([300, 129], [300, 1500], 16), ([128, 1], [2047, 2048], 8), ([65, 97], [96, 1000], 8), ([33, 34], [33, 66], 24)])
def test_attend_prompts_of_long_sequences(counts, lens, hq, dtype, int8):
    g = gen(51)
    cache, blocks = fill_cache(g, dtype, 2, 8, 16, 128, 4096, int8)
    check_attend(g, cache, blocks, counts, lens, hq, dtype)


@pytest.mark.parametrize("int8", [False, True])
def test_attend_many_rows_that_see_nothing(int8):
    g = gen(52)
    counts, lens = [4, 2, 64, 0, 64], [4, 60, 64, 0, 700]
    mask = torch.zeros(134, dtype=torch.int64, device="cuda")
    mask[1], mask[3] = 2, 5
    mask[6 + 63] = -(1 << 63)  # the last bit
    cache, blocks = fill_cache(g, BF16, 5, 8, 16, 128, 2048, int8)
    q, got = check_attend(g, cache, blocks, counts, lens, 16, BF16, mask=mask)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (got[6:6 + 63] == 0).all() and got[6 + 63].abs().max() > 0


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("mask", [False, True])
def test_attend_many_rows_nothing_from_behind_the_end(int8, mask):
    g, rng = gen(53), np.random.default_rng(53)
    counts, lens = [40, 33, 64], [137, 48, 900]
    cache, blocks = fill_cache(g, F16, 3, 8, 16, 128, 4096, int8)
    words = trees(rng, counts) if mask else None
    q, want = check_attend(g, cache, blocks, counts, lens, 32, F16, mask=words)
    bad = [math.nan, math.inf, -math.inf]
    for b, n in enumerate(lens):
        page = int(blocks[b, n // 16])
        if int8:
            cache.k_scale[page, :, n % 16:], cache.v_scale[page, :, n % 16:] = bad[b], math.nan
        else:
            cache.k[page, :, n % 16:], cache.v[page, :, n % 16:] = bad[b], bad[2 - b]
        blocks[b, n // 16 + 1:] = [-1, 1 << 30, -(1 << 31)][b]
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    words = None if words is None else torch.cat((words, words[:2]))
    got = cache.attend(q, index([0, 40, 73, 137]), index(lens), blocks, 64, mask=words)
    assert torch.equal(got[:137], want[:137])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_many_rows_values_that_are_not_finite(dtype):
    """An infinity in a drafted token's value, and a NaN in another's, reach the rows that see them and no others."""
    g, rng = gen(54), np.random.default_rng(54)
    cache, blocks = fill_cache(g, dtype, 1, 8, 16, 128, 8192, False)
    mask = trees(rng, [50])
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, dtype, 50, 32, 128)
    args = (q, index([0, 50]), index([1050]), blocks, 50)
    want = cache.attend(*args, mask=mask)
    for new, head, i, value in ((7, 2, 9, math.inf), (30, 5, 126, math.nan)):
        at = 1000 + new
        cache.v[blocks[0, at // 16].long(), head, at % 16, i] = value
        got = cache.attend(*args, mask=mask)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[((mask >> new) & 1).bool(), 4 * head:4 * head + 4, i] = True
        assert 0 < hit.sum() < 200 and not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want[~hit])
        cache.v[blocks[0, at // 16].long(), head, at % 16, i] = 0
        want = cache.attend(*args, mask=mask)


def test_attend_many_rows_pages_that_are_not_there():
    g = gen(55)
    cache, blocks = fill_cache(g, BF16, 2, 8, 16, 128, 4096, False)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, BF16, 80, 16, 128)
    holes = blocks.clone()
    holes[:, 2], holes[:, 4] = -1, cache.k.shape[0]
    packed = torch.cat((blocks[:, [0, 1, 3]], blocks[:, 5:], blocks[:, [2, 4]]), 1).contiguous()
    a = cache.attend(q, index([0, 40, 80]), index([400, 370]), holes, 40)
    b = cache.attend(q, index([0, 40, 80]), index([368, 338]), packed, 40)
    assert (a.double() - b.double()).abs().max() <= 2 ** -7 * b.abs().max()


@pytest.mark.parametrize("int8", [False, True])
def test_pages_beyond_32_bits(int8):
    """A cache of more than 2^32 bytes and 2^31 elements: tokens go to its last pages and are read there."""
    g = gen(70)
    pages = 36000 if not int8 else 70000
    cache = hipq.KvCache(*(torch.empty((pages, 8, 64, 128), dtype=torch.int8 if int8 else BF16, device="cuda") for _ in range(2)),
                         *(torch.empty((pages, 8, 64), device="cuda") if int8 else None for _ in range(2)))
    assert cache.k.numel() > (1 << 31) and cache.k.numel() * cache.k.element_size() > (1 << 32)
    blocks = torch.tensor([[pages - 1, 1, pages // 2]], dtype=torch.int32, device="cuda")
    n = 150
    at = torch.arange(n, device="cuda")
    slots = (blocks[0, at // 64] * 64 + at % 64).to(torch.int32)
    k, v = randn(g, BF16, n, 8, 128), randn(g, BF16, n, 8, 128)
    cache.append(k, k, v, slots, slots, None)
    if not int8:
        assert torch.equal(tokens_of(cache.v, blocks[0], n), v.transpose(0, 1))
    check_attend(g, cache, blocks, [3], [n], 16, BF16)


@pytest.mark.parametrize("heads, hq, n", [(2, 4, 100), (1, 4, 5000), (8, 64, 4000)])
def test_attend_rows_that_are_not_there(heads, hq, n):
    """Starts in front of the first row, behind the last, falling, at both ends of 32 bits: no row outside is read or written, and the rows of a sequence that is
    in order are what they are among others in order."""
    g = gen(n)
    cache, blocks = fill_cache(g, BF16, 8, heads, 16, 128, n, False)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, BF16, 30, hq, 128)
    top, low = (1 << 31) - 1, -(1 << 31)
    call = lambda starts, lens: cache.attend(q, index(starts), index(lens), blocks, 12, out=torch.full_like(q, 11.0))  # noqa: E731
    want = call([0, 0, 3, 12, 12, 12, 12, 12, 12], [n] * 8)[3:12]
    for starts, end in (([top, low, 3, 12, low, low + 7, -5, -9, low], 12), ([low, low, 3, 12, top, low, 0, -1, low], 24)):
        got = call(starts, [n, top, n, n, low, -1, n, top])
        assert torch.equal(got[3:12], want) and (got[end:] == 11).all() and torch.isfinite(got).all()


def test_attend_over_its_queries():
    """The outputs may lie where the queries lay."""
    g = gen(71)
    for longest in (100, 3000):
        cache, blocks = fill_cache(g, BF16, 2, 2, 16, 128, longest, False)
        q = randn(g, BF16, 20, 8, 128)
        index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        a = (index([0, 9, 20]), index([longest, longest - 30]), blocks, 11)
        want = cache.attend(q, *a)
        assert torch.equal(cache.attend(q, *a, out=q), want)


def test_attend_subnormal_value_scales():
    """Value scales down to the smallest float32: finite outputs, zeros where float16 has none so small."""
    g = gen(72)
    cache, blocks = fill_cache(g, F16, 1, 2, 16, 64, 200, True)
    cache.v_scale.fill_(1e-42)
    q = randn(g, F16, 1, 4, 64)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    assert (cache.attend(q, index([0, 1]), index([200]), blocks, 1) == 0).all()


@pytest.mark.parametrize("int8", [False, True])
def test_attend_long(int8):
    """Split over many work-groups; very different scores; a bound that cuts a length off."""
    g = gen(10)
    cache, blocks = fill_cache(g, BF16, 2, 1, 64, 128, 20000, int8)
    check_attend(g, cache, blocks, [1, 2], [20000, 19999], 4, BF16)
    check_attend(g, cache, blocks, [1, 2], [20000, 17], 4, BF16, scale=2.0)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, BF16, 2, 4, 128)
    assert torch.equal(cache.attend(q, index([0, 1, 2]), index([20000, 300]), blocks, 1, longest=300), cache.attend(q, index([0, 1, 2]), index([300, 300]), blocks, 1, longest=300))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attend_value_scales_of_any_size(dtype):
    """An int8 cache whose values differ by many orders of magnitude from token to token."""
    g = gen(11)
    cache, blocks = fill_cache(g, dtype, 2, 1, 16, 64, 300, True)
    cache.v_scale.copy_(10.0 ** (torch.rand(cache.v_scale.shape, device="cuda", generator=g) * 4 - 3 if dtype == BF16 else torch.rand(cache.v_scale.shape, device="cuda", generator=g) * 2 - 1))
    check_attend(g, cache, blocks, [1, 1], [300, 123], 4, dtype)
    cache.v_scale.mul_(1e-6)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = randn(g, dtype, 2, 4, 64)
    small = cache.attend(q, index([0, 1, 2]), index([300, 123]), blocks, 1)
    assert torch.isfinite(small).all()


# ---- sampling --------------------------------------------------------------------------------------------------------------
def check_sample(logits, u, t=None, k=None, p=None, m=None):
    r = logits.shape[0]
    f = lambda v, d: torch.tensor(v, dtype=d, device="cuda") if v is not None else None  # noqa: E731
    got = hipq.sample(logits, f(u, F32), f(t, F32), f(k, torch.int32), f(p, F32), f(m, F32)).tolist()
    x = logits.cpu()
    n = lambda v, i, d: d if v is None else float(np.float32(v[i]))  # noqa: E731
    want = [ref.sample(x[i], n(u, i, 0), n(t, i, 1.0), 0 if k is None else k[i], n(p, i, 1.0), n(m, i, 0.0)) for i in range(r)]
    assert got == want, [(i, a, b) for i, (a, b) in enumerate(zip(got, want)) if a != b][:5]
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("v", [1, 2, 7, 64, 1000, 4097, 50257])
def test_sample_filters(v, dtype):
    rng, g = np.random.default_rng(v), gen(v)
    r = 24
    x = (torch.randn((r, v), device="cuda", generator=g) * 2.5).to(dtype)
    u = rng.random(r).astype(np.float32).tolist()
    t = rng.uniform(0.3, 2, r).tolist()
    k = [0, 1, 2, 5, 50, 300, v, v + 1] * 3
    p = rng.uniform(0.05, 1.05, r).tolist()
    m = np.maximum(0, rng.uniform(-0.1, 0.1, r)).tolist()
    check_sample(x, u)
    check_sample(x, u, t=t)
    check_sample(x, u, t=t, k=k)
    check_sample(x, u, t=t, p=p)
    check_sample(x, u, t=t, m=m)
    check_sample(x, u, t=t, k=k, p=p, m=m)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_ties(dtype):
    """Rows of one score, of two, of few: the first by index are kept, and more of them than a list holds."""
    rng = np.random.default_rng(1)
    v = 9000
    x = torch.stack([torch.zeros(v), torch.arange(v) % 2 * 1.0, torch.arange(v) % 5 * 0.25, (torch.arange(v) >= 4500) * 3.0, torch.arange(v) % 3 * -1e-3]).repeat(8, 1).to(dtype).cuda()
    r = x.shape[0]
    u = rng.random(r).tolist()
    k = [1, 7, 4500, 4501, 8999, 100, 6000, 3, 5000, 0] * 4
    p = rng.uniform(0.01, 0.99, r).tolist()
    check_sample(x, u, k=k)
    check_sample(x, u, p=p)
    check_sample(x, u, k=k, p=p, m=[0.5, 0.0] * 20)


def test_sample_ends_of_uniform_and_odd_parameters():
    x = torch.tensor([[0.0, 1.0, 2.0, 3.0]] * 10).cuda()
    check_sample(x, [0.0, 1 - 2 ** -24, 0.5, 0.1, 0.9, 0.3, 0.6, 0.0, 0.99, 0.2], t=[1, 1, 0, -1, 1, 1, 1e-6, 1e6, 1, 1], k=[0, 0, 2, 1, -3, 2, 0, 0, 4, 1],
                 p=[1, 1, 1, 1, 0, 0.0, 1, 1, 2, 1], m=[0, 0, 0, 0, 0, 0, 0, 0, 1.0, 5.0])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_sample_infinities_and_nan(dtype):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, nan, -inf, nan], [-inf, 1, nan, 2], [inf, 1, inf, 2], [inf, -inf, nan, 2], [-inf, -inf, 0, -inf], [0.0, -0.0, -inf, 0.0]] * 3, dtype=dtype).cuda()
    r = x.shape[0]
    got = check_sample(x, [0.0, 0.7, 0.6, 0.9, 0.99, 0.5] * 3, t=[1.0] * 12 + [0.0] * 6, k=[0] * 6 + [2] * 12, p=[1] * 6 + [0.9] * 12)
    assert got[0] == -1 and got[2] == 2 and got[12] == -1


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sample_last_token_that_top_p_keeps(dtype):
    """Rows with top-p alone whose border is a heavy token, which is the answer as often as not: left out by any part of the work-group, it
    would make another token of the row.  Every call gives the same."""
    rng = np.random.default_rng(12)
    r, v = 320, 700
    x = torch.from_numpy(rng.standard_normal((r, v)) * 0.1 - 9.0)
    heavy = rng.integers(2, 6, r)
    for i in range(r):  # the heavy tokens weigh about the same, the others all together 700 e^-9 of one
        x[i, torch.from_numpy(rng.choice(v, heavy[i], replace=False))] = torch.from_numpy(rng.uniform(-0.2, 0.2, heavy[i]))
    x, u, p = x.to(dtype).cuda(), rng.random(r).astype(np.float32).tolist(), (rng.uniform(0.2, 0.95, r)).tolist()
    first = check_sample(x, u, p=p)
    f = lambda n: torch.tensor(n, dtype=F32, device="cuda")  # noqa: E731
    for _ in range(20):
        assert hipq.sample(x, f(u), top_p=f(p)).tolist() == first


def test_sample_rows_with_gaps_and_odd_addresses():
    g = gen(4)
    wide = (torch.randn((9, 1003), device="cuda", generator=g) * 2).to(BF16)
    check_sample(wide[:, 1:1000], np.linspace(0, 0.99, 9).tolist(), k=[40] * 9, p=[0.9] * 9)


def test_sample_large_vocabulary():
    g = gen(5)
    x = torch.randn((4, 200001), device="cuda", generator=g) * 3
    check_sample(x, [0.1, 0.5, 0.9, 0.999], t=[1.0, 0.7, 1.5, 1.0], k=[0, 0, 20000, 50], p=[0.95, 0.999, 0.9, 0.8], m=[0, 1e-3, 0, 0])


def test_sample_millions_of_rows():
    """More rows than one launch has: 2^22 and some of them, the last with filters of their own."""
    g, r = gen(13), (1 << 22) + 3
    x, u = (torch.randn((r, 2), device="cuda", generator=g) * 2).to(F16), torch.rand(r, device="cuda", generator=g)
    p = torch.ones(r, device="cuda")
    p[-2:] = 0.0  # the first alone
    w = torch.softmax(x.double(), 1)
    want = (u.double() >= w[:, 0]).long()  # (a number as near to a border as 2^-40 may fall on either side: none does)
    want[-2:] = x[-2:].argmax(1)
    assert ((u.double() - w[:, 0]).abs() > 2.0 ** -36).all()
    assert torch.equal(hipq.sample(x, u, top_p=p), want)
    k = torch.zeros(r, dtype=torch.int32, device="cuda")
    k[-2:] = 1
    assert torch.equal(hipq.sample(x, u, temperature=torch.ones(r, device="cuda"), top_k=k, min_p=torch.zeros(r, device="cuda")), want)


# ---- together, on streams and in graphs ------------------------------------------------------------------------------------
def decoder(g, dtype, hidden=256, hq=4, hkv=2, dim=64, inner=320, vocab=1000, page=16, pages=40, int8=False):
    mk = lambda n, k, **kw: hipq.LinearW4(ref.pack_rows(torch.randint(0, 16, (n, k), dtype=torch.uint8, device="cuda", generator=g)),  # noqa: E731
                                          (torch.rand((n, k // 32), device="cuda", generator=g) * 0.01 + 0.005).to(dtype), 32, **kw)
    return dict(qkv=mk((hq + 2 * hkv) * dim, hidden), out=mk(hidden, hq * dim), up=mk(2 * inner, hidden, activation="silu"), down=mk(hidden, inner), head=mk(vocab, hidden),
                cache=new_cache(dtype, pages, hkv, page, dim, int8), table=hipq.rotation_table(500, dim), hq=hq, hkv=hkv, dim=dim, page=page,
                norm=torch.ones(dim, dtype=dtype, device="cuda"))


def rms(x):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


def decode_step(d, x, positions, slots, starts, lens, blocks, most, u, mask=None):
    n = x.shape[0]
    qkv = d["qkv"](rms(x)).view(n, d["hq"] + 2 * d["hkv"], d["dim"])
    q, k, v = qkv[:, :d["hq"]], qkv[:, d["hq"]:d["hq"] + d["hkv"]], qkv[:, d["hq"] + d["hkv"]:]
    q = d["cache"].append(q, k, v, positions, slots, d["table"], q_norm=d["norm"], k_norm=d["norm"])
    a = d["cache"].attend(q, starts, lens, blocks, most, mask=mask)
    x = x + d["out"](a.view(n, -1))
    x = x + d["down"](d["up"](rms(x)))
    logits = d["head"](rms(x))
    return logits, hipq.sample(logits, u, top_k=torch.full((n,), 50, dtype=torch.int32, device="cuda"), top_p=torch.full((n,), 0.9, device="cuda"))


def places(b, n_from, n_to, blocks, page):
    at = torch.arange(n_from, n_to, device="cuda")
    return (blocks[:, at // page] * page + (at % page).to(torch.int32)).reshape(-1).to(torch.int32), at.to(torch.int32).repeat(b)


@pytest.mark.parametrize("int8", [False, True])
def test_a_prompt_at_once_and_token_by_token(int8):
    """A step of everything together: the last token's scores are the same whether the prompt goes in as one piece, token by token, or as a
    chain written as a tree, up to the roundings of 16-bit activations on the way."""
    b, n = 3, 37
    results = []
    for way in ("once", "single", "tree"):
        g = gen(20)
        d = decoder(g, BF16, int8=int8)
        x = randn(g, BF16, b, n, 256)
        blocks = torch.randperm(40, device="cuda", generator=g)[:b * 3].view(b, 3).to(torch.int32)
        u = torch.full((b * n,), 0.3, device="cuda")
        if way == "single":
            for i in range(n):
                slots, positions = places(b, i, i + 1, blocks, 16)
                logits, token = decode_step(d, x[:, i].contiguous(), positions, slots, torch.arange(b + 1, dtype=torch.int32, device="cuda"),
                                            torch.full((b,), i + 1, dtype=torch.int32, device="cuda"), blocks, 1, u[:b])
        else:
            slots, positions = places(b, 0, n, blocks, 16)
            mask = None if way == "once" else (2 ** torch.arange(1, n + 1, dtype=torch.int64, device="cuda") - 1).repeat(b)
            logits, token = decode_step(d, x.view(b * n, 256), positions, slots, torch.arange(b + 1, dtype=torch.int32, device="cuda") * n,
                                        torch.full((b,), n, dtype=torch.int32, device="cuda"), blocks, n, u, mask)
            logits, token = logits.view(b, n, -1)[:, -1], token.view(b, n)[:, -1]
        for i in range(b):
            assert int(token[i]) == ref.sample(logits[i].cpu(), float(np.float32(0.3)), 1.0, 50, float(np.float32(0.9)), 0.0)
        results.append(logits.double())
    spread = results[0].std()
    # one layer: five roundings to bfloat16 (2^-8) between the inputs and the scores, each spread over many terms
    assert (results[1] - results[0]).abs().max() < 8 * 2 ** -8 * spread and (results[2] - results[0]).abs().max() < 8 * 2 ** -8 * spread


def test_a_captured_step_replayed():
    """A decoding step in a graph: replays with new inputs in the same memory, eager work of the same operators between them."""
    g = gen(30)
    b = 4
    d = decoder(g, BF16)
    blocks = torch.randperm(40, device="cuda", generator=g)[:b * 3].view(b, 3).to(torch.int32)
    x, u = randn(g, BF16, b, 256), torch.rand(b, device="cuda", generator=g)
    lens, positions, slots = (torch.zeros(b, dtype=torch.int32, device="cuda") for _ in range(3))
    starts = torch.arange(b + 1, dtype=torch.int32, device="cuda")

    def place(i):
        s, p = places(b, i, i + 1, blocks, 16)
        slots.copy_(s), positions.copy_(p), lens.fill_(i + 1)
    place(0)
    decode_step(d, x, positions, slots, starts, lens, blocks, 1, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, tokens = decode_step(d, x, positions, slots, starts, lens, blocks, 1, u)
    for i in range(6):
        place(i)
        x.copy_(randn(g, BF16, b, 256))
        u.copy_(torch.rand(b, device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        seen, chosen = logits.clone(), tokens.clone()
        want, want_tokens = decode_step(d, x, positions, slots, starts, lens, blocks, 1, u)
        assert torch.equal(seen, want) and torch.equal(chosen, want_tokens)


def test_two_streams_at_once():
    """The same plan and cache on two streams: workspaces are a call's own."""
    g = gen(40)
    w = weights(g, BF16, 512, 512, 128)
    plan = hipq.LinearW4(ref.pack_rows(w[0]), w[1], 128, zeros=w[2], bias=w[3])
    cache, blocks = fill_cache(g, BF16, 2, 2, 16, 64, 3000, False)
    index = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    starts, lens = index([0, 1, 2]), index([3000, 2500])
    xs, qs = [randn(g, BF16, 400, 512) for _ in range(2)], [randn(g, BF16, 2, 4, 64) for _ in range(2)]
    want = [(plan(x), cache.attend(q, starts, lens, blocks, 1)) for x, q in zip(xs, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append((plan(xs[s]), cache.attend(qs[s], starts, lens, blocks, 1)))
    torch.cuda.synchronize()
    for s in range(2):
        for y, o in got[s]:
            assert torch.equal(y, want[s][0]) and torch.equal(o, want[s][1])
