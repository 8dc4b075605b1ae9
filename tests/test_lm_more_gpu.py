"""Experts, the cache held to a budget and penalties on the GPU, against their formulas in 64 bits (lm_more_reference.py)."""
import math

import numpy as np
import pytest
import torch

import lm_more_reference as more
import lm_reference as ref
from lm_bounds import rms, rounded
from nart_amd import hipq

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, dtype, *shape):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def whole(g, lo, hi, dtype, *shape):
    return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=g)


# ---- experts --------------------------------------------------------------------------------------------------------
class Layer:
    """The weights of a layer of experts, unpacked, and its plan."""

    def __init__(self, g, dtype, experts, k, inner, n, top, group=128, zeros=True, act="silu", scores="softmax", normalize=True):
        scales = lambda *shape: (torch.rand(shape, device="cuda", generator=g) * 0.02 + 0.002).to(dtype)  # noqa: E731
        points = lambda *shape: whole(g, 0, 16, torch.uint8, *shape) if zeros else None  # noqa: E731
        self.up, self.down = whole(g, 0, 16, torch.uint8, experts, 2 * inner, k), whole(g, 0, 16, torch.uint8, experts, n, inner)
        self.up_scales, self.down_scales = scales(experts, 2 * inner, -(-k // group)), scales(experts, n, -(-inner // group))
        self.up_zeros, self.down_zeros = points(experts, 2 * inner, -(-k // group)), points(experts, n, -(-inner // group))
        self.how = dict(act=act, scores=scores, normalize=normalize)
        self.top, self.group, self.experts, self.k, self.dtype = top, group, experts, k, dtype
        pack = lambda q: ref.pack_rows(q.flatten(0, 1)).view(q.shape[0], q.shape[1], -1)  # noqa: E731
        self.plan = hipq.ExpertsW4(pack(self.up), self.up_scales, pack(self.down), self.down_scales, top, group, gate_up_zeros=self.up_zeros, down_zeros=self.down_zeros,
                                   activation=act, scores=scores, normalize=normalize)

    def want(self, x, logits):
        return more.experts(x, logits, self.up, self.up_scales, self.down, self.down_scales, self.top, self.group, self.up_zeros, self.down_zeros, **self.how)

    def check(self, x, logits, y=None):
        got = self.plan(x, logits, y)
        want, off, spread = self.want(x, logits)
        ok, far = ref.within(got, want, off)
        assert ok, "%s: %g too far" % (self.plan.kernel(x.shape[0]), far)
        if want.numel() >= 1000:  # roundings are independent: 1.2 times what those of the hidden rows and of the result leave (lm_bounds.py)
            far, may = rms(got.double() - want), 1.2 * torch.sqrt(rms(rounded(want, got.dtype)).square() + rms(spread).square())
            assert far <= may, "%g away, %g allowed" % (far, may)
        return got


@pytest.mark.parametrize("m", [1, 2, 3, 8, 15, 16, 17, 33, 64, 65, 100, 129, 300, 700])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_experts_rows(m, dtype):
    g = gen(m)
    layer = Layer(g, dtype, 5, 288, 160, 200, 2)
    layer.check(randn(g, dtype, m, 288), randn(g, F32, m, 5))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("experts, top, k, inner, n", [(1, 1, 32, 32, 1), (2, 2, 64, 96, 17), (7, 3, 160, 32, 130), (65, 6, 96, 288, 33), (3, 1, 1056, 544, 257), (16, 16, 128, 64, 48)])
@pytest.mark.parametrize("m", [1, 5, 40, 400])
def test_experts_shapes(m, experts, top, k, inner, n, group):
    g = gen(n + k + m)
    dtype = BF16 if n % 2 else F16
    layer = Layer(g, dtype, experts, k, inner, n, top, group, zeros=n != 17, act="gelu" if n == 33 else "silu", scores="sigmoid" if top == 3 else "softmax", normalize=k != 96)
    layer.check(randn(g, dtype, m, k), randn(g, F32, m, experts))


@pytest.mark.parametrize("dtype, group, zeros", [(BF16, 128, False), (F16, 128, True), (BF16, 64, True), (F16, 64, False), (BF16, 32, True), (F16, 32, False)])
@pytest.mark.parametrize("m, experts, top, kernel", [(3, 8, 2, "w4_experts_stream_4"), (24, 40, 3, "w4_experts_stream_4"), (16, 8, 4, "w4_experts_stream_16"), (60, 30, 3, "w4_experts_stream_16"), (40, 8, 2, "w4_experts_16x128"), (60, 4, 2, "w4_experts_32x128"), (100, 4, 2, "w4_experts_64x128"), (1500, 4, 2, "w4_experts_128x256")])
def test_experts_kernels(m, experts, top, kernel, dtype, group, zeros):
    """Every kernel, with reductions that end inside a block and are shared by work-groups."""
    g = gen(m + group)
    layer = Layer(g, dtype, experts, 1056, 2080, 300, top, group, zeros)
    layer.check(randn(g, dtype, m, 1056), randn(g, F32, m, experts))
    assert layer.plan.kernel(m) == kernel


@pytest.mark.parametrize("scores, normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("logits", [F32, F16, BF16])
@pytest.mark.parametrize("m", [6, 150])
def test_experts_scores(scores, normalize, logits, m):
    """Equal scores, infinite ones, NaN, tokens with fewer experts than `top` and with none, large and small scores."""
    g = gen(7)
    layer = Layer(g, BF16, 70, 64, 64, 40, 4, 64, scores=scores, normalize=normalize)
    x, s = randn(g, BF16, m, 64), (randn(g, F32, m, 70) * 3).to(logits)
    s[0] = 0.5                 # all the same: the first four
    s[1] = -math.inf
    s[1, 69] = -50.0           # one expert
    s[2] = math.nan
    s[2, 3] = s[2, 66] = 2.0   # two
    s[3] = -math.inf           # none
    s[4, 5] = s[4, 64] = math.inf
    s[5] = -200.0 - torch.arange(70, device="cuda")  # sigmoids that are 0 in 32 bits
    got = layer.check(x, s)
    assert (got[3] == 0).all()


@pytest.mark.parametrize("m", [4, 130])
def test_experts_all_of_one(m):
    """Every token chooses the same experts; the others have no rows.  And one of 1024 experts, 16 of them for a token."""
    g = gen(m)
    layer = Layer(g, BF16, 9, 96, 64, 80, 2, 32)
    s = randn(g, F32, m, 9)
    s[:, 8] += 100
    s[:, 3] += 100
    layer.check(randn(g, BF16, m, 96), s)
    layer = Layer(g, F16, 1024, 32, 32, 16, 16, 32)
    layer.check(randn(g, F16, m, 32), randn(g, F32, m, 1024))


@pytest.mark.parametrize("m, experts, top", [(1, 5, 2), (9, 40, 3), (40, 60, 4), (60, 7, 1), (300, 3, 1)])
def test_experts_wide_outputs(m, experts, top):
    """More tiles of outputs than CUs, which other numbers of waves compute."""
    g = gen(m)
    layer = Layer(g, BF16, experts, 64, 160, 4200, top, 32)
    layer.check(randn(g, BF16, m, 64), randn(g, F32, m, experts))


@pytest.mark.parametrize("m, experts, top", [(3000, 5, 3), (9000, 300, 1)])
def test_experts_many_pairs(m, experts, top):
    """More pairs than one work-group numbers at once."""
    g = gen(m)
    layer = Layer(g, F16, experts, 64, 32, 40, top, 64)
    layer.check(randn(g, F16, m, 64), randn(g, F32, m, experts))


@pytest.mark.parametrize("dtype, group, zeros", [(BF16, 128, False), (F16, 128, True), (BF16, 64, True), (F16, 64, False), (BF16, 32, True), (F16, 32, False)])
@pytest.mark.parametrize("experts, top", [(4, 4), (64, 6), (70, 5), (256, 16), (257, 3)])
def test_experts_of_one_token(experts, top, dtype, group, zeros):
    """One token, which has kernels of its own: ordinary scores, equal ones, fewer experts than `top`, none, the last ones alone."""
    g = gen(experts + group)
    layer = Layer(g, dtype, experts, 288, 160, 100, top, group, zeros, scores="sigmoid" if top == 5 else "softmax", normalize=top != 6)
    x = randn(g, dtype, 1, 288)
    for kind in range(5):
        s = randn(g, F32, 1, experts)
        if kind == 1:
            s[:] = 0.25
        elif kind == 2:
            s[:, 1:] = -math.inf
        elif kind == 3:
            s[:] = math.nan
        elif kind == 4:
            s[:, -top:] += 50
        got = layer.check(x, s)
        if kind == 3:
            assert (got == 0).all()


@pytest.mark.parametrize("dtype, group, zeros", [(BF16, 128, False), (F16, 64, True), (BF16, 32, True)])
@pytest.mark.parametrize("experts, top", [(3, 1), (8, 4), (64, 6), (70, 16), (256, 16), (257, 5)])
@pytest.mark.parametrize("m", [2, 3, 4, 5])
def test_experts_of_up_to_four_tokens(m, experts, top, dtype, group, zeros):
    """They have kernels of their own: experts that they share, all, some and none of them, tokens without any, rows with gaps between them."""
    g = gen(experts + group + m)
    layer = Layer(g, dtype, experts, 288, 160, 100, top, group, zeros, scores="sigmoid" if top == 5 else "softmax", normalize=top != 6)
    x = randn(g, dtype, m, 320)[:, :288]
    for kind in range(4):
        s = randn(g, F32, m, experts + 3)[:, 1:experts + 1]
        if kind == 1:
            s[:] = s[:1].clone()       # the same for all
        elif kind == 2:
            s[0] = -math.inf           # none
            s[m - 1, 1:] = math.nan    # one
        elif kind == 3:
            s[:, -1] += 50             # one that all have
        got = layer.check(x, s)
        if kind == 2:
            assert (got[0] == 0).all()


@pytest.mark.parametrize("m, experts", [(3, 4), (14, 4), (40, 30), (60, 3), (200, 4), (900, 4)])
def test_experts_rows_that_are_not_finite(m, experts):
    """An infinity or NaN in a row of x stays in its token's result."""
    g = gen(m)
    layer = Layer(g, BF16, experts, 256, 128, 90, 2, 64)
    x, s = randn(g, BF16, m, 256), randn(g, F32, m, experts)
    clean = layer.plan(x, s)
    x[1, 5], x[m - 1, 200] = math.inf, math.nan
    got = layer.plan(x, s)
    assert torch.isnan(got[1]).all() and torch.isnan(got[m - 1]).all()
    same = [i for i in range(m) if i not in (1, m - 1)]
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("m", [1, 5, 24, 200])
def test_experts_rows_with_gaps(m):
    g = gen(m)
    x, y, s = randn(g, BF16, m, 400), torch.full((m + 2, 77), 7.0, dtype=BF16, device="cuda"), randn(g, BF16, m, 30)
    Layer(g, BF16, 6, 320, 64, 70, 2, 64).check(x[:, 16:16 + 320], s[:, 5:11], y=y[1:m + 1, 3:73])
    assert (y[0] == 7).all() and (y[m + 1] == 7).all() and (y[:, :3] == 7).all() and (y[:, 73:] == 7).all()


def test_experts_more_dimensions_and_no_rows():
    g = gen(1)
    layer = Layer(g, BF16, 4, 64, 64, 40, 2, 32)
    x, s = randn(g, BF16, 2, 3, 64), randn(g, F32, 2, 3, 4)
    assert torch.equal(layer.plan(x, s).view(6, 40), layer.plan(x.view(6, 64), s.view(6, 4)))
    assert layer.plan(x[:0, 0], s[:0, 0]).shape == (0, 40)


@pytest.mark.parametrize("m", [1, 3, 9, 40, 200, 900])
def test_experts_same_result_every_time(m):
    """Also in a captured graph, with other calls and other inputs between its replays, and on another stream."""
    g = gen(m)
    layer = Layer(g, BF16, 12, 512, 256, 300, 3)
    x, s = randn(g, BF16, m, 512), randn(g, F32, m, 12)
    first = layer.plan(x, s)
    y = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.plan(x, s, y)
    for i in range(4):
        other_x, other_s = randn(g, BF16, m, 512), randn(g, F32, m, 12)
        want = layer.plan(other_x, other_s)
        before = x.clone(), s.clone()
        x.copy_(other_x), s.copy_(other_s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        x.copy_(before[0]), s.copy_(before[1])
        assert torch.equal(layer.plan(x, s), first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = layer.plan(x, s)
    stream.synchronize()
    assert torch.equal(again, first)


@pytest.mark.parametrize("sizes", [(1, 3), (2, 30), (4, 200), (60, 900)])
def test_experts_two_calls_at_once(sizes):
    """One layer on two streams, and in two graphs that are replayed side by side."""
    g = gen(sum(sizes))
    layer = Layer(g, BF16, 12, 512, 256, 300, 3)
    inputs = [(randn(g, BF16, m, 512), randn(g, F32, m, 12)) for m in sizes]
    want = [layer.plan(x, s) for x, s in inputs]
    outputs, streams, graphs = [torch.zeros_like(w) for w in want], [torch.cuda.Stream() for _ in sizes], [torch.cuda.CUDAGraph() for _ in sizes]
    for (x, s), y, graph in zip(inputs, outputs, graphs):
        with torch.cuda.graph(graph):
            for _ in range(3):
                layer.plan(x, s, y)
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for (x, s), stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                got.append(layer.plan(x, s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    for _ in range(4):
        for y in outputs:
            y.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(outputs, want))


# ---- penalties --------------------------------------------------------------------------------------------------------
def check_penalized(x, out=None, **kw):
    before = x.clone()
    got = hipq.penalize(x, out=out, **kw)
    want, off = more.penalize(before, **{k: None if v is None else v.cpu() for k, v in kw.items()})
    finite = torch.isfinite(want)
    got = got.cpu()
    assert torch.equal(got.double()[~finite].nan_to_num(nan=7.0), want[~finite].nan_to_num(nan=7.0))
    untouched = finite & (off == 0)
    if "bias" not in kw:
        assert torch.equal(got.double()[untouched], want[untouched])
    ok, far = ref.within(got[finite], want[finite], off[finite])
    assert ok, far
    return got


def everything(g, rows, vocab, longest, biases):
    lens = whole(g, 0, longest + 1, torch.int32, rows)
    return dict(tokens=(torch.rand((rows, longest), device="cuda", generator=g).pow(3) * vocab).to(torch.int32), lens=lens,
                prompt_lens=(lens * torch.rand(rows, device="cuda", generator=g)).to(torch.int32), repetition=torch.rand(rows, device="cuda", generator=g) + 0.7,
                frequency=torch.rand(rows, device="cuda", generator=g) - 0.2, presence=torch.rand(rows, device="cuda", generator=g) - 0.2,
                bias_tokens=whole(g, 0, vocab, torch.int32, rows, biases), bias=randn(g, F32, rows, biases) * 5,
                allowed=whole(g, -2 ** 31, 2 ** 31, torch.int64, rows, -(-vocab // 32)).to(torch.int32))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows, vocab, longest, biases", [(1, 1, 1, 1), (3, 7, 20, 2), (2, 33, 5, 40), (5, 4096, 100, 9), (4, 4097, 3000, 300), (1, 50257, 700, 5), (7, 16383, 40, 1),
                                                          (300, 20001, 60, 3), (513, 130, 9, 2)])
def test_penalize(rows, vocab, longest, biases, dtype):
    g = gen(rows + vocab)
    kw = everything(g, rows, vocab, longest, biases)
    x = randn(g, dtype, rows, vocab) * 3
    got = check_penalized(x, **kw)
    assert torch.equal(hipq.penalize(x, out=x, **kw).cpu(), got)  # in place


@pytest.mark.parametrize("which", [(), ("tokens",), ("tokens", "lens", "repetition"), ("tokens", "frequency"), ("tokens", "presence", "prompt_lens"), ("bias_tokens", "bias"), ("allowed",)])
def test_penalize_parts(which):
    g = gen(len(which))
    kw = everything(g, 6, 9000, 50, 7)
    check_penalized(randn(g, BF16, 6, 9000), **{k: kw[k] for k in which})


def test_penalize_rows_with_gaps():
    """Rows of scores, tokens, biases and bits inside wider ones; what lies between the results' rows stays."""
    g = gen(3)
    kw = everything(g, 4, 3001, 30, 6)
    wide = lambda t: torch.cat((t, t[:, :5]), 1)[:, :t.shape[1]]  # noqa: E731
    for name in ("tokens", "bias_tokens", "bias", "allowed"):
        kw[name] = wide(kw[name])
    x, out = randn(g, F16, 4, 3010)[:, 3:3004], torch.full((6, 3006), 7.0, dtype=F16, device="cuda")
    check_penalized(x, out=out[1:5, 2:3003], **kw)
    assert (out[0] == 7).all() and (out[5] == 7).all() and (out[:, :2] == 7).all() and (out[:, 3003:] == 7).all()


def test_penalize_edges():
    """Tokens outside of the vocabulary, lengths below zero and beyond the history, the same bias twice, nothing allowed, scores that are not finite, numbers of occurrences
    beyond 16 bits."""
    g = gen(4)
    x = randn(g, F32, 6, 500)
    x[0, 3], x[0, 4], x[0, 5] = math.inf, -math.inf, math.nan
    tokens = whole(g, 0, 500, torch.int32, 6, 70000)
    tokens[:, :8] = torch.tensor([3, 4, 5, -1, 500, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32)
    tokens[1] = 17
    lens = torch.tensor([8, 70000, -5, 100000, 0, 1], dtype=torch.int32, device="cuda")
    value = lambda v: torch.full((6,), v, device="cuda")  # noqa: E731
    at = torch.tensor([[9, 9, -1, 500, 9]] * 6, dtype=torch.int32, device="cuda")
    allowed = torch.full((6, 16), -1, dtype=torch.int32, device="cuda")
    allowed[5] = 0
    got = check_penalized(x, tokens=tokens, lens=lens, prompt_lens=torch.tensor([0, 0, 0, 50000, 0, 7], dtype=torch.int32, device="cuda"), repetition=value(1.25),
                          frequency=value(0.01), presence=value(0.5), bias_tokens=at, bias=randn(g, F32, 6, 5), allowed=allowed)
    assert (got[5] == -math.inf).all()
    assert hipq.penalize(x[:0]).shape == (0, 500) and hipq.penalize(x[:, :0]).shape == (6, 0)


def test_penalize_and_sample_in_a_graph():
    """A masked row goes to the token that is left; replays follow what the inputs hold then."""
    g = gen(5)
    rows, vocab = 5, 1000
    x, kw = randn(g, BF16, rows, vocab), everything(g, rows, vocab, 20, 3)
    out, tokens, uniform = torch.zeros_like(x), torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.rand(rows, device="cuda", generator=g)
    graph = torch.cuda.CUDAGraph()
    hipq.penalize(x, out=out, **kw)
    hipq.sample(out, uniform, out=tokens)
    with torch.cuda.graph(graph):
        hipq.penalize(x, out=out, **kw)
        hipq.sample(out, uniform, out=tokens)
    for only in (3, 999, 31, 32):
        x.copy_(randn(g, BF16, rows, vocab))
        kw["allowed"][0] = 0
        kw["allowed"][0, only // 32] = np.array([1 << only % 32], dtype=np.uint32).view(np.int32)[0].item()
        graph.replay()
        torch.cuda.synchronize()
        assert tokens[0] == only
        assert torch.equal(out, hipq.penalize(x, **kw)) and torch.equal(tokens, hipq.sample(out, uniform))


# ---- the cache ----------------------------------------------------------------------------------------------------------
class Sequences:
    """Sequences of given lengths in a paged cache full of other things."""

    def __init__(self, g, dtype, lens, heads, dim, page, int8, spare=3, more=0):
        rng = np.random.default_rng(len(lens) + sum(lens))
        self.lens, self.page, self.heads, self.dim = lens, page, heads, dim
        per = max(1, -(-max(lens) // page)) + more
        self.pages = len(lens) * per + spare
        self.blocks = rng.permutation(self.pages)[:len(lens) * per].reshape(len(lens), per)
        self.rest = np.setdiff1d(np.arange(self.pages), self.blocks)
        shape = (self.pages, heads, page)
        if int8:
            k, v = (whole(g, -127, 128, torch.int8, *shape, dim) for _ in range(2))
            self.scales = [torch.rand(shape, device="cuda", generator=g) * 0.02 + 0.002 for _ in range(2)]
        else:
            k, v = randn(g, dtype, *shape, dim), randn(g, dtype, *shape, dim)
            self.scales = [None, None]
        self.cache = hipq.KvCache(k, v, *self.scales)
        self.weights = torch.exp(2 * randn(g, F32, *shape))
        self.ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731

    def of(self, pool, b):
        """A sequence's tokens: [heads, len, ...]."""
        n = self.lens[b]
        x = pool[torch.from_numpy(self.blocks[b, :-(-n // self.page)]).long().cuda()]
        return x.transpose(0, 1).reshape(self.heads, x.shape[0] * self.page, *x.shape[3:])[:, :n]

    def all(self, pool):
        return None if pool is None else [self.of(pool, b) for b in range(len(self.lens))]


def check_weighed(g, s, dtype, counts, group, tree=False, scale=None, q_gap=0):
    total = sum(counts)
    q = randn(g, dtype, total + 2, s.heads * group + q_gap, s.dim)[:, :s.heads * group]  # rows of no sequence behind
    starts = [0] + list(np.cumsum(counts))
    mask = None
    if tree:
        rng = np.random.default_rng(total)
        words = rng.integers(0, 2 ** 63, total + 2, dtype=np.int64)
        words[::5] = 0  # rows that see no new token
        mask = torch.from_numpy(words).cuda()
    kw = dict(mask=mask, scale=scale)
    before = s.weights.clone()
    out = torch.full_like(before, 7.0)
    got = s.cache.weigh(q, s.ints(starts), s.ints(s.lens), s.ints(s.blocks), max(counts), s.weights, out=out, **kw)
    assert got is out and torch.equal(before, s.weights)
    want = more.weigh(q, s.all(s.cache.k), starts, s.lens, mask, scale or s.dim ** -0.5, group, s.all(before), s.all(s.cache.k_scale))
    left = torch.ones(before.shape, dtype=torch.bool, device="cuda")
    for b, n in enumerate(s.lens):
        if want[b] is None or n == 0:
            continue
        w, off = want[b]
        have = s.of(out, b).double()
        ok = (have - w).abs() <= off
        assert ok.all(), "sequence %d: %g away, %g allowed" % (b, ((have - w).abs() - off).max() + off[~ok].max(), off[~ok].max())
        for i, p in enumerate(s.blocks[b, :-(-n // s.page)]):
            left[p, :, :min(s.page, n - i * s.page)] = False
    assert (out[left] == 7).all()
    again = s.cache.weigh(q, s.ints(starts), s.ints(s.lens), s.ints(s.blocks), max(counts), s.weights, **kw)  # in place
    assert again is s.weights and torch.equal(again[~left], out[~left]) and torch.equal(again[left], before[left])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens, counts, heads, group, dim, page", [
    ([1], [1], 1, 1, 64, 16), ([2, 33, 0, 17], [1, 1, 0, 1], 2, 4, 128, 16), ([700, 1, 90, 300], [1, 1, 0, 1], 2, 8, 64, 48), ([2500, 31], [3, 31], 1, 5, 128, 64),
    ([64, 65, 300], [64, 40, 1], 2, 3, 256, 32), ([5000], [2], 3, 1, 256, 128), ([1300, 200], [100, 129], 1, 7, 128, 64), ([130, 20], [70, 20], 4, 16, 64, 16)])
@pytest.mark.parametrize("tree", [False, True])
def test_weigh(lens, counts, heads, group, dim, page, int8, dtype, tree):
    if tree and max(counts) > 64:
        pytest.skip("a mask has 64 bits")
    g = gen(sum(lens))
    check_weighed(g, Sequences(g, dtype, lens, heads, dim, page, int8), dtype, counts, group, tree, scale=0.3 if dim == 64 else None, q_gap=group % 3)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("new, group", [(1, 2), (1, 16), (2, 16), (30, 4)])
def test_weigh_long(new, group, int8):
    """Sequences shared by work-groups, as many of them as there may be."""
    g = gen(new)
    check_weighed(g, Sequences(g, BF16, [70001, 16385, 40000], 1, 128, 64, int8), BF16, [new, new // 2 + 1, 1], group)


@pytest.mark.parametrize("new", [1, 40])
def test_weigh_blocks_outside(new):
    """Tokens of blocks outside the cache are not there; lengths beyond `longest` and beyond the blocks end there."""
    g = gen(2)
    s = Sequences(g, BF16, [100, 90], 2, 64, 16, False)
    q = randn(g, BF16, 2 * new, 2, 64)
    starts, blocks = [0, new, 2 * new], s.blocks.copy()
    blocks[0, 1], blocks[1, 2] = -1, s.pages
    out = s.cache.weigh(q, s.ints(starts), s.ints(s.lens), s.ints(blocks), new, s.weights, out=torch.full_like(s.weights, 7.0))
    gone = {0: 1, 1: 2}
    for b in range(2):
        keep = np.array([t for t in range(s.lens[b]) if t // 16 != gone[b]])
        k, old = (s.of(x, b)[:, torch.from_numpy(keep).cuda()] for x in (s.cache.k, s.weights))
        seen = torch.from_numpy(keep[None] - (s.lens[b] - new) <= np.arange(new)[:, None]).cuda()
        for h in range(2):
            x = torch.where(seen, q[starts[b]:starts[b + 1], h].double() @ k[h].double().t() / 8, -math.inf)
            want = torch.softmax(x, -1).sum(0) + torch.where(torch.from_numpy(keep < s.lens[b] - new).cuda(), old[h].double(), 0.0)
            assert ((s.of(out, b)[h, torch.from_numpy(keep).cuda()].double() - want).abs() <= 2.0 ** -17 * want).all()
        page = torch.from_numpy(s.blocks[b, gone[b]:gone[b] + 1]).long().cuda()
        assert (out[page] == 7).all()
    short = s.cache.weigh(q, s.ints(starts), s.ints([1000, 1 << 30]), s.ints(s.blocks), new, s.weights, out=torch.full_like(s.weights, 7.0), longest=50)
    s.lens = [50, 50]
    same = s.cache.weigh(q, s.ints(starts), s.ints(s.lens), s.ints(s.blocks), new, s.weights, out=torch.full_like(s.weights, 7.0))
    assert torch.equal(short, same)


def test_weigh_rows_that_are_not_finite():
    """A row of NaN makes the weights of what it sees NaN, and no others."""
    g = gen(3)
    for new in (2, 50):
        s = Sequences(g, BF16, [200], 1, 64, 16, False)
        q = randn(g, BF16, new, 1, 64)
        q[0] = math.nan
        s.cache.weigh(q, s.ints([0, new]), s.ints([200]), s.ints(s.blocks), new, s.weights)
        got = s.of(s.weights, 0)[0]
        assert torch.isnan(got[:200 - new + 1]).all() and torch.isfinite(got[200 - new + 1:]).all()


def same(a, b):
    """Equal, and NaN in the same places."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()) if a.is_floating_point() else torch.equal(a, b)


def check_evicted(s, budget, recent, first, in_place, longest=None):
    pools = [p for p in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale, s.weights) if p is not None]
    tokens = [s.all(p) for p in pools]
    tokens = [[x.clone() for x in pool] for pool in tokens]
    before = [p.clone() for p in pools]
    lens = [min(n, longest) if longest else n for n in s.lens]
    want = more.evict([w[:, :n] for w, n in zip(tokens[-1], lens)], lens, budget, recent, first)
    need = -(-min(budget, max(max(lens), 1)) // s.page)
    to = s.blocks if in_place else np.random.default_rng(1).permutation(s.rest)[:len(lens) * need].reshape(len(lens), need)
    given = s.ints(s.lens)
    blocks = s.ints(s.blocks)
    left, kept = s.cache.evict(s.weights, given, blocks, budget, recent=recent, first=first, to=None if in_place else s.ints(to), longest=longest, left=given if in_place else None)
    assert left.tolist() == [min(n, budget) for n in lens]
    touched = torch.zeros((s.pages, s.heads, s.page), dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        many = min(n, budget)
        assert (kept[b, :, many:] == -1).all()
        assert np.array_equal(kept[b, :, :many].cpu().numpy(), want[b][:, :many])
        if many == 0:
            continue
        j = np.arange(many)
        at, place = torch.from_numpy(to[b][j // s.page]).long().cuda(), torch.from_numpy(j % s.page).cuda()
        index = torch.from_numpy(want[b]).long().cuda()
        touched[at, :, place] = True
        for pool, mine in zip(pools, tokens):
            have = pool[at, :, place].transpose(0, 1)
            x = mine[b]
            assert same(have, torch.gather(x, 1, index if x.dim() == 2 else index[..., None].expand(-1, -1, x.shape[2])))
    for pool, was in zip(pools, before):
        assert same(pool[~touched], was[~touched])


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens, budget, recent, first, heads, dim, page", [
    ([1], 1, 0, 0, 1, 64, 16), ([5, 0, 40], 4, 1, 1, 2, 64, 16), ([300, 17, 100, 101], 100, 30, 4, 3, 128, 48), ([1000, 2000], 999, 999, 0, 1, 128, 64), ([700], 50, 0, 50, 2, 256, 16),
    ([5000, 4097, 9000], 4096, 100, 3, 2, 64, 128), ([20000], 19999, 5000, 0, 1, 128, 32), ([40000, 33000], 3001, 17, 0, 2, 64, 64), ([100], 700, 20, 4, 2, 128, 16)])
def test_evict(lens, budget, recent, first, heads, dim, page, int8, in_place):
    g = gen(sum(lens))
    s = Sequences(g, BF16, lens, heads, dim, page, int8, spare=len(lens) * (-(-budget // page) + 1))
    check_evicted(s, budget, recent, first, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("what", ["equal", "few values", "zeros", "not finite", "either sign", "close"])
def test_evict_ties(what, in_place):
    g = gen(9)
    s = Sequences(g, F16, [6000, 501, 77], 2, 64, 32, False, spare=60)
    w = s.weights
    if what == "equal":
        w.fill_(0.25)
    elif what == "few values":
        w.copy_(whole(g, 0, 3, torch.int32, *w.shape).float())
    elif what == "zeros":
        w.copy_(torch.where(torch.rand(w.shape, device="cuda", generator=g) < 0.97, 0.0, w))
        w[::2] *= -1  # zeros of either sign are equal
    elif what == "not finite":
        u = torch.rand(w.shape, device="cuda", generator=g)
        w.copy_(torch.where(u < 0.3, math.nan, torch.where(u < 0.8, -math.inf, torch.where(u < 0.85, math.inf, w))))
    elif what == "either sign":
        w.copy_(randn(g, F32, *w.shape))
    else:
        w.copy_(1 + whole(g, 0, 200, torch.int32, *w.shape).float() * 2.0 ** -23)
    check_evicted(s, 500, 20, 5, in_place)


def test_evict_longest_and_blocks_outside():
    g = gen(4)
    s = Sequences(g, BF16, [300, 200], 2, 64, 16, False, spare=40)
    check_evicted(s, 40, 5, 0, False, longest=100)
    # tokens of blocks that are not there are the lightest, and are not moved
    s = Sequences(g, BF16, [300, 200], 1, 64, 16, False, spare=40)
    blocks, to = s.blocks.copy(), s.rest[:8].reshape(2, 4)
    blocks[0, 2], blocks[1, 12] = -1, s.pages + 7
    to[1, 0] = -5
    before = s.weights.clone()
    w = [s.of(before, b).clone() for b in range(2)]
    w[0][:, 32:48] = math.nan
    w[1][:, 192:] = math.nan
    want = more.evict(w, s.lens, 64, 10, 0)
    left, kept = s.cache.evict(s.weights, s.ints(s.lens), s.ints(blocks), 64, recent=10, to=s.ints(to))
    assert left.tolist() == [64, 64] and all(np.array_equal(kept[b].cpu().numpy(), want[b]) for b in range(2))
    changed = (s.weights != before).any(-1).any(-1).nonzero().flatten().tolist()
    assert set(changed) <= set(to.flatten().tolist()) - {-5}
    for j in range(16, 64):  # of the second sequence, in blocks that are there
        t = want[1][0, j]
        if t < 192:
            assert s.weights[int(to[1, j // 16]), 0, j % 16] == w[1][0, t]


def test_weigh_and_evict_in_a_graph():
    """A step of a conversation, captured: attention, its weights, and every few steps the budget; replayed with other tokens it gives what eager calls give."""
    g = gen(6)
    s = Sequences(g, BF16, [400, 90], 2, 128, 16, False)
    q, starts, lens, blocks = randn(g, BF16, 2, 8, 128), s.ints([0, 1, 2]), s.ints(s.lens), s.ints(s.blocks)
    out, kept = torch.zeros_like(q), torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda")
    pools = (s.cache.k, s.cache.v, s.weights, lens)
    start = [p.clone() for p in pools]

    def step():
        s.cache.attend(q, starts, lens, blocks, 1, out=out)
        s.cache.weigh(q, starts, lens, blocks, 1, s.weights)
        s.cache.evict(s.weights, lens, blocks, 64, recent=8, left=lens, kept=kept)

    def reset():
        for p, was in zip(pools, start):
            p.copy_(was)
    step()
    reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        q.copy_(randn(g, BF16, 2, 8, 128))
        reset()
        step()
        want = [p.clone() for p in (*pools, out, kept)]
        reset()
        out.zero_(), kept.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*pools, out, kept), want))
        assert lens.tolist() == [64, 64]


# ---- together --------------------------------------------------------------------------------------------------------------
def test_conversations_with_a_budget():
    """Steps of a small model as a program makes them: queries, keys and values by 4-bit products into the cache, attention and its weights, the cache held to a budget,
    experts, penalties on the scores, the next token.  Each operator is held against its formula on what it was given."""
    g = gen(11)
    b, heads, kv, dim, hidden, vocab, budget = 3, 4, 2, 64, 256, 300, 40
    s = Sequences(g, BF16, [60, 33, 41], kv, dim, 16, False, more=3)
    s.weights.zero_()
    table = hipq.rotation_table(500, dim)
    quant = lambda rows, k: (whole(g, 0, 256, torch.uint8, rows, k // 2), (torch.rand((rows, k // 64), device="cuda", generator=g) * 0.01).to(BF16))  # noqa: E731
    wqkv, wo, head = (hipq.LinearW4(*quant(*shape), 64) for shape in (((heads + 2 * kv) * dim, hidden), (hidden, heads * dim), (vocab, hidden)))
    layer = Layer(g, BF16, 6, hidden, 96, hidden, 2, 64, scores="sigmoid")
    router, embedding = randn(g, BF16, hidden, 6) * 0.1, randn(g, BF16, vocab, hidden)
    position, lens, blocks, starts = s.ints([100, 80, 200]), s.ints(s.lens), s.ints(s.blocks), s.ints(range(b + 1))
    history, count = torch.full((b, 20), -1, dtype=torch.int32, device="cuda"), s.ints([0] * b)
    value = lambda v: torch.full((b,), v, device="cuda")  # noqa: E731
    kept = torch.zeros((b, kv, budget), dtype=torch.int32, device="cuda")
    token = whole(g, 0, vocab, torch.int64, b)
    rows = torch.arange(b, device="cuda")
    evicted = 0
    for step in range(12):
        x = embedding[token]
        qkv = wqkv(x).view(b, heads + 2 * kv, dim)
        slots = (blocks.gather(1, (lens[:, None] // 16).long())[:, 0] * 16 + lens % 16).to(torch.int32)
        q = s.cache.append(qkv[:, :heads], qkv[:, heads:-kv], qkv[:, -kv:], position, slots, table)
        lens += 1
        position += 1
        s.lens = lens.tolist()
        o = s.cache.attend(q, starts, lens, blocks, 1)
        want, off = ref.attend(q, s.all(s.cache.k), s.all(s.cache.v), list(range(b + 1)), s.lens, None, dim ** -0.5, heads // kv)
        assert ref.within(o, want, off)[0]
        before = s.all(s.weights.clone())
        s.cache.weigh(q, starts, lens, blocks, 1, s.weights)
        for (w, off), have in zip(more.weigh(q, s.all(s.cache.k), list(range(b + 1)), s.lens, None, dim ** -0.5, heads // kv, before), s.all(s.weights)):
            assert ((have.double() - w).abs() <= off).all()
        if max(s.lens) > 48:
            tokens, long = [t.clone() for t in s.all(s.cache.v)], list(s.lens)
            want = more.evict([t.clone() for t in s.all(s.weights)], s.lens, budget, 8, 2)
            s.cache.evict(s.weights, lens, blocks, budget, recent=8, first=2, left=lens, kept=kept)
            s.lens = lens.tolist()
            assert s.lens == [min(n, budget) for n in long]
            for i in range(b):
                assert np.array_equal(kept[i, :, :s.lens[i]].cpu().numpy(), want[i])
                assert torch.equal(s.of(s.cache.v, i), torch.gather(tokens[i], 1, torch.from_numpy(want[i]).cuda()[..., None].expand(-1, -1, dim)))
            evicted += 1
        x = x + wo(o.flatten(1))
        x = x + layer.check(x, (x @ router).float())
        scores = head(x)
        kw = dict(tokens=history, lens=count, repetition=value(1.3), frequency=value(0.2), presence=value(0.1))
        scores = check_penalized(scores, **kw).cuda()
        token = hipq.sample(scores, torch.rand(b, device="cuda", generator=g), temperature=value(0.8))
        history[rows, count.long()] = token.to(torch.int32)
        count += 1
    assert evicted >= 2 and (history[:, :12] >= 0).all()
