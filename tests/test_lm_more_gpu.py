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
@pytest.mark.parametrize("m, experts, top, kernel", [(40, 8, 2, "w4_experts_16x128"), (60, 4, 2, "w4_experts_32x128"), (100, 4, 2, "w4_experts_64x128"), (300, 4, 2, "w4_experts_128x256")])
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


@pytest.mark.parametrize("m", [1, 9, 40, 200, 900])
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
