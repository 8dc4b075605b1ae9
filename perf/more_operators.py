"""What the operators around the language-model core are measured on: layers of experts, a cache held to a budget, penalties before sampling.

Four kinds of work, each over the range of sizes that programs have which serve quantized language models:

  experts   hipq.ExpertsW4: a mixture-of-experts layer with 4-bit weights, from one token to a prompt's
  weigh     hipq.KvCache.weigh: the attention that every token in the paged cache receives from the new ones, accumulated
  evict     hipq.KvCache.evict: the heaviest and the latest tokens of every sequence and head, moved to other pages
  penalize  hipq.penalize: penalties for repeated tokens, biases and a grammar's bits on the scores of every row

With `own` false everything is computed in its plain form by elementary torch operations, in 32 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token, two of eight large experts: the weights are read once, and little else counts
        dict(name="experts_m1", kind="experts", m=1, experts=8, top=2, k=4096, inner=14336, n=4096, group=128, zeros=False, act="silu", scores="softmax",
             normalize=True, dtype="bf16"),
        # one token, few of many small experts: the smallest layers, where latency counts
        dict(name="experts_m1_small", kind="experts", m=1, experts=64, top=6, k=2048, inner=1408, n=2048, group=128, zeros=False, act="silu", scores="softmax",
             normalize=False, dtype="bf16"),
        # a batch of decoding sequences over many small experts, nearly all of them chosen by one or two tokens
        dict(name="experts_m24", kind="experts", m=24, experts=64, top=6, k=2048, inner=1408, n=2048, group=64, zeros=True, act="silu", scores="softmax",
             normalize=False, dtype="fp16"),
        # a prompt, odd sizes, the smallest groups, scores by themselves
        dict(name="experts_m333_ragged", kind="experts", m=333, experts=13, top=3, k=1056, inner=1120, n=1000, group=32, zeros=True, act="gelu", scores="sigmoid",
             normalize=True, dtype="bf16"),
        # a long prompt
        dict(name="experts_m2048", kind="experts", m=2048, experts=32, top=4, k=4096, inner=2048, n=4096, group=128, zeros=False, act="silu", scores="softmax",
             normalize=True, dtype="bf16"),
        # one token of 8 sequences of up to 2000
        dict(name="weigh_b8", kind="weigh", b=8, new=1, hq=32, hkv=8, d=128, longest=2000, page=64, int8=False, dtype="bf16"),
        # the last 32 tokens of a long prompt over it, in an int8 cache
        dict(name="weigh_b1_window_i8", kind="weigh", b=1, new=32, hq=32, hkv=8, d=128, longest=30000, page=48, int8=True, dtype="bf16"),
        # one token of two very long sequences
        dict(name="weigh_b2_long", kind="weigh", b=2, new=1, hq=64, hkv=8, d=128, longest=131072, page=128, int8=False, dtype="fp16"),
        # half of a few conversations' tokens
        dict(name="evict_b4", kind="evict", b=4, hkv=8, d=128, longest=4096, budget=2048, recent=256, first=4, page=64, int8=False, dtype="bf16"),
        # a quarter of two very long ones, in an int8 cache
        dict(name="evict_b2_long_i8", kind="evict", b=2, hkv=8, d=128, longest=131072, budget=32000, recent=1000, first=0, page=48, int8=True, dtype="bf16"),
        # the answer to one user: all there is
        dict(name="penalize_r1", kind="penalize", r=1, v=32000, longest=1500, bias=8, allowed=True, repetition=True, dtype="bf16"),
        # a large batch over a large vocabulary with long histories
        dict(name="penalize_r256", kind="penalize", r=256, v=128000, longest=4000, bias=0, allowed=True, repetition=True, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("experts", "experts", "weigh", "evict", "penalize"))
    half = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "experts":
        experts = _log(rng, 4, 160)
        top = min(experts, rng.choice((1, 2, 2, 4, 6, 8)))
        most = (350 << 20) // (3 * experts)  # a third of the weights of an expert
        k = 32 * _log(rng, 16, max(16, min(160, most // (32 * 256))))
        inner = 32 * _log(rng, 8, max(8, min(448, most // (32 * k))))
        n = rng.choice((k, k, _log(rng, 200, max(200, k))))
        m = _log(rng, 1, max(1, min(2048, (1 << 36) // (top * k * inner))))
        return dict(kind=kind, m=m, experts=experts, top=top, k=k, inner=inner, n=n, group=rng.choice((32, 64, 128, 128)), zeros=rng.random() < 0.5,
                    act=rng.choice(("silu", "silu", "gelu")), scores=rng.choice(("softmax", "softmax", "sigmoid")), normalize=rng.random() < 0.5, dtype=half)
    if kind == "penalize":
        v = _log(rng, 1000, 150000)
        return dict(kind=kind, r=_log(rng, 1, min(256, (32 << 20) // v)), v=v, longest=_log(rng, 1, 4000), bias=rng.choice((0, 0, _log(rng, 1, 300))),
                    allowed=rng.random() < 0.5, repetition=rng.random() < 0.7, dtype=rng.choice(("bf16", "fp16", "fp32")))
    hkv = rng.choice((1, 2, 4, 8, 8))
    d = rng.choice((64, 128, 128, 256))
    int8 = rng.random() < 0.4
    b = _log(rng, 1, 48)
    page = rng.choice((16, 48, 64, 128))
    if kind == "weigh":
        new = rng.choice((1, 1, 1, _log(rng, 2, 64)))
        hq = hkv * rng.choice((1, 4, 6, 8))
        most = max(new + 1, min(131072, (128 << 20) // (b * hkv * d), (1 << 28) // (b * hq * new)))
        return dict(kind=kind, b=b, new=new, hq=hq, hkv=hkv, d=d, longest=_log(rng, new + 1, most), page=page, int8=int8, dtype=half)
    longest = _log(rng, 40, max(40, min(131072, (96 << 20) // (b * hkv * d))))
    budget = _log(rng, max(1, longest // 10), longest)
    recent = rng.randrange(budget + 1) // rng.choice((1, 4, 16))
    return dict(kind=kind, b=b, hkv=hkv, d=d, longest=longest, budget=budget, recent=recent, first=min(budget - recent, rng.choice((0, 0, 4))), page=page,
                int8=int8, dtype=half)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, dtype, *shape):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)


def _uniform(gen, lo, hi, *shape):
    return torch.rand(shape, device="cuda", generator=gen, dtype=torch.float32) * (hi - lo) + lo


def _whole(gen, lo, hi, dtype, *shape):
    return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=gen)


def _experts(case, gen):
    t, (m, e, k, inner, n, group) = TYPES[case["dtype"]], (case[f] for f in ("m", "experts", "k", "inner", "n", "group"))
    zeros = (lambda *shape: _whole(gen, 5, 12, torch.uint8, *shape)) if case["zeros"] else (lambda *shape: None)
    s = dict(x=_randn(gen, t, m, k), group=group, top=case["top"], act=case["act"], scores=case["scores"], normalize=case["normalize"],
             logits=_randn(gen, torch.float32, m, e) * 1.5 + _randn(gen, torch.float32, e),  # some experts are chosen more often
             gate_up=_whole(gen, 0, 256, torch.uint8, e, 2 * inner, k // 2), gate_up_scales=_uniform(gen, 0.004, 0.012, e, 2 * inner, -(-k // group)).to(t),
             gate_up_zeros=zeros(e, 2 * inner, -(-k // group)),
             down=_whole(gen, 0, 256, torch.uint8, e, n, inner // 2), down_scales=_uniform(gen, 0.004, 0.012, e, n, -(-inner // group)).to(t),
             down_zeros=zeros(e, n, -(-inner // group)))
    if own:  # the plan that such a program keeps: the weights in the kernels' order
        from nart_amd import hipq
        s["plan"] = hipq.ExpertsW4(s["gate_up"], s["gate_up_scales"], s["down"], s["down_scales"], s["top"], group, gate_up_zeros=s["gate_up_zeros"],
                                   down_zeros=s["down_zeros"], activation=s["act"], scores=s["scores"], normalize=s["normalize"])
    return s


def _pool(case, gen, pages):
    t, (hkv, d, page) = TYPES[case["dtype"]], (case[f] for f in ("hkv", "d", "page"))
    if case["int8"]:
        kc, vc = (_whole(gen, -127, 128, torch.int8, pages, hkv, page, d) for _ in range(2))
        return dict(kc=kc, vc=vc, ks=_uniform(gen, 0.008, 0.024, pages, hkv, page), vs=_uniform(gen, 0.008, 0.024, pages, hkv, page))
    return dict(kc=_randn(gen, t, pages, hkv, page, d), vc=_randn(gen, t, pages, hkv, page, d), ks=None, vs=None)


def _counts(case):
    """New tokens of every sequence: from all that a call allows down to half of them."""
    return np.array([case["new"] - 5 * i % (case["new"] // 2 + 1) for i in range(case["b"])])


def _int32(array):
    return torch.from_numpy(np.ascontiguousarray(array, dtype=np.int32)).cuda()


def _weigh(case, seed, gen):
    b, page, rng = case["b"], case["page"], np.random.default_rng(seed)
    counts = _counts(case)
    lens = np.maximum(rng.integers(max(1, case["longest"] // 2), case["longest"] + 1, b), counts)
    lens[-1] = case["longest"]
    per = -(-int(lens.max()) // page)  # pages of the longest sequence
    s = _pool(case, gen, b * per)
    s |= dict(q=_randn(gen, TYPES[case["dtype"]], int(counts.sum()), case["hq"], case["d"]), starts=_int32(np.concatenate(([0], np.cumsum(counts)))), lens=_int32(lens),
              blocks=_int32(rng.permutation(b * per).reshape(b, per)), new=case["new"], longest=int(lens.max()),
              weights=_uniform(gen, 0, 2, b * per, case["hkv"], page), out=torch.zeros((b * per, case["hkv"], page), device="cuda"))
    if own:
        from nart_amd import hipq
        s["cache"] = hipq.KvCache(s["kc"], s["vc"], s["ks"], s["vs"])
    return s


def _evict(case, seed, gen):
    b, page, rng = case["b"], case["page"], np.random.default_rng(seed)
    lens = rng.integers(max(1, case["longest"] // 2), case["longest"] + 1, b)
    lens[-1] = case["longest"]
    per, to = -(-int(lens.max()) // page), -(-case["budget"] // page)
    s = _pool(case, gen, b * (per + to))
    # what tokens receive spreads over orders of magnitude, and some receive nothing
    weights = torch.exp(3 * _randn(gen, torch.float32, b * (per + to), case["hkv"], page))
    s |= dict(weights=torch.where(weights < 0.01, 0.0, weights), lens=_int32(lens), blocks=_int32(rng.permutation(b * per).reshape(b, per)),
              to=_int32(b * per + rng.permutation(b * to).reshape(b, to)), budget=case["budget"], recent=case["recent"], first=case["first"], longest=int(lens.max()),
              kept=torch.zeros((b, case["hkv"], case["budget"]), dtype=torch.int32, device="cuda"), left=torch.zeros(b, dtype=torch.int32, device="cuda"), b=b)
    for name in ("kc", "vc", "ks", "vs", "weights"):  # the pages that the kept ones move to are those behind the sequences'
        if s[name] is not None:
            s[name][b * per:] = 0
        s["to_" + name] = None if s[name] is None else s[name][b * per:]
    if case["int8"]:
        s |= {name + "_values": torch.empty(s["to_" + name].shape, dtype=TYPES[case["dtype"]], device="cuda") for name in ("kc", "vc")}
    if own:
        from nart_amd import hipq
        s["cache"] = hipq.KvCache(s["kc"], s["vc"], s["ks"], s["vs"])
    return s


def _penalize(case, gen):
    r, v, longest = case["r"], case["v"], case["longest"]
    lens = _whole(gen, longest // 2, longest + 1, torch.int32, r)
    s = dict(logits=(_randn(gen, torch.float32, r, v) * 2.5).to(TYPES[case["dtype"]]),
             # a text's tokens: some come often, most never
             tokens=torch.clamp(_uniform(gen, 0, 1, r, longest).pow(4) * v, max=v - 1).to(torch.int32), lens=lens, prompt_lens=(lens * _uniform(gen, 0, 1, r)).to(torch.int32),
             repetition=_uniform(gen, 1, 1.5, r) if case["repetition"] else None, frequency=_uniform(gen, 0, 0.5, r), presence=_uniform(gen, 0, 0.5, r),
             bias_tokens=None, bias=None, allowed=None, out=torch.empty((r, v), dtype=TYPES[case["dtype"]], device="cuda"))
    if case["bias"]:  # of different tokens
        s |= dict(bias=_randn(gen, torch.float32, r, case["bias"]) * 4,
                  bias_tokens=((torch.arange(case["bias"], device="cuda") * (v // case["bias"]) + _whole(gen, 0, v, torch.int64, r, 1)) % v).to(torch.int32))
    if case["allowed"]:
        s["allowed"] = _whole(gen, -2 ** 31, 2 ** 31, torch.int64, r, -(-v // 32)).to(torch.int32)
    return s


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    if kind == "experts":
        s = _experts(case, gen)
    elif kind == "weigh":
        s = _weigh(case, seed, gen)
    elif kind == "evict":
        s = _evict(case, seed, gen)
    else:
        s = _penalize(case, gen)
    return dict(s, kind=kind)


# ---- one pass: the plain forms ----------------------------------------------------------------------------------------
def _activate(x, act):
    return x * torch.sigmoid(x) if act == "silu" else 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _dense(s, name, e):
    q, scales, zeros = s[name][e], s[name + "_scales"][e], s[name + "_zeros"]
    rows, half = q.shape
    q = torch.stack((q & 15, q >> 4), 2).view(rows, 2 * half).float()
    spread = lambda t: t.float().repeat_interleave(s["group"], 1)[:, :2 * half]  # noqa: E731
    return (q - (8.0 if zeros is None else spread(zeros[e]))) * spread(scales)


def _plain_experts(s):
    chosen, which = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    chosen, which = chosen[:, :s["top"]], which[:, :s["top"]]
    if s["scores"] == "sigmoid":
        w = torch.sigmoid(chosen)
    else:
        most = s["logits"].amax(1, keepdim=True)
        w = torch.exp(chosen - most) / torch.exp(s["logits"] - most).sum(1, keepdim=True)
    if s["normalize"]:
        w = w / w.sum(1, keepdim=True)
    y = torch.zeros((s["x"].shape[0], s["down"].shape[1]), device="cuda")
    order = torch.argsort(which.flatten(), stable=True)
    counts = torch.bincount(which.flatten(), minlength=s["logits"].shape[1]).tolist()
    at = 0
    for e, count in enumerate(counts):  # expert by expert, those that a token has chosen
        if count:
            pairs = order[at:at + count]
            rows = pairs // s["top"]
            gate, up = (s["x"][rows].float() @ _dense(s, "gate_up", e).t()).chunk(2, 1)
            h = _activate(gate, s["act"]) * up
            y.index_add_(0, rows, (h @ _dense(s, "down", e).t()) * w.flatten()[pairs][:, None])
            at += count
    return y.to(s["x"].dtype)


def _plain_weigh(s):
    total, hq, d = s["q"].shape
    pages, hkv, page, _ = s["kc"].shape
    b, per = s["blocks"].shape
    group, new, n = hq // hkv, s["new"], per * page
    k = s["kc"][s["blocks"]].float()
    if s["ks"] is not None:
        k = k * s["ks"][s["blocks"]][..., None]
    k = k.transpose(1, 2).reshape(b, hkv, n, d)
    starts, lens = s["starts"].long(), s["lens"].long()
    counts = starts[1:] - starts[:-1]
    rows = torch.arange(new, device="cuda")
    there = rows < counts[:, None]                             # b, new
    at = torch.clamp(starts[:-1, None] + rows, max=total - 1)  # the row of q
    q = s["q"].float()[at].view(b, new, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, new * group, d)
    scores = (q @ k.transpose(-1, -2) * (1 / math.sqrt(d))).view(b, hkv, new, group, n)
    token = torch.arange(n, device="cuda")
    fresh = token - (lens - counts)[:, None]                   # b, n: the index among the new tokens, below zero before them
    seen = (fresh[:, None] <= rows[:, None]) & (token < lens[:, None])[:, None]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True) * there[:, None, :, None, None]
    before = torch.where(fresh[:, None] >= 0, 0.0, s["weights"][s["blocks"]].transpose(1, 2).reshape(b, hkv, n))
    got = (p.sum((2, 3)) + before) * (token < lens[:, None])[:, None]
    s["out"][s["blocks"]] = got.view(b, hkv, per, page).transpose(1, 2)
    return s["out"]


def _plain_evict(s):
    pages, hkv, page, d = s["kc"].shape
    b, per = s["blocks"].shape
    n, budget = per * page, s["budget"]
    lens = s["lens"].long()[:, None, None]
    token = torch.arange(n, device="cuda")
    w = s["weights"][s["blocks"]].transpose(1, 2).reshape(b, hkv, n)
    rank = torch.where((token < s["first"]) | (token >= lens - s["recent"]), math.inf, w)
    rank = torch.where(token < lens, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    left = torch.clamp(s["lens"], max=budget)
    j = torch.arange(budget, device="cuda")
    there = j < left[:, None]                                   # b, budget
    kept = torch.sort(torch.where(order < lens, order, n), dim=-1).values
    at = torch.clamp(kept[..., :j.shape[0]], max=n - 1)
    seq, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[None, :, None]
    source = s["blocks"].long()[seq, at // page], head, at % page
    target = s["to"].long()[:, None][:, :, j // page].expand(b, hkv, -1), head.expand(b, hkv, j.shape[0]), (j % page).expand(b, hkv, -1)
    inside = there[:, None].expand(b, hkv, -1)
    target = tuple(t[inside] for t in target)
    for name in ("kc", "vc", "ks", "vs", "weights"):
        if s[name] is not None:
            s[name][target] = s[name][source][inside]
    s["kept"].copy_(torch.where(inside, kept[..., :j.shape[0]], -1))
    s["left"].copy_(left)


def _plain_penalize(s):
    x = s["logits"].float()
    rows, v = x.shape
    place = torch.arange(s["tokens"].shape[1], device="cuda")
    there = place < s["lens"][:, None]
    fresh = there & (place >= s["prompt_lens"][:, None])
    tokens = s["tokens"].long()
    count = torch.zeros_like(x).scatter_add_(1, tokens, fresh.float())
    if s["repetition"] is not None:
        seen = torch.zeros_like(x).scatter_add_(1, tokens, there.float()) > 0
        rep = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - count * s["frequency"][:, None] - (count > 0) * s["presence"][:, None]
    if s["bias"] is not None:
        x = x.scatter_add(1, s["bias_tokens"].long(), s["bias"])
    if s["allowed"] is not None:
        bits = (s["allowed"][..., None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x = torch.where(bits.view(rows, -1)[:, :v] > 0, x, -math.inf)
    s["out"].copy_(x)
    return s["out"]


def run(state):
    s, kind = state, state["kind"]
    if kind == "experts":
        return s["plan"](s["x"], s["logits"]) if own else _plain_experts(s)
    if kind == "weigh":
        if own:
            return s["cache"].weigh(s["q"], s["starts"], s["lens"], s["blocks"], s["new"], s["weights"], out=s["out"], longest=s["longest"])
        return _plain_weigh(s)
    if kind == "evict":
        if own:
            s["cache"].evict(s["weights"], s["lens"], s["blocks"], s["budget"], recent=s["recent"], first=s["first"], to=s["to"], longest=s["longest"], left=s["left"],
                             kept=s["kept"])
        else:
            _plain_evict(s)
        if s["ks"] is None:
            return s["to_kc"], s["to_vc"], s["to_weights"], s["kept"], s["left"]
        return (torch.mul(s["to_kc"], s["to_ks"][..., None], out=s["kc_values"]), torch.mul(s["to_vc"], s["to_vs"][..., None], out=s["vc_values"]), s["to_weights"],
                s["kept"], s["left"])
    if own:
        from nart_amd import hipq
        return hipq.penalize(s["logits"], s["tokens"], s["lens"], s["prompt_lens"], repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                             bias_tokens=s["bias_tokens"], bias=s["bias"], allowed=s["allowed"], out=s["out"])
    return _plain_penalize(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "experts":
        m, e, top, k, inner, n = (case[f] for f in ("m", "experts", "top", "k", "inner", "n"))
        used = e * (1 - (1 - top / e) ** m)  # experts that some token chooses
        scales = 3 if case["zeros"] else 2
        groups = 2 * inner * -(-k // case["group"]) + n * -(-inner // case["group"])
        return {"bytes": int(used * ((2 * inner * k + n * inner) // 2 + groups * scales)) + 2 * m * (k + n) + 4 * m * e, "flops": 2 * m * top * inner * (2 * k + n)}
    if kind == "penalize":
        r, v = case["r"], case["v"]
        return {"bytes": r * (2 * v * (4 if case["dtype"] == "fp32" else 2) + 3 * case["longest"] + 8 * case["bias"] + (v // 8 if case["allowed"] else 0)), "flops": 0}
    b, hkv, d = (case[f] for f in ("b", "hkv", "d"))
    wide = d + 4 if case["int8"] else 2 * d
    tokens = 0.75 * case["longest"] * b  # lengths are spread over the upper half
    if kind == "weigh":
        rows = int(_counts(case).sum())
        return {"bytes": int(tokens * hkv * (wide + 8)) + rows * case["hq"] * d * 2, "flops": int(2 * tokens * rows / b * case["hq"] * d)}
    kept = min(case["budget"], 0.75 * case["longest"]) * b
    # the values that an int8 cache stands for are read off for the comparison: no part of what a pass has to do
    return {"bytes": int(hkv * (4 * tokens + kept * (4 * wide + 8))), "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _product(x, q, scales, zeros, group):
    """x times 4-bit rows, group by group: what is left of the zero point, times the scale."""
    total = torch.zeros((x.shape[0], q.shape[0]), dtype=torch.float64, device="cuda")
    k = 2 * q.shape[1]
    for g, at in enumerate(range(0, k, group)):
        to = min(k, at + group)
        part = q[:, at // 2:to // 2].to(torch.int16)
        zero = 8 if zeros is None else zeros[:, g:g + 1].to(torch.int16)
        xs = x[:, at:to]
        total += (xs[:, 0::2] @ ((part % 16) - zero).double().t() + xs[:, 1::2] @ ((part // 16) - zero).double().t()) * scales[:, g].double()
    return total


def _exact_experts(s):
    x, logits = s["x"].double(), s["logits"].double().cpu().numpy()
    m, experts = logits.shape
    which = np.argsort(-logits, axis=1, kind="stable")[:, :s["top"]]
    if s["scores"] == "sigmoid":
        share = 1 / (1 + np.exp(-logits))
    else:
        share = np.exp(logits - logits.max(1, keepdims=True))
        share = share / share.sum(1, keepdims=True)
    share = np.take_along_axis(share, which, 1)
    if s["normalize"]:
        share = share / share.sum(1, keepdims=True)
    y = torch.zeros((m, s["down"].shape[1]), dtype=torch.float64, device="cuda")
    for e in range(experts):
        rows, slots = np.nonzero(which == e)
        if len(rows):
            at = torch.from_numpy(rows).cuda()
            both = _product(x[at], s["gate_up"][e], s["gate_up_scales"][e], None if s["gate_up_zeros"] is None else s["gate_up_zeros"][e], s["group"])
            g, u = both[:, :both.shape[1] // 2], both[:, both.shape[1] // 2:]
            g = g / (1 + torch.exp(-g)) if s["act"] == "silu" else g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
            o = _product(g * u, s["down"][e], s["down_scales"][e], None if s["down_zeros"] is None else s["down_zeros"][e], s["group"])
            y[at] += o * torch.from_numpy(share[rows, slots]).cuda()[:, None]  # a token has an expert once
    return y


def _exact_weigh(s):
    hq, d = s["q"].shape[1:]
    hkv, page = s["kc"].shape[1:3]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):  # sequence by sequence, without what its pages hold behind its end
        lo, hi = starts[b], starts[b + 1]
        new, at = hi - lo, s["blocks"][b, :-(-n // page)].long()
        k = s["kc"][at].double()
        k = k if s["ks"] is None else k * s["ks"][at].double()[..., None]
        k = k.permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n]
        hidden = torch.from_numpy(~np.tri(new, dtype=bool)).cuda()
        got = s["weights"][at].double().transpose(0, 1).reshape(hkv, -1)
        got[:, n:] = 0
        got[:, n - new:n] = 0
        for h in range(hkv):
            q = s["q"][lo:hi, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            a = (q.reshape(-1, d) @ k[h].t() / d ** 0.5).view(new, -1, n)
            a[..., n - new:].masked_fill_(hidden[:, None], -math.inf)
            got[h, :n] += torch.softmax(a, -1).sum((0, 1))
        out[at] = got.view(hkv, -1, page).transpose(0, 1)
    return out


def _exact_evict(s):
    page, hkv = s["kc"].shape[2], s["kc"].shape[1]
    blocks, to, lens = s["blocks"].cpu().numpy(), s["to"].cpu().numpy(), s["lens"].tolist()
    base = s["kc"].shape[0] - s["to_kc"].shape[0]
    weights = s["weights"].cpu().numpy()
    kept = np.full(s["kept"].shape, -1, np.int32)
    names = [name for name in ("kc", "vc", "ks", "vs", "weights") if s[name] is not None]
    out = {name: torch.zeros(s["to_" + name].shape, dtype=torch.float64, device="cuda") for name in names}
    for b, n in enumerate(lens):
        many = min(n, s["budget"])
        for h in range(hkv):
            w = weights[blocks[b], h].reshape(-1)[:n]
            if n > s["budget"]:
                middle = np.arange(s["first"], n - s["recent"])
                heavy = middle[np.argsort(-w[middle], kind="stable")[:s["budget"] - s["first"] - s["recent"]]]
                at = np.sort(np.concatenate((np.arange(s["first"]), heavy, np.arange(n - s["recent"], n))))
            else:
                at = np.arange(n)
            kept[b, h, :many] = at
            j = np.arange(many)
            source, target = (torch.from_numpy(np.ascontiguousarray(p)).long().cuda() for p in (blocks[b][at // page], to[b][j // page] - base))
            inside, place = torch.from_numpy(at % page).cuda(), torch.from_numpy(j % page).cuda()
            for name in names:
                out[name][target, h, place] = s[name][source, h, inside].double()
    left = torch.tensor([min(n, s["budget"]) for n in lens], dtype=torch.int32)
    if s["ks"] is not None:
        out["kc"] *= out["ks"][..., None]
        out["vc"] *= out["vs"][..., None]
    return out["kc"], out["vc"], out["weights"], torch.from_numpy(kept), left


def _exact_penalize(s):
    x = s["logits"].double().cpu().numpy().copy()
    tokens, lens, prompt = (s[name].cpu().numpy() for name in ("tokens", "lens", "prompt_lens"))
    number = lambda name, r: float(s[name][r])  # noqa: E731
    for r in range(x.shape[0]):
        if s["repetition"] is not None:
            at, by = np.unique(tokens[r, :lens[r]]), number("repetition", r)
            x[r, at] = np.where(x[r, at] > 0, x[r, at] / by, x[r, at] * by)
        at, count = np.unique(tokens[r, prompt[r]:lens[r]], return_counts=True)
        x[r, at] -= count * number("frequency", r) + number("presence", r)
        if s["bias"] is not None:
            x[r, s["bias_tokens"][r].cpu().numpy()] += s["bias"][r].double().cpu().numpy()
        if s["allowed"] is not None:
            bits = np.unpackbits(s["allowed"][r].cpu().numpy().view(np.uint8), bitorder="little")[:x.shape[1]]
            x[r, bits == 0] = -math.inf
    return torch.from_numpy(x)


def exact(case, seed):
    s = prepare(case, seed)
    return {"experts": _exact_experts, "weigh": _exact_weigh, "evict": _exact_evict, "penalize": _exact_penalize}[s["kind"]](s)
