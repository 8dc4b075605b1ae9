"""What the language-model operators are measured on: the calls that a program makes which serves a quantized language model.

Five kinds of work, each over the range of sizes that such programs have:

  linear   hipq.LinearW4: a product with 4-bit weights and group scales, from one row to a prompt's
  gated    the same plan with two projections, the activation and their product
  append   hipq.KvCache.append: norms of queries and keys (optional), the rotation, keys and values into the paged cache
  attend   hipq.KvCache.attend: one token, a chain or a tree of drafted tokens of each sequence over the paged cache
  sample   hipq.sample: a token of every row of scores from given uniform numbers

With `own` false everything is computed in its plain form by elementary torch operations, in 32 bits (sampling in 64: a sum next to
its border decides which token it is).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token through a square projection: the smallest call, where latency counts
        dict(name="linear_m1", kind="linear", m=1, n=4096, k=4096, group=128, zeros=False, bias=False, act="", dtype="bf16"),
        # a batch of decoding sequences through the gated pair of a feed-forward block, zero points and small groups
        dict(name="gated_m17", kind="gated", m=17, n=14336, k=4096, group=64, zeros=True, bias=False, act="silu", dtype="bf16"),
        # a short prompt through a layer of odd sizes with a bias, the smallest groups
        dict(name="linear_m100_ragged", kind="linear", m=100, n=5000, k=5504, group=32, zeros=True, bias=True, act="", dtype="bf16"),
        # a prompt through a large layer
        dict(name="linear_m2048", kind="linear", m=2048, n=8192, k=8192, group=128, zeros=False, bias=False, act="", dtype="fp16"),
        # one new token of 32 sequences into the cache
        dict(name="append_t32", kind="append", t=32, hq=32, hkv=8, d=128, rot=128, interleaved=False, norm=False, int8=False, page=64,
             far=8192, dtype="bf16"),
        # a prompt's tokens with norms into an int8 cache, a part of each head rotated, pairs side by side
        dict(name="append_t5000_i8", kind="append", t=5000, hq=40, hkv=8, d=128, rot=64, interleaved=True, norm=True, int8=True, page=32,
             far=131072, dtype="fp16"),
        # one token of 8 sequences of up to 2000
        dict(name="attend_b8", kind="attend", b=8, new=1, tree=False, hq=32, hkv=8, d=128, longest=2000, page=64, int8=False, dtype="bf16"),
        # trees of up to 32 drafted tokens of 16 sequences of up to 8000 in an int8 cache
        dict(name="attend_tree_b16_i8", kind="attend", b=16, new=32, tree=True, hq=32, hkv=8, d=128, longest=8000, page=32, int8=True,
             dtype="bf16"),
        # one token of two very long sequences
        dict(name="attend_b2_long", kind="attend", b=2, new=1, tree=False, hq=64, hkv=8, d=128, longest=131072, page=128, int8=False,
             dtype="fp16"),
        # the answer to one user
        dict(name="sample_r1", kind="sample", r=1, v=32000, filters=True, dtype="bf16"),
        # an odd vocabulary for a small batch, temperature alone
        dict(name="sample_r24_plain", kind="sample", r=24, v=50257, filters=False, dtype="fp16"),
        # a large batch over a large vocabulary in 32 bits
        dict(name="sample_r256", kind="sample", r=256, v=128000, filters=True, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "gated", "append", "attend", "attend", "sample"))
    half = rng.choice(("bf16", "bf16", "fp16"))
    if kind in ("linear", "gated"):
        k = 32 * _log(rng, 16, 512)
        n = _log(rng, 200, min(32768, (96 << 20) // k) // (2 if kind == "gated" else 1))
        m = _log(rng, 1, max(1, min(2048, (1 << 36) // (n * k))))
        return dict(kind=kind, m=m, n=n, k=k, group=rng.choice((32, 64, 128, 128)), zeros=rng.random() < 0.5, bias=rng.random() < 0.3,
                    act=rng.choice(("silu", "gelu")) if kind == "gated" else "", dtype=half)
    hkv = rng.choice((1, 2, 4, 8, 8))
    d = rng.choice((64, 128, 128, 256))
    if kind == "append":
        hq = hkv * rng.choice((1, 4, 5, 8))
        t = _log(rng, 1, min(8192, (48 << 20) // ((hq + 2 * hkv) * d)))
        return dict(kind=kind, t=t, hq=hq, hkv=hkv, d=d, rot=rng.choice((d, d, d // 2)), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.5, int8=rng.random() < 0.4, page=rng.choice((16, 48, 64, 128)), far=_log(rng, t + 1, 131072), dtype=half)
    if kind == "attend":
        b = _log(rng, 1, 48)
        new = rng.choice((1, 1, 1, _log(rng, 2, 64)))
        hq = hkv * rng.choice((1, 4, 6, 8))
        most = max(new + 1, min(131072, (96 << 20) // (b * hkv * d), (1 << 28) // (b * hq * new)))
        return dict(kind=kind, b=b, new=new, tree=new > 1 and rng.random() < 0.7, hq=hq, hkv=hkv, d=d, longest=_log(rng, new + 1, most),
                    page=rng.choice((16, 48, 64, 128)), int8=rng.random() < 0.4, dtype=half)
    v = _log(rng, 1000, 150000)
    return dict(kind=kind, r=_log(rng, 1, min(256, (32 << 20) // v)), v=v, filters=rng.random() < 0.7, dtype=rng.choice(("bf16", "fp16", "fp32")))


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, dtype, *shape):
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)


def _uniform(gen, lo, hi, *shape):
    return torch.rand(shape, device="cuda", generator=gen, dtype=torch.float32) * (hi - lo) + lo


def _linear(case, gen):
    t, group = TYPES[case["dtype"]], case["group"]
    rows, k = case["n"] * (2 if case["act"] else 1), case["k"]
    groups = -(-k // group)
    s = dict(x=_randn(gen, t, case["m"], k),
             q=torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device="cuda", generator=gen),
             scales=_uniform(gen, 0.004, 0.012, rows, groups).to(t),
             zeros=torch.randint(5, 12, (rows, groups), dtype=torch.uint8, device="cuda", generator=gen) if case["zeros"] else None,
             bias=_randn(gen, t, rows) if case["bias"] else None, group=group, act=case["act"] or None)
    if own:  # the plan that such a program keeps: the weights in the kernels' order
        from nart_amd import hipq
        s["plan"] = hipq.LinearW4(s["q"], s["scales"], group, zeros=s["zeros"], bias=s["bias"], activation=s["act"])
    return s


def _cache(k, v, k_scale, v_scale):
    from nart_amd import hipq
    return hipq.KvCache(k, v, k_scale, v_scale)


def _append(case, gen):
    t, (n, hq, hkv, d, page, rot) = TYPES[case["dtype"]], (case[f] for f in ("t", "hq", "hkv", "d", "page", "rot"))
    pages = -(-n // page) + 2
    qkv = _randn(gen, t, n, (hq + 2 * hkv) * d).view(n, hq + 2 * hkv, d)
    place = torch.int8 if case["int8"] else t
    angle = torch.arange(case["far"], dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** -(
        torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    s = dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:],
             positions=torch.randint(0, case["far"], (n,), device="cuda", generator=gen).to(torch.int32),
             slots=torch.randperm(pages * page, device="cuda", generator=gen)[:n].to(torch.int32),
             table=torch.cat((angle.cos(), angle.sin()), 1).float(),
             q_norm=_uniform(gen, 0.5, 1.5, d).to(t) if case["norm"] else None, k_norm=_uniform(gen, 0.5, 1.5, d).to(t) if case["norm"] else None,
             interleaved=case["interleaved"], out=torch.zeros((n, hq, d), dtype=t, device="cuda"),
             kc=torch.zeros((pages, hkv, page, d), dtype=place, device="cuda"), vc=torch.zeros((pages, hkv, page, d), dtype=place, device="cuda"),
             ks=None, vs=None)
    if case["int8"]:
        s |= dict(ks=torch.zeros((pages, hkv, page), device="cuda"), vs=torch.zeros((pages, hkv, page), device="cuda"),
                  k_values=torch.empty((pages, hkv, page, d), dtype=t, device="cuda"), v_values=torch.empty((pages, hkv, page, d), dtype=t, device="cuda"))
    if own:
        s["cache"] = _cache(s["kc"], s["vc"], s["ks"], s["vs"])
    return s


def _counts(case):
    """New tokens of every sequence: from all that a call allows down to half of them."""
    return np.array([case["new"] - 5 * i % (case["new"] // 2 + 1) for i in range(case["b"])])


def _attend(case, seed, gen):
    t, (b, new, hq, hkv, d, page) = TYPES[case["dtype"]], (case[f] for f in ("b", "new", "hq", "hkv", "d", "page"))
    rng = np.random.default_rng(seed)
    counts = _counts(case)
    lens = np.maximum(rng.integers(max(1, case["longest"] // 2), case["longest"] + 1, b), counts)
    lens[-1] = case["longest"]
    per = -(-int(lens.max()) // page)  # pages of the longest sequence
    blocks = rng.permutation(b * per).reshape(b, per).astype(np.int32)
    pages = b * per
    mask = None
    if case["tree"]:  # every drafted token but the first hangs on an earlier one
        words = np.zeros(int(counts.sum()), np.uint64)
        at = 0
        for c in counts:
            for i in range(c):
                words[at + i] = np.uint64(1 << i) | (words[at + rng.integers(max(0, i - 6), i)] if i else np.uint64(0))
            at += c
        mask = torch.from_numpy(words.view(np.int64)).cuda()
    if case["int8"]:
        kc, vc = (torch.randint(-127, 128, (pages, hkv, page, d), dtype=torch.int8, device="cuda", generator=gen) for _ in range(2))
        ks, vs = (_uniform(gen, 0.008, 0.024, pages, hkv, page) for _ in range(2))
    else:
        kc, vc, ks, vs = _randn(gen, t, pages, hkv, page, d), _randn(gen, t, pages, hkv, page, d), None, None
    total = int(counts.sum())
    s = dict(q=_randn(gen, t, total, hq, d), kc=kc, vc=vc, ks=ks, vs=vs, starts=torch.from_numpy(np.concatenate(([0], np.cumsum(counts))).astype(np.int32)).cuda(),
             lens=torch.from_numpy(lens.astype(np.int32)).cuda(), blocks=torch.from_numpy(blocks).cuda(), new=new, longest=int(lens.max()), mask=mask,
             out=torch.zeros((total, hq, d), dtype=t, device="cuda"))
    if own:
        s["cache"] = _cache(kc, vc, ks, vs)
    return s


def _sample(case, gen):
    r = case["r"]
    s = dict(logits=_randn(gen, torch.float32, r, case["v"]).mul_(2.5).to(TYPES[case["dtype"]]), uniform=_uniform(gen, 0, 1, r),
             temperature=_uniform(gen, 0.6, 1.2, r), top_k=None, top_p=None, min_p=None)
    if case["filters"]:  # every request has its own: some without top-k, some without min-p, one row in sixteen greedy
        k = torch.randint(1, 400, (r,), device="cuda", generator=gen)
        s |= dict(top_k=torch.where(k < 200, k, 0).to(torch.int32), top_p=_uniform(gen, 0.6, 1, r),
                  min_p=torch.clamp(_uniform(gen, -0.03, 0.03, r), min=0), temperature=torch.where(torch.arange(r, device="cuda") % 16 == 15, 0.0, s["temperature"]))
    return s


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    if kind in ("linear", "gated"):
        s = _linear(case, gen)
    elif kind == "append":
        s = _append(case, gen)
    elif kind == "attend":
        s = _attend(case, seed, gen)
    else:
        s = _sample(case, gen)
    return dict(s, kind=kind)


# ---- one pass: the plain forms ----------------------------------------------------------------------------------------
def _activate(x, act):
    return x * torch.sigmoid(x) if act == "silu" else 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_linear(s):
    rows, half = s["q"].shape
    q = torch.stack((s["q"] & 15, s["q"] >> 4), 2).view(rows, 2 * half).float()
    spread = lambda t: t.float().repeat_interleave(s["group"], 1)[:, :2 * half]  # noqa: E731
    w = (q - (8.0 if s["zeros"] is None else spread(s["zeros"]))) * spread(s["scales"])
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["act"]:
        gate, up = y.chunk(2, 1)
        y = _activate(gate, s["act"]) * up
    return y.to(s["x"].dtype)


def _plain_rotate(x, weight, cos, sin, interleaved):
    x = x.float()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    rot = 2 * cos.shape[-1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_place(x, slots, place, scales):
    pages, heads, page, d = place.shape
    at = slots.long()
    if scales is None:
        place[at // page, :, at % page] = x.to(place.dtype)
        return
    scale = x.abs().amax(-1) / 127
    place[at // page, :, at % page] = torch.round(x / torch.where(scale > 0, scale, 1.0)[..., None]).to(torch.int8)
    scales[at // page, :, at % page] = scale


def _plain_append(s):
    cos, sin = s["table"][s["positions"].long()].chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    s["out"].copy_(_plain_rotate(s["q"], s["q_norm"], cos, sin, s["interleaved"]))
    _plain_place(_plain_rotate(s["k"], s["k_norm"], cos, sin, s["interleaved"]), s["slots"], s["kc"], s["ks"])
    _plain_place(s["v"].float(), s["slots"], s["vc"], s["vs"])


def _plain_attend(s):
    total, hq, d = s["q"].shape
    pages, hkv, page, _ = s["kc"].shape
    b, per = s["blocks"].shape
    group, new, n = hq // hkv, s["new"], per * page

    def gathered(pool, scales):
        x = pool[s["blocks"]].float() if scales is None else pool[s["blocks"]].float() * scales[s["blocks"]][..., None]
        return x.transpose(1, 2).reshape(b, hkv, n, d)

    starts, lens = s["starts"].long(), s["lens"].long()
    counts = starts[1:] - starts[:-1]
    rows = torch.arange(new, device="cuda")
    there = rows < counts[:, None]                             # b, new
    at = torch.clamp(starts[:-1, None] + rows, max=total - 1)  # the row of q
    q = s["q"].float()[at].view(b, new, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, new * group, d)
    scores = q @ gathered(s["kc"], s["ks"]).transpose(-1, -2) * (1 / math.sqrt(d))
    token = torch.arange(n, device="cuda")
    drafted = token - (lens - counts)[:, None]                 # b, n: the index among the new tokens, below zero before them
    if s["mask"] is None:
        seen = drafted[:, None] <= rows[:, None]
    else:
        seen = (drafted < 0)[:, None] | ((s["mask"][at][..., None] >> torch.clamp(drafted, 0, 63)[:, None]) & 1 > 0)
    seen = seen & (token < lens[:, None])[:, None]             # b, new, n
    scores = scores.view(b, hkv, new, group, n).masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (p / p.sum(-1, keepdim=True)).view(b, hkv, new * group, n) @ gathered(s["vc"], s["vs"])
    o = o.view(b, hkv, new, group, d).permute(0, 2, 1, 3, 4).reshape(b, new, hq, d)
    s["out"].copy_(o[there])
    return s["out"]


def _plain_sample(s):
    x = s["logits"].double()
    rows, v = x.shape
    t = s["temperature"].double()[:, None]
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ordered - ordered[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(v, device="cuda")
    keep = (t > 0) | (rank == 0)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & (rank < torch.where(k > 0, k, v))
        kept = w * keep
        before = kept.cumsum(1) - kept
        keep = keep & ((before < s["top_p"].double()[:, None] * kept.sum(1, keepdim=True)) | (rank == 0)) & (w >= s["min_p"].double()[:, None])
    c = torch.zeros_like(x).scatter_(1, order, w * keep).cumsum(1)
    return torch.clamp((c <= s["uniform"].double()[:, None] * c[:, -1:]).sum(1), max=v - 1)


def run(state):
    s, kind = state, state["kind"]
    if kind in ("linear", "gated"):
        return s["plan"](s["x"]) if own else _plain_linear(s)
    if kind == "append":
        if own:
            s["cache"].append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["table"], out=s["out"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                              eps=1e-6, interleaved=s["interleaved"])
        else:
            _plain_append(s)
        if s["ks"] is None:
            return s["out"], s["kc"], s["vc"]
        return s["out"], torch.mul(s["kc"], s["ks"][..., None], out=s["k_values"]), torch.mul(s["vc"], s["vs"][..., None], out=s["v_values"])
    if kind == "attend":
        if own:
            return s["cache"].attend(s["q"], s["starts"], s["lens"], s["blocks"], s["new"], mask=s["mask"], out=s["out"], longest=s["longest"])
        return _plain_attend(s)
    if own:
        from nart_amd import hipq
        return hipq.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return _plain_sample(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("linear", "gated"):
        m, n, k = case["m"], case["n"], case["k"]
        rows, groups = n * (2 if case["act"] else 1), -(-k // case["group"])
        return {"bytes": rows * k // 2 + rows * groups * (3 if case["zeros"] else 2) + 2 * rows * case["bias"] + 2 * m * (k + n), "flops": 2 * m * rows * k}
    if kind == "append":
        t, hq, hkv, d = (case[f] for f in ("t", "hq", "hkv", "d"))
        # the values that an int8 cache stands for are read off for the comparison: no part of what a pass has to do
        return {"bytes": t * (4 * hq * d + 4 * hkv * d + 2 * hkv * (d + 4 if case["int8"] else 2 * d) + 4 * case["rot"] + 8), "flops": 0}
    if kind == "attend":
        b, hq, hkv, d = (case[f] for f in ("b", "hq", "hkv", "d"))
        tokens = 0.75 * case["longest"] * b  # lengths are spread over the upper half
        rows = int(_counts(case).sum())
        return {"bytes": tokens * hkv * 2 * (d + 4 if case["int8"] else 2 * d) + rows * hq * d * 4, "flops": 4 * tokens * rows / b * hq * d}
    return {"bytes": case["r"] * (case["v"] * (4 if case["dtype"] == "fp32" else 2) + 12), "flops": 0}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_linear(s):
    x, rows, k = s["x"].double(), s["q"].shape[0], 2 * s["q"].shape[1]
    q = s["q"].to(torch.int64)
    total = torch.zeros((x.shape[0], rows), dtype=torch.float64, device="cuda")
    for g, at in enumerate(range(0, k, s["group"])):  # group by group: what is left of the zero point, times the scale
        to = min(k, at + s["group"])
        part = q[:, at // 2:to // 2]
        zero = 8 if s["zeros"] is None else s["zeros"][:, g:g + 1].to(torch.int64)
        xs = x[:, at:to]
        total += (xs[:, 0::2] @ ((part % 16) - zero).double().t() + xs[:, 1::2] @ ((part // 16) - zero).double().t()) * s["scales"][:, g].double()
    if s["bias"] is not None:
        total += s["bias"].double()
    if s["act"]:
        n = rows // 2
        g = total[:, :n]
        g = g / (1 + torch.exp(-g)) if s["act"] == "silu" else g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
        total = g * total[:, n:]
    return total


def _exact_append(s):
    n, hq, d = s["q"].shape
    pages, hkv, page, _ = s["kc"].shape
    rot = s["table"].shape[1]
    turn = torch.complex(*(s["table"].double()[s["positions"].long()].view(n, 1, 2, rot // 2).unbind(2)))
    first = torch.arange(rot // 2, device="cuda") * (2 if s["interleaved"] else 1)
    second = first + (1 if s["interleaved"] else rot // 2)

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / d + 1e-6) * weight.double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def cached(x):
        if s["ks"] is not None:
            most = x.abs().amax(-1, keepdim=True)
            x = torch.round(x * 127 / most) * (most / 127)
        flat = torch.zeros((pages * page, hkv, d), dtype=torch.float64, device="cuda")
        flat[s["slots"].long()] = x
        return flat.view(pages, page, hkv, d).transpose(1, 2).contiguous()

    return turned(s["q"], s["q_norm"]), cached(turned(s["k"], s["k_norm"])), cached(s["v"].double())


def _exact_attend(s):
    total, hq, d = s["q"].shape
    hkv, page = s["kc"].shape[1:3]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    words = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint64)
    out = torch.zeros((total, hq, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):  # sequence by sequence, without what its pages hold behind its end
        lo, hi = starts[b], starts[b + 1]
        at = s["blocks"][b, :-(-n // page)].long()

        def tokens(pool, scales):
            x = pool[at].double()
            x = x if scales is None else x * scales[at].double()[..., None]
            return x.permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n]

        k, v = tokens(s["kc"], s["ks"]), tokens(s["vc"], s["vs"])
        new = hi - lo
        if words is None:
            seen = np.tri(new, dtype=bool)
        else:
            seen = (words[lo:hi, None] >> np.arange(new, dtype=np.uint64)) % 2 == 1
        hidden = torch.from_numpy(~seen).cuda()
        for h in range(hkv):
            q = s["q"][lo:hi, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            a = (q.reshape(-1, d) @ k[h].t() / d ** 0.5).view(new, -1, n)
            a[..., n - new:].masked_fill_(hidden[:, None], -math.inf)
            out[lo:hi, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.softmax(a, -1) @ v[h]
    return out


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    u, t = s["uniform"].double().tolist(), s["temperature"].double().tolist()
    got = []
    for r in range(x.shape[0]):
        if t[r] <= 0:
            got.append(int(np.argmax(x[r])))
            continue
        w = np.exp((x[r] - x[r].max()) / t[r])
        keep = np.arange(x.shape[1])
        if s["top_k"] is not None:
            order = np.argsort(-x[r], kind="stable")
            k = int(s["top_k"][r])
            order = order[:k] if k > 0 else order
            run_up = np.concatenate(([0.0], np.cumsum(w[order])))
            many = max(1, int(np.searchsorted(run_up[:-1], float(s["top_p"][r]) * run_up[-1], side="left")))
            keep = order[:many]
            keep = np.sort(keep[w[keep] >= float(s["min_p"][r])])
        c = np.cumsum(w[keep])
        got.append(int(keep[min(len(keep) - 1, int(np.searchsorted(c, u[r] * c[-1], side="right")))]))
    return torch.tensor(got, dtype=torch.int64)


def exact(case, seed):
    s = prepare(case, seed)
    make = {"linear": _exact_linear, "gated": _exact_linear, "append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}
    return make[s["kind"]](s)
