"""The language-model operators in 64 bits, written from their formulas, and the bounds that follow for a kernel's results.  A kernel sums in 32
bits: every addition or product may be off by 2^-23 of its result (half of that where it rounds to nearest), and the result is rounded once."""
import math

import torch

STEP32 = 2.0 ** -23


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def pack_rows(q):
    """uint8 [N, K] of 0..15 -> [N, K / 2], the lower half first."""
    return q[:, 0::2] | (q[:, 1::2] << 4)


def activate(x, name):
    t = x if name == "silu" else 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    return x / (1 + torch.exp(-t))


def linear(x, q, scales, group, zeros=None, bias=None, act=None):
    """(y, how far y may be off): q unpacked."""
    x, n, k = x.double(), q.shape[0], q.shape[1]
    y = torch.zeros((x.shape[0], n), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)  # of what is summed on the way: x (16 + q) and (16 + z) x
    for g, at in enumerate(range(0, k, group)):
        xs, w = x[:, at:at + group], q[:, at:at + group].double()
        z = 8.0 if zeros is None else zeros[:, g:g + 1].double()
        s = scales[:, g].double()
        y += (xs @ (w - z).t()) * s
        size += (xs.abs() @ (w + z + 32).t()) * s.abs()
    off = STEP32 * (2 * group + math.ceil(k / group) + 4) * size
    if bias is not None:
        y, off = y + bias.double(), off + STEP32 * (y.abs() + bias.double().abs())
    if act:
        (gate, up), (off_gate, off_up) = y.chunk(2, 1), off.chunk(2, 1)
        a = activate(gate, act)
        # both activations change by at most 1.13 times what their argument does; the exponential and the division are good to 2^-20 of
        # what they give (the argument of the exponential is rounded: 2^-23 of up to 88 / log2(e) and more, where the result is about 0)
        off_a = 1.13 * off_gate + 2.0 ** -20 * (a.abs() + 1e-3)
        y, off = a * up, off_a * up.abs() + a.abs() * off_up + off_a * off_up
    return y, off


def within(got, want, off):
    """Is every value of `got` rounded from something at most `off` away from `want`?"""
    h = half_step(got.dtype)
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[got.dtype]  # half of the smallest step
    far = (got.double() - want).abs() - (off + h * (want.abs() + off) + tiny)
    return bool((far <= 0).all()), float(far.max()) if far.numel() else 0.0


def rotate(x, weight, eps, cos, sin, interleaved):
    """(y, how far): x [tokens, heads, dim], cos and sin [tokens, rot / 2]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    half = cos.shape[-1]
    rot = 2 * half
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    y, size = x.clone(), x.abs()
    a, b = ((slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, half), slice(half, rot)))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    size = size.clone()
    both = x[..., a].abs() + x[..., b].abs()
    size[..., a] = size[..., b] = both
    return y, (STEP32 * 24 if weight is not None else STEP32 * 3) * size  # a norm: 16 additions and shuffled sums, a root, a quotient, products


def attend(q, k, v, starts, lens, mask, scale, group, k_scale=None, v_scale=None, dtype=None):
    """(o, how far): q [tokens, q heads, dim]; k, v: lists of [heads, len, dim] (codes with scales [heads, len])."""
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(o)
    dim = q.shape[-1]
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        new = hi - lo
        if new == 0:
            continue
        fresh = torch.arange(n, device=q.device) - (n - new)
        row = torch.arange(new, device=q.device)[:, None]
        if mask is None:
            seen = fresh <= row
        else:
            seen = (fresh < 0) | (((mask[lo:hi, None] >> fresh.clamp(0, 63)) & 1) > 0)
        for h in range(k[b].shape[0]):
            qs = q[lo:hi, h * group:(h + 1) * group].double()
            kh, vh = k[b][h].double(), v[b][h].double()
            ks = 1.0 if k_scale is None else k_scale[b][h].double()
            vs = 1.0 if v_scale is None else v_scale[b][h].double()[:, None]
            x = (qs @ kh.t()) * ks * scale
            x = torch.where(seen[:, None], x, -math.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            o[lo:hi, h * group:(h + 1) * group] = p @ torch.where(torch.isfinite(vh), vh * vs, 0.0)
            # a score's error, which is the relative error of its weight: dim products and the scaling, codes raised by 128
            size = (qs.abs() @ (kh.abs() + (0 if k_scale is None else 256)).t()) * ks * abs(scale)
            d = (STEP32 * (dim + 6) * torch.where(seen[:, None], size, 0.0)).amax(-1, keepdim=True) + 2.0 ** -20
            spread = p @ (torch.where(torch.isfinite(vh), vh, 0.0).abs() * vs)
            raised = p @ ((torch.zeros_like(vh) if v_scale is None else torch.full_like(vh, 256.0)) * vs)
            # weights are rounded to the type of q (twice as far for sums that are rescaled), sums of n terms in 32 bits
            off[lo:hi, h * group:(h + 1) * group] = spread * (half_step(dtype or q.dtype) + 3 * d) + STEP32 * (n + 64) * (spread + raised)
    return o, off


def sample(x, u, t, k, p, m):
    """One row: the token (numpy-free, 64 bits)."""
    x = torch.where(torch.isnan(x.double()), -math.inf, x.double())
    top = x.max()
    if top == -math.inf:
        return -1
    order = torch.sort(x, descending=True, stable=True).indices
    if not t > 0:
        return int(order[0])
    w = torch.where(x == top, 1.0, torch.exp((x - top) / t))
    w = torch.where(x == -math.inf, 0.0, w)
    ws = w[order]
    if 0 < k < x.numel():
        ws = ws.clone()
        ws[k:] = 0
    keep = ws > 0
    if p < 1:
        keep &= (ws.cumsum(0) - ws) < p * ws.sum()
    keep &= ws >= min(m, 1.0)
    keep[0] = True
    c = torch.zeros_like(w).scatter_(0, order, ws * keep).cumsum(0)
    return min(int((c <= u * c[-1]).sum()), x.numel() - 1)
