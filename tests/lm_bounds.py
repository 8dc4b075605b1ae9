"""How far results of the language-model operators spread around their formulas in 64 bits, beside the worst cases of lm_reference.py: roundings
to 16 bits are independent and go either way, so what they leave behind grows like the root of their squares' sum.  A kernel that loses a tile,
rounds a weight once more than it says or keeps a sum in 16 bits stays within the worst case of a long sum, and far outside of this."""
import math

import torch

from lm_reference import half_step


def rms(x, *dims):
    return x.square().mean(dims).sqrt() if dims else x.square().mean().sqrt()


def rounded(want, dtype):
    """What rounding leaves of results in 64 bits: at least half of the type's smallest step, where it is coarser than their own."""
    return want.to(dtype).double() - want


def linear_spread(x, q, scales, group, zeros=None, bias=None, act=None):
    """(y, root mean square of what sums in 32 bits may be off), for x of either sign.  Every group sums `group` terms of at most 63 |x|; their
    signs make a running sum of at most 63 sqrt(sum x^2), and each addition rounds it by up to 2^-24 of itself, independently of the others:
    sqrt(group) 2^-24 63 sqrt(sum x^2) of a group, once more for the sums of x."""
    x, k = x.double(), q.shape[1]
    y = torch.zeros((x.shape[0], q.shape[0]), dtype=torch.float64, device=x.device)
    var = torch.zeros_like(y)
    for g, at in enumerate(range(0, k, group)):
        xs, w, s = x[:, at:at + group], q[:, at:at + group].double(), scales[:, g].double()
        y += (xs @ (w - (8.0 if zeros is None else zeros[:, g:g + 1].double())).t()) * s
        var += 2 * group * (2.0 ** -24 * 63 * s).square() * xs.square().sum(1, keepdim=True)
    # the running sum over the groups
    var += math.ceil(k / group) * (2.0 ** -24 * y.abs()).square()
    off = var.sqrt()
    if bias is not None:
        y = y + bias.double()
    if act:
        (gate, up), (off_gate, off_up) = y.chunk(2, 1), off.chunk(2, 1)
        t = gate if act == "silu" else 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        a = gate / (1 + torch.exp(-t))
        y, off = a * up, 1.13 * off_gate * up.abs() + a.abs() * off_up + 2.0 ** -20 * (a * up).abs()
    return y, off


def check_linear_spread(got, x, q, scales, group, zeros=None, bias=None, act=None):
    """The results' distance from the formula is that of one rounding: 1.2 times over all (they are 1000 and more, a root mean square of which is
    good to 5 %; a second rounding of the same size would make it 1.41 times)."""
    want, off = linear_spread(x, q, scales, group, zeros, bias, act)
    assert want.numel() >= 1000
    far, may = rms(got.double() - want), 1.2 * torch.sqrt(rms(rounded(want, got.dtype)).square() + rms(off).square())
    assert far <= may, "%g away, %g allowed" % (far, may)


def attend_spread(q, k, v, starts, lens, mask, scale, group, k_scale=None, v_scale=None, exact=False):
    """(o, root mean square of what the weights' roundings make of it): arguments of lm_reference.attend.  A weight p_t is off by
      * its rounding to 16 bits: evenly spread over half a step, so 1 / sqrt(3) of it as a root mean square at most,
      * in float16 up to 2^-32 of the largest weight (over codes: times value scale), where that is more,
      * its score's sum of `dim` products and the scaling: sqrt(dim + 6) roundings of 2^-24 of the products' sum,
    each times its value.  Sums in 32 bits: 2^-20 of sum p |v|.  exact: weights are not rounded."""
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    var = torch.zeros_like(o)
    dim, h = q.shape[-1], 0.0 if exact else half_step(q.dtype)
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        new = hi - lo
        if new == 0 or n == 0:
            continue
        fresh = torch.arange(n, device=q.device) - (n - new)
        row = torch.arange(new, device=q.device)[:, None]
        seen = fresh <= row if mask is None else (fresh < 0) | (((mask[lo:hi, None] >> fresh.clamp(0, 63)) & 1) > 0)
        for head in range(k[b].shape[0]):
            qs = q[lo:hi, head * group:(head + 1) * group].double()
            ks = 1.0 if k_scale is None else k_scale[b][head].double()
            vs = torch.ones(n, dtype=torch.float64, device=q.device) if v_scale is None else v_scale[b][head].double()
            kh, codes = k[b][head].double(), v[b][head].double()
            x = torch.where(seen[:, None], (qs @ kh.t()) * ks * scale, -math.inf)
            p = torch.softmax(x, -1).nan_to_num(0.0)  # rows that see nothing
            w = p * vs
            o[lo:hi, head * group:(head + 1) * group] = w @ codes
            size = (qs.abs() @ kh.abs().t()) * ks * abs(scale)
            d = 2.0 ** -24 * math.sqrt(dim + 6) * torch.where(seen[:, None], size, 0.0) + 2.0 ** -22
            tiny = 2.0 ** -32 * w.amax(-1, keepdim=True) if q.dtype == torch.float16 and not exact else 0.0
            rel = (w * torch.sqrt(h * h / 3 + d * d)).square() + (tiny * seen[:, None]) ** 2 / 3
            var[lo:hi, head * group:(head + 1) * group] = rel @ codes.square() + (2.0 ** -20 * (w @ codes.abs())).square()
    return o, var.sqrt()


def check_attend_spread(got, want, off, rows=None):
    """Root mean squares over a head's elements, and over all.  A weight's rounding is the same for all elements of a head, so where few tokens
    make the result it does not average: up to half a step, sqrt(3) times the root mean square, for each, and what the values of two tokens have
    in common, some 2 / sqrt(64) of it: 2.2 times together.  Over `rows` heads of rows that are independent (by default all of them) squares
    of roundings average: their own spread is 0.9 of their mean, half of that for the root, four times that for the worst of many tests."""
    far, one = got.double() - want, torch.sqrt(off.square() + rounded(want, got.dtype).square())
    smallest = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    rows = want[..., 0].numel() if rows is None else rows
    for what, limit in ((rms(far, -1) / (rms(one, -1) + smallest), 2.2), (rms(far) / (rms(one) + smallest), min(2.2, 1.1 + 1.8 / math.sqrt(rows)))):
        assert torch.isfinite(what).all() and what.max() <= limit, "%g times what roundings leave, %g allowed" % (what.max(), limit)
