"""Experts, weights of the cache's tokens, eviction and penalties in 64 bits, written from their formulas, with the bounds that follow for a kernel's results
(as in lm_reference.py: a sum or product in 32 bits is off by 2^-23 of its size at most, a rounding by half a step)."""
import math

import numpy as np
import torch

import lm_reference as ref
from lm_reference import STEP32, half_step


def choose(logits, top, scores, normalize):
    """(experts [tokens, top], -1 where there is none; their shares)."""
    x = logits.double().cpu().numpy()
    which, share = np.full((x.shape[0], top), -1), np.zeros((x.shape[0], top))
    for t, row in enumerate(x):
        row = np.where(np.isnan(row), -np.inf, row)
        order = np.argsort(-row, kind="stable")[:top]
        order = order[row[order] > -np.inf]
        if len(order) == 0:
            continue
        most = row[order[0]]
        with np.errstate(over="ignore", invalid="ignore"):
            if scores == "softmax":
                w = np.where(row == most, 1.0, np.exp(row - most))
                w = w[order] / (w[order] if normalize else w).sum()
            else:
                low = min(most, 0.0) if normalize else 0.0  # both terms times e^low
                w = 1 / (np.exp(low) + np.exp(low - row[order]))
                w = w / w.sum() if normalize else w
        which[t, :len(order)], share[t, :len(order)] = order, w
    return which, share


def experts(x, logits, gate_up, gate_up_scales, down, down_scales, top, group, gate_up_zeros=None, down_zeros=None, act="silu", scores="softmax", normalize=True):
    """(y, how far y may be off, its root mean square from the hidden rows' rounding): gate_up and down unpacked."""
    which, share = choose(logits, top, scores, normalize)
    y = torch.zeros((x.shape[0], down.shape[1]), dtype=torch.float64, device=x.device)
    off, var = torch.zeros_like(y), torch.zeros_like(y)
    half = half_step(x.dtype)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    for e in range(gate_up.shape[0]):
        rows, slots = np.nonzero(which == e)
        if len(rows) == 0:
            continue
        at, w = torch.from_numpy(rows).to(x.device), torch.from_numpy(share[rows, slots]).to(x.device)[:, None]
        pick = lambda t: None if t is None else t[e]  # noqa: E731
        h, h_off = ref.linear(x[at], gate_up[e], gate_up_scales[e], group, pick(gate_up_zeros), None, act)
        o, o_off = ref.linear(h, down[e], down_scales[e], group, pick(down_zeros))
        zero = 8.0 if down_zeros is None else down_zeros[e].double().repeat_interleave(group, 1)[:, :down.shape[2]]
        dense = (down[e].double() - zero) * down_scales[e].double().repeat_interleave(group, 1)[:, :down.shape[2]]
        h_off = h_off + half * (h.abs() + h_off) + tiny
        o_off = o_off + h_off @ dense.abs().t()
        y[at] += w * o
        # a share: exponentials and a division, good to 2^-20, scores up to some hundreds; below 2^-126, the smallest normal number of 32 bits, it is 0
        off[at] += w * (o_off + (2.0 ** -20 + STEP32 * (top + 2)) * (o.abs() + o_off)) + 2.0 ** -126 * (o.abs() + o_off)
        var[at] += (w * torch.sqrt((h * half).square() @ dense.square().t() / 3)).square()
    return y, off, var.sqrt()


def penalize(x, tokens=None, lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None, bias_tokens=None, bias=None, allowed=None):
    """(scores, how far): one row after the other, entry by entry."""
    y = x.double().cpu().numpy().copy()
    off = np.zeros_like(y)
    rows, vocab = y.shape
    value = lambda t, r, otherwise: otherwise if t is None else float(t[r])  # noqa: E731
    for r in range(rows):
        seen, count = {}, {}
        if tokens is not None:
            n = tokens.shape[1] if lens is None else min(int(lens[r]), tokens.shape[1])
            for i, t in enumerate(tokens[r, :max(n, 0)].tolist()):
                if 0 <= t < vocab:
                    seen[t] = True
                    if i >= value(prompt_lens, r, 0):
                        count[t] = count.get(t, 0) + 1
        for t in seen:
            by = value(repetition, r, 1.0)
            if repetition is not None:
                y[r, t] = y[r, t] / by if y[r, t] > 0 else y[r, t] * by
            off[r, t] = STEP32 * abs(y[r, t])
            if t in count:
                less = count[t] * value(frequency, r, 0.0) + value(presence, r, 0.0)
                y[r, t] -= less
                off[r, t] += STEP32 * (2 * abs(less) + abs(y[r, t]))
        if bias is not None:
            last = {}
            for t, b in zip(bias_tokens[r].tolist(), bias[r].tolist()):
                last[t] = b
            for t, b in last.items():
                if 0 <= t < vocab:
                    y[r, t] += b
                    off[r, t] += STEP32 * abs(y[r, t])
        if allowed is not None:
            bits = np.unpackbits(np.ascontiguousarray(allowed[r].cpu().numpy()).view(np.uint8), bitorder="little")[:vocab]
            y[r, bits == 0] = -np.inf
            off[r, bits == 0] = 0
    return torch.from_numpy(y), torch.from_numpy(off)


def weigh(q, k, starts, lens, mask, scale, group, old, k_scale=None):
    """[(weights [heads, len], how far)] of each sequence with new tokens, None of others: k: lists of [heads, len, dim] (codes with scales [heads, len]), old: of [heads, len]."""
    got = []
    dim = q.shape[-1]
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        new = hi - lo
        if new == 0:
            got.append(None)
            continue
        fresh = torch.arange(n, device=q.device) - (n - new)
        row = torch.arange(new, device=q.device)[:, None]
        seen = fresh <= row if mask is None else (fresh < 0) | (((mask[lo:hi, None] >> fresh.clamp(0, 63)) & 1) > 0)
        before = torch.where(fresh < 0, old[b].double(), 0.0)
        w, off = before.clone(), STEP32 * before.abs()
        for h in range(k[b].shape[0]):
            qs, kh = q[lo:hi, h * group:(h + 1) * group].double(), k[b][h].double()
            ks = 1.0 if k_scale is None else k_scale[b][h].double()
            x = torch.where(seen[:, None], (qs @ kh.t()) * ks * scale, -math.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
            p = p / torch.where(p.sum(-1, keepdim=True) > 0, p.sum(-1, keepdim=True), 1.0)
            # a score's error is the relative error of its weight and, as largest of a row, of the sum (as for attention); the logarithm of the sum, and what is taken
            # off in its place, are as large as the scores, and rounded
            size = (qs.abs() @ kh.abs().t()) * ks * abs(scale)
            d = (STEP32 * (dim + 10) * torch.where(seen[:, None], size, 0.0)).amax(-1, keepdim=True) + 2.0 ** -20
            w[h] += p.sum((0, 1))
            # sums of n terms in 32 bits, and of the rows
            off[h] += (p * (3 * d + STEP32 * 64)).sum((0, 1)) + STEP32 * new * group * w[h].abs()
        got.append((w, off))
    return got


def evict(weights, lens, budget, recent, first):
    """For each sequence [heads, min(len, budget)]: the places of the tokens that stay.  weights: lists of [heads, len]."""
    got = []
    for w, n in zip(weights, lens):
        rows = []
        for h in range(w.shape[0]):
            if n <= budget:
                rows.append(np.arange(n))
                continue
            x = w[h].double().cpu().numpy()
            middle = np.arange(first, n - recent)
            key = np.where(np.isnan(x[middle]), -np.inf, x[middle])
            order = np.lexsort((middle, -key, np.isnan(x[middle])))  # numbers before NaN, the heaviest first, of equal ones the first
            rows.append(np.sort(np.concatenate((np.arange(first), middle[order[:budget - first - recent]], np.arange(n - recent, n)))))
        got.append(np.stack(rows) if rows else np.zeros((0, 0), int))
    return got
