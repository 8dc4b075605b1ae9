"""The spreads of lm_bounds.py, on the CPU: results that are computed as the kernels say they compute them keep to them, results with a mistake
that the worst case of a sum would hide do not."""
import numpy as np
import pytest
import torch

import lm_bounds
import lm_reference as ref

BF16, F16 = torch.bfloat16, torch.float16


def normals(rng, dtype, *shape):
    return torch.from_numpy(rng.standard_normal(shape)).to(dtype)


# ---- products ----------------------------------------------------------------------------------------------------------
def product(x, q, scales, group, zeros, how):
    x, y = x.float(), 0
    for g, at in enumerate(range(0, q.shape[1], group)):
        w, s = q[:, at:at + group].float() - zeros[:, g:g + 1].float(), scales[:, g].float()
        if how == "rounded weights":
            y = y + x[:, at:at + group] @ (w * s[:, None]).to(scales.dtype).float().t()
        else:
            y = y + (x[:, at:at + group] @ w.t()) * s
        if how == "16-bit sums":
            y = y.to(scales.dtype).float()
        if how == "sums of x with a wrong zero" and g == 1:
            y = y + x[:, at:at + group].sum(1, keepdim=True) * s * 2.0 ** -4
    return y.to(scales.dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("k, group", [(1056, 128), (4128, 128), (2112, 64), (1024, 32)])
def test_products(k, group, dtype):
    rng = np.random.default_rng(k)
    groups = -(-k // group)
    x, q = normals(rng, dtype, 16, k), torch.from_numpy(rng.integers(0, 16, (96, k)).astype(np.uint8))
    scales, zeros = torch.from_numpy(rng.random((96, groups)) * 0.02 + 0.002).to(dtype), torch.from_numpy(rng.integers(0, 16, (96, groups)).astype(np.uint8))
    lm_bounds.check_linear_spread(product(x, q, scales, group, zeros, ""), x, q, scales, group, zeros)
    for how in ("rounded weights", "16-bit sums", "sums of x with a wrong zero"):
        with pytest.raises(AssertionError, match="away"):
            lm_bounds.check_linear_spread(product(x, q, scales, group, zeros, how), x, q, scales, group, zeros)


# ---- attention ---------------------------------------------------------------------------------------------------------
def tiles(q, k, v, ks, vs, scale, how):
    """One row over the cache with weights in 16 bits."""
    dtype, n = q.dtype, k.shape[0]
    s = ((k.double() @ q.double()) * (1 if ks is None else ks.double()) * scale * 1.4426950408889634).float()
    p = torch.exp2(s - s.max().ceil())
    w = p if vs is None else p * vs
    shift = 1.0
    if dtype == F16:
        shift = 2.0 ** 7 if vs is None else 2.0 ** 7 / 2.0 ** float(torch.log2(w.max()).floor())
        if how == "weights by the largest scale":
            shift = 1 / float(vs.max())
        if how == "weights of 1 and less":
            shift = 1.0
    w = (w * shift).to(dtype).float() / shift
    total = (w if vs is None else p).clone()
    if how in ("a tile lost", "the first tile lost", "the last tokens lost"):
        at = {"a tile lost": n // 64 * 32, "the first tile lost": 0, "the last tokens lost": n - 32}[how]
        w[at:at + 32], total[at:at + 32] = 0, 0
    o = (w.double() @ v.double()) / total.double().sum()
    return (o * (1.01 if how == "scaled" else 1)).to(dtype)


MISTAKES = ["a tile lost", "the first tile lost", "the last tokens lost", "scaled"]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [700, 4096, 20000])
def test_attention(n, int8, dtype):
    rng, dim, rows = np.random.default_rng(n), 128, 4
    q = normals(rng, dtype, rows, 1, dim)
    k, v = (torch.from_numpy(rng.integers(-127, 128, (n, dim)).astype(np.int8)) if int8 else normals(rng, dtype, n, dim) for _ in range(2))
    ks, vs = (torch.from_numpy(rng.random(n).astype(np.float32) * 0.02 + 0.001) if int8 else None for _ in range(2))
    one = lambda t: None if t is None else t[None]  # noqa: E731
    many = lambda t: None if t is None else [one(t)] * rows  # noqa: E731
    want, off = lm_bounds.attend_spread(q, many(k), many(v), list(range(rows + 1)), [n] * rows, None, dim ** -0.5, 1, many(ks), many(vs))
    worst = ref.attend(q, many(k), many(v), list(range(rows + 1)), [n] * rows, None, dim ** -0.5, 1, many(ks), many(vs))[0]
    assert torch.allclose(want, worst, rtol=1e-12, atol=1e-14)
    run = lambda how: torch.stack([tiles(q[r, 0], k, v, ks, vs, dim ** -0.5, how) for r in range(rows)])[:, None]  # noqa: E731
    lm_bounds.check_attend_spread(run(""), want, off)
    for how in MISTAKES:
        with pytest.raises(AssertionError, match="roundings leave"):
            lm_bounds.check_attend_spread(run(how), want, off)


# one score far above the rest, one value scale many times the others'
@pytest.mark.parametrize("n, gap, ratio", [(8192, 9, 4096), (131072, 12, 256), (131072, 15, 16)])
def test_attention_float16_codes_of_many_sizes(n, gap, ratio):
    rng, dim = np.random.default_rng(n), 64
    q = torch.ones((1, 1, dim), dtype=F16)
    k = torch.full((n, dim), 1, dtype=torch.int8)
    ks = torch.from_numpy((rng.standard_normal(n) * 0.5).astype(np.float32))
    ks[n // 3] = gap
    v = torch.from_numpy(rng.integers(1, 128, (n, dim)).astype(np.int8))
    vs = torch.from_numpy(rng.random(n).astype(np.float32) * 0.01 + 0.01)
    vs[n // 2] *= ratio
    args = (q, [k[None]], [v[None]], [0, 1], [n], None, 1 / dim, 1, [ks[None]], [vs[None]])
    want, off = lm_bounds.attend_spread(*args)
    lm_bounds.check_attend_spread(tiles(q[0, 0], k, v, ks, vs, 1 / dim, "")[None, None], want, off)
    with pytest.raises(AssertionError, match="roundings leave"):
        lm_bounds.check_attend_spread(tiles(q[0, 0], k, v, ks, vs, 1 / dim, "weights by the largest scale")[None, None], want, off)


def test_attention_float16_long_tail():
    """The same over 16 bits: many tokens of small weights that have a mean of their own."""
    rng, dim, n = np.random.default_rng(3), 64, 131072
    q, k, v = torch.ones((1, 1, dim), dtype=F16), torch.zeros((n, dim), dtype=F16), normals(rng, F16, n, dim) + 1
    k[n // 3], v[n // 3] = 17.4, -1
    args = (q, [k[None]], [v[None]], [0, 1], [n], None, 1 / dim, 1)
    want, off = lm_bounds.attend_spread(*args)
    lm_bounds.check_attend_spread(tiles(q[0, 0], k, v, None, None, 1 / dim, "")[None, None], want, off)
    with pytest.raises(AssertionError, match="roundings leave"):
        lm_bounds.check_attend_spread(tiles(q[0, 0], k, v, None, None, 1 / dim, "weights of 1 and less")[None, None], want, off)
