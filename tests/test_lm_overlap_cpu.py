"""Outputs that lie over inputs which other work-groups still read are refused, without a GPU (as in test_lm_cpu.py)."""
import ctypes as C
import os
import random
import subprocess
import sys

import pytest

import test_lm_cpu as base
from test_lm_cpu import P, ROOT, stub  # noqa: F401


def bytes_of(at, width, *steps):
    """The bytes of rows of `width` bytes: steps of (how many, bytes apart)."""
    starts = [at]
    for n, step in steps:
        starts = [s + i * step for s in starts for i in range(n)]
    return {b for s in starts for b in range(s, s + width)}


def products():
    from nart_amd import hipq
    lib, rng, met = hipq.lib(), random.Random(1), [0, 0]
    plans = {(n, k): base.plan(N=n, K=k)[1] for n in (1, 8, 40) for k in (32, 64)}
    for _ in range(6000):
        (n, k), m = rng.choice(list(plans)), rng.choice((1, 1, 2, 3, 7))
        xs = k + 8 * rng.choice((0, 1, 5, 12))
        ys = rng.choice((xs, n + rng.randrange(60))) if xs >= n else n + rng.randrange(60)
        y = P + 2 * rng.randrange(-3 * ys, m * xs + 40)
        over = bool(bytes_of(P, 2 * k, (m, 2 * xs)) & bytes_of(y, 2 * n, (m, 2 * ys)))
        rc = lib.hipq_w4_run(plans[n, k], P, xs, y, ys, m, None, 0, None)
        assert (rc != 0) == over, (n, k, m, xs, ys, y - P, lib.hipq_last_error())
        assert not over or b"over x" in lib.hipq_last_error()
        met[over] += 1
    assert min(met) > 1000, met
    # all rows between each other, and far too many to look at one by one
    run = lambda y, ys: lib.hipq_w4_run(plans[8, 32], P, 64, y, ys, 1 << 24, P << 20, 1 << 60, None)  # noqa: E731
    assert run(P + 64, 64) == 0 and run(P + 112, 64) == 0 and run(P + 114, 64) != 0 and run(P + 62, 64) != 0


CASES = [products]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c.__name__)
def test_outputs_over_inputs(case, stub):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, case.__name__], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stdout[-4000:]


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    base.STUB = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    globals()[sys.argv[2]]()
