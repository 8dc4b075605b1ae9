"""A launch has under 2^32 work-items side by side: of more, only what is left over 2^32 would run, without an error.  What the entry points launch at
the ends of their ranges, without a GPU (as in test_lm_cpu.py)."""
import ctypes as C
import os
import subprocess
import sys

import pytest

import test_lm_cpu as base
from test_lm_cpu import F16, P, ROOT


def launched(rc):
    """The launches of one call, as (work-items side by side, rows of them)."""
    n = C.c_long.in_dll(base.STUB, "stub_launches")
    grids = (C.c_uint64 * 64).in_dll(base.STUB, "stub_grids")
    assert rc == 0, base.hipq.lib().hipq_last_error()
    got = [(grids[2 * i], grids[2 * i + 1]) for i in range(n.value)]
    n.value = 0
    assert got and all(0 < x < 1 << 32 and 0 < y < 1 << 16 for x, y in got), got
    return got


def samples():
    run = lambda rows: launched(base.hipq.lib().hipq_sample(P, F16, rows, 7, 7, P, None, None, None, None, P, None))  # noqa: E731
    for rows in (1, 1 << 21, (1 << 22) - 1, 1 << 22, (1 << 22) + 3, 1 << 24):
        assert sum(x for x, _ in run(rows)) == 1024 * rows


def sums_of_x():
    """Of 2^35 numbers, eight for each work-item."""
    lib = base.hipq.lib()
    for K, M in ((2048, 1 << 24), (16384, 1 << 21), (16384, (1 << 21) - 1), (4096, 1024)):
        plan = base.plan(N=2048, K=K)[1]
        launched(0)
        assert lib.hipq_w4_plan_kernel(plan, M) == b"w4_tile_128x256"
        (side, rows), *_ = launched(lib.hipq_w4_run(plan, P, K, 1 << 50, 2048, M, P << 20, 1 << 60, None))
        items = -(-M // 128) * 128 * K // 8
        assert items <= side * rows < items + side


CASES = [samples, sums_of_x]


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    folder = tmp_path_factory.mktemp("hip")
    source = folder / "stub.c"
    source.write_text('#define hipLaunchKernel launch_one\n#include "%s"\n#undef hipLaunchKernel\n' % os.path.join(ROOT, "tests", "hip_stub.c") + """
int stub_device;
int hipGetDevice(int *d) { return *d = stub_device, kSuccess; }
int hipFuncSetAttribute(const void *f, int a, int v) { return (void)f, (void)a, (void)v, kSuccess; }
long stub_launches;
uint64_t stub_grids[64];
int hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds, void *st)
{
    if (stub_launches < 32) {
        stub_grids[2 * stub_launches] = (uint64_t)g.x * b.x, stub_grids[2 * stub_launches + 1] = g.y;
        stub_launches++;
    }
    return launch_one(f, g, b, args, lds, st);
}
""")
    so = str(folder / "stub.so")
    subprocess.check_call(["gcc", "-O1", "-std=gnu11", "-Wall", "-fPIC", "-shared", str(source), "-o", so])
    return so


@pytest.mark.parametrize("case", CASES, ids=lambda c: c.__name__)
def test_grids(case, stub):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, case.__name__], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stdout[-4000:]


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    base.STUB = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    from nart_amd import hipq
    base.hipq = hipq
    globals()[sys.argv[2]]()
