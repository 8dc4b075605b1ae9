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


def products():
    """A work-group of 512 for 128 rows of 256 outputs: 2^23 are too many."""
    lib = base.hipq.lib()
    plans = {n: base.plan(N=n, K=32)[1] for n in (16384, 16128, 1 << 20)}
    gated = base.plan(N=8192, K=32, activation=1)[1]
    launched(0)
    run = lambda plan, M: lib.hipq_w4_run(plan, P, 32, 1 << 50, 1 << 20, M, P << 20, 1 << 60, None)  # noqa: E731
    for n, M in ((16384, (1 << 24) - 256), (16128, 1 << 24), (1 << 20, 1 << 17)):
        launched(run(plans[n], M))
        refused(run(plans[n], 1 << 24), b"outputs") if n != 16128 else None
    launched(run(gated, (1 << 24) - 256))
    refused(run(gated, 1 << 24), b"outputs")


def refused(rc, message):
    assert rc != 0 and message in base.hipq.lib().hipq_last_error(), (rc, base.hipq.lib().hipq_last_error())
    assert C.c_long.in_dll(base.STUB, "stub_launches").value == 0


def attention():
    """A work-group for each sequence, head, block of rows and part: 2^24 of 256 are too many."""
    lib = base.hipq.lib()

    def run(sequences, heads, most_new=1, dim=64, blocks=1, longest=16):
        c = base.cache(dict(heads=heads, dim=dim))
        d = base.hipq.KvAttendDesc(q=P, o=P, q_token=heads * dim, q_head=dim, o_token=heads * dim, o_head=dim, starts=P, lens=P, blocks=P, blocks_stride=blocks,
                                   sequences=sequences, tokens=sequences, q_heads=heads, blocks_per_sequence=blocks, most_new=most_new, longest=longest, scale=0.1)
        return lib.hipq_kv_attend(C.byref(c), C.byref(d), P, 1 << 60, None)
    for sequences, heads, more in ((1 << 20, 15, {}), (1 << 12, 4095, {}), (1 << 10, 512, dict(most_new=1 << 9)), (300, 64, dict(dim=128, most_new=4096, longest=1 << 14, blocks=1 << 10))):
        launched(run(sequences, heads, **more))
    for sequences, heads, more in ((1 << 20, 16, {}), (1 << 12, 4096, {}), (1 << 20, 64, {}), (1 << 10, 512, dict(most_new=1 << 10))):
        refused(run(sequences, heads, **more), b"work-groups")


def new_tokens():
    """A work-item for eight elements of a token, for each eight of its heads."""
    lib = base.hipq.lib()

    def run(tokens, heads, dim=256):
        c = base.cache(dict(heads=heads, dim=dim))
        d = base.hipq.KvAppendDesc(k=P, v=P, k_head=dim, v_head=dim, positions=P, slots=P, tokens=tokens, eps=1e-6)
        return lib.hipq_kv_append(C.byref(c), C.byref(d), None)
    for tokens, heads in ((1 << 24, 28), (1 << 20, 508), (5, 4096)):
        (side, rows), = launched(run(tokens, heads))
        assert side >= tokens * 32 * -(-2 * heads // 8) or tokens == 5
    for tokens, heads in ((1 << 24, 32), (1 << 24, 4096), (1 << 20, 512)):
        refused(run(tokens, heads), b"tokens of")


CASES = [samples, sums_of_x, products, attention, new_tokens]


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
