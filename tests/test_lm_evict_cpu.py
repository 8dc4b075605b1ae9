"""What an eviction writes may not lie over what its launches read, without a GPU (as in test_lm_cpu.py)."""
import ctypes as C
import importlib.util
import os
import random
import subprocess
import sys
import sysconfig

import pytest

import test_lm_cpu as base
from test_lm_cpu import P, ROOT, Tensor, stub  # noqa: F401
from test_lm_overlap_cpu import bytes_of


class At(Tensor):
    def __init__(self, at, *args, **kw):
        super().__init__(*args, **kw)
        self.at = at

    def data_ptr(self):
        return self.at

    def bytes(self):
        """Of its entries, the last dimension of which has no gaps."""
        return bytes_of(self.at, 4 * self.shape[-1], *((n, 4 * s) for n, s in zip(self.shape[:-1], self.strides[:-1])))


def evictions():
    from nart_amd import hipq
    hipq.lib()
    path = os.path.join(os.path.dirname(hipq.LIB_PATH), "hipq_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
    spec = importlib.util.spec_from_file_location("hipq_calls", path)
    calls = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(calls)
    calls.init(lambda: 0, lambda device: 0)
    calls.types("float32", "float16", "bfloat16", "int32", "int64", "uint8", "int8")
    kernels, rng, met = C.c_long.in_dll(base.STUB, "stub_kernels"), random.Random(1), {}
    k = At(P << 8, "bfloat16", 5, 2, 16, 64)
    cache = calls.kv_cache(k, k, None, None)
    for _ in range(6000):
        b, budget, far = rng.choice((1, 2, 3)), rng.choice((1, 7, 20)), rng.choice((100, 400, 3000))
        at = lambda far=far: P + 4 * rng.randrange(far)  # noqa: E731
        t = dict(weights=At(P + 16 * rng.randrange(far // 4), "float32", 5, 2, 16), lens=At(at(), "int32", b), blocks=At(at(), "int32", b, 2, stride=(rng.choice((2, 3, 40)), 1)),
                 to=At(at(), "int32", b, 2, stride=(rng.choice((2, 3, 40)), 1)), left=At(at(), "int32", b), kept=At(at(), "int32", b, 2, budget))
        if rng.random() < 0.5:
            t["left"] = t["lens"]
        bytes_ = {name: x.bytes() for name, x in t.items()}
        over = {frozenset((name, other)) for name in ("weights", "left", "kept") for other in t if other != name and bytes_[name] & bytes_[other]}
        if t["left"].at == t["lens"].at:
            over.discard(frozenset(("left", "lens")))
        before = kernels.value
        if b > 1 and t["to"].at == t["blocks"].at and t["to"].strides != t["blocks"].strides:
            continue  # refused for another reason
        try:
            rc = calls.kv_evict(cache, 0, t["weights"], t["lens"], t["blocks"], t["to"], t["left"], t["kept"], budget, 0, 0, None, None)
        except ValueError as e:
            names = str(e).split(" lies over ")
            assert frozenset(names) in over and kernels.value == before, (e, over)
            met[frozenset(names)] = met.get(frozenset(names), 0) + 1
        else:
            assert rc == 0 and not over and kernels.value == before + 2, (over, hipq.lib().hipq_last_error())
            met[None] = met.get(None, 0) + 1
    assert len(met) == 13 and met[None] > 300, met  # twelve pairs


CASES = [evictions]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c.__name__)
def test_outputs_over_inputs(case, stub):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, case.__name__], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-4000:]


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    base.STUB = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    globals()[sys.argv[2]]()
