"""What experts, weighing, eviction and penalties refuse, and what they launch at the ends of their ranges, without a GPU (as in test_lm_cpu.py and
test_lm_grids_cpu.py, in processes of their own over tests/hip_stub.c)."""
import ctypes as C
import os
import subprocess
import sys

import pytest

import test_lm_cpu as base
import test_lm_grids_cpu as grids
from test_lm_cpu import BF16, CACHES, F16, F32, P, ROOT, Refusals, Tensor, cache, changed
from test_lm_grids_cpu import stub  # noqa: F401


def layer(**kw):
    from nart_amd import hipq
    d, h = hipq.W4ExpertsDesc(experts=4, top=2, N=512, K=512, inner=256, group=128, type=BF16, activation=1, scores=0, normalize=1), C.c_void_p()
    changed(d, kw)
    a = dict(gate_up=P, gate_up_scales=P, gate_up_zeros=None, down=P, down_scales=P, down_zeros=None)
    a.update(kw)
    rc = hipq.lib().hipq_w4_experts_create(C.byref(d), a["gate_up"], a["gate_up_scales"], a["gate_up_zeros"], a["down"], a["down_scales"], a["down_zeros"], None, C.byref(h))
    return rc, h


def layers_of_experts():
    from nart_amd import hipq

    def call(**kw):
        rc, h = layer(**kw)
        if rc == 0:
            hipq.lib().hipq_w4_experts_destroy(h)
        return rc
    r = Refusals(call, 2)
    r.takes(2, experts=1, top=1, N=1, K=32, inner=32, group=32, type=F16, activation=2, scores=1, normalize=0, gate_up_zeros=P, down_zeros=P)
    r.takes(2, experts=1024, top=16, N=16, K=32, inner=32)
    for type in (F32, 3, -1):
        r.refuses("neither float16 nor bfloat16", type=type)
    for group in (0, 16, 256):
        r.refuses("groups of", group=group)
    for activation in (-1, 0, 3):
        r.refuses("activation", activation=activation)
    for scores in (-1, 2):
        r.refuses("scores", scores=scores)
    r.refuses("normalize", normalize=2)
    for experts in (0, -1, 1025):
        r.refuses("experts", experts=experts, top=1)
    for top in (0, -1, 5):
        r.refuses("experts of a token", top=top)
    r.refuses("experts of a token", top=17, experts=20)
    for N in (0, -1, (1 << 20) + 1):
        r.refuses("outputs", N=N)
    for K in (0, 16, 33, (1 << 20) + 32):
        r.refuses("inputs", K=K)
        r.refuses("hidden values", inner=K)
    for name in ("gate_up", "gate_up_scales", "down", "down_scales"):
        r.refuses("null pointer", **{name: None})
    for name in ("gate_up_zeros", "down_zeros"):
        r.refuses("zero points for one", **{name: P})


def runs_of_experts():
    from nart_amd import hipq
    lib = hipq.lib()
    rc, h = layer()
    assert rc == 0
    need = {M: lib.hipq_w4_experts_workspace(h, M) for M in (1, 8, 40, 200, 2000)}
    assert all(n > 0 for n in need.values()) and lib.hipq_w4_experts_workspace(h, 0) == 0 and lib.hipq_w4_experts_workspace(None, 1) == 0

    def call(plan=h, x=P, x_stride=512, logits=P << 10, logits_type=F32, logits_stride=4, y=P << 11, y_stride=512, M=8, workspace=P << 12, size=1 << 40):
        return lib.hipq_w4_experts_run(plan, x, x_stride, logits, logits_type, logits_stride, y, y_stride, M, workspace, size, None)
    r = Refusals(call, 3)
    r.takes(0, M=0, x=None, y=None, logits=None, workspace=None)
    r.takes(2, M=1, x_stride=0, y_stride=0, logits_stride=0)
    r.takes(3, x_stride=520, y_stride=513, y=(P << 11) + 2, logits_stride=5, size=need[8])
    r.takes(3, logits_type=BF16, logits=(P << 10) + 2)
    assert lib.hipq_w4_experts_kernel(h, 1) == b"w4_experts_stream_4" and lib.hipq_w4_experts_kernel(None, 1) == b""
    for M in (-1, (1 << 20) + 1):
        r.refuses("rows", M=M)
        assert lib.hipq_w4_experts_kernel(h, M) == b"" and lib.hipq_w4_experts_workspace(h, M) == 0
    r.refuses("null plan", plan=None)
    for name in ("x", "logits", "y"):
        r.refuses("null pointer", **{name: None})
    for changes in (dict(x=P + 8), dict(x_stride=516)):
        r.refuses("multiples of 16 bytes", **changes)
    for changes in (dict(y=(P << 11) + 1), dict(logits=(P << 10) + 2), dict(logits_type=F16, logits=(P << 10) + 1)):
        r.refuses("aligned", **changes)
    for logits_type in (-1, 3):
        r.refuses("logits of type", logits_type=logits_type)
    for changes in (dict(x_stride=504), dict(y_stride=511), dict(logits_stride=3), dict(x_stride=0)):
        r.refuses("overlap", **changes)
    r.refuses("elements apart", x_stride=1 << 29)
    r.refuses("y lies over x", y=P + 512)
    r.refuses("y lies over the logits", logits=(P << 11) + 100)
    for changes in (dict(workspace=None), dict(size=need[8] - 1), dict(workspace=(P << 12) + 8)):
        r.refuses("workspace of %d bytes" % need[8], **changes)
    C.c_int.in_dll(base.STUB, "stub_device").value = 1
    r.refuses("the plan is on device 0, the current one is 1")
    C.c_int.in_dll(base.STUB, "stub_device").value = 0
    lib.hipq_w4_experts_destroy(h)
    lib.hipq_w4_experts_destroy(None)
    rc, h = layer(inner=1 << 20, K=32, N=1)
    assert rc == 0 and lib.hipq_w4_experts_workspace(h, 1023) > 0 and lib.hipq_w4_experts_workspace(h, 1024) == 0
    assert b"hidden values each" in lib.hipq_last_error()


def weights_of_the_cache():
    from nart_amd import hipq
    lib = hipq.lib()

    def desc(kw):
        d = hipq.KvWeighDesc(q=P, q_token=1024, q_head=128, starts=P, lens=P, blocks=P, mask=None, weights=P, out=P, blocks_stride=10, sequences=2, tokens=6, q_heads=8,
                             blocks_per_sequence=10, most_new=3, longest=160, scale=0.1)
        return changed(d, kw)

    def call(workspace=P, size=1 << 40, **kw):
        address = kw.pop("c_k", None)
        c = cache(kw)
        c.k = address or c.k
        d = desc(kw)
        assert not kw, kw
        return lib.hipq_kv_weigh(C.byref(c), C.byref(d), workspace, size, None)
    r = Refusals(call, 2)
    for changes in (dict(sequences=0), dict(tokens=0), dict(most_new=0), dict(longest=0), dict(pages=0), dict(blocks_per_sequence=0, blocks=None)):
        r.takes(0, q=None, weights=None, **changes)
    for changes in (dict(mask=P), dict(quantized=1), dict(dim=256), dict(dim=64, type=F16), dict(longest=1 << 30), dict(sequences=1, blocks_stride=0), dict(out=P << 8),
                    dict(mask=P, most_new=64), dict(most_new=20, q_heads=4), dict(most_new=200, q_heads=4)):
        r.takes(3 if changes.get("most_new") == 200 else 2, **changes)
    for message, changes in CACHES:
        r.refuses(message, **changes)
    for name in ("q", "starts", "lens", "blocks", "weights", "out"):
        r.refuses("null pointer", **{name: None})
    r.refuses("weigh: 6 query heads", q_heads=6)
    r.refuses("64 new tokens", mask=P, most_new=65)
    for changes in (dict(most_new=-1), dict(most_new=(1 << 20) + 1)):
        r.refuses("new tokens of a sequence", **changes)
    r.refuses("longest", longest=-1)
    r.refuses("overlap", blocks_stride=9)
    for scale in (0.0, -0.1, float("nan"), float("inf")):
        r.refuses("scale", scale=scale)
    for changes in (dict(q=P + 8), dict(q_token=1020), dict(q_head=4), dict(weights=P + 8, out=P + 8)):
        r.refuses("16 bytes", **changes)
    for out in (P + 16, P - 16, P + 4 * 10 * 4 * 16 - 16):
        r.refuses("lies over", out=out)
    r.takes(2, out=P + 4 * 10 * 4 * 16)
    r.refuses("work-groups", sequences=1 << 20, heads=64, q_heads=4096, blocks_stride=1 << 20, most_new=64)
    kw = {}
    c, d = cache(kw), desc(kw)
    need = lib.hipq_kv_weigh_workspace(C.byref(c), C.byref(d))
    assert need > 0 and lib.hipq_kv_weigh_workspace(C.byref(c), None) == 0
    for changes in (dict(workspace=None), dict(size=need - 1), dict(workspace=P + 4)):
        r.refuses("workspace of %d bytes" % need, **changes)
    assert lib.hipq_kv_weigh(C.byref(c), None, None, 0, None) != 0


def evictions():
    from nart_amd import hipq
    lib = hipq.lib()

    def desc(kw):
        d = hipq.KvEvictDesc(weights=P, lens=P, blocks=P, to=2 * P, blocks_stride=10, to_stride=4, kept=P, left=P, sequences=2, blocks_per_sequence=10, to_per_sequence=4, longest=160,
                             budget=64, recent=8, first=4)
        return changed(d, kw)

    def call(workspace=None, size=0, **kw):
        address = kw.pop("c_k", None)
        c = cache(kw)
        c.k = address or c.k
        d = desc(kw)
        assert not kw, kw
        return lib.hipq_kv_evict(C.byref(c), C.byref(d), workspace, size, None)
    r = Refusals(call, 2)
    r.takes(0, sequences=0, weights=None, lens=None)
    for changes in (dict(to=P, to_stride=10), dict(to=P, to_stride=10, to_per_sequence=10), dict(quantized=1), dict(dim=64, quantized=1), dict(dim=256), dict(pages=0), dict(budget=1, recent=0, first=1),
                    dict(budget=1 << 30, to_per_sequence=10, to_stride=10), dict(longest=0, weights=None, blocks=None, to=None), dict(recent=64, first=0), dict(longest=10, to_per_sequence=1),
                    dict(sequences=1, blocks_stride=0, to_stride=0), dict(sequences=1, to=P, blocks_stride=0, to_stride=4)):
        r.takes(2, **changes)
    for message, changes in CACHES:
        r.refuses(message, **changes)
    for name in ("weights", "lens", "blocks", "to", "kept", "left"):
        r.refuses("null pointer", **{name: None})
    for budget in (0, -1, (1 << 30) + 1):
        r.refuses("budget", budget=budget)
    for changes in (dict(recent=-1), dict(first=-1), dict(recent=61), dict(first=57), dict(recent=2 ** 31 - 1, first=2 ** 31 - 1)):
        r.refuses("first and", **changes)
    r.refuses("longest", longest=-1)
    r.refuses("sequences", sequences=-1)
    for changes in (dict(blocks_stride=9), dict(to_stride=3)):
        r.refuses("overlap", **changes)
    r.refuses("in place", to=P, to_stride=4)
    r.refuses("blocks for 64 tokens", to_per_sequence=3)
    r.refuses("16 bytes", weights=P + 4)
    r.refuses("sequences of", sequences=1 << 20, heads=4, blocks_stride=10)
    long = dict(blocks_per_sequence=2000, blocks_stride=2000, longest=30000)
    kw = dict(long)
    c, d = cache(kw), desc(kw)
    need = lib.hipq_kv_evict_workspace(C.byref(c), C.byref(d))
    assert need > 0
    r.takes(5, workspace=P, size=need, **long)
    for changes in (dict(), dict(workspace=P, size=need - 1), dict(workspace=P + 4, size=need + 4), dict(size=need)):
        r.refuses("workspace of %d bytes" % need, **long, **changes)


def penalties():
    from nart_amd import hipq

    def call(**kw):
        d = hipq.PenalizeDesc(logits=P, out=P << 8, stride=1000, out_stride=1000, tokens=P, lens=P, prompt_lens=P, repetition=P, frequency=P, presence=P, bias_tokens=P, bias=P, allowed=P,
                              tokens_stride=20, bias_stride=5, allowed_stride=32, type=F32, rows=3, vocab=1000, longest=20, biases=5)
        changed(d, kw)
        assert not kw, kw
        return hipq.lib().hipq_penalize(C.byref(d), None)
    r = Refusals(call, 1)
    for changes in (dict(rows=0), dict(vocab=0)):
        r.takes(0, logits=None, out=None, **changes)
    for changes in (dict(out=P), dict(rows=1, stride=0, out_stride=0, tokens_stride=0, bias_stride=0, allowed_stride=0), dict(tokens=None, longest=0), dict(bias=None, bias_tokens=None, biases=0),
                    dict(lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None, allowed=None), dict(type=BF16, logits=P + 2), dict(type=F16, out_stride=1001),
                    dict(vocab=1 << 20, stride=1 << 20, out_stride=1 << 20, out=P << 12, allowed_stride=1 << 15)):
        r.takes(1, **changes)
    for type in (-1, 3):
        r.refuses("type", type=type)
    for rows in (-1, (1 << 24) + 1):
        r.refuses("rows", rows=rows)
    for vocab in (-1, (1 << 20) + 1):
        r.refuses("scores of a row", vocab=vocab)
    for longest in (-1, 1 << 30):
        r.refuses("histories", longest=longest)
    for biases in (-1, 1 << 30):
        r.refuses("biases", biases=biases)
    for name in ("logits", "out"):
        r.refuses("null pointer", **{name: None})
    for changes in (dict(logits=P + 2), dict(out=(P << 8) + 1, type=F16)):
        r.refuses("aligned", **changes)
    for changes in (dict(stride=999), dict(out_stride=999), dict(tokens_stride=19), dict(bias_stride=4), dict(allowed_stride=31)):
        r.refuses("overlap", **changes)
    r.refuses("no tokens", tokens=None)
    for name in ("bias", "bias_tokens"):
        r.refuses("belong together", **{name: None})
    for changes in (dict(out=P + 4), dict(out=P, out_stride=1004), dict(out=P + 4000 * 2 + 3996)):
        r.refuses("lies over", **changes)


def calls_with_tensors():
    import importlib.util
    import sysconfig
    from nart_amd import hipq
    lib = hipq.lib()
    path = os.path.join(os.path.dirname(hipq.LIB_PATH), "hipq_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
    spec = importlib.util.spec_from_file_location("hipq_calls", path)
    calls = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(calls)
    calls.init(lambda: 0, lambda device: 0)
    f32, f16, bf16, i32, i64, u8, i8 = names = ["float32", "float16", "bfloat16", "int32", "int64", "uint8", "int8"]
    calls.types(*names)
    kernels = C.c_long.in_dll(base.STUB, "stub_kernels")

    def trial(launches, call, **valid):
        def run(launches, **changes):
            before = kernels.value
            assert call(**dict(valid, **changes)) == 0, lib.hipq_last_error()
            assert kernels.value - before == launches, (changes, kernels.value - before)

        def refuse(message, **changes):
            before = kernels.value
            try:
                rc = call(**dict(valid, **changes))
            except ValueError as e:
                assert message in str(e), (changes, e)
            else:
                assert rc and message in lib.hipq_last_error().decode(), (changes, rc, lib.hipq_last_error())
            assert kernels.value == before, changes
        run(launches)
        return run, refuse

    # experts
    rc, h = layer(N=640)
    assert calls.experts_workspace(h.value, 4) > 0
    work = lambda: Tensor(u8, 1 << 20)  # noqa: E731
    run, refuse = trial(2, lambda x, logits, y, w: calls.experts_run(h.value, BF16, 640, 512, 4, x, logits, y, w), x=Tensor(bf16, 4, 512), logits=Tensor(f32, 4, 4), y=Tensor(bf16, 4, 640, stride=(700, 1)), w=work())
    run(0, x=Tensor(bf16, 0, 512), y=Tensor(bf16, 0, 640), logits=Tensor(f32, 0, 4), w=None)
    run(2, logits=Tensor(bf16, 4, 4, stride=(9, 1)))
    refuse("x: bfloat16 is expected", x=Tensor(f16, 4, 512))
    refuse("logits: float32 or float16 or bfloat16", logits=Tensor(i32, 4, 4))
    refuse("logits: 4 entries", logits=Tensor(f32, 3, 4))
    refuse("logits: 4 entries", logits=Tensor(f32, 4, 5))
    refuse("y: 640 entries", y=Tensor(bf16, 4, 512))
    refuse("logits is on device 1", logits=Tensor(f32, 4, 4, device=1))
    refuse("workspace", w=Tensor(u8, 16))
    lib.hipq_w4_experts_destroy(h)

    # the cache
    quant, scales, k = Tensor(i8, 9, 4, 16, 128), Tensor(f32, 9, 4, 16), Tensor(bf16, 9, 4, 16, 128)
    c, c8 = calls.kv_cache(k, k, None, None), calls.kv_cache(quant, quant, scales, scales)
    asked = []

    def allocate(count):
        asked.append(count)
        return Tensor(u8, count)
    q = Tensor(bf16, 5, 8, 128)
    run, refuse = trial(2, lambda cache, device, q, weights, out, starts, lens, blocks, mask, most_new, longest, scale: calls.kv_weigh(
        cache, device, q, weights, out, starts, lens, blocks, mask, most_new, longest, scale, allocate), cache=c, device=0, q=q, weights=scales, out=scales, starts=Tensor(i32, 3),
        lens=Tensor(i32, 2), blocks=Tensor(i32, 2, 6), mask=None, most_new=3, longest=None, scale=0.1)
    assert len(asked) == 1 and asked[0] > 0
    run(2, cache=c8, mask=Tensor(i64, 5), q=Tensor(f16, 5, 8, 128))
    run(2, longest=1 << 40)
    run(0, most_new=0)
    refuse("the cache is on device 2", device=2)
    refuse("q: bfloat16 is expected, which the cache has", q=Tensor(f16, 5, 8, 128))
    refuse("weights: float32", weights=Tensor(bf16, 9, 4, 16))
    refuse("weights: 9 entries", weights=Tensor(f32, 8, 4, 16))
    refuse("out: 16 entries", out=Tensor(f32, 9, 4, 8))
    refuse("out has gaps", out=Tensor(f32, 9, 4, 16, stride=(128, 32, 1)))
    refuse("starts: 3 entries", starts=Tensor(i32, 2))
    refuse("blocks: rows overlap", blocks=Tensor(i32, 2, 6, stride=(0, 1)))
    refuse("mask: 5 entries", mask=Tensor(i64, 2))
    refuse("longest", longest=-5)
    refuse("too many", blocks=Tensor(i32, 2, 1 << 28, stride=(1 << 28, 1)))
    for most_new in (-1, -(1 << 40), 1 << 40):
        refuse("new tokens of a sequence", most_new=most_new)

    del asked[:]
    run, refuse = trial(2, lambda cache, device, weights, lens, blocks, to, left, kept, budget, recent, first, longest: calls.kv_evict(
        cache, device, weights, lens, blocks, to, left, kept, budget, recent, first, longest, allocate), cache=c, device=0, weights=scales, lens=Tensor(i32, 2), blocks=Tensor(i32, 2, 6),
        to=Tensor(i32, 2, 3), left=Tensor(i32, 2), kept=Tensor(i32, 2, 4, 40), budget=40, recent=5, first=0, longest=None)
    run(2, cache=c8, to=Tensor(i32, 2, 6))
    assert not asked
    run(5, blocks=Tensor(i32, 2, 2000))
    assert len(asked) == 1 and asked[0] > 0
    refuse("the cache is on device 2", device=2)
    refuse("weights: 4 entries", weights=Tensor(f32, 9, 5, 16))
    refuse("lens: int32", lens=Tensor(i64, 2))
    refuse("left: 2 entries", left=Tensor(i32, 3))
    refuse("kept: 40 entries", kept=Tensor(i32, 2, 4, 39))
    refuse("kept: 4 entries", kept=Tensor(i32, 2, 3, 40))
    refuse("to: 2 entries", to=Tensor(i32, 1, 3))
    refuse("blocks for 40 tokens", to=Tensor(i32, 2, 2))
    refuse("blocks: rows overlap", to=Tensor(i32, 2, 3, stride=(0, 1)))
    refuse("budget", budget=0, kept=Tensor(i32, 2, 4, 0))
    refuse("first and", recent=41)
    refuse("longest", longest=-1)

    # penalties
    run, refuse = trial(1, lambda x, out, tokens, lens, prompt, rep, freq, pres, at, bias, allowed: calls.penalize(x, out, tokens, lens, prompt, rep, freq, pres, at, bias, allowed),
                        x=Tensor(f32, 3, 50), out=Tensor(f32, 3, 50), tokens=Tensor(i32, 3, 7), lens=Tensor(i32, 3), prompt=Tensor(i32, 3), rep=Tensor(f32, 3), freq=Tensor(f32, 3),
                        pres=Tensor(f32, 3), at=Tensor(i32, 3, 4), bias=Tensor(f32, 3, 4), allowed=Tensor(i32, 3, 2))
    nothing = dict(tokens=None, lens=None, prompt=None, rep=None, freq=None, pres=None, at=None, bias=None, allowed=None)
    run(1, **nothing)
    run(1, tokens=Tensor(i32, 3, 7, stride=(70, 1)), allowed=Tensor(i32, 3, 2, stride=(5, 1)))
    run(1, tokens=Tensor(i32, 3, 0), at=Tensor(i32, 3, 0), bias=Tensor(f32, 3, 0))
    run(0, x=Tensor(f32, 3, 0), out=Tensor(f32, 3, 0), allowed=None)
    refuse("logits: float32 or float16 or bfloat16", x=Tensor(i32, 3, 50))
    refuse("out: float32", out=Tensor(bf16, 3, 50))
    refuse("out: 50 entries", out=Tensor(f32, 3, 51))
    refuse("tokens: int32", tokens=Tensor(i64, 3, 7))
    refuse("tokens: 3 entries", tokens=Tensor(i32, 2, 7))
    refuse("tokens: a tensor is expected", tokens=None)
    refuse("tokens: a tensor is expected", **dict(nothing, rep=Tensor(f32, 3)))
    refuse("lens: 3 entries", lens=Tensor(i32, 4))
    refuse("repetition: float32", rep=Tensor(bf16, 3))
    refuse("presence: 3 entries", pres=Tensor(f32, 1))
    refuse("bias: 4 entries", bias=Tensor(f32, 3, 5))
    refuse("belong together", bias=None)
    refuse("as far apart", bias=Tensor(f32, 3, 4, stride=(9, 1)))
    refuse("allowed: 2 entries", allowed=Tensor(i32, 3, 1))
    refuse("allowed is not on the GPU", allowed=Tensor(i32, 3, 2, device=-1))
    refuse("overlap", x=Tensor(f32, 3, 50, stride=(0, 1)), out=Tensor(f32, 3, 50, stride=(60, 1)))


def launches_at_the_ends():
    """A launch has under 2^32 work-items side by side, and under 2^16 such rows."""
    from nart_amd import hipq
    lib, launched = hipq.lib(), grids.launched
    for d in (dict(N=1 << 20, K=32, inner=32), dict(N=16, K=4096, inner=1024), dict(N=16, K=32, inner=32, experts=1024, top=16)):
        rc, h = layer(**d)
        launched(rc)
        for M in (1, 64, 128, 129, 4096, 1 << 17, 1 << 20):
            need = lib.hipq_w4_experts_workspace(h, M)
            if need:
                launched(lib.hipq_w4_experts_run(h, P, d["K"], P << 30, F32, 1024, 1 << 56, 1 << 20, M, P << 20, 1 << 60, None))
            else:
                grids.refused(lib.hipq_w4_experts_run(h, P, d["K"], P << 30, F32, 1024, 1 << 56, 1 << 20, M, P << 20, 1 << 60, None), b"rows")
        lib.hipq_w4_experts_destroy(h)

    def penalize(rows, vocab, type=F16):
        d = hipq.PenalizeDesc(logits=P, out=1 << 60, stride=vocab, out_stride=vocab, type=type, rows=rows, vocab=vocab)
        return lib.hipq_penalize(C.byref(d), None)
    for rows, vocab in ((1, 1), (1 << 24, 1 << 20), (1 << 24, 7), (1 << 20, 8193), (255, 16384), (1, 1 << 20)):
        total = sum(x * y for x, y in launched(penalize(rows, vocab)))
        assert total * 16 >= rows * vocab

    def weigh(sequences, heads, most_new=1, dim=64, blocks=1, longest=16):
        c = cache(dict(heads=heads, dim=dim))
        d = hipq.KvWeighDesc(q=P, q_token=heads * dim, q_head=dim, starts=P, lens=P, blocks=P, weights=P, out=P, blocks_stride=blocks, sequences=sequences, tokens=sequences, q_heads=heads,
                             blocks_per_sequence=blocks, most_new=most_new, longest=longest, scale=0.1)
        return lib.hipq_kv_weigh(C.byref(c), C.byref(d), P, 1 << 60, None)
    for sequences, heads, more in ((1 << 20, 15, {}), (1 << 12, 4095, {}), (300, 64, dict(dim=128, most_new=4096, longest=1 << 14, blocks=1 << 10)), (1, 1, dict(longest=1 << 30, blocks=1 << 26))):
        launched(weigh(sequences, heads, **more))
    for sequences, heads, more in ((1 << 20, 16, {}), (1 << 12, 4096, {}), (1 << 10, 512, dict(most_new=1 << 10))):
        grids.refused(weigh(sequences, heads, **more), b"work-groups")

    def evict(sequences, heads, blocks=1, budget=16, dim=64):
        c = cache(dict(heads=heads, dim=dim))
        d = hipq.KvEvictDesc(weights=P, lens=P, blocks=P, to=2 * P, blocks_stride=blocks, to_stride=blocks, kept=P, left=P, sequences=sequences, blocks_per_sequence=blocks, to_per_sequence=blocks,
                             longest=1 << 30, budget=budget)
        return lib.hipq_kv_evict(C.byref(c), C.byref(d), P, 1 << 60, None)
    for args in ((1 << 20, 3), (1, 1, 1 << 26), (1, 4, 1 << 26, 1 << 29), (1 << 18, 7, 1, 16, 256)):
        launched(evict(*args))
    for args in ((1 << 20, 4), (1 << 12, 4096), (1 << 10, 64, 1 << 15), (1 << 19, 4, 1, 16, 256)):
        grids.refused(evict(*args), b"sequences of")


CASES = [layers_of_experts, runs_of_experts, weights_of_the_cache, evictions, penalties, calls_with_tensors, launches_at_the_ends]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c.__name__)
def test_refusals(case, stub):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, case.__name__], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-4000:]


@pytest.mark.parametrize("changes, message", [
    (dict(activation=None), "activation"), (dict(scores="max"), "scores"), (dict(gate_up=(2, 128)), "gate_up: uint8 with three dimensions"), (dict(down=(2, 8, 20)), "down:"), (dict(down=(3, 8, 32)), "down:"),
    (dict(gate_up_scales=(2, 128, 2)), "gate_up_scales: torch.bfloat16 of shape"), (dict(down_scales=(2, 8, 1)), "down_scales"), (dict(group=48), "group"), (dict(top=3), "top"), (dict(top=0), "top"),
    (dict(gate_up_zeros=(2, 128, 1)), "zeros: for both"), (dict(gate_up_zeros=(2, 128, 2), down_zeros=(2, 8, 2)), "gate_up_zeros")])
def test_constructor_refuses(changes, message):
    torch = pytest.importorskip("torch")
    from nart_amd import hipq
    shapes = dict(gate_up=(2, 128, 16), gate_up_scales=(2, 128, 1), gate_up_zeros=None, down=(2, 8, 32), down_scales=(2, 8, 2), down_zeros=None)
    shapes.update({n: v for n, v in changes.items() if n in shapes})
    t = {n: None if s is None else torch.zeros(s, dtype=torch.bfloat16 if "scales" in n else torch.uint8) for n, s in shapes.items()}
    with pytest.raises(ValueError, match=message):
        hipq.ExpertsW4(t["gate_up"], t["gate_up_scales"], t["down"], t["down_scales"], changes.get("top", 2), changes.get("group", 32), gate_up_zeros=t["gate_up_zeros"], down_zeros=t["down_zeros"],
                       **{n: v for n, v in changes.items() if n in ("activation", "scores")})


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    base.STUB = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    from nart_amd import hipq
    base.hipq = grids.base.hipq = hipq
    globals()[sys.argv[2]]()
