"""What the operators of language models refuse, without a GPU: the C entries and the calls with tensors, each in a process of its own in
which tests/hip_stub.c stands in for the HIP runtime.  A call that is taken launches its kernels, one that is refused none."""
import ctypes as C
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = 0, 1, 2
P = 1 << 20  # an address, never touched


class Refusals:
    """call(**changes): the entry with valid arguments but for the changes."""

    def __init__(self, call, launches):
        from nart_amd import hipq
        self.call, self.kernels, self.error = call, C.c_long.in_dll(STUB, "stub_kernels"), lambda: hipq.lib().hipq_last_error().decode()
        self.takes(launches)

    def takes(self, launches, **changes):
        before = self.kernels.value
        assert self.call(**changes) == 0, (changes, self.error())
        assert self.kernels.value - before == launches, (changes, self.kernels.value - before)

    def refuses(self, message, **changes):
        before = self.kernels.value
        assert self.call(**changes) != 0, changes
        assert message in self.error(), (changes, self.error())
        assert self.kernels.value == before, changes


def plan(N=512, K=512, group=128, type=BF16, activation=0, **kw):
    from nart_amd import hipq
    d, h = hipq.W4Desc(N=N, K=K, group=group, type=type, activation=activation), C.c_void_p()
    a = dict(q=P, scales=P, zeros=None, bias=None)
    a.update(kw)
    rc = hipq.lib().hipq_w4_plan_create(C.byref(d), a["q"], a["scales"], a["zeros"], a["bias"], None, C.byref(h))
    return rc, h


def plans_of_4_bit_weights():
    from nart_amd import hipq

    def call(**kw):
        rc, h = plan(**kw)
        if rc == 0:
            hipq.lib().hipq_w4_plan_destroy(h)
        return rc
    r = Refusals(call, 1)
    for group in (32, 64, 128):
        r.takes(1, group=group, K=32, N=1, zeros=P, bias=P, type=F16, activation=2)
    for type in (F32, 3, -1):
        r.refuses("neither float16 nor bfloat16", type=type)
    for group in (0, 16, 96, 256, -32):
        r.refuses("groups of", group=group)
    for activation in (-1, 3):
        r.refuses("activation", activation=activation)
    for N in (0, -1, (1 << 26) + 1):
        r.refuses("outputs", N=N)
    for K in (0, 16, 33, 48, -32, (1 << 24) + 32):
        r.refuses("inputs", K=K)
    for name in ("q", "scales"):
        r.refuses("null pointer", **{name: None})


def runs_of_4_bit_weights():
    from nart_amd import hipq
    lib = hipq.lib()
    rc, h = plan(K=2048)
    assert rc == 0

    def call(plan=h, x=P, x_stride=2048, y=4 * P, y_stride=512, M=8, workspace=None, size=0):
        return lib.hipq_w4_run(plan, x, x_stride, y, y_stride, M, workspace, size, None)
    need = lib.hipq_w4_workspace(h, 8)
    assert need == 0
    r = Refusals(call, 1)
    r.takes(0, M=0, x=None, y=None)
    r.takes(1, M=1, x_stride=0, y_stride=0)
    r.takes(1, x_stride=2056, y_stride=513, y=4 * P + 2)
    for M in (-1, (1 << 24) + 1):
        r.refuses("rows", M=M)
        assert lib.hipq_w4_plan_kernel(h, M) == b"" and lib.hipq_w4_workspace(h, M) == 0
    assert lib.hipq_w4_plan_kernel(None, 1) == b"" and lib.hipq_w4_workspace(None, 1) == 0 and lib.hipq_w4_plan_kernel(h, 0) != b""
    r.refuses("null plan", plan=None)
    for name in ("x", "y"):
        r.refuses("null pointer", **{name: None})
    for changes in (dict(x=P + 8), dict(x_stride=2052)):
        r.refuses("multiples of 16 bytes", **changes)
    r.refuses("aligned", y=4 * P + 1)
    r.refuses("over x", y=P)
    for changes in (dict(x_stride=2040), dict(y_stride=511), dict(x_stride=-2048), dict(y_stride=0)):
        r.refuses("overlap", **changes)
    r.refuses("elements apart", x_stride=1 << 23)
    need = lib.hipq_w4_workspace(h, 200)
    assert need > 0
    r.takes(2, M=200, workspace=P, size=need)
    for changes in (dict(), dict(workspace=P, size=need - 1), dict(workspace=P + 8, size=need + 8), dict(size=need)):
        r.refuses("workspace of %d bytes" % need, M=200, **changes)
    C.c_int.in_dll(STUB, "stub_device").value = 1
    r.refuses("the plan is on device 0, the current one is 1")
    C.c_int.in_dll(STUB, "stub_device").value = 0
    lib.hipq_w4_plan_destroy(h)
    lib.hipq_w4_plan_destroy(None)


def changed(struct, kw, but=()):
    for n, v in list(kw.items()):
        if n in dict(struct._fields_) and n not in but:
            setattr(struct, n, kw.pop(n))
    return struct


def cache(kw):
    from nart_amd import hipq
    c = changed(hipq.KvCacheStruct(k=P, v=P, k_scale=P, v_scale=P, pages=10, heads=4, page=16, dim=128, type=BF16, quantized=0), kw, ("k", "v"))
    if kw.pop("no_scales", False):
        c.k_scale = c.v_scale = None
    return c


CACHES = [("neither float16 nor bfloat16", dict(type=F32)), ("quantized", dict(quantized=2)), ("heads of", dict(dim=96)), ("heads of", dict(dim=512)),
          ("pages of", dict(page=8)), ("pages of", dict(page=24)), ("pages of", dict(page=0)), ("pages of", dict(page=1 << 17)), ("heads", dict(heads=0)),
          ("pages", dict(pages=-1)), ("pages", dict(pages=1 << 27)), ("null pointer", dict(quantized=1, no_scales=True)), ("16 bytes", dict(c_k=P + 8))]


def new_tokens_of_the_cache():
    from nart_amd import hipq

    def call(**kw):
        address = kw.pop("c_k", None)
        c = cache(kw)
        c.k = address or c.k
        d = hipq.KvAppendDesc(q=P, k=P, v=P, q_token=1024, q_head=128, k_token=512, k_head=128, v_token=512, v_head=128, out_token=1024, out_head=128, q_out=P,
                              positions=P, slots=P, table=P, tokens=5, q_heads=8, table_rows=100, rot=128, interleaved=0, eps=1e-6)
        changed(d, kw)
        assert not kw, kw
        return hipq.lib().hipq_kv_append(C.byref(c), C.byref(d), None)
    r = Refusals(call, 1)
    for changes in (dict(tokens=0, q=None, k=None, v=None), dict(pages=0)):
        r.takes(0, **changes)
    for changes in (dict(q_heads=0, q=None, q_out=None), dict(rot=0, table=None), dict(rot=16, interleaved=1), dict(quantized=1), dict(q_norm=P, k_norm=P, eps=0.0)):
        r.takes(1, **changes)
    for message, changes in CACHES:
        r.refuses(message, **changes)
    for rot in (8, 24, 144, -16):
        r.refuses("rotated elements", rot=rot)
    for changes in (dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(positions=None), dict(slots=None)):
        r.refuses("null pointer", **changes)
    r.refuses("no table", table=None)
    r.refuses("interleaved", interleaved=2)
    for eps in (-1e-6, float("nan")):
        r.refuses("eps", eps=eps)
    for tokens in (-1, (1 << 24) + 1):
        r.refuses("tokens", tokens=tokens)
    r.refuses("query heads", q_heads=-1)
    for name in ("q", "v", "q_out", "table", "k_norm"):
        r.refuses("16 bytes", **{name: P + 8})
    for name in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "out_token", "out_head"):
        r.refuses("multiples of 8", **{name: 1028})
    r.refuses("tokens of", tokens=1 << 24, q_heads=65536, dim=256)  # more work-groups than a grid has


def attention_over_the_cache():
    from nart_amd import hipq
    lib = hipq.lib()

    def desc(kw):
        d = hipq.KvAttendDesc(q=P, o=P, q_token=1024, q_head=128, o_token=1024, o_head=128, starts=P, lens=P, blocks=P, mask=None, blocks_stride=10,
                              sequences=2, tokens=6, q_heads=8, blocks_per_sequence=10, most_new=3, longest=160, scale=0.1)
        return changed(d, kw)

    def call(workspace=None, size=0, **kw):
        address = kw.pop("c_k", None)
        c = cache(kw)
        c.k = address or c.k
        d = desc(kw)
        assert not kw, kw
        return lib.hipq_kv_attend(C.byref(c), C.byref(d), workspace, size, None)
    r = Refusals(call, 1)
    for changes in (dict(sequences=0), dict(tokens=0), dict(most_new=0)):
        r.takes(0, q=None, o=None, **changes)
    for changes in (dict(mask=P), dict(mask=P, most_new=64), dict(blocks=None, blocks_per_sequence=0, longest=0), dict(pages=0), dict(quantized=1), dict(dim=256),
                    dict(dim=64, type=F16), dict(longest=0), dict(longest=1 << 30), dict(sequences=1, blocks_stride=0)):
        r.takes(1, **changes)
    for message, changes in CACHES:
        r.refuses(message, **changes)
    for changes in (dict(q=None), dict(o=None), dict(starts=None), dict(lens=None), dict(blocks=None)):
        r.refuses("null pointer", **changes)
    for q_heads in (0, 6, -4):
        r.refuses("query heads", q_heads=q_heads)
    r.refuses("64 new tokens", mask=P, most_new=65)
    for most_new in (-1, (1 << 20) + 1):
        r.refuses("new tokens of a sequence", most_new=most_new)
    r.refuses("rows of a sequence", most_new=1 << 20, q_heads=128)
    r.refuses("sequences", sequences=-1)
    r.refuses("new tokens", tokens=-1)
    r.refuses("longest", longest=-1)
    r.takes(1, blocks_per_sequence=1 << 26, blocks_stride=1 << 26)
    for n in (-1, (1 << 26) + 1, 1 << 27):
        r.refuses("blocks of a sequence", blocks_per_sequence=n)
    r.refuses("overlap", blocks_stride=9)
    for scale in (0.0, -0.1, float("nan"), float("inf")):
        r.refuses("scale", scale=scale)
    for changes in (dict(q=P + 8), dict(o=P + 8), dict(q_token=1020), dict(q_head=4), dict(o_token=1028), dict(o_head=132)):
        r.refuses("16 bytes", **changes)
    r.refuses("work-groups", sequences=1 << 20, heads=64, q_heads=4096, blocks_stride=1 << 20, most_new=64)
    long = dict(blocks_per_sequence=500, blocks_stride=500, longest=8000)
    kw = dict(long)
    c, d = cache(kw), desc(kw)
    need = lib.hipq_kv_attend_workspace(C.byref(c), C.byref(d))
    assert need > 0
    r.takes(2, workspace=P, size=need, **long)
    for changes in (dict(), dict(workspace=P, size=need - 1), dict(workspace=P + 4, size=need + 4), dict(size=need)):
        r.refuses("workspace of %d bytes" % need, **long, **changes)


def samples():
    from nart_amd import hipq

    def call(logits=P, type=F32, rows=3, vocab=1000, stride=1000, uniform=P, tokens=P):
        return hipq.lib().hipq_sample(logits, type, rows, vocab, stride, uniform, None, None, None, None, tokens, None)
    r = Refusals(call, 1)
    r.takes(0, rows=0, logits=None)
    for changes in (dict(rows=1, stride=0), dict(vocab=1), dict(vocab=1 << 20, stride=1 << 20), dict(type=BF16, logits=P + 2), dict(type=F16, stride=1001), dict(logits=P + 4)):
        r.takes(1, **changes)
    for type in (-1, 3):
        r.refuses("type", type=type)
    for rows in (-1, (1 << 24) + 1):
        r.refuses("rows", rows=rows)
    for vocab in (0, -1, (1 << 20) + 1):
        r.refuses("scores", vocab=vocab)
    for name in ("logits", "uniform", "tokens"):
        r.refuses("null pointer", **{name: None})
    for changes in (dict(logits=P + 2), dict(type=F16, logits=P + 1)):
        r.refuses("aligned", **changes)
    r.refuses("overlap", stride=999)


class Tensor:
    """What the extension asks a tensor for."""

    def __init__(self, dtype, *shape, stride=None, device=0):
        self.dtype, self.shape, self.device = dtype, shape, device
        self.strides, n = [], 1
        for s in reversed(shape):
            self.strides.insert(0, n)
            n *= s
        self.strides = tuple(self.strides if stride is None else stride)

    def stride(self):
        return self.strides

    def get_device(self):
        return self.device

    def data_ptr(self):
        return P * (1 + len(self.dtype)) * (1 + self.shape[-1])


def calls_with_tensors():
    """The checks of dtypes, shapes, strides and devices in front of the C entries."""
    import importlib.util
    import sysconfig
    from nart_amd import hipq
    hipq.lib()
    path = os.path.join(os.path.dirname(hipq.LIB_PATH), "hipq_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
    spec = importlib.util.spec_from_file_location("hipq_calls", path)
    calls = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(calls)
    calls.init(lambda: 0, lambda device: 0)
    f32, f16, bf16, i32, i64, u8, i8 = names = ["float32", "float16", "bfloat16", "int32", "int64", "uint8", "int8"]
    calls.types(*names)
    kernels = C.c_long.in_dll(STUB, "stub_kernels")

    def trial(call, **valid):
        def run(launches, **changes):
            before = kernels.value
            assert call(**dict(valid, **changes)) == 0, hipq.lib().hipq_last_error()
            assert kernels.value - before == launches, changes

        def refuse(message, **changes):
            before = kernels.value
            try:
                rc = call(**dict(valid, **changes))
            except ValueError as e:
                assert message in str(e), (changes, e)
            else:
                assert rc and message in hipq.lib().hipq_last_error().decode(), (changes, rc)
            assert kernels.value == before, changes
        run(1)
        return run, refuse

    # products
    rc, h = plan(N=512, K=256)
    run, refuse = trial(lambda x, y, w: calls.w4_run(h.value, BF16, 512, 256, x, y, w), x=Tensor(bf16, 4, 256), y=Tensor(bf16, 4, 512), w=None)
    run(0, x=Tensor(bf16, 0, 256), y=Tensor(bf16, 0, 512))
    run(1, x=Tensor(bf16, 4, 256, stride=(264, 1)), y=Tensor(bf16, 4, 512, stride=(600, 1)))
    run(1, x=Tensor(bf16, 1, 256, stride=(3, 1)), y=Tensor(bf16, 1, 512))
    refuse("x: bfloat16 is expected", x=Tensor(f16, 4, 256))
    refuse("y: bfloat16 is expected", y=Tensor(f32, 4, 512))
    refuse("x: 256 entries", x=Tensor(bf16, 4, 128))
    refuse("y: 4 entries", y=Tensor(bf16, 3, 512))
    refuse("x: 2 dimensions", x=Tensor(bf16, 1, 4, 256))
    refuse("x: the last dimension has gaps", x=Tensor(bf16, 4, 256, stride=(1, 4)))
    refuse("x is not on the GPU", x=Tensor(bf16, 4, 256, device=-1))
    refuse("y is on device 1", y=Tensor(bf16, 4, 512, device=1))
    refuse("overlap", x=Tensor(bf16, 4, 256, stride=(0, 1)))
    refuse("too large", x=Tensor(bf16, 1 << 31, 256, stride=(0, 1)))
    hipq.lib().hipq_w4_plan_destroy(h)

    # the cache
    k, scales = Tensor(bf16, 9, 4, 16, 128), Tensor(f32, 9, 4, 16)
    quant = Tensor(i8, 9, 4, 16, 128)
    c, c8 = calls.kv_cache(k, k, None, None), calls.kv_cache(quant, quant, scales, scales)
    for message, a in (("k: float16 or bfloat16 or int8", (Tensor(f32, 9, 4, 16, 128), k, None, None)), ("v: bfloat16", (k, quant, None, None)),
                       ("v: 4 entries", (k, Tensor(bf16, 9, 2, 16, 128), None, None)), ("as wide", (k, Tensor(bf16, 9, 4, 16, 64), None, None)),
                       ("k has gaps", (Tensor(bf16, 9, 4, 16, 128, stride=(16384, 4096, 128, 1)), k, None, None)), ("4 dimensions", (Tensor(bf16, 9, 16, 128), k, None, None)),
                       ("scales belong", (k, k, scales, scales)), ("k_scale: 16 entries", (quant, quant, Tensor(f32, 9, 4, 8), scales)),
                       ("v_scale: float32", (quant, quant, scales, Tensor(bf16, 9, 4, 16))), ("not on the GPU", (k, Tensor(bf16, 9, 4, 16, 128, device=-1), None, None))):
        with pytest.raises(ValueError, match=message):
            calls.kv_cache(*a)
    with pytest.raises(ValueError, match="k_scale"):
        calls.kv_cache(quant, quant, None, None)

    # new tokens
    q, kv, index, table = Tensor(bf16, 5, 8, 128), Tensor(bf16, 5, 4, 128), Tensor(i32, 5), Tensor(f32, 100, 128)
    run, refuse = trial(lambda cache, device, q, k, v, positions, slots, table, out, q_norm, k_norm, eps, interleaved: calls.kv_append(
        cache, device, q, k, v, positions, slots, table, out, q_norm, k_norm, eps, interleaved), cache=c, device=0, q=q, k=kv, v=kv, positions=index, slots=index,
        table=table, out=q, q_norm=None, k_norm=None, eps=1e-6, interleaved=0)
    run(1, cache=c8)
    run(1, cache=c8, **{n: Tensor(f16, 5, h, 128) for n, h in (("q", 8), ("k", 4), ("v", 4), ("out", 8))})
    run(1, table=None, q_norm=Tensor(bf16, 128))
    run(1, q=Tensor(bf16, 5, 8, 128, stride=(2048, 128, 1)), k=Tensor(bf16, 5, 4, 128, stride=(0, 128, 1)))
    run(0, **{n: Tensor(bf16, 0, h, 128) for n, h in (("q", 8), ("k", 4), ("v", 4), ("out", 8))}, positions=Tensor(i32, 0), slots=Tensor(i32, 0))
    refuse("the cache is on device 1", device=1)
    refuse("q: bfloat16 is expected, which the cache has", q=Tensor(f16, 5, 8, 128))
    refuse("k: 4 entries", k=Tensor(bf16, 5, 8, 128))
    refuse("v: 5 entries", v=Tensor(bf16, 4, 4, 128))
    refuse("q: 128 entries", q=Tensor(bf16, 5, 8, 64))
    refuse("out: 8 entries", out=Tensor(bf16, 5, 4, 128))
    refuse("out: rows overlap", out=Tensor(bf16, 5, 8, 128, stride=(0, 128, 1)))
    refuse("slots: int32", slots=Tensor(i64, 5))
    refuse("positions: 5 entries", positions=Tensor(i32, 6))
    refuse("table: float32", table=Tensor(bf16, 100, 128))
    refuse("table has gaps", table=Tensor(f32, 100, 128, stride=(256, 1)))
    refuse("rotated elements", table=Tensor(f32, 100, 40))
    refuse("rotated elements", table=Tensor(f32, 100, 256))
    refuse("q_norm: 128 entries", q_norm=Tensor(bf16, 64))
    refuse("k_norm: bfloat16", k_norm=Tensor(f32, 128))
    refuse("interleaved", interleaved=5)
    refuse("multiples of 8", v=Tensor(bf16, 5, 4, 128, stride=(513, 128, 1)))

    # attention
    asked = []

    def allocate(count):
        asked.append(count)
        return Tensor(u8, count)
    run, refuse = trial(lambda cache, device, q, out, starts, lens, blocks, mask, most_new, longest, scale: calls.kv_attend(
        cache, device, q, out, starts, lens, blocks, mask, most_new, longest, scale, allocate), cache=c, device=0, q=q, out=q, starts=Tensor(i32, 3),
        lens=Tensor(i32, 2), blocks=Tensor(i32, 2, 6), mask=None, most_new=3, longest=None, scale=0.1)
    assert not asked
    run(1, cache=c8, mask=Tensor(i64, 5))
    run(1, longest=1 << 40)
    run(1, blocks=Tensor(i32, 2, 6, stride=(50, 1)))
    run(2, blocks=Tensor(i32, 2, 600))
    assert len(asked) == 1 and asked[0] > 0
    run(0, most_new=0)
    refuse("the cache is on device 2", device=2)
    refuse("starts: 3 entries", starts=Tensor(i32, 2))
    refuse("lens: int32", lens=Tensor(i64, 2))
    refuse("blocks: 2 entries", blocks=Tensor(i32, 3, 6))
    refuse("blocks: rows overlap", blocks=Tensor(i32, 2, 6, stride=(0, 1)))
    refuse("blocks: the last dimension has gaps", blocks=Tensor(i32, 2, 6, stride=(1, 2)))
    refuse("mask: int64", mask=Tensor(i32, 5))
    refuse("mask: 5 entries", mask=Tensor(i64, 2))
    refuse("out: 8 entries", out=Tensor(bf16, 5, 4, 128))
    refuse("out: rows overlap", out=Tensor(bf16, 5, 8, 128, stride=(1024, 0, 1)))
    refuse("query heads", q=Tensor(bf16, 5, 6, 128), out=Tensor(bf16, 5, 6, 128))
    refuse("longest", longest=-5)
    for most_new in (-1, -(1 << 40), 1 << 40, (1 << 32) + 3):
        refuse("new tokens of a sequence", most_new=most_new)
    refuse("64 new tokens", most_new=65, mask=Tensor(i64, 5))
    refuse("scale", scale=0.0)
    refuse("too many", blocks=Tensor(i32, 2, 1 << 28, stride=(1 << 28, 1)))

    # sampling
    run, refuse = trial(lambda logits, u, t, k, p, m, out: calls.sample(logits, u, t, k, p, m, out), logits=Tensor(f32, 3, 50), u=Tensor(f32, 3), t=None, k=None, p=None,
                        m=None, out=Tensor(i64, 3))
    run(1, logits=Tensor(bf16, 3, 50, stride=(77, 1)), t=Tensor(f32, 3), k=Tensor(i32, 3), p=Tensor(f32, 3), m=Tensor(f32, 3))
    run(0, logits=Tensor(f32, 0, 50), u=Tensor(f32, 0), out=Tensor(i64, 0))
    refuse("logits: float32 or float16 or bfloat16", logits=Tensor(i32, 3, 50))
    refuse("uniform: float32", u=Tensor(bf16, 3))
    refuse("uniform: 3 entries", u=Tensor(f32, 1))
    refuse("temperature: 3 entries", t=Tensor(f32, 2))
    refuse("top_k: int32", k=Tensor(i64, 3))
    refuse("top_p: the last dimension has gaps", p=Tensor(f32, 3, stride=(0,)))
    refuse("min_p is not on the GPU", m=Tensor(f32, 3, device=-1))
    refuse("out: int64", out=Tensor(i32, 3))
    refuse("overlap", logits=Tensor(f32, 3, 50, stride=(0, 1)))
    refuse("scores", logits=Tensor(f32, 3, (1 << 20) + 1))


CASES = [plans_of_4_bit_weights, runs_of_4_bit_weights, new_tokens_of_the_cache, attention_over_the_cache, samples, calls_with_tensors]


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    folder = tmp_path_factory.mktemp("hip")
    source = folder / "stub.c"
    source.write_text('#include "%s"\nint stub_device;\nint hipGetDevice(int *d) { return *d = stub_device, kSuccess; }\n'
                      "int hipFuncSetAttribute(const void *f, int a, int v) { return (void)f, (void)a, (void)v, kSuccess; }\n" % os.path.join(ROOT, "tests", "hip_stub.c"))
    so = str(folder / "stub.so")
    subprocess.check_call(["gcc", "-O1", "-std=gnu11", "-Wall", "-fPIC", "-shared", str(source), "-o", so])
    return so


@pytest.mark.parametrize("case", CASES, ids=lambda c: c.__name__)
def test_refusals(case, stub):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, case.__name__], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                       timeout=120)
    assert r.returncode == 0, r.stdout[-4000:]


@pytest.mark.parametrize("changes, message", [
    (dict(activation="relu"), "activation"), (dict(q=(8, 16, 2)), "two dimensions"), (dict(scales=(8, 2)), "scales: torch.bfloat16 of shape"),
    (dict(group=48), "group"), (dict(q=(0, 16)), "no rows"), (dict(q=(7, 16), activation="silu"), "even number"), (dict(zeros=(8, 3)), "zeros"), (dict(bias=(9,)), "bias")])
def test_constructor_refuses(changes, message):
    torch = pytest.importorskip("torch")
    from nart_amd import hipq
    shapes = dict(dict(q=(8, 16), scales=(8, 1), zeros=None, bias=None), **{n: v for n, v in changes.items() if n in ("q", "scales", "zeros", "bias")})
    t = {n: None if s is None else torch.zeros(s, dtype=torch.uint8 if n in ("q", "zeros") else torch.bfloat16) for n, s in shapes.items()}
    with pytest.raises(ValueError, match=message):
        hipq.LinearW4(t["q"], t["scales"], changes.get("group", 32), zeros=t["zeros"], bias=t["bias"], activation=changes.get("activation"))


if __name__ == "__main__":
    sys.path.insert(0, ROOT)
    STUB = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    globals()[sys.argv[2]]()
