"""What the long-context entry points refuse, on the CPU: their host side compiled with stand-ins for the device
(tests/native/longctx_host.cpp).  Each case changes one argument of a call that is taken; a refused call launches
nothing and says why."""
import ctypes
import os
import shutil
import subprocess

import pytest

from zhip import hip

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
M = 1 << 20


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    so = str(tmp_path_factory.mktemp("host") / "longctx_host.so")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O1", "-fPIC", "-std=c++17", "-shared", "-Wl,-Bsymbolic",
                    "-Wno-unused-result", "-Wno-unused-value", "-I" + os.path.join(REPO, "include"),
                    "-I" + os.path.join(REPO, "ziggy-llm_amd", "csrc"), "-o", so,
                    os.path.join(REPO, "tests", "native", "longctx_host.cpp")], check=True)
    L = ctypes.CDLL(so)
    for n in ("fake_context", "fake_buffer"):
        getattr(L, n).restype = ctypes.c_void_p
    for n in ("ziggy_hip_kv8_codes_length", "ziggy_hip_kv8_scales_length"):
        getattr(L, n).restype = ctypes.c_size_t
    return Host(L)


class Host:
    def __init__(self, L):
        self.L, self.next = L, 1 << 32
        self.ctx = ctypes.c_void_p(L.fake_context(0, ctypes.c_size_t(64 << 20)))

    def buffer(self, n, device=0, at=None):
        if at is None:
            at, self.next = self.next, self.next + (n + 4095) // 4096 * 4096 + 4096
        return ctypes.c_void_p(self.L.fake_buffer(self.ctx, device, ctypes.c_size_t(at), ctypes.c_size_t(n)))

    def call(self, name, *args):
        err = ctypes.create_string_buffer(256)
        before = self.L.fake_launches()
        st = getattr(self.L, name)(*args, err, ctypes.c_size_t(256))
        launched = self.L.fake_launches() - before
        if st:
            assert st == 6 and launched == 0 and err.value, (name, st, launched, err.value)
        else:
            assert launched > 0 and not err.value
        return st == 0


Z, U, F = ctypes.c_size_t, ctypes.c_uint32, ctypes.c_float


def try_all(host, call, good, bad):
    """call(**good) is taken; with any one of `bad` in place of its own it is refused."""
    assert call(**good)
    for change in bad:
        assert not call(**{**good, **change}), change


def test_rope(host):
    x, y, at, fac = host.buffer(4 * 1000), host.buffer(4 * 1000), host.buffer(40), host.buffer(4 * 32)
    d = dict(head_dim=64, rope_dim=64, style=0, base=10000.0, scaling=0, factor=1.0, original_context=0, low=1.0, high=4.0,
             magnitude=1.0)

    def call(src=x, soff=0, ss=0, dst=y, doff=0, ds=0, pos=at, first=0, factors=fac, rows=5, heads=3, ctx=host.ctx, **desc):
        return host.call("ziggy_hip_rope_rows_f32", ctx, ctypes.byref(hip.RopeDesc(**{**d, **desc})), src, Z(soff), Z(ss), dst,
                         Z(doff), Z(ds), pos, U(first), factors, U(rows), U(heads))

    nan, inf = float("nan"), float("inf")
    try_all(host, call, {}, [
        dict(ctx=None), dict(src=None), dict(dst=None), dict(rows=0), dict(heads=0), dict(heads=1 << 17), dict(rows=1 << 31),
        dict(rows=6), dict(head_dim=0), dict(head_dim=63), dict(head_dim=514), dict(rope_dim=0), dict(rope_dim=66), dict(rope_dim=63),
        dict(style=2), dict(scaling=4), dict(base=0.0), dict(base=-1.0), dict(base=nan), dict(base=inf), dict(magnitude=nan),
        dict(scaling=1, factor=0.0), dict(scaling=1, factor=nan), dict(scaling=1, factor=inf), dict(scaling=2, factor=4.0),
        dict(scaling=3, original_context=100, low=4.0, high=4.0), dict(scaling=3, original_context=100, low=0.0),
        dict(scaling=2, original_context=100, high=inf), dict(scaling=2, original_context=100, base=1.0),
        dict(soff=2), dict(doff=6), dict(soff=4 * 50), dict(ss=191), dict(ds=100), dict(ss=300), dict(ss=1 << 61), dict(ds=(1 << 62) + 1),
        dict(soff=(1 << 64) - 4), dict(pos=host.buffer(16)), dict(factors=host.buffer(124)),
        dict(src=host.buffer(4 * 1000, device=1)), dict(dst=host.buffer(4 * 1000, device=1)), dict(pos=host.buffer(40, device=1)),
        dict(dst=x, doff=4), dict(dst=x, ss=192, ds=196), dict(pos=None, first=0xFFFFFFFF), dict(dst=at), dict(pos=y), dict(factors=y)])
    assert call(dst=x) and call(dst=x, ss=193, ds=193) and call(pos=None, first=0xFFFFFFFB) and call(factors=None)
    assert call(scaling=2, original_context=100) and call(scaling=3, original_context=100) and call(scaling=1, factor=2.0)
    assert host.call("ziggy_hip_rope_rows_f32", host.ctx, None, x, Z(0), Z(0), y, Z(0), Z(0), at, U(0), None, U(1), U(1)) is False


def cache(host, layers=2, kvh=4, hd=64, context=100, device=0, less=(0, 0, 0, 0), **buffers):
    codes, scales = layers * kvh * -(-context // 32) * 32 * hd, layers * kvh * -(-context // 32) * 4
    b = [host.buffer(max(n - l, 1), device) for n, l in zip((codes, scales, codes, scales), less)]
    for i, v in buffers.items():
        b["k_codes k_scales v_codes v_scales".split().index(i)] = v
    return hip.Kv8CacheDesc(*b, layers, kvh, hd, context)


def bad_caches(host):
    some = host.buffer(4 * M)
    out = [dict(c=None)]
    out += [dict(c=cache(host, **k)) for k in (dict(hd=32), dict(hd=80), dict(hd=512), dict(device=1),
                                               *(dict(less=tuple(int(i == j) for j in range(4))) for i in range(4)))]
    out += [dict(c=cache(host, k_codes=some, v_codes=some)), dict(c=cache(host, k_codes=some, v_scales=some)), dict(c=cache(host, v_codes=None))]
    for k in ("layers", "head_count_kv", "context_length"):
        for v in (0, 0xFFFFFFFF):
            c = cache(host)
            setattr(c, k, v)
            out.append(dict(c=c))
    return out


def test_kv8_lengths(host):
    f, g = host.L.ziggy_hip_kv8_codes_length, host.L.ziggy_hip_kv8_scales_length
    assert f(2, 8, 128, 100) == 2 * 8 * 128 * 128 and g(2, 8, 128, 100) == 2 * 8 * 4 * 4
    assert f(1, 1, 64, 1) == 64 * 32 and g(1, 1, 64, 1) == 4
    assert f(80, 8, 128, 1 << 20) == 80 * 8 * 128 << 20
    for bad in ((0, 1, 64, 1), (1, 0, 64, 1), (1, 1, 0, 1), (1, 1, 63, 1), (1, 1, 64, 0), (1, 1, 64, 0xFFFFFFFF), (0xFFFFFFFF, 1024, 256, 0x7FFFFFE0)):
        assert f(*bad) == 0 and g(*bad) == 0


def test_store_and_load(host):
    x, good = host.buffer(4 * M), cache(host)
    k, v = host.buffer(4 * 256 * 100), host.buffer(4 * 256 * 100)

    def store(c=good, k=k, ko=0, v=v, vo=0, stride=0, layer=1, position=0, rows=100, ctx=host.ctx):
        return host.call("ziggy_hip_kv8_store", ctx, ctypes.byref(c) if c else None, k, Z(ko), v, Z(vo), Z(stride), U(layer), U(position), U(rows))

    def load(c=good, k=k, v=v, layer=1, position=0, rows=100, ctx=host.ctx):
        return host.call("ziggy_hip_kv8_load_f32", ctx, ctypes.byref(c) if c else None, k, v, U(layer), U(position), U(rows))

    both = bad_caches(host) + [dict(ctx=None), dict(k=None), dict(v=None), dict(layer=2), dict(rows=0), dict(rows=101), dict(position=1),
                               dict(position=100, rows=1), dict(position=0xFFFFFFFF, rows=2), dict(k=host.buffer(4 * 256 * 100 - 1)),
                               dict(v=host.buffer(4 * 256 * 100 - 1)), dict(k=host.buffer(4 * M, device=2)), dict(k=ctypes.c_void_p(good.k_codes), rows=1),
                               dict(v=ctypes.c_void_p(good.k_codes), rows=1)]
    try_all(host, store, {}, both + [dict(ko=1), dict(vo=2), dict(ko=4), dict(stride=255), dict(stride=257), dict(stride=1 << 62), dict(ko=(1 << 64) - 4)])
    try_all(host, load, {}, both + [dict(v=k)])
    assert store(k=x, v=x, ko=1024, vo=2048, stride=1000) and store(position=99, rows=1) and load(position=99, rows=1)


def test_attention(host):
    good, q, out = cache(host), host.buffer(4 * 8 * 64 * 30), host.buffer(4 * 8 * 64 * 30)

    def call(c=good, q=q, stride=0, out=out, heads=8, layer=0, position=70, queries=30, window=0, scale=0.1, ctx=host.ctx):
        return host.call("ziggy_hip_kv8_attention_f32", ctx, ctypes.byref(c) if c else None, q, Z(stride), out, U(heads), U(layer),
                         U(position), U(queries), U(window), F(scale))

    try_all(host, call, {}, bad_caches(host) + [
        dict(ctx=None), dict(q=None), dict(out=None), dict(heads=0), dict(heads=6), dict(heads=9), dict(heads=260, queries=1), dict(layer=2),
        dict(queries=0), dict(queries=31), dict(position=71), dict(position=0xFFFFFFFF, queries=2), dict(scale=float("nan")),
        dict(scale=float("inf")), dict(stride=511), dict(stride=513), dict(stride=1 << 62), dict(out=q), dict(out=host.buffer(4 * 8 * 64 * 30 - 4)),
        dict(q=host.buffer(4 * 8 * 64 * 30 - 4)), dict(q=host.buffer(M, device=1)), dict(out=host.buffer(M, device=1)),
        dict(out=ctypes.c_void_p(good.v_codes), queries=1)])
    assert call(window=1) and call(window=0xFFFFFFFF) and call(position=0, queries=1, heads=4) and call(scale=-1.0)


def test_attention_score_scale(host):
    """A scale whose product with log2 e passes binary32 is refused, the largest below it taken."""
    good, q, out = cache(host), host.buffer(4 * 8 * 64), host.buffer(4 * 8 * 64)
    for scale, taken in ((3e38, False), (-2.4e38, False), (2.3e38, True), (-2.3e38, True), (float("-inf"), False)):
        assert taken == host.call("ziggy_hip_kv8_attention_f32", host.ctx, ctypes.byref(good), q, Z(0), out, U(8), U(0), U(70), U(1), U(0), F(scale))


def test_sampling(host):
    x, u, out, rec = host.buffer(4 * 1000 * 7), host.buffer(56), host.buffer(28), host.buffer(4 * 7 * 20)

    def call(x=x, stride=0, rec=rec, n=20, u=u, out=out, rows=7, vocab=1000, ctx=host.ctx, **o):
        return host.call("ziggy_hip_sample_rows_f32", ctx, x, Z(stride), rec, U(n),
                         ctypes.byref(hip.SamplingOptions(**{**dict(temperature=1.0, repeat_penalty=1.1), **o})), u, out, U(rows), U(vocab))

    nan = float("nan")
    try_all(host, call, {}, [
        dict(ctx=None), dict(x=None), dict(u=None), dict(out=None), dict(rec=None), dict(rows=0), dict(rows=8), dict(vocab=0), dict(vocab=1001),
        dict(stride=999), dict(stride=1001), dict(stride=1 << 62), dict(n=21), dict(n=0xFFFFFFFF), dict(u=host.buffer(55)),
        dict(out=host.buffer(27)), dict(x=host.buffer(M, device=1)), dict(out=x), dict(out=u), dict(out=rec), dict(temperature=nan),
        dict(temperature=float("inf")), dict(repeat_penalty=nan), dict(top_p=nan), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=nan),
        dict(min_p=1.5), dict(min_p=-1.0)])
    assert call(top_k=1000) and call(top_k=0xFFFFFFFF) and call(rec=None, n=0) and call(temperature=-1.0) and call(top_p=0.0, min_p=1.0)
    big, many = host.buffer(4 * 262145), host.buffer(8 * M)
    assert call(x=big, vocab=262144, rows=1) and not call(x=big, vocab=262145, rows=1)
    assert call(x=many, vocab=2000, rows=7, top_k=1024) and not call(x=many, vocab=2000, rows=7, top_k=1025)
    assert host.call("ziggy_hip_sample_rows_f32", host.ctx, x, Z(0), None, U(0), None, u, out, U(1), U(10)) is False


def test_wrapped_memory(host):
    base, size = 0x10000000, 0x1000000

    def wrap(at, n, ctx=host.ctx, out=True):
        h, err = ctypes.c_void_p(1), ctypes.create_string_buffer(256)
        st = host.L.ziggy_hip_wrap_buffer(ctx, ctypes.c_void_p(at), Z(n), ctypes.byref(h) if out else None, err, Z(256))
        assert st in (0, 6) and bool(err.value) == bool(st) and (not out or bool(h.value) == (st == 0))
        return st == 0

    assert wrap(base, size) and wrap(base + 16, size - 16) and wrap(base + size - 16, 1)
    for bad in ((base, size + 1), (base + 16, size), (base + 8, 8), (base - 16, 32), (0, 16), (base, 0), (base + size, 16), (base, (1 << 64) - 1)):
        assert not wrap(*bad), bad
    assert not wrap(base, 16, ctx=None) and not wrap(base, 16, out=False)
    assert not wrap(base, 16, ctx=ctypes.c_void_p(host.L.fake_context(1, Z(1 << 20))))


def test_the_callers_device_stays_current(host):
    other = ctypes.c_void_p(host.L.fake_context(3, Z(64 << 20)))
    x, y = host.buffer(4096, device=3), host.buffer(4096, device=3)
    assert host.L.fake_device() == 0
    assert host.call("ziggy_hip_rope_rows_f32", other, ctypes.byref(hip.RopeDesc(64)), x, Z(0), Z(0), y, Z(0), Z(0), None, U(0), None, U(1), U(1))
    assert host.L.fake_device() == 0


def test_null_context_in_the_library():
    with pytest.raises(hip.HipError) as e:
        hip._call("ziggy_hip_kv8_load_f32", None, None, None, None, 0, 0, 1)
    assert e.value.status == 6
