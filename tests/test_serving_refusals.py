"""What the entry points that serve several sequences refuse, on the CPU: their host side compiled with stand-ins for the
device (tests/native/serving_host.cpp).  Each case changes one argument of a call that is taken; a refused call launches
nothing and says why."""
import ctypes
import os
import shutil
import subprocess

import pytest

from tests.test_longctx_refusals import F, M, U, Z, Host, try_all
from zhip import hip

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    so = str(tmp_path_factory.mktemp("host") / "serving_host.so")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O1", "-fPIC", "-std=c++17", "-shared", "-Wl,-Bsymbolic",
                    "-Wno-unused-result", "-Wno-unused-value", "-I" + os.path.join(REPO, "include"),
                    "-I" + os.path.join(REPO, "ziggy-llm_amd", "csrc"), "-o", so,
                    os.path.join(REPO, "tests", "native", "serving_host.cpp")], check=True)
    L = ctypes.CDLL(so)
    for n in ("fake_context", "fake_buffer"):
        getattr(L, n).restype = ctypes.c_void_p
    for n in ("ziggy_hip_kv4_codes_length", "ziggy_hip_kv4_scales_length"):
        getattr(L, n).restype = ctypes.c_size_t
    return Host(L)


def ref(x):
    return ctypes.byref(x) if x is not None else None


def rope(**changes):
    return hip.RopeDesc(**{**dict(head_dim=64, rope_dim=64, style=1, base=10000.0), **changes})


def heads(host, desc=True, factors=None, q_norm=None, k_norm=None, eps=1e-6, offset=0.0, **changes):
    return hip.HeadsDesc(ctypes.pointer(rope(**changes)) if desc else None, factors, q_norm, k_norm, eps, offset)


def bad_heads(host):
    small = host.buffer(4 * 64 - 1)
    out = [heads(host, **k) for k in (
        dict(head_dim=62), dict(head_dim=0), dict(head_dim=1024), dict(rope_dim=0), dict(rope_dim=66), dict(rope_dim=3), dict(style=2),
        dict(scaling=4), dict(base=0.0), dict(base=NAN), dict(magnitude=INF), dict(scaling=1, factor=0.0), dict(scaling=2, factor=4.0),
        dict(eps=-1e-6), dict(eps=NAN), dict(eps=INF), dict(offset=NAN), dict(offset=INF), dict(q_norm=small), dict(k_norm=small),
        dict(q_norm=host.buffer(256, device=1)), dict(k_norm=host.buffer(256, device=1)), dict(factors=host.buffer(127)),
        dict(factors=host.buffer(128, device=1)))]
    return [dict(d=h) for h in out]


def test_norm_rope(host):
    x, y, at = host.buffer(4 * 1000), host.buffer(4 * 1000), host.buffer(40)
    w, fac = host.buffer(256), host.buffer(128)
    good = heads(host, q_norm=w, k_norm=w, factors=fac)

    def call(d=good, src=x, soff=0, ss=0, dst=y, doff=0, ds=0, pos=at, first=0, rows=5, q=2, k=1, ctx=host.ctx):
        return host.call("ziggy_hip_norm_rope_rows_f32", ctx, ref(d), src, Z(soff), Z(ss), dst, Z(doff), Z(ds), pos, U(first), U(rows), U(q), U(k))

    # (another head size alone asks for rows of another width, which may fit: taken or not, it is no refusal of the size)
    try_all(host, call, {}, [b for b in bad_heads(host) if b["d"].rope.contents.head_dim != 62] + [
        dict(ctx=None), dict(d=None), dict(d=heads(host, desc=False)), dict(src=None), dict(dst=None), dict(rows=0), dict(q=0, k=0), dict(q=1 << 17),
        dict(k=1 << 17), dict(q=0xFFFFFFFF, k=2), dict(rows=6), dict(rows=1 << 31), dict(soff=2), dict(doff=6), dict(soff=4 * 50), dict(ss=191),
        dict(ds=100), dict(ss=300), dict(ss=1 << 61), dict(ds=(1 << 62) + 1), dict(soff=(1 << 64) - 4), dict(pos=host.buffer(16)),
        dict(src=host.buffer(4000, device=1)), dict(dst=host.buffer(4000, device=1)), dict(pos=host.buffer(40, device=1)),
        dict(dst=x, doff=4), dict(dst=x, ss=192, ds=196), dict(pos=None, first=0xFFFFFFFF), dict(dst=at), dict(pos=y),
        dict(d=heads(host, q_norm=y)), dict(d=heads(host, k_norm=y)), dict(d=heads(host, factors=y))])
    assert call(dst=x) and call(dst=x, ss=193, ds=193) and call(pos=None, first=0xFFFFFFFB) and call(q=3, k=0) and call(q=0, k=3)
    assert call(d=heads(host)) and call(d=heads(host, q_norm=w)) and call(d=heads(host, eps=0.0, offset=1.0))


def cache(host, layers=2, kvh=4, hd=64, pages=10, device=0, less=(0, 0, 0, 0), **buffers):
    codes = layers * kvh * pages * 32 * hd
    b = [host.buffer(max(n - l, 1), device) for n, l in zip((codes, codes // 16, codes, codes // 16), less)]
    for i, v in buffers.items():
        b["k_codes k_scales v_codes v_scales".split().index(i)] = v
    return hip.Kv4CacheDesc(*b, layers, kvh, hd, pages)


def batch(host, sequences=3, per=5, rows=20, max_rows=0, max_length=0, device=(0, 0, 0), less=(0, 0, 0), **buffers):
    b = [host.buffer(max(n - l, 1), d) for n, l, d in zip((4 * min(sequences, 9) * min(per, 1000), 4 * min(sequences, 9) + 4, 4 * min(sequences, 9)), less, device)]
    for i, v in buffers.items():
        b["page_table row_starts lengths".split().index(i)] = v
    return hip.BatchDesc(*b, sequences, per, rows, max_rows, max_length)


def bad_caches_and_batches(host, good):
    some = host.buffer(4 * M)
    out = [dict(c=None), dict(b=None), dict(layer=2), dict(ctx=None)]
    out += [dict(c=cache(host, **k)) for k in (dict(hd=32), dict(hd=80), dict(hd=512), dict(device=1),
                                               *(dict(less=tuple(int(i == j) for j in range(4))) for i in range(4)))]
    out += [dict(c=cache(host, k_codes=some, v_codes=some)), dict(c=cache(host, k_codes=some, v_scales=some)), dict(c=cache(host, v_codes=None))]
    for k in ("layers", "head_count_kv", "pages"):
        for v in (0, 0xFFFFFFFF):
            c = cache(host)
            setattr(c, k, v)
            out.append(dict(c=c))
    out += [dict(b=batch(host, **k)) for k in (
        dict(sequences=0), dict(per=0), dict(rows=0), dict(sequences=65537), dict(per=(1 << 24) + 1), dict(rows=0x80000000), dict(rows=1 << 30),
        dict(less=(1, 0, 0)), dict(less=(0, 1, 0)), dict(less=(0, 0, 1)), dict(device=(1, 0, 0)), dict(device=(0, 1, 0)), dict(device=(0, 0, 1)),
        dict(page_table=None), dict(row_starts=None), dict(lengths=None), dict(page_table=ctypes.c_void_p(good.v_codes)),
        dict(row_starts=ctypes.c_void_p(good.k_scales)), dict(lengths=ctypes.c_void_p(good.k_codes)))]
    return out


def test_kv4_lengths(host):
    f, g = host.L.ziggy_hip_kv4_codes_length, host.L.ziggy_hip_kv4_scales_length
    assert f(2, 8, 128, 100) == 2 * 8 * 100 * 64 * 64 and g(2, 8, 128, 100) == 2 * 8 * 100 * 64 * 4
    assert f(1, 1, 64, 1) == 64 * 32 and g(1, 1, 64, 1) == 128 and f(1, 3, 96, 7) == 3 * 7 * 64 * 48 and g(1, 3, 96, 7) == 3 * 7 * 64 * 3
    for bad in ((0, 1, 64, 1), (1, 0, 64, 1), (1, 1, 0, 1), (1, 1, 63, 1), (1, 1, 64, 0), (1, 1, 64, (1 << 24) + 1), (1, 1025, 64, 1),
                (0xFFFFFFFF, 1024, 256, 1 << 24)):
        assert f(*bad) == 0 and g(*bad) == 0


def test_append(host):
    good, src, q_out = cache(host), host.buffer(4 * 20 * 1100), host.buffer(4 * 20 * 512)
    tables = batch(host)
    w = host.buffer(256)

    def call(c=good, layer=1, b=tables, d=heads(host, q_norm=w, k_norm=w), src=src, k=2048, v=4 * 768, stride=1100, q=8, qo=0, out=q_out, oo=0, os=0, ctx=host.ctx):
        return host.call("ziggy_hip_kv4_append", ctx, ref(c), U(layer), ref(b), ref(d), src, Z(k), Z(v), Z(stride), U(q), Z(qo), out, Z(oo), Z(os))

    try_all(host, call, {}, bad_caches_and_batches(host, good) + bad_heads(host) + [
        dict(src=None), dict(out=None), dict(src=host.buffer(4 * 22000 - 1), v=4 * 844), dict(k=2), dict(v=4 * 845), dict(k=(1 << 64) - 4), dict(stride=255),
        dict(stride=511), dict(stride=1105), dict(stride=1 << 62), dict(q=1 << 17), dict(q=9), dict(qo=3), dict(qo=4 * 589), dict(oo=2), dict(oo=4), dict(os=511),
        dict(os=1 << 62), dict(src=host.buffer(4 * 22000, device=1)), dict(out=host.buffer(4 * 20 * 512, device=1)), dict(src=ctypes.c_void_p(good.k_codes)),
        dict(out=ctypes.c_void_p(good.v_codes), b=batch(host, rows=1)), dict(out=src, oo=4), dict(out=src, oo=0), dict(out=src, oo=4 * 100, qo=4 * 600, os=1100),
        dict(out=src, oo=2048, os=1100), dict(out=src, oo=1024, os=1100, qo=1024), dict(out=w, b=batch(host, rows=1), q=1), dict(d=heads(host, k_norm=ctypes.c_void_p(good.k_codes))),
        dict(d=heads(host, factors=ctypes.c_void_p(good.v_scales)))])
    assert call(out=src, os=1100) and call(q=0, out=None) and call(d=None) and call(d=heads(host, desc=False, k_norm=w)) and call(os=600, b=batch(host, rows=17))
    assert call(out=src, os=1100, oo=2048, qo=2048, k=0, v=1024) and call(b=batch(host, max_rows=100, max_length=0xFFFFFFFF))
    assert call(b=batch(host, sequences=9, per=1000, rows=1, max_rows=1))


def test_append_alone_without_a_gap(host):
    """A stride of 0: rows of one kv row each, keys and values in parts of the buffer of their own."""
    good, src = cache(host), host.buffer(4 * 2 * 20 * 256)
    args = [host.ctx, ref(good), U(0), ref(batch(host)), None, src, Z(0), Z(4 * 20 * 256), Z(0), U(0), Z(0), None, Z(0), Z(0)]
    assert host.call("ziggy_hip_kv4_append", *args)
    args[7] = Z(4 * 20 * 256 + 4)
    assert not host.call("ziggy_hip_kv4_append", *args)


def test_load(host):
    good, tables = cache(host), batch(host)
    k, v = host.buffer(4 * 20 * 256), host.buffer(4 * 20 * 256)

    def call(c=good, layer=1, b=tables, k=k, v=v, ctx=host.ctx):
        return host.call("ziggy_hip_kv4_load_f32", ctx, ref(c), U(layer), ref(b), k, v)

    try_all(host, call, {}, bad_caches_and_batches(host, good) + [
        dict(k=None), dict(v=None), dict(v=k), dict(k=host.buffer(4 * 20 * 256 - 1)), dict(v=host.buffer(4 * 20 * 256 - 1)),
        dict(k=host.buffer(M, device=1)), dict(k=ctypes.c_void_p(good.k_codes), b=batch(host, rows=1)), dict(b=batch(host, page_table=v)),
        dict(b=batch(host, row_starts=k)), dict(b=batch(host, lengths=k))])


def test_attention(host):
    good, tables = cache(host), batch(host)
    q, out = host.buffer(4 * 8 * 64 * 20), host.buffer(4 * 8 * 64 * 20)

    def call(c=good, layer=0, b=tables, q=q, qo=0, stride=0, out=out, heads=8, window=0, scale=0.1, ctx=host.ctx):
        return host.call("ziggy_hip_kv4_attention_f32", ctx, ref(c), U(layer), ref(b), q, Z(qo), Z(stride), out, U(heads), U(window), F(scale))

    try_all(host, call, {}, bad_caches_and_batches(host, good) + [
        dict(q=None), dict(out=None), dict(heads=0), dict(heads=6), dict(heads=9), dict(heads=260, b=batch(host, rows=1)), dict(scale=NAN), dict(scale=INF),
        dict(scale=-INF), dict(scale=2.4e38), dict(scale=-3e38), dict(stride=511), dict(stride=513), dict(stride=1 << 62), dict(qo=2), dict(qo=4), dict(out=q),
        dict(out=host.buffer(4 * 8 * 64 * 20 - 4)), dict(q=host.buffer(4 * 8 * 64 * 20 - 4)), dict(q=host.buffer(M, device=1)), dict(out=host.buffer(M, device=1)),
        dict(out=ctypes.c_void_p(good.v_codes), b=batch(host, rows=1)), dict(b=batch(host, page_table=out)), dict(b=batch(host, row_starts=out)),
        dict(b=batch(host, lengths=out))])
    assert call(window=1) and call(window=0xFFFFFFFF) and call(scale=-1.0) and call(scale=0.0) and call(scale=2.3e38) and call(b=batch(host, rows=10), stride=1024)
    assert call(heads=256, b=batch(host, rows=1, max_rows=7, max_length=9), q=host.buffer(M), out=host.buffer(M))


def test_logprobs(host):
    x, tok, out, ent = host.buffer(4 * 7 * 1000), host.buffer(28), host.buffer(28), host.buffer(28)
    ids, top = host.buffer(4 * 7 * 20), host.buffer(4 * 7 * 20)

    def call(x=x, stride=0, tok=tok, out=out, ent=ent, k=20, ids=ids, top=top, rows=7, vocab=1000, ctx=host.ctx):
        return host.call("ziggy_hip_token_logprobs_f32", ctx, x, Z(stride), tok, out, ent, U(k), ids, top, U(rows), U(vocab))

    try_all(host, call, {}, [
        dict(ctx=None), dict(x=None), dict(tok=None), dict(out=None), dict(ids=None), dict(top=None), dict(rows=0), dict(rows=8), dict(vocab=0), dict(vocab=1001),
        dict(k=21), dict(k=65, rows=1), dict(k=20, vocab=19), dict(stride=999), dict(stride=1001), dict(stride=1 << 62), dict(tok=host.buffer(27)),
        dict(out=host.buffer(27)), dict(ent=host.buffer(27)), dict(x=host.buffer(M, device=1)), dict(tok=host.buffer(28, device=1)), dict(ent=host.buffer(28, device=1)),
        dict(out=x), dict(out=tok), dict(ent=out), dict(ent=x), dict(ids=top), dict(ids=x), dict(top=x), dict(top=ent), dict(ids=tok)])
    assert call(ent=None) and call(k=0, ids=None, top=None) and call(k=64, rows=2) and call(rows=6, stride=1100)
    big = host.buffer(4 * 262145)
    assert call(x=big, vocab=262144, rows=1) and not call(x=big, vocab=262145, rows=1)


def test_the_callers_device_stays_current(host):
    other = ctypes.c_void_p(host.L.fake_context(3, Z(64 << 20)))
    x, y = host.buffer(4096, device=3), host.buffer(4096, device=3)
    assert host.L.fake_device() == 0
    assert host.call("ziggy_hip_norm_rope_rows_f32", other, ref(heads(host)), x, Z(0), Z(0), y, Z(0), Z(0), None, U(0), U(1), U(1), U(0))
    assert host.L.fake_device() == 0


def test_freed_buffers_and_null_contexts_in_the_binding():
    class Gone:
        h = None

    b = hip.Batch.__new__(hip.Batch)
    b.buffers, b._desc = (Gone(),), hip.BatchDesc()
    with pytest.raises(hip.HipError, match="freed"):
        b.desc
    with pytest.raises(hip.HipError) as e:
        hip._call("ziggy_hip_kv4_load_f32", None, None, 0, None, None, None)
    assert e.value.status == 6


def test_more_rows_and_sequences_than_a_launch_has(host):
    x, y = host.buffer(1 << 40), host.buffer(1 << 40)
    for rows, taken in ((1 << 25, True), ((1 << 25) + 1, False)):
        args = [host.ctx, ref(heads(host, head_dim=2, rope_dim=2)), x, Z(0), Z(0), y, Z(0), Z(0), None, U(0), U(rows), U(1), U(0)]
        assert host.call("ziggy_hip_norm_rope_rows_f32", *args) == taken
        b = batch(host, rows=rows)
        assert host.call("ziggy_hip_kv4_load_f32", host.ctx, ref(cache(host)), U(0), ref(b), x, y) == taken
        assert host.call("ziggy_hip_kv4_append", host.ctx, ref(cache(host)), U(0), ref(b), None, x, Z(0), Z(1024), Z(512), U(0), Z(0), None, Z(0), Z(0)) == taken
    for kvh, heads_, sequences, rows, taken in ((64, 64, 1 << 15, 8, True), (64, 64, (1 << 15) + 1, 8, False), (4, 16, 2, 1 << 25, True), (4, 20, 2, 1 << 25, False)):
        c, b = cache(host, kvh=kvh), batch(host, sequences=sequences, rows=rows, page_table=x, row_starts=host.buffer(1 << 20), lengths=host.buffer(1 << 20))
        q, out = host.buffer(1 << 42), host.buffer(1 << 42)
        assert host.call("ziggy_hip_kv4_attention_f32", host.ctx, ref(c), U(0), ref(b), q, Z(0), Z(0), out, U(heads_), U(0), F(0.1)) == taken


def test_outputs_behind_a_cache_in_its_buffers(host):
    """What counts is where the arrays end, not the buffers that they lie in."""
    at, codes = 1 << 41, 2 * 4 * 10 * 32 * 64
    arena = host.buffer(1 << 24, at=at)
    c, b = cache(host, k_codes=arena), batch(host)
    q = host.buffer(4 * 8 * 64 * 20)
    for off, taken in ((codes, True), (codes - 4, False)):
        out = host.buffer(4 * 8 * 64 * 20, at=at + off)
        assert host.call("ziggy_hip_kv4_attention_f32", host.ctx, ref(c), U(0), ref(b), q, Z(0), Z(0), out, U(8), U(0), F(0.1)) == taken
