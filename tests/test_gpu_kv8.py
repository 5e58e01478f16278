"""The 8-bit K/V cache's store and read-back against a plain form, code for code and scale for scale: every
code is the exact quotient's nearest integer, so nothing is tolerated."""
import numpy as np
import pytest

from tests import longctx_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu


def upload(ctx, layers, context):
    heads, _, hd = layers[0].codes[0].shape
    kc, ks, vc, vs = oracle.kv8_device(layers, context)
    return hip.Kv8Cache(ctx.buffer(kc), ctx.buffer(ks), ctx.buffer(vc), ctx.buffer(vs), len(layers), heads, hd, context)


def same(cache, layers, context):
    want = oracle.kv8_device(layers, context)
    got = [b.read(a.dtype) for b, a in zip(cache.buffers, want)]
    for name, g, w in zip(("k codes", "k scales", "v codes", "v scales"), got, want):
        assert np.array_equal(g, w, equal_nan=g.dtype == np.float32), (name, np.flatnonzero(g != w)[:8])


def values(rng, rows, heads, hd):
    x = rng.normal(0, 1, (rows, heads, hd)).astype(np.float32)
    x[:, :, ::31] *= 6
    x[rng.random((rows, heads, hd)) < 0.1] = 0
    return x


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("position,rows", [(0, 1), (0, 32), (0, 31), (5, 1), (31, 1), (31, 2), (17, 60), (64, 33), (40, 100), (96, 4)])
def test_store(hip_ctx, hd, position, rows):
    print("kv8 store", hd, position, rows, flush=True)
    rng = np.random.default_rng(hd + position * 100 + rows)
    heads, context = 3, 150
    layers = [oracle.Kv8(heads, context, hd, rng) for _ in range(2)]
    cache = upload(hip_ctx, layers, context)
    k, v = values(rng, rows, heads, hd), values(rng, rows, heads, hd)
    hip_ctx.kv8_store(cache, hip_ctx.buffer(k), hip_ctx.buffer(v), 1, position, rows)
    layers[1].store(k, v, position)
    same(cache, layers, context)  # the other layer, and the rows around, as they were


@pytest.mark.parametrize("first", [0, 9])
def test_one_row_at_a_time(hip_ctx, first):
    """Decoding: rows whose scale grows within the block, and rows whose does not."""
    rng = np.random.default_rng(first)
    heads, hd, context = 2, 128, 80
    layers = [oracle.Kv8(heads, context, hd, rng)]
    cache = upload(hip_ctx, layers, context)
    for t in range(first, context):
        k, v = values(rng, 1, heads, hd) * (1 + t % 7), values(rng, 1, heads, hd) / (1 + t % 5)
        hip_ctx.kv8_store(cache, hip_ctx.buffer(k), hip_ctx.buffer(v), 0, t, 1)
        layers[0].store(k, v, t)
        same(cache, layers, context)


@pytest.mark.parametrize("size", [1e-45, 3e-44, 1.3e-38, 1e-37, 1e-30, 1e-20, 1.0, 1e20, 3.3e38])
def test_sizes(hip_ctx, size):
    """From the smallest denormal to the largest value: scales below the reciprocal's range among them."""
    rng = np.random.default_rng(3)
    heads, hd, context = 1, 64, 64
    layers = [oracle.Kv8(heads, context, hd, rng)]
    cache = upload(hip_ctx, layers, context)
    k = (np.clip(rng.normal(0, 0.4, (40, heads, hd)), -1, 1) * size).astype(np.float32)
    v = np.zeros_like(k)
    hip_ctx.kv8_store(cache, hip_ctx.buffer(k), hip_ctx.buffer(v), 0, 0, 40)
    layers[0].store(k, v, 0)
    same(cache, layers, context)


def test_ties_go_to_even(hip_ctx):
    """Values half a step between codes, and one ulp to either side."""
    heads, hd, context = 1, 128, 32
    scale = np.float32(0.0123)
    top = np.float32(scale * np.float32(127))
    while np.float32(top * np.float32(1 / 127)) != scale:
        top = np.nextafter(top, np.float32(np.inf))
    half = (np.arange(-126, 126) + 0.5) * float(scale)
    mid = half.astype(np.float32)
    k = np.zeros((32, heads, hd), np.float32)
    flat = np.concatenate([mid, np.nextafter(mid, np.float32(9)), np.nextafter(mid, np.float32(-9)),
                           (np.arange(-64, 64) * 2.0 ** -3 + 2.0 ** -4).astype(np.float32)[:100]])
    k.reshape(-1)[:flat.size] = flat
    k[31, 0, 127] = top
    v = np.zeros_like(k)
    exact = np.zeros_like(k)  # a power-of-two scale: true ties
    exact.reshape(-1)[:252] = np.arange(-126, 126) + 0.5
    exact[31, 0, 127] = 127
    for a in (k, exact):
        layers = [oracle.Kv8(heads, context, hd)]
        cache = upload(hip_ctx, layers, context)
        hip_ctx.kv8_store(cache, hip_ctx.buffer(a), hip_ctx.buffer(v), 0, 0, 32)
        layers[0].store(a, v, 0)
        same(cache, layers, context)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_row_that_is_not_finite_marks_its_block(hip_ctx, bad):
    rng = np.random.default_rng(8)
    heads, hd, context = 2, 64, 96
    layers = [oracle.Kv8(heads, context, hd, rng)]
    cache = upload(hip_ctx, layers, context)
    k, v = values(rng, 96, heads, hd), values(rng, 96, heads, hd)
    k[40, 1, 5] = bad
    v[70, 0, 0] = bad
    kb, vb = hip_ctx.buffer(k), hip_ctx.buffer(v)
    hip_ctx.kv8_store(cache, kb, vb, 0, 0, 96)
    out = [hip_ctx.empty(k.nbytes) for _ in range(2)]
    hip_ctx.kv8_load(cache, *out, 0, 0, 96)
    layers[0].store(k, v, 0)
    for w, (o, marked) in enumerate(zip(out, ((1, 1), (2, 0)))):
        got = o.read().reshape(96, heads, hd)
        want = np.zeros(got.shape, bool)
        want[32 * marked[0]:32 * marked[0] + 32, marked[1]] = True
        assert np.array_equal(np.isnan(got), want)
        assert np.array_equal(got[~want], layers[0].rows(w, 0, 96)[~want])
    # one more row leaves the block marked, a new beginning clears it
    one = values(rng, 1, heads, hd)
    hip_ctx.kv8_store(cache, hip_ctx.buffer(one), hip_ctx.buffer(one), 0, 41, 1)
    hip_ctx.kv8_load(cache, *out, 0, 0, 96)
    assert np.isnan(out[0].read().reshape(96, heads, hd)[32:64, 1]).all()
    k[40, 1, 5] = 1
    hip_ctx.kv8_store(cache, hip_ctx.buffer(k[32:64]), hip_ctx.buffer(v[32:64]), 0, 32, 32)
    hip_ctx.kv8_load(cache, *out, 0, 0, 64)
    assert np.isfinite(out[0].read().reshape(96, heads, hd)[:64]).all()


@pytest.mark.parametrize("hd,stride,koff,voff", [(64, 4 * 192 + 1, 1, 200), (128, 4 * 384, 384, 768), (96, 700, 0, 300), (256, 1600, 2, 771)])
def test_strided_rows_of_one_buffer(hip_ctx, hd, stride, koff, voff):
    rng = np.random.default_rng(hd)
    heads, context, rows = 3 if hd < 256 else 2, 100, 50
    layers = [oracle.Kv8(heads, context, hd, rng)]
    cache = upload(hip_ctx, layers, context)
    x = rng.normal(0, 1, rows * stride + 2000).astype(np.float32)
    at = np.arange(rows)[:, None] * stride + np.arange(heads * hd)
    k, v = (x[at + o].reshape(rows, heads, hd) for o in (koff, voff))
    xb = hip_ctx.buffer(x)
    hip_ctx.kv8_store(cache, xb, xb, 0, 13, rows, row_stride=stride, k_off=4 * koff, v_off=4 * voff)
    layers[0].store(k, v, 13)
    same(cache, layers, context)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("position,rows", [(0, 1), (7, 3), (31, 2), (0, 70), (33, 64)])
def test_load(hip_ctx, hd, position, rows):
    rng = np.random.default_rng(hd + rows)
    heads, context = 5, 100
    layers = [oracle.Kv8(heads, context, hd, rng) for _ in range(3)]
    cache = upload(hip_ctx, layers, context)
    n = rows * heads * hd
    out = [hip_ctx.buffer(np.full(n + 9, 5, np.float32)) for _ in range(2)]
    hip_ctx.kv8_load(cache, *out, 2, position, rows)
    for w in range(2):
        got = out[w].read()
        assert np.array_equal(got[:n].reshape(rows, heads, hd), layers[2].rows(w, position, rows))
        assert np.all(got[n:] == 5)


def test_empty_cache_and_lengths(hip_ctx):
    cache = hip_ctx.kv8_cache(2, 4, 128, 1000)
    assert cache.buffers[0].nbytes == cache.buffers[2].nbytes == 2 * 4 * 1024 * 128
    assert cache.buffers[1].nbytes == cache.buffers[3].nbytes == 2 * 4 * 32 * 4
