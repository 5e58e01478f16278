"""The long-context operators where offsets pass 32 bits: caches of more than 4 GiB a head, rows a GiB apart."""
import numpy as np
import pytest

from tests import longctx_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu

STRIDE = 1 << 28  # floats: rows 1 GiB apart


def spread(ctx, rows):
    """A buffer whose rows (given dense) are STRIDE apart."""
    b = ctx.empty(4 * ((len(rows) - 1) * STRIDE + rows[0].size))
    for i, r in enumerate(rows):
        b.write(np.ascontiguousarray(r, np.float32), 4 * i * STRIDE)
    return b


@pytest.mark.parametrize("queries", [1, 5, 100])
def test_cache_positions_past_four_gib(hip_ctx, queries):
    """Rows and a window at position 18 million of heads of 256 (codes 4.6 GB into a head), as near the start."""
    heads, kvh, hd, far = 4, 2, 256, 18 << 20
    print("far cache", queries, flush=True)
    rng = np.random.default_rng(queries)
    rows, window = 150 + queries, 140
    k, v = (rng.normal(0, 1, (rows, kvh, hd)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 1, (queries, heads, hd)).astype(np.float32)
    near = oracle.Kv8(kvh, rows, hd)
    near.store(k, v, 0)
    want, bound = oracle.kv8_attention(near, q, rows - queries, hd ** -0.5, window)
    cache = hip_ctx.kv8_cache(1, kvh, hd, far + 300)
    assert cache.buffers[0].nbytes > 9 << 30
    hip_ctx.kv8_store(cache, hip_ctx.buffer(k), hip_ctx.buffer(v), 0, far, rows)
    ko, vo = hip_ctx.empty(k.nbytes), hip_ctx.empty(v.nbytes)
    hip_ctx.kv8_load(cache, ko, vo, 0, far, rows)
    out = hip_ctx.empty(q.nbytes)
    hip_ctx.kv8_attention(cache, hip_ctx.buffer(q), out, heads, 0, far + rows - queries, queries, window=window)
    for got, which in ((ko, 0), (vo, 1)):
        assert np.array_equal(got.read().reshape(k.shape), near.rows(which, 0, rows))
    err = np.abs(out.read().reshape(want.shape) - want)
    assert np.all(err <= bound), (err / bound).max()
    for b in cache.buffers:
        b.free()


def test_layers_past_four_gib(hip_ctx):
    """The last of 40 layers of 8 heads of 128 by 131072 positions, 5.3 GB of codes before it, by itself."""
    heads, kvh, hd, context, layers = 8, 8, 128, 131072, 40
    rng = np.random.default_rng(3)
    n = 70
    k, v = (rng.normal(0, 1, (n, kvh, hd)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 1, (1, heads, hd)).astype(np.float32)
    near = oracle.Kv8(kvh, n, hd)
    near.store(k, v, 0)
    cache = hip_ctx.kv8_cache(layers, kvh, hd, context)
    for layer in (layers - 1, layers - 9, 0):
        hip_ctx.kv8_store(cache, hip_ctx.buffer(-k if layer == 0 else k), hip_ctx.buffer(-v if layer == 0 else v), layer, 0, n)
    want, bound = oracle.kv8_attention(near, q, n - 1, hd ** -0.5)
    out = hip_ctx.empty(q.nbytes)
    for layer in (layers - 1, layers - 9):
        hip_ctx.kv8_attention(cache, hip_ctx.buffer(q), out, heads, layer, n - 1)
        assert np.all(np.abs(out.read().reshape(want.shape) - want) <= bound)
    for b in cache.buffers:
        b.free()


def test_rows_a_gib_apart(hip_ctx):
    rng = np.random.default_rng(5)
    rows, heads, hd = 6, 4, 64
    x = rng.normal(0, 1, (rows, heads, hd)).astype(np.float32)
    far = spread(hip_ctx, x)
    dense, out = hip_ctx.buffer(x), hip_ctx.empty(x.nbytes)
    d = hip.RopeDesc(hd, style=1)
    hip_ctx.rope_rows(d, dense, out, rows, heads, first_position=7)
    want = out.read()
    hip_ctx.rope_rows(d, far, out, rows, heads, first_position=7, src_stride=STRIDE)
    assert np.array_equal(out.read(), want)
    hip_ctx.rope_rows(d, far, far, rows, heads, first_position=7, src_stride=STRIDE, dst_stride=STRIDE)

    a, b = (hip_ctx.kv8_cache(1, heads, hd, 64) for _ in range(2))
    hip_ctx.kv8_store(a, out, out, 0, 0, rows)
    hip_ctx.kv8_store(b, far, far, 0, 0, rows, row_stride=STRIDE)
    got = [hip_ctx.empty(x.nbytes) for _ in range(4)]
    hip_ctx.kv8_load(a, got[0], got[1], 0, 0, rows)
    hip_ctx.kv8_load(b, got[2], got[3], 0, 0, rows)
    assert np.array_equal(got[0].read(), got[2].read()) and np.array_equal(got[1].read(), got[3].read())

    hip_ctx.kv8_store(a, dense, dense, 0, 0, rows)
    hip_ctx.kv8_attention(a, out, got[0], heads, 0, 0, rows)
    hip_ctx.kv8_attention(a, far, got[1], heads, 0, 0, rows, q_stride=STRIDE)
    assert np.array_equal(got[0].read(), got[1].read())

    tokens, u = hip_ctx.empty(4 * rows), hip_ctx.buffer(rng.random(rows))
    for o in (hip.SamplingOptions(temperature=0.7, top_k=20), hip.SamplingOptions(temperature=0.7, top_p=0.8)):
        hip_ctx.sample_rows(out, tokens, u, o, rows, heads * hd)
        want = tokens.read(np.uint32)
        hip_ctx.sample_rows(far, tokens, u, o, rows, heads * hd, row_stride=STRIDE)
        assert np.array_equal(tokens.read(np.uint32), want)
    far.free()


def test_more_rows_than_four_gib(hip_ctx):
    """130000 rows of 64 heads of 128, 4.3 GB, rotated in place: the last ones as by themselves."""
    rows, heads, hd, n = 131100, 64, 128, 9
    rng = np.random.default_rng(9)
    x = rng.normal(0, 1, (n, heads, hd)).astype(np.float32)
    b = hip_ctx.empty(4 * rows * heads * hd)
    at = 4 * (rows - n) * heads * hd
    assert at > 1 << 32
    b.write(x, at)
    d = hip.RopeDesc(hd, style=0, base=500000.0)
    hip_ctx.rope_rows(d, b, b, rows, heads)
    alone = hip_ctx.buffer(x)
    hip_ctx.rope_rows(d, alone, alone, n, heads, first_position=rows - n)
    got, want = hip_ctx.empty(x.nbytes), alone.read()
    hip_ctx.rope_rows(hip.RopeDesc(hd, 2, magnitude=1.0), b, got, n, heads, src_off=at, positions=hip_ctx.buffer(np.zeros(n, np.uint32)))
    assert np.array_equal(got.read(), want)
    b.free()
