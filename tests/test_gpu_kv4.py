"""The paged 4-bit cache's append and read-back against a plain form, byte for byte: a code is the nearest of eight
values and a scale a power of two, so nothing is tolerated."""
import numpy as np
import pytest

from tests import serving_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu


def same(got, cache, what=""):
    for name, g, w in zip(("k codes", "k scales", "v codes", "v scales"), (b.read(np.uint8) for b in got.buffers), cache.device()):
        assert np.array_equal(g, w), (what, name, np.flatnonzero(g != w)[:8], np.count_nonzero(g != w))


def values(rng, rows, heads, hd):
    x = rng.normal(0, 1, (rows, heads, hd)).astype(np.float32)
    x[:, :, ::31] *= 6
    x[rng.random((rows, heads, hd)) < 0.1] = 0
    return x


def append(ctx, got, cache, layer, batch, x, heads_desc=None, turned=None, **limits):
    """x [rows][3][heads][hd]: what lies beside, K and V.  `turned`: K as the oracle has it (in 64 bits)."""
    rows, _, heads, hd = x.shape
    w = 4 * heads * hd
    ctx.kv4_append(got, layer, batch.on(ctx, **limits), heads_desc, ctx.buffer(x), w, 2 * w, row_stride=3 * heads * hd)
    k = x[:, 1] if turned is None else turned.astype(np.float32)
    for r, s, p in batch.positions():
        cache.put(layer, *batch.place(s, p), k[r], x[r, 2])


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("rows,lengths", [([1], [1]), ([1], [64]), ([1], [65]), ([64], [64]), ([5], [70]), ([130], [130]), ([1, 1, 1], [9, 200, 64]),
                                          ([0, 3, 0, 0, 77, 1, 0], [10, 63, 0, 130, 77, 129, 64])])
def test_append(hip_ctx, hd, rows, lengths):
    print("kv4 append", hd, rows, lengths, flush=True)
    rng = np.random.default_rng(hd + sum(lengths))
    heads = 3
    batch = oracle.Batch(rows, lengths, rng)
    cache = oracle.Kv4(2, batch.pool, heads, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    x = np.stack([values(rng, batch.n, heads, hd) for _ in range(3)], axis=1)
    append(hip_ctx, got, cache, 1, batch, x)
    same(got, cache)  # the other layer, and the positions around, as they were
    k, v = hip_ctx.buffer(np.full((batch.n + 1, heads, hd), 5, np.float32)), hip_ctx.buffer(np.full((batch.n + 1, heads, hd), 5, np.float32))
    hip_ctx.kv4_load(got, 1, batch.on(hip_ctx, rows=batch.n + 1), k, v)
    for w, b in enumerate((k, v)):
        y = b.read().reshape(-1, heads, hd)
        assert np.all(y[-1] == 5)  # no sequence's row
        for r, s, p in batch.positions():
            assert np.array_equal(y[r], cache.rows(1, *batch.place(s, p))[w])


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("hd,rd", [(64, 64), (96, 48), (96, 2), (128, 128), (128, 90), (256, 256), (256, 100)])
def test_keys_normalised_and_turned_on_the_way(hip_ctx, hd, rd, style):
    print("kv4 turned", hd, rd, style, flush=True)
    rng = np.random.default_rng(hd * 3 + rd)
    heads, q_heads = 2, 6
    batch = oracle.Batch([3, 70, 1], [1003, 90, 1], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    x = values(rng, batch.n, q_heads + 2 * heads, hd)
    weights = [rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2)]
    d = hip.Heads(hip.RopeDesc(hd, rd, style, 500000.0), *map(hip_ctx.buffer, weights), eps=1e-5, weight_offset=0.25)
    src, out = hip_ctx.buffer(x), hip_ctx.buffer(np.full((batch.n + 1, q_heads * hd + 4), 7, np.float32))
    hip_ctx.kv4_append(got, 0, batch.on(hip_ctx), d, src, 4 * q_heads * hd, 4 * (q_heads + heads) * hd, (q_heads + 2 * heads) * hd,
                       q_heads, 0, out, 16, q_heads * hd + 4)
    at = np.array([p for _, _, p in batch.positions()])
    f = oracle.rope_frequencies(rd, 500000.0)
    k, _ = oracle.rope(oracle.norm(x[:, q_heads:q_heads + heads], weights[1], 1e-5, 0.25), at, f, rd, style)
    q, pair = oracle.rope(oracle.norm(x[:, :q_heads], weights[0], 1e-5, 0.25), at, f, rd, style)
    for r, s, p in batch.positions():
        cache.put(0, *batch.place(s, p), k[r].astype(np.float32), x[r, q_heads + heads:])
    same(got, cache)
    y = out.read().reshape(batch.n + 1, -1)
    assert np.all(y[-1, 4:] == 7) and np.all(y[:-1].reshape(-1)[:4] == 7) and np.all(y[1:-1, :4] == 7)
    err = np.abs(y[:-1, 4:].reshape(q.shape) - q)
    assert np.all(err <= 8 * 2.0 ** -24 * np.maximum(pair, np.abs(q)))  # as for norm_rope_rows
    # the queries in place give the same bits, and leave what lies beside them
    hip_ctx.kv4_append(got, 0, batch.on(hip_ctx), d, src, 4 * q_heads * hd, 4 * (q_heads + heads) * hd, (q_heads + 2 * heads) * hd,
                       q_heads, 0, src, 0, (q_heads + 2 * heads) * hd)
    z = src.read().reshape(x.shape)
    assert np.array_equal(z[:, :q_heads].reshape(batch.n, -1), y[:-1, 4:]) and np.array_equal(z[:, q_heads:], x[:, q_heads:])
    same(got, cache)


@pytest.mark.parametrize("shift", [0, 1, 2])
def test_rows_off_the_vector_loads(hip_ctx, shift):
    rng = np.random.default_rng(shift)
    heads, hd = 2, 64
    batch = oracle.Batch([4, 2], [70, 2], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    width = 2 * heads * hd + 1 + shift
    x = rng.normal(0, 1, (batch.n, width)).astype(np.float32)
    held = np.concatenate([np.zeros(shift, np.float32), x.reshape(-1)])
    hip_ctx.kv4_append(got, 0, batch.on(hip_ctx), None, hip_ctx.buffer(held), 4 * shift, 4 * (shift + heads * hd), width)
    for r, s, p in batch.positions():
        k, v = (x[r, i * heads * hd:(i + 1) * heads * hd].reshape(heads, hd) for i in range(2))
        cache.put(0, *batch.place(s, p), k, v)
    same(got, cache)


def test_one_row_at_a_time_and_taken_back(hip_ctx):
    """A position depends on no other: rows stored one by one, and stored again, are those stored at once."""
    rng = np.random.default_rng(9)
    heads, hd, n = 2, 128, 70
    batch = oracle.Batch([n], [n], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    x = np.stack([values(rng, n, heads, hd) for _ in range(3)], axis=1)
    for t in range(n):
        one = oracle.Batch([1], [t + 1], rng)
        one.table = batch.table
        append(hip_ctx, got, cache, 0, one, 1e6 * values(rng, 3, heads, hd)[None])
        append(hip_ctx, got, cache, 0, one, x[t:t + 1])
        same(got, cache, t)


@pytest.mark.parametrize("size", [1e-45, 1e-38, 3e-30, 1e-28, 1e-20, 1.0, 1e20, 1e28, 4e28, 3e38])
def test_sizes(hip_ctx, size):
    """From the smallest denormal to the largest value: past both ends of the scales among them."""
    rng = np.random.default_rng(3)
    heads, hd = 1, 64
    batch = oracle.Batch([40], [40], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd)
    got = oracle.upload(hip_ctx, cache)
    x = (np.clip(rng.normal(0, 0.4, (40, 3, heads, hd)), -1, 1) * size).astype(np.float32)
    x[5:9, 1:] = 0
    append(hip_ctx, got, cache, 0, batch, x)
    same(got, cache)


def test_ties_go_to_the_even_code(hip_ctx):
    """Values half way between two of the eight, and one step of binary32 to either side; the scales' own border."""
    rng = np.random.default_rng(3)
    heads, hd = 1, 256
    half = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7], np.float32)
    near = np.concatenate([half, np.nextafter(half, np.float32(0)), np.nextafter(half, np.float32(9))[:-1], [0.0]]).astype(np.float32)
    row = np.concatenate([np.tile(np.concatenate([near, [7.0, 6.5, 3.0, 1.0, 0.1]]).astype(np.float32), 1)[:32]] * 8)
    x = np.zeros((64, 3, heads, hd), np.float32)
    for r in range(64):
        x[r, 1, 0] = np.roll(row, r) * np.float32(2.0) ** (r - 30)
        x[r, 2, 0] = -np.roll(row, 3 * r) * np.float32(2.0) ** (20 - r)
    for i, v in enumerate((7.0, np.nextafter(np.float32(7), np.float32(8)), np.nextafter(np.float32(7), np.float32(0)))):
        x[i, 1:, 0, :32] = v  # the largest that 2^0 serves, and its neighbours
    batch = oracle.Batch([64], [64], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd)
    got = oracle.upload(hip_ctx, cache)
    append(hip_ctx, got, cache, 0, batch, x)
    same(got, cache)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_value_that_is_not_finite_marks_its_position(hip_ctx, bad):
    rng = np.random.default_rng(8)
    heads, hd = 2, 64
    batch = oracle.Batch([70], [70], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    x = np.stack([values(rng, 70, heads, hd) for _ in range(3)], axis=1)
    x[40, 1, 1, 5] = bad
    x[66, 2, 0, 63] = bad
    append(hip_ctx, got, cache, 0, batch, x)
    same(got, cache)
    out = [hip_ctx.empty(4 * 70 * heads * hd) for _ in range(2)]
    hip_ctx.kv4_load(got, 0, batch.on(hip_ctx), *out)
    for o in out:
        nan = np.isnan(o.read().reshape(70, heads, hd))
        assert nan[40, 1].all() and nan[66, 0].all() and nan.sum() == 2 * hd
    x[[40, 66]] = 1.0  # stored again, the mark is gone
    append(hip_ctx, got, cache, 0, batch, x)
    same(got, cache)


def test_what_is_passed_over(hip_ctx):
    """Pages that the pool doesn't have, rows and positions past the limits, rows ahead of position 0, tables that
    don't ascend: nothing of them is stored, and no query row of theirs ahead of position 0 is touched."""
    rng = np.random.default_rng(4)
    heads, hd = 2, 64
    batch = oracle.Batch([4, 5, 3, 2], [66, 3, 300, 130], rng)
    cache = oracle.Kv4(1, batch.pool, heads, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    batch.table[0, 1], batch.table[3, 2] = batch.pool, 0xFFFFFFFF  # positions 64 .. and 128 ..
    x = np.stack([values(rng, batch.n, heads, hd) for _ in range(3)], axis=1)
    w = heads * hd
    q = hip_ctx.buffer(np.full((batch.n, w), 7, np.float32))
    hip_ctx.kv4_append(got, 0, batch.on(hip_ctx, max_rows=4, max_length=299), None, hip_ctx.buffer(x), 4 * w, 8 * w, 3 * w, heads, 0, q)
    k, v = (hip_ctx.buffer(np.full((batch.n, w), 7, np.float32)) for _ in range(2))
    hip_ctx.kv4_load(got, 0, batch.on(hip_ctx, max_rows=4, max_length=299), k, v)
    rows = [k.read().reshape(x[:, 0].shape), v.read().reshape(x[:, 0].shape)]
    turned = q.read().reshape(x[:, 0].shape)
    for r, s, p in batch.positions():
        i = r - int(batch.starts[s])
        stored = i < 4 and 0 <= p < 299 and not (s == 0 and p >= 64) and not (s == 3 and p >= 128)
        if stored:
            cache.put(0, *batch.place(s, p), x[r, 1], x[r, 2])
        for y, want in zip(rows, cache.rows(0, *batch.place(s, p)) if stored else (7, 7)):
            assert np.all(y[r] == want), (r, s, p)
        assert np.array_equal(turned[r], x[r, 0] if i < 4 and p >= 0 else np.full_like(x[r, 0], 7))
    same(got, cache)
    batch.starts = np.array([3, 1, 0xFFFFFFFF, 2, 9], np.uint32)  # none but sequence 1 has rows, four at most
    batch.lengths = [66, 13, 300, 130]
    hip_ctx.kv4_append(got, 0, batch.on(hip_ctx, rows=14, max_rows=4), None, hip_ctx.buffer(x), 4 * w, 8 * w, 3 * w)
    kept = [b.read(np.uint8) for b in got.buffers]
    again = oracle.upload(hip_ctx, cache)
    total = sum(np.count_nonzero(a != b.read(np.uint8)) for a, b in zip(kept, again.buffers))
    assert total <= 4 * heads * (hd + hd // 16)  # four positions' bytes at most


def test_far_pages(hip_ctx):
    """Pages past 2^32 bytes of codes."""
    rng = np.random.default_rng(6)
    heads, hd, pages = 8, 256, 70000  # 70000 * 8 * 8192 bytes of codes: 4.6 GB
    got = hip_ctx.kv4_cache(1, heads, hd, pages)
    batch = oracle.Batch([2, 3], [65, 70], rng)
    batch.table[:] = np.array([[69999, 65536, 0xFFFFFFFF], [3, 68000, 0xFFFFFFFF]], np.uint32)[:, :batch.table.shape[1]]
    x = np.stack([values(rng, batch.n, heads, hd) for _ in range(3)], axis=1)
    w = heads * hd
    hip_ctx.kv4_append(got, 0, batch.on(hip_ctx), None, hip_ctx.buffer(x), 4 * w, 8 * w, 3 * w)
    k, v = hip_ctx.empty(4 * batch.n * w), hip_ctx.empty(4 * batch.n * w)
    hip_ctx.kv4_load(got, 0, batch.on(hip_ctx), k, v)
    for i, b in ((1, k), (2, v)):
        assert np.array_equal(b.read().reshape(batch.n, heads, hd), oracle.of_four_bits(*oracle.in_four_bits(x[:, i])).astype(np.float32))
    for b in got.buffers:
        b.free()
