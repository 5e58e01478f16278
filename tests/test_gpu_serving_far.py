"""The operators that serve several sequences where offsets pass 32 bits and tables are long: pages and layers past
4 GiB of codes, rows a GiB apart, thousands of sequences."""
import numpy as np
import pytest

from tests import serving_oracle as oracle
from tests.test_gpu_kv4 import same
from tests.test_gpu_longctx_far import STRIDE, spread
from zhip import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [[1, 1], [5, 1], [150, 2]])
def test_pages_and_layers_past_four_gib(hip_ctx, rows):
    """The last of three layers of 24000 pages of 8 heads of 256 (4.7 GB of codes ahead of its last pages)."""
    print("far pages", rows, flush=True)
    rng = np.random.default_rng(sum(rows))
    heads, kvh, hd, pages, layer = 16, 8, 256, 24000, 2
    got = hip_ctx.kv4_cache(3, kvh, hd, pages)
    assert got.buffers[0].nbytes > 4 << 30
    batch = oracle.Batch(rows, [n + 60 for n in rows], rng)
    near = batch.table.copy()
    used = near != 0xFFFFFFFF
    far = np.array([23999, 23998, 20000, 5, 23001, 22000, 23997], np.uint32)
    batch.table[used] = far[near[used]]
    cache = oracle.Kv4(1, batch.pool, kvh, hd)
    full = oracle.Batch.__new__(oracle.Batch)  # every position is a row once
    full.rows = full.lengths = batch.lengths
    full.starts = np.concatenate([[0], np.cumsum(batch.lengths)]).astype(np.uint32)
    full.n, full.table = int(full.starts[-1]), batch.table
    x = rng.normal(0, 1, (2, full.n, kvh, hd)).astype(np.float32)
    src, w = hip_ctx.buffer(x), 4 * full.n * kvh * hd
    hip_ctx.kv4_append(got, layer, full.on(hip_ctx), None, src, 0, w)
    k, v = hip_ctx.empty(w), hip_ctx.empty(w)
    hip_ctx.kv4_load(got, layer, full.on(hip_ctx), k, v)
    for i, b in enumerate((k, v)):
        assert np.array_equal(b.read().reshape(x[i].shape), oracle.of_four_bits(*oracle.in_four_bits(x[i])).astype(np.float32))
    for r, s, p in full.positions():
        cache.put(0, int(near[s, p // oracle.PAGE]), p % oracle.PAGE, x[0, r], x[1, r])
    q = rng.normal(0, 1, (batch.n, heads, hd)).astype(np.float32)
    out = hip_ctx.empty(q.nbytes)
    hip_ctx.kv4_attention(got, layer, batch.on(hip_ctx), hip_ctx.buffer(q), out, heads)
    batch.table = near
    want, bound = oracle.attention(cache, 0, batch, q, hd ** -0.5)
    assert np.all(np.abs(out.read().reshape(want.shape) - want) <= bound)
    for b in got.buffers:
        b.free()


def test_rows_a_gib_apart(hip_ctx):
    rng = np.random.default_rng(5)
    heads, kvh, hd = 4, 2, 64
    batch = oracle.Batch([4, 2], [70, 65], rng)
    width = (heads + 2 * kvh) * hd
    x = rng.normal(0, 1, (batch.n, width)).astype(np.float32)
    dense, far = hip_ctx.buffer(x), spread(hip_ctx, x)
    desc = hip.Heads(hip.RopeDesc(hd, hd, 1, 10000.0), hip_ctx.buffer(rng.normal(1, 0.2, hd).astype(np.float32)))
    a, b = hip_ctx.empty(x.nbytes), hip_ctx.empty(x.nbytes)
    on = batch.on(hip_ctx)
    hip_ctx.norm_rope_rows(desc, dense, a, batch.n, heads, kvh, first_position=9, src_stride=width)
    hip_ctx.norm_rope_rows(desc, far, b, batch.n, heads, kvh, first_position=9, src_stride=STRIDE)
    assert np.array_equal(a.read()[:batch.n * (heads + kvh) * hd], b.read()[:batch.n * (heads + kvh) * hd])
    empty = oracle.Kv4(1, batch.pool, kvh, hd, rng)
    one, two = (oracle.upload(hip_ctx, empty) for _ in range(2))
    k, v = 4 * heads * hd, 4 * (heads + kvh) * hd
    hip_ctx.kv4_append(one, 0, on, desc, dense, k, v, width, heads, 0, dense, 0, width)
    hip_ctx.kv4_append(two, 0, on, desc, far, k, v, STRIDE, heads, 0, far, 0, STRIDE)
    for g, h in zip(one.buffers, two.buffers):
        assert np.array_equal(g.read(np.uint8), h.read(np.uint8))
    hip_ctx.kv4_attention(one, 0, on, dense, a, heads, q_stride=width)
    hip_ctx.kv4_attention(two, 0, on, far, b, heads, q_stride=STRIDE)
    assert np.array_equal(a.read()[:batch.n * heads * hd], b.read()[:batch.n * heads * hd])
    logits = rng.normal(0, 2, (batch.n, 500)).astype(np.float32)
    far.free()
    far, tokens = spread(hip_ctx, logits), hip_ctx.buffer(rng.integers(0, 500, batch.n).astype(np.uint32))
    outs = [[hip_ctx.empty(4 * batch.n), hip_ctx.empty(4 * batch.n), hip_ctx.empty(4 * 3 * batch.n), hip_ctx.empty(4 * 3 * batch.n)] for _ in range(2)]
    for (lp, en, ti, tl), src, stride in zip(outs, (hip_ctx.buffer(logits), far), (0, STRIDE)):
        hip_ctx.token_logprobs(src, tokens, lp, batch.n, 500, en, 3, ti, tl, stride)
    for g, h in zip(*outs):
        assert np.array_equal(g.read(np.uint32), h.read(np.uint32))
    far.free()


@pytest.mark.parametrize("sequences", [66, 1023, 1025, 4097, 9000])
def test_thousands_of_sequences(hip_ctx, sequences):
    """Lengths and rows of all kinds, some none, one with a prompt; what they append and attend to."""
    print("sequences", sequences, flush=True)
    rng = np.random.default_rng(sequences)
    heads, kvh, hd = 2, 1, 64
    rows = rng.choice([0, 1, 1, 2, 5], sequences)
    lengths = np.maximum(rows, rng.choice([1, 3, 40, 64, 65], sequences))
    rows[sequences // 3], lengths[sequences // 3] = 90, 200
    rows[sequences // 2], lengths[sequences // 2] = 40, 64
    rows[-1], lengths[-1] = 1, 2500
    batch = oracle.Batch(rows, lengths, rng)
    cache = oracle.Kv4(1, batch.pool, kvh, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    x = rng.normal(0, 1, (2, batch.n, kvh, hd)).astype(np.float32)
    on = batch.on(hip_ctx)
    hip_ctx.kv4_append(got, 0, on, None, hip_ctx.buffer(x), 0, 4 * batch.n * kvh * hd)
    page, slot = (np.array(i) for i in zip(*(batch.place(s, p) for _, s, p in batch.positions())))
    for w in range(2):
        cache.codes[w][0, page, slot], cache.scales[w][0, page, slot] = oracle.in_four_bits(x[w])
    same(got, cache)
    q = rng.normal(0, 1, (batch.n, heads, hd)).astype(np.float32)
    out = hip_ctx.buffer(np.full((batch.n + 1, heads, hd), 7, np.float32))
    hip_ctx.kv4_attention(got, 0, batch.on(hip_ctx, rows=batch.n + 1), hip_ctx.buffer(np.concatenate([q, q[:1]])), out, heads)
    want, bound = oracle.attention(cache, 0, batch, q, hd ** -0.5)
    y = out.read().reshape(-1, heads, hd)
    assert np.all(y[-1] == 7) and np.all(np.abs(y[:-1] - want) <= bound)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,kvh,rows", [(2, 2, 1), (4, 2, 2), (12, 2, 2), (5, 1, 3), (8, 2, 8), (6, 1, 9), (3, 1, 60)])
@pytest.mark.parametrize("sequences", [64, 65, 100])
def test_every_width_of_a_batch(hip_ctx, sequences, heads, kvh, rows, hd):
    """Up to 1, 4, 16, 32 columns and more, some sequences long enough to be split, with the table of many sequences and
    without; the widths that the batch names, and no word of them."""
    print("width", sequences, heads, kvh, rows, hd, flush=True)
    rng = np.random.default_rng(sequences + rows)
    n = rng.integers(0, rows + 1, sequences)
    n[7] = rows
    lengths = np.maximum(n, rng.integers(1, 70, sequences))
    lengths[7], lengths[-3] = 2100, 700
    batch = oracle.Batch(n, lengths, rng)
    cache = oracle.Kv4(1, batch.pool, kvh, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    q = rng.normal(0, 0.7, (batch.n, heads, hd)).astype(np.float32)
    src, want, bound = hip_ctx.buffer(q), *oracle.attention(cache, 0, batch, q, hd ** -0.5, 1500)
    for limits in (dict(max_rows=rows, max_length=2100), dict()):
        out = hip_ctx.buffer(np.full(q.shape, 7, np.float32))
        hip_ctx.kv4_attention(got, 0, batch.on(hip_ctx, **limits), src, out, heads, 1500)
        off = np.abs(out.read().reshape(q.shape) - want)
        assert np.all(off <= bound), (limits, np.argwhere(~(off <= bound))[:4])


def test_thousands_of_long_sequences_share_pages(hip_ctx):
    """3000 sequences of a row over the same 2000 positions: splits and workspace at their most; all rows alike."""
    rng = np.random.default_rng(4)
    heads, kvh, hd, sequences, length = 4, 2, 128, 3000, 2000
    one = oracle.Batch([1], [length], rng)
    cache = oracle.Kv4(1, one.pool, kvh, hd, rng)
    q = rng.normal(0, 1, (1, heads, hd)).astype(np.float32)
    table = np.repeat(one.table, sequences, axis=0)
    on = hip.Batch(hip_ctx.buffer(table), hip_ctx.buffer(np.arange(sequences + 1, dtype=np.uint32)),
                   hip_ctx.buffer(np.full(sequences, length, np.uint32)), sequences, table.shape[1], sequences, 1)
    out = hip_ctx.empty(4 * sequences * q.size)
    hip_ctx.kv4_attention(oracle.upload(hip_ctx, cache), 0, on, hip_ctx.buffer(np.repeat(q, sequences, axis=0)), out, heads)
    want, bound = oracle.attention(cache, 0, one, q, hd ** -0.5)
    assert np.all(np.abs(out.read().reshape(sequences, heads, hd) - want) <= bound)


def test_tables_of_many_sequences_that_hold_nonsense(hip_ctx):
    """Nothing outside the buffers is touched, and rows that belong to no sequence keep their output."""
    rng = np.random.default_rng(13)
    heads, hd, rows, sequences = 4, 64, 50, 300
    cache = oracle.Kv4(1, 9, 2, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    q = hip_ctx.buffer(rng.normal(0, 1, (rows, heads * hd)).astype(np.float32))
    words = lambda: rng.integers(0, 1 << 32, sequences + 1, dtype=np.uint64).astype(np.uint32)
    for starts in (words(), words() % (rows + 5), np.sort(words() % rows), np.full(sequences + 1, 0xFFFFFFFF, np.uint32),
                   np.tile(np.array([0, 0xFFFFFFFF], np.uint32), sequences)[:sequences + 1]):
        for lengths in (words()[1:], np.full(sequences, 0xFFFFFFFF, np.uint32), words()[1:] % 300):
            table = rng.integers(0, 1 << 32, (sequences, 3), dtype=np.uint64).astype(np.uint32)
            table[::2] %= 12
            b = hip.Batch(hip_ctx.buffer(table), hip_ctx.buffer(starts), hip_ctx.buffer(lengths), sequences, 3, rows)
            out = hip_ctx.buffer(np.full((rows, heads * hd), 7, np.float32))
            hip_ctx.kv4_attention(got, 0, b, q, out, heads)
            y = out.read().reshape(rows, -1)
            if starts.min() >= rows:
                assert np.all(y == 7)
    assert all(np.array_equal(b.read(np.uint8), w) for b, w in zip(got.buffers, cache.device()))
