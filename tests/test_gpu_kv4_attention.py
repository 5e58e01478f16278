"""ziggy_hip_kv4_attention_f32 against a 64-bit form (the tolerance: serving_oracle.attention)."""
import numpy as np
import pytest

from tests import serving_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu


def attend(ctx, rows, lengths, heads, kvh, hd, window=0, scale=None, layers=1, layer=0, stride=0, off=0, rng=None, cache=None, q=None,
           batch=None, hidden=(), **limits):
    print("kv4 attention", rows[:8], lengths[:8], heads, kvh, hd, window, flush=True)
    rng = rng or np.random.default_rng(sum(lengths) + heads + hd)
    batch = batch or oracle.Batch(rows, lengths, rng)
    cache = cache or oracle.Kv4(layers, batch.pool, kvh, hd, rng)
    scale = hd ** -0.5 if scale is None else scale
    width = heads * hd
    if q is None:
        q = rng.normal(0, 0.7, (batch.n, heads, hd)).astype(np.float32)
    held = np.full((batch.n, stride or width), 3, np.float32)
    held[:, :width] = q.reshape(batch.n, -1)
    held = np.concatenate([np.zeros(off, np.float32), held.reshape(-1)])
    out = ctx.buffer(np.full((batch.n + 1, width), 7, np.float32))
    src = ctx.buffer(np.concatenate([held, np.zeros(stride or width, np.float32)]))
    ctx.kv4_attention(oracle.upload(ctx, cache), layer, batch.on(ctx, rows=batch.n + 1, **limits), src, out, heads, window, scale, q_off=4 * off,
                      q_stride=stride)
    got = out.read().reshape(batch.n + 1, heads, hd)
    assert np.all(got[-1] == 7)  # a row behind the last sequence
    want, bound = oracle.attention(cache, layer, batch, q, scale, window, hidden)
    return got[:-1], want, bound


def check(*args, **more):
    got, want, bound = attend(*args, **more)
    off = np.abs(got - want)
    assert np.all(off <= bound), ((off / np.maximum(bound, 1e-300)).max(), np.argwhere(~(off <= bound))[:4])
    return got


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 200, 1000])
def test_one_row(hip_ctx, hd, length):
    check(hip_ctx, [1], [length], 4, 2, hd)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (3, 3), (5, 1), (7, 1), (16, 2), (17, 1), (64, 1), (12, 4), (40, 8)])
def test_groups(hip_ctx, hd, heads, kvh):
    check(hip_ctx, [1, 1], [150, 37], heads, kvh, hd)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [2, 5, 16, 17, 33, 64, 65, 130, 259])
def test_many_rows(hip_ctx, hd, rows):
    check(hip_ctx, [rows], [rows], 3, 1, hd)
    check(hip_ctx, [rows], [rows + 75], 4, 2, hd)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_batches(hip_ctx, hd):
    check(hip_ctx, [1] * 9, [5, 64, 65, 700, 1, 128, 31, 2, 1500], 8, 2, hd)
    check(hip_ctx, [0, 1, 0, 4, 70, 0, 1, 2], [90, 300, 0, 4, 71, 64, 1, 129], 6, 3, hd)
    check(hip_ctx, [200, 1, 1, 33], [300, 900, 5, 33], 4, 1, hd)


@pytest.mark.parametrize("sequences", [63, 64, 65, 130, 200])
def test_many_sequences(hip_ctx, sequences):
    rng = np.random.default_rng(sequences)
    check(hip_ctx, list(rng.integers(0, 3, sequences - 1)) + [2], list(rng.integers(2, 90, sequences)), 2, 1, 64)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 5000, 0xFFFFFFFF])
def test_windows(hip_ctx, hd, window):
    check(hip_ctx, [1, 40, 3], [333, 190, 3], 4, 2, hd, window=window)
    check(hip_ctx, [150], [400], 4, 2, hd, window=window)


def test_layers_strides_and_offsets(hip_ctx):
    check(hip_ctx, [3, 1], [100, 70], 4, 2, 128, layers=3, layer=2)
    for stride, off in ((4 * 64 + 4, 4), (4 * 64 + 3, 0), (4 * 64 + 1, 5), (0, 1)):
        check(hip_ctx, [3, 70], [100, 170], 4, 2, 64, stride=stride, off=off)


@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-30, 0.7])
def test_scales(hip_ctx, scale):
    check(hip_ctx, [2, 1, 50], [90, 400, 81], 4, 2, 64, scale=scale)


def test_long_contexts(hip_ctx):
    check(hip_ctx, [1], [20000], 4, 1, 128)
    check(hip_ctx, [3, 1], [9000, 12345], 2, 1, 64)
    check(hip_ctx, [1, 1, 1], [30000, 40, 3000], 2, 2, 64)


def test_limits_that_the_batch_names(hip_ctx):
    check(hip_ctx, [1, 3, 2], [500, 90, 700], 4, 2, 64, max_rows=3, max_length=700)
    check(hip_ctx, [1, 1], [500, 90], 4, 2, 64, max_rows=1)


def test_a_result_depends_on_its_inputs_alone(hip_ctx):
    rng = np.random.default_rng(2)
    batch = oracle.Batch([1, 5, 90], [3000, 700, 900], rng)
    cache, q = oracle.Kv4(1, batch.pool, 2, 128, rng), rng.normal(0, 1, (96, 8, 128)).astype(np.float32)
    first = attend(hip_ctx, [], [], 8, 2, 128, batch=batch, cache=cache, q=q, rng=rng)[0]
    for _ in range(3):
        check(hip_ctx, [70, 1], [70, 5000], 4, 2, 64)  # something else through the same workspace
        assert np.array_equal(first, attend(hip_ctx, [], [], 8, 2, 128, batch=batch, cache=cache, q=q, rng=rng)[0])


def test_scales_far_apart(hip_ctx):
    """Values of 2^90 that no row sees, or that have no weight, beside values of 2^-90: nothing of them gets in, whatever
    they are, and what is seen keeps its bits.  Sums past binary32's largest mean come out as the mean."""
    rng = np.random.default_rng(5)
    batch = oracle.Batch([40], [200], rng)
    for hd in (64, 128):
        cache = oracle.Kv4(1, batch.pool, 1, hd, rng)
        big = [batch.place(0, t) for t in range(165, 200)]
        for page, slot in big:
            cache.scales[1][0, page, slot] = 219  # rows before 165 don't see them
        q = rng.normal(0, 0.5, (40, 2, hd)).astype(np.float32)
        got, want, _ = attend(hip_ctx, [], [], 2, 1, hd, batch=batch, cache=cache, q=q, rng=rng)
        small = slice(0, 5)  # positions 160 .. 164
        assert np.all(np.abs(got[small] - want[small]) <= 1e-4 * np.abs(want[small]).max())
        assert np.all(np.abs(got[5:] - want[5:]) <= 1e-4 * np.abs(want[5:]).max(axis=(1, 2), keepdims=True))
        for page, slot in [batch.place(0, t) for t in range(200)]:
            cache.scales[1][0, page, slot] = 219
            cache.codes[1][0, page, slot] = 7  # all 6 2^92
        got, want, _ = attend(hip_ctx, [], [], 2, 1, hd, batch=batch, cache=cache, q=q, rng=rng)
        assert np.all(np.abs(got / (6 * 2.0 ** 92) - 1) < 1e-5)
        # weightless: one key so near the queries that the others' weights are 0 in binary32
        for t in range(200):
            page, slot = batch.place(0, t)
            cache.scales[1][0, page, slot] = 37 if t == 7 else 219
            cache.scales[0][0, page, slot] = 127
            cache.codes[0][0, page, slot] = 7 if t == 7 else 0
        got, want, _ = attend(hip_ctx, [], [], 2, 1, hd, batch=batch, cache=cache, q=np.full_like(q, 3), rng=rng, scale=1.0)
        assert np.all(np.abs(got - want) <= 1e-5 * np.abs(want).max()) and np.abs(want).max() < 1e-20


def test_small_weights_beside_a_dominant_key(hip_ctx):
    """A weight of 2^-60 on a value of 2^60 counts as much as the dominant key's own."""
    rng = np.random.default_rng(6)
    hd = 64
    batch = oracle.Batch([1], [300], rng)
    cache = oracle.Kv4(1, batch.pool, 1, hd, rng)
    for t in range(300):
        page, slot = batch.place(0, t)
        cache.scales[0][0, page, slot] = 127
        cache.codes[0][0, page, slot] = 0
        cache.codes[0][0, page, slot, 0] = 2 if t == 11 else 0  # a score of 60 in powers of two
        cache.scales[1][0, page, slot] = 187 if t in (200, 250) else 127
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = 60 * np.log(2)
    check(hip_ctx, [], [], 1, 1, hd, batch=batch, cache=cache, q=q, rng=rng, scale=1.0)
    got, want, _ = attend(hip_ctx, [], [], 1, 1, hd, batch=batch, cache=cache, q=q, rng=rng, scale=1.0)
    # the score's 2^-24 of 60 and the exponential's 2^-21 on each of the two kinds of terms, of at most 6 each
    assert np.all(np.abs(got - want) <= (2 * 60 * 2.0 ** -23 + 2.0 ** -20) * 18)


@pytest.mark.parametrize("rows,length", [(1, 2), (1, 70), (3, 130), (1, 5000), (9, 200), (80, 100)])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_every_bit_of_a_weight_counts(hip_ctx, hd, rows, length):
    """One value of 1 among zeros, and one key that sees the query's first value: the output is w / (w + n - 1),
    w = exp(q k scale).  Tolerance: the score is one exact product, rounded with the scale to 2^-22 of itself; the
    exponential and its pieces 2^-21; the sums of n - 1 ones are exact, the others' 2^-22: a piece lost, or taken
    twice, would be 2^-16 or 2^-8."""
    for group in (1, 4, 16):
        rng = np.random.default_rng(hd + rows + group)
        batch = oracle.Batch([rows], [length], rng)
        cache = oracle.Kv4(1, batch.pool, 1, hd)
        for t in range(length):
            page, slot = batch.place(0, t)
            cache.scales[0][0, page, slot] = cache.scales[1][0, page, slot] = 127
            cache.codes[0][0, page, slot, 0] = 2 if t == 1 else 0  # 1 and 0
            cache.codes[1][0, page, slot] = 2 if t == 1 else 0
        q = np.zeros((rows, group, hd), np.float32)
        q[..., 0] = rng.uniform(-6, 6, (rows, group))
        got, _, _ = attend(hip_ctx, [], [], group, 1, hd, batch=batch, cache=cache, q=q, rng=rng, scale=0.7)
        score = q[..., :1].astype(np.float64) * float(np.float32(0.7))
        others = np.arange(length - rows, length)[:, None, None]  # positions in sight but the one
        want = np.where(others >= 1, np.exp(score) / (np.exp(score) + others), 0.0)
        off = np.abs(got - want)
        assert np.all(off <= (np.abs(score) * 2.0 ** -21 + 2.0 ** -20) * want), (off / np.maximum(want, 1e-300)).max()


@pytest.mark.parametrize("rows,lengths", [([1], [300]), ([1] * 5, [64, 900, 20, 300, 3000]), ([4], [500]), ([40], [200]), ([200], [300])])
def test_errors_over_all_outputs(hip_ctx, rows, lengths):
    """The worst case of the bound above is far from what happens: roundings go both ways.  A score's 3 hd products add up
    with as many roundings, each of at most 2^-24 of the sum so far (2^-24 / sqrt(3) of it in the mean), which in the
    mean over scores is at most R = sqrt(sum (q k scale)^2): sqrt(hd) 2^-24 R together.  The scale's roundings and the
    maximum's add 2^-22 R.  That is a weight's error relative to itself; the exponential's is 2^-22, the sums' and the
    outputs' less.  An output's error is the sum of w error (v - output), in the mean of squares as large beside the
    output, a sum of w v of values of either sign, as the weights' errors are beside 1; 1.5 times that for what the mean
    over few rows leaves open.  (Products of 128: 6 10^-6 here; a weight's third piece taken twice is 9 10^-6.)"""
    for heads, kvh, hd in ((4, 4, 128), (8, 2, 128), (16, 1, 64), (2, 1, 256)):
        rng = np.random.default_rng(heads + hd)
        batch = oracle.Batch(rows, lengths, rng)
        cache = oracle.Kv4(1, batch.pool, kvh, hd, rng)
        q = rng.normal(0, 0.7, (batch.n, heads, hd)).astype(np.float32)
        got, want, _ = attend(hip_ctx, rows, lengths, heads, kvh, hd, batch=batch, cache=cache, q=q, rng=rng)
        squares = []
        for r, s, p in batch.positions():
            at = np.arange(p + 1)
            k, _ = cache.rows(0, batch.table[s, at // 64].astype(int), at % 64)
            squares.append((np.repeat(k ** 2, heads // kvh, axis=1) * q[r].astype(np.float64) ** 2).sum(axis=2).mean() / hd)
        size = np.sqrt(np.mean(squares))
        assert np.linalg.norm(got - want) <= 1.5 * ((np.sqrt(hd) + 4) * 2.0 ** -24 * size + 2.0 ** -21) * np.linalg.norm(want), (heads, kvh, hd, size)


def test_marked_positions(hip_ctx):
    """A position with a NaN: rows that see it are NaN throughout (its kv head's), the others as without it."""
    rng = np.random.default_rng(7)
    batch = oracle.Batch([60, 1], [100, 70], rng)
    for hd in (64, 256):
        cache = oracle.Kv4(1, batch.pool, 2, hd, rng)
        q = rng.normal(0, 0.7, (61, 4, hd)).astype(np.float32)
        want, bound = oracle.attention(cache, 0, batch, q, hd ** -0.5, 0)
        page, slot = batch.place(0, 75)
        k = rng.normal(0, 1, (2, hd)).astype(np.float32)
        k[0, 3] = np.nan
        kept = [c[0, page, slot, 1].copy() for c in (*cache.codes, *cache.scales)]
        cache.put(0, page, slot, k, np.abs(k))
        for c, x in zip((*cache.codes, *cache.scales), kept):  # head 1 as before
            c[0, page, slot, 1] = x
        got = attend(hip_ctx, [], [], 4, 2, hd, batch=batch, cache=cache, q=q, rng=rng)[0]
        sees = np.zeros((61, 4), bool)
        sees[35:60, :2] = True  # positions 75 .. 99
        assert np.isnan(got[sees]).all()
        assert np.all(np.abs(got - want)[~sees] <= bound[~sees])


def test_bytes_that_were_never_stored(hip_ctx):
    """Whatever lies behind the last position, before the window, on the sequence's own pages or on others."""
    rng = np.random.default_rng(8)
    for rows, lengths, window in (([1, 1], [37, 100], 0), ([1], [200], 50), ([50, 3], [50, 70], 0), ([70], [150], 33), ([1], [4000], 100)):
        batch = oracle.Batch(rows, lengths, rng)
        for hd in (64, 96):
            cache = oracle.Kv4(1, batch.pool, 2, hd, rng)
            seen = np.zeros((batch.pool, 64), bool)
            for _, s, p in batch.positions():
                for t in range(max(0, p + 1 - window) if window else 0, p + 1):
                    seen[batch.place(s, t)] = True
            for w in range(2):
                cache.codes[w][0][~seen] = 15
                cache.scales[w][0][~seen] = 255
            check(hip_ctx, [], [], 4, 2, hd, batch=batch, cache=cache, window=window, rng=rng)


def test_rows_that_nothing_is_left_for(hip_ctx):
    """Rows ahead of position 0, and rows all of whose pages the pool doesn't have: zeros; missing pages inside a
    context are passed over; rows past max_rows are left as they were."""
    rng = np.random.default_rng(9)
    heads, hd = 4, 64
    batch = oracle.Batch([5, 2, 1, 90], [3, 100, 64, 300], rng)
    cache = oracle.Kv4(1, batch.pool, 2, hd, rng)
    table = batch.table.copy()
    hidden = {(1, 0), (2, 0), (3, 1), (3, 4)}
    for s, p in hidden:
        table[s, p] = batch.pool + 5 if s else 0xFFFFFFFF
    kept, batch.table = batch.table, table
    src = rng.normal(0, 1, (batch.n, heads, hd)).astype(np.float32)
    out = hip_ctx.buffer(np.full((batch.n, heads * hd), 7, np.float32))
    hip_ctx.kv4_attention(oracle.upload(hip_ctx, cache), 0, batch.on(hip_ctx), hip_ctx.buffer(src), out, heads)
    got = out.read().reshape(src.shape)
    batch.table = kept
    want, bound = oracle.attention(cache, 0, batch, src, hd ** -0.5, 0, hidden)
    assert np.all(want[:2] == 0) and np.all(got[:2] == 0) and np.all(got[7] == 0)
    assert np.all(np.abs(got - want) <= bound)
    out = hip_ctx.buffer(np.full((batch.n, heads * hd), 7, np.float32))
    hip_ctx.kv4_attention(oracle.upload(hip_ctx, cache), 0, batch.on(hip_ctx, max_rows=3), hip_ctx.buffer(src), out, heads)
    again = out.read().reshape(src.shape)
    for r, s, p in batch.positions():
        assert np.all(again[r] == 7) if r - int(batch.starts[s]) >= 3 else not np.any(again[r] == 7)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_queries_that_are_not_finite_stay_their_own(hip_ctx, bad):
    rng = np.random.default_rng(10)
    for rows, lengths in (([1, 3], [90, 70]), ([70], [120])):
        batch = oracle.Batch(rows, lengths, rng)
        cache = oracle.Kv4(1, batch.pool, 1, 64, rng)
        q = rng.normal(0, 1, (batch.n, 3, 64)).astype(np.float32)
        q[2, 1, 9] = bad
        got, want, bound = attend(hip_ctx, [], [], 3, 1, 64, batch=batch, cache=cache, q=q, rng=rng)
        assert np.isnan(got[2, 1]).all()
        fine = np.ones((batch.n, 3), bool)
        fine[2, 1] = False
        assert np.all(np.abs(got - want)[fine] <= bound[fine])


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e4])
def test_queries_of_any_size(hip_ctx, size):
    """1e4: scores in the thousands, where one key takes everything."""
    rng = np.random.default_rng(11)
    batch = oracle.Batch([1, 40], [300, 60], rng)
    cache = oracle.Kv4(1, batch.pool, 2, 128, rng)
    q = (size * rng.normal(0, 1, (41, 4, 128))).astype(np.float32)
    check(hip_ctx, [], [], 4, 2, 128, batch=batch, cache=cache, q=q, rng=rng)


def test_tables_that_hold_nonsense(hip_ctx):
    """Nothing outside the buffers is touched, and rows that belong to no sequence keep their output."""
    rng = np.random.default_rng(12)
    heads, hd, rows = 4, 64, 20
    cache = oracle.Kv4(1, 9, 2, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    q = hip_ctx.buffer(rng.normal(0, 1, (rows, heads * hd)).astype(np.float32))
    for starts in ([7, 3, 0xFFFFFFFF, 0, 5], [0xFFFFFFFF] * 5, [20, 20, 20, 20, 20], [0, 0xFFFFFFFF, 2, 3, 4]):
        for lengths in ([0xFFFFFFFF] * 4, [0, 1 << 31, 5, 0x7FFFFFFF]):
            table = rng.integers(0, 1 << 32, (4, 3), dtype=np.uint64).astype(np.uint32)
            table[::2] %= 12
            b = hip.Batch(hip_ctx.buffer(table), hip_ctx.buffer(np.array(starts, np.uint32)), hip_ctx.buffer(np.array(lengths, np.uint32)), 4, 3, rows)
            out = hip_ctx.buffer(np.full((rows, heads * hd), 7, np.float32))
            hip_ctx.kv4_attention(got, 0, b, q, out, heads, window=40)
            y = out.read().reshape(rows, -1)
            if min(starts) >= rows:
                assert np.all(y == 7)
    assert all(np.array_equal(b.read(np.uint8), w) for b, w in zip(got.buffers, cache.device()))
