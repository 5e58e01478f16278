"""The operators that serve several sequences at values and sizes far from a model's ordinary ones."""
import numpy as np
import pytest

from tests import serving_oracle as oracle
from tests.test_gpu_kv4_attention import attend
from zhip import hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e7, -1e7, 1e10, -3e13, 1e25, -1e30])
@pytest.mark.parametrize("rows,lengths", [([1], [1]), ([1], [70]), ([1, 1], [3000, 9]), ([3], [130]), ([9], [200]), ([90], [300]),
                                          ([30, 1], [2000, 64])])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_of_any_size(hip_ctx, hd, rows, lengths, size):
    """Queries and keys of one value each: positions with the same key have the same score, to the bit, and those with
    another have one so far below that their weight is 0.  The output is the mean of the values at the keys that are
    best, whatever the scores are, and every row has one such key at least.
    Tolerance: weights are 1 exactly, or one power of two for all of a column; the sums of n terms are off by n 2^-23 and
    n 2^-24, the factors of the maximum and of the splits by 2^-20."""
    for group in (1, 3, 12):
        rng = np.random.default_rng(hd + group + sum(lengths))
        batch = oracle.Batch(rows, lengths, rng)
        cache = oracle.Kv4(1, batch.pool, 1, hd, rng)
        cache.scales[0][:] = 127
        first = cache.codes[0][..., 0].copy()
        cache.codes[0][:] = 0
        cache.codes[0][..., 0] = first
        q = np.zeros((batch.n, group, hd), np.float32)
        # of many sizes; one column in four a model's own, near 1
        q[..., 0] = size * rng.uniform(0.5, 2, (batch.n, group))
        ordinary = rng.random((batch.n, group)) < 0.25
        q[ordinary, 0] = rng.normal(0, 1, ordinary.sum())
        got, plain, bound = attend(hip_ctx, [], [], group, 1, hd, batch=batch, cache=cache, q=q, rng=rng)
        assert np.all(np.abs(got - plain)[ordinary] <= bound[ordinary])
        for r, s, p in batch.positions():
            at = np.arange(p + 1)
            k, v = cache.rows(0, batch.table[s, at // 64].astype(int), at % 64)
            best = k[:, 0, 0] * np.sign(size)
            v = v[best == best.max(), 0]
            off = np.abs(got[r] - v.mean(axis=0))[~ordinary[r]]
            assert np.all(off <= (2.0 ** -20 + (p + 1) * 2.0 ** -21) * np.abs(v).max()), (group, r, off.max())


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("size,weight,eps", [(1e-40, 1, 0.0), (1e-42, 1, 0.0), (3e-39, 1, 0.0), (1e37, 1, 1e-6), (1e30, 1e-20, 1e-6),
                                             (1e-30, 1e20, 0.0), (1e-42, 1e-30, 0.0), (1e37, 1e30, 0.0)])
def test_norms_of_any_size(hip_ctx, style, size, weight, eps):
    """Heads and weights from denormal to the largest: the factor 1 / sqrt(mean x^2) alone, or times a weight, may be
    no binary32 number where the normalised value is.
    Tolerance: as for ordinary heads (the factor's rounding, the normalised value's, the weight's sum with the offset, its product,
    and the rotation's three: 8 2^-24 of the pair)."""
    rng = np.random.default_rng(17)
    heads, rows = 5, 3
    for hd, rd, extra in ((128, 128, 0), (96, 48, 0), (64, 64, 1), (512, 6, 0)):
        x = (size * rng.normal(0, 1, (rows, heads, hd))).astype(np.float32)
        w = [(weight * rng.normal(1, 0.2, hd)).astype(np.float32) for _ in range(2)]
        held = np.concatenate([x.reshape(rows, -1), np.zeros((rows, extra), np.float32)], axis=1)
        src = hip_ctx.buffer(held)
        d = hip.Heads(hip.RopeDesc(hd, rd, style), *(hip_ctx.buffer(v) for v in w), eps=eps)
        hip_ctx.norm_rope_rows(d, src, src, rows, 3, 2, first_position=5, src_stride=held.shape[1], dst_stride=held.shape[1])
        got = src.read().reshape(held.shape)[:, :heads * hd].reshape(x.shape)
        y = np.concatenate([oracle.norm(x[:, :3], w[0], eps), oracle.norm(x[:, 3:], w[1], eps)], axis=1)
        want, pair = oracle.rope(y, np.arange(5, 5 + rows), oracle.rope_frequencies(rd, 10000.0), rd, style)
        pair = np.maximum(pair, np.abs(want))
        off = np.abs(got - want)
        assert np.all(off <= 8 * 2.0 ** -24 * pair + 2.0 ** -149), (hd, rd, (off / pair).max())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,lengths,window", [([100], [100], 0), ([70], [700], 0), ([100], [20000], 1024), ([90], [90], 33), ([300], [9000], 100),
                                                 ([90, 65, 1], [100, 1500, 70], 0), ([120, 1, 80], [6000, 90, 80], 500)])
def test_room_that_a_batch_does_not_use(hip_ctx, hd, rows, lengths, window):
    """Prompts whose pages could hold far more positions than they have: right, and to the bit as with the limit that
    fits, as the parts of a sum follow what the rows see and not what they might.  A window far into a context too."""
    heads, kvh = 8, 2
    rng = np.random.default_rng(hd + sum(lengths))
    batch = oracle.Batch(rows, lengths, rng, extra_pages=1500)
    cache = oracle.Kv4(1, batch.pool, kvh, hd, rng)
    got = oracle.upload(hip_ctx, cache)
    q = rng.normal(0, 0.7, (batch.n, heads, hd)).astype(np.float32)
    src, y = hip_ctx.buffer(q), []
    for limit in (max(lengths), 0, 2 * max(lengths)):
        print("room", rows, lengths, window, hd, limit, flush=True)
        out = hip_ctx.buffer(np.full(q.shape, 7, np.float32))
        hip_ctx.kv4_attention(got, 0, batch.on(hip_ctx, max_rows=max(rows), max_length=limit), src, out, heads, window)
        y.append(out.read().reshape(q.shape))
    want, bound = oracle.attention(cache, 0, batch, q, hd ** -0.5, window)
    assert np.all(np.abs(y[0] - want) <= bound)
    assert np.array_equal(y[0], y[1]) and np.array_equal(y[0], y[2])


def pool_of(cache, kvh, hd):
    """K and V of every position of the pool [kv head][page x position][hd], in 64 bits."""
    k, v = (oracle.of_four_bits(cache.codes[w][0], cache.scales[w][0]).transpose(2, 0, 1, 3).reshape(kvh, -1, hd) for w in range(2))
    return k, v


def near(got, x, k, v, seen, scale):
    """Outputs [columns][hd] of one kv head for queries x [columns][hd], seen [columns][positions].
    Tolerance: weights are off by 2 e of themselves for scores off by e (the score's own and the maximum's, as
    serving_oracle.attention has them) and by 2^-20, the sums of n terms, three pieces each, by 3 n 2^-24 of the sum of
    their magnitudes; the quotient of two such sums by twice that.  Of sum w |v|, not of the largest value: a few keys in
    tens of thousands have nearly all the weight."""
    z = x.astype(np.float64) @ k.T * float(np.float32(scale))
    e = (3 * k.shape[1] + 8) * 2.0 ** -23 * (np.abs(x.astype(np.float64)) @ np.abs(k).T).max(axis=1) * scale
    z[~seen] = -np.inf
    w = np.exp(z - z.max(axis=1, keepdims=True))
    w /= w.sum(axis=1, keepdims=True)
    bound = 2 * (2 * e + 2.0 ** -20 + 3 * 2.0 ** -24 * seen.sum(axis=1))[:, None] * (w @ np.abs(v))
    off = np.abs(got - w @ v)
    assert np.all(off <= bound), ((off / bound).max(), np.argwhere(~(off <= bound))[:4])


def with_loud_first_page(pages, kvh, hd, rng):
    """A pool whose page 0, which no sequence has, would take all the weight if it were seen in place of a missing one."""
    cache = oracle.Kv4(1, pages, kvh, hd, rng)
    cache.scales[0][0, 0] = 140
    return cache


@pytest.mark.parametrize("sequences,group,hd", [(64, 1, 64), (64, 8, 64), (100, 1, 128), (64, 24, 64)])
def test_long_lists_of_pages_of_single_rows(hip_ctx, sequences, group, hd):
    """Sequences so long, and so many, that a wavefront goes through its list of 64 blocks' pages several times (300 blocks
    of 39990 positions): every page from the list of its own time, and pages that the pool lacks on both sides of the
    lists' ends.  The sequences read the same pages, each in an order of its own."""
    rng = np.random.default_rng(sequences + group)
    kvh, length, scale = 8, 39990, hd ** -0.5
    pages = -(-length // 64)
    cache = with_loud_first_page(pages + 1, kvh, hd, rng)
    table = np.stack([rng.permutation(pages) + 1 for _ in range(sequences)]).astype(np.uint32)
    seen = np.ones((sequences, pages + 1, 64), bool)
    seen[:, 0] = False
    for s in range(sequences):
        seen[s, table[s, -1], length % 64:] = False
        for p in np.concatenate([rng.permutation(pages - 1)[:20], [126, 127, 128, 129, 130, 255, 256, 257, 384, 512, 513]]):
            seen[s, table[s, p] if table[s, p] <= pages else 0] = False
            table[s, p] = pages + 1 + rng.integers(0, 1 << 31)
    q = rng.normal(0, 0.7, (sequences, kvh * group, hd)).astype(np.float32)
    print("lists", sequences, group, hd, flush=True)
    on = hip.Batch(hip_ctx.buffer(table), hip_ctx.buffer(np.arange(sequences + 1, dtype=np.uint32)),
                   hip_ctx.buffer(np.full(sequences, length, np.uint32)), sequences, pages, sequences, 1, length)
    out = hip_ctx.empty(q.nbytes)
    hip_ctx.kv4_attention(oracle.upload(hip_ctx, cache), 0, on, hip_ctx.buffer(q), out, kvh * group)
    got = out.read().reshape(sequences, kvh, group, hd)
    k, v = pool_of(cache, kvh, hd)
    some = range(0, sequences, 1 if group == 1 else 7)
    for h in range(kvh):
        near(np.concatenate([got[s, h] for s in some]), np.concatenate([q[s, h * group:(h + 1) * group] for s in some]), k[h], v[h],
             np.repeat(seen.reshape(sequences, -1)[list(some)], group, axis=0), scale)


@pytest.mark.parametrize("rows,length,heads,kvh,hd", [(1024, 9390, 64, 8, 64), (70, 140000, 2, 1, 64), (70, 143000, 2, 1, 256)])
def test_long_lists_of_pages_of_prompts(hip_ctx, rows, length, heads, kvh, hd):
    """The same for a prompt's tiles: so many that each goes through all 147 pages, and splits of more than 64 pages."""
    rng = np.random.default_rng(rows + hd)
    group, scale, pages = heads // kvh, hd ** -0.5, -(-length // 64)
    cache = with_loud_first_page(pages + 1, kvh, hd, rng)
    order = (rng.permutation(pages) + 1).astype(np.uint32)
    table, here = order.copy(), np.ones(length, bool)
    for p in np.concatenate([rng.permutation(pages - rows // 64 - 2)[:pages // 30], [63, 64, 65, 66, 127, 128, 129]]):
        table[p] = pages + 1 + rng.integers(0, 1 << 31)
        here[64 * p:64 * p + 64] = False
    q = rng.normal(0, 0.7, (rows, heads, hd)).astype(np.float32)
    print("prompt lists", rows, length, hd, flush=True)
    on = hip.Batch(hip_ctx.buffer(table), hip_ctx.buffer(np.array([0, rows], np.uint32)), hip_ctx.buffer(np.array([length], np.uint32)),
                   1, pages, rows, rows, length)
    out = hip_ctx.empty(q.nbytes)
    hip_ctx.kv4_attention(oracle.upload(hip_ctx, cache), 0, on, hip_ctx.buffer(q), out, heads)
    got = out.read().reshape(q.shape)
    k, v = pool_of(cache, kvh, hd)
    at = (order[np.arange(length) // 64].astype(int) * 64 + np.arange(length) % 64)
    some = np.unique(np.concatenate([[0, 1, rows - 1], rng.integers(0, rows, 12)]))
    seen = (np.arange(length) <= (length - rows + some)[:, None]) & here
    for h in range(kvh):
        mine = slice(h * group, (h + 1) * group)
        near(got[some, mine].reshape(-1, hd), q[some, mine].reshape(-1, hd), k[h][at], v[h][at], np.repeat(seen, group, axis=0), scale)


@pytest.mark.parametrize("rows,length", [(1, 2), (3, 50), (12, 200), (80, 90)])
def test_scores_past_the_range(hip_ctx, rows, length):
    """One key whose score is above binary32's largest, or below its least, beside keys of 0, and rows that see it alone.
    Below: without weight, so the mean of the other values in sight (to n 2^-23 and n 2^-24 of the largest), zeros where
    there are none.  Above: NaN."""
    rng = np.random.default_rng(rows)
    hd = 64
    batch = oracle.Batch([rows], [length], rng)
    cache = oracle.Kv4(1, batch.pool, 1, hd, rng)
    cache.codes[0][:] = 0
    first = length - rows  # what the first row sees last
    page, slot = batch.place(0, first)
    cache.codes[0][0, page, slot, 0, 3] = 7
    cache.scales[0][0, page, slot] = 219
    q = np.zeros((rows, 2, hd), np.float32)
    q[:, 0, 3], q[:, 1, 3] = -3e38, 3e38
    for window in (0, 1):
        got = attend(hip_ctx, [], [], 2, 1, hd, batch=batch, cache=cache, q=q, rng=rng, scale=0.5, window=window)[0]
        for r in range(rows):
            at = np.arange(max(0, first + r + 1 - window) if window else 0, first + r + 1)
            v = cache.rows(0, batch.table[0, at // 64].astype(int), at % 64)[1][at != first, 0]
            want = v.mean(axis=0) if len(v) else np.zeros(hd)
            assert np.all(np.abs(got[r, 0] - want) <= (2.0 ** -20 + at.size * 2.0 ** -21) * np.abs(v).max(initial=0))
            assert np.isnan(got[r, 1]).all() == (first in at)
