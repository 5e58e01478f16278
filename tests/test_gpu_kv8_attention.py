"""Attention over the 8-bit cache against a 64-bit form, element by element within the bound that its 32-bit sums
allow (longctx_oracle.kv8_attention derives it).  Blocks that no query sees hold NaN scales."""
import numpy as np
import pytest

from tests import longctx_oracle as oracle
from tests.test_gpu_kv8 import upload
from zhip import hip

pytestmark = pytest.mark.gpu


def attend(ctx, heads, kvh, hd, position, queries=1, window=0, layer=0, layers=1, context=None, scale=None, sharp=1.0,
           stride=0, spoil=True, seed=0):
    print("kv8 attention", heads, kvh, hd, position, queries, window, layer, flush=True)
    rng = np.random.default_rng(seed + heads * 1000 + hd + position + queries)
    n = position + queries
    context = context or n + 40
    ls = [oracle.Kv8(kvh, context, hd, rng) for _ in range(layers)]
    c = ls[layer]
    if spoil:
        first = max(0, position + 1 - window) if window else 0
        for w in range(2):
            c.scales[w][:, :first // 32] = np.nan
            c.scales[w][:, (n - 1) // 32 + 1:] = np.inf
            # rows behind the last query's, in its own block
            c.codes[w][:, n:] = 127
    cache = upload(ctx, ls, context)
    width = heads * hd
    stride = stride or width
    qf = rng.normal(0, sharp, queries * stride).astype(np.float32)
    q = qf[np.arange(queries)[:, None] * stride + np.arange(width)].reshape(queries, heads, hd)
    out = ctx.buffer(np.full(queries * width + 64, 3, np.float32))
    scale = hd ** -0.5 if scale is None else scale
    ctx.kv8_attention(cache, ctx.buffer(qf), out, heads, layer, position, queries, window=window, scale=scale, q_stride=stride)
    got = out.read()
    assert np.all(got[queries * width:] == 3)
    want, bound = oracle.kv8_attention(c, q, position, scale, window)
    err = np.abs(got[:queries * width].reshape(want.shape) - want)
    assert np.all(err <= bound), (err / bound).max()
    return cache, q, got[:queries * width]


@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (32, 4, 64), (6, 6, 96), (8, 1, 256), (1, 1, 64), (5, 1, 128), (24, 2, 96), (16, 1, 128),
                                          (64, 1, 64), (34, 2, 256)])
@pytest.mark.parametrize("position", [0, 1, 30, 31, 32, 33, 63, 64, 150, 511, 1000])
def test_one_query(hip_ctx, heads, kvh, hd, position):
    attend(hip_ctx, heads, kvh, hd, position)


@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (4, 4, 64), (8, 2, 256), (12, 4, 96)])
@pytest.mark.parametrize("position", [4111, 8191, 20000])
def test_one_query_far_out(hip_ctx, heads, kvh, hd, position):
    attend(hip_ctx, heads, kvh, hd, position, layer=1, layers=2)


@pytest.mark.parametrize("position,window", [(0, 1), (100, 1), (100, 32), (100, 33), (100, 101), (100, 102), (4000, 64), (4000, 65),
                                             (4000, 1023), (5000, 4096), (37, 4294967295)])
@pytest.mark.parametrize("queries", [1, 5])
def test_windows(hip_ctx, position, window, queries):
    attend(hip_ctx, 8, 2, 128, position, queries, window)


@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (8, 8, 64), (7, 1, 96), (4, 2, 256)])
@pytest.mark.parametrize("position,queries", [(0, 2), (0, 9), (31, 2), (50, 16), (1500, 9), (0, 17), (20, 40), (3, 100)])
def test_several_queries(hip_ctx, heads, kvh, hd, position, queries):
    attend(hip_ctx, heads, kvh, hd, position, queries)


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 1, 64), (3, 3, 96), (2, 1, 256)])
@pytest.mark.parametrize("position,queries,window", [(0, 300, 0), (77, 257, 0), (900, 130, 0), (64, 200, 50), (2000, 70, 333), (10, 128, 129)])
def test_prompts(hip_ctx, heads, kvh, hd, position, queries, window):
    attend(hip_ctx, heads, kvh, hd, position, queries, window)


@pytest.mark.parametrize("queries", [1, 9, 90])
def test_strided_queries_and_scales(hip_ctx, queries):
    attend(hip_ctx, 4, 2, 64, 200, queries, stride=4 * 64 + 3, scale=0.3, sharp=3.0)
    attend(hip_ctx, 4, 2, 128, 200, queries, stride=1000, scale=-0.1)
    attend(hip_ctx, 4, 2, 128, 200, queries, scale=0.0)


@pytest.mark.parametrize("queries", [1, 70])
@pytest.mark.parametrize("position", [400, 6000])
def test_small_weights_beside_a_dominant_key_keep_their_value(hip_ctx, queries, position):
    """One key whose score is 13 above thousands of others (weights of 2e-6 beside 1), with a value of 0 in the
    output's dims: what is left is the sum of the small ones.  Bound: a weight is held to 2^-21 of itself, its
    score's error (longctx_oracle) added, or to 2^-38 of the largest."""
    heads, kvh, hd = 2, 1, 64
    n = position + queries
    rng = np.random.default_rng(position)
    c = oracle.Kv8(kvh, n, hd, rng)
    c.scales[0][:] = np.float32(1 / 64)
    c.scales[1][:] = np.float32(1 / 64)
    c.codes[0][:] = rng.integers(-2, 3, c.codes[0].shape)
    c.codes[1][:] = rng.integers(30, 100, c.codes[1].shape)
    c.codes[0][:, 3] = 13
    c.codes[1][:, 3] = 0
    q = np.full((queries, heads, hd), 1.0, np.float32)
    cache = upload(hip_ctx, [c], n)
    out = hip_ctx.empty(q.nbytes)
    hip_ctx.kv8_attention(cache, hip_ctx.buffer(q), out, heads, 0, position, queries, scale=1.0)
    want, _ = oracle.kv8_attention(c, q, position, 1.0)
    got = out.read().reshape(want.shape)
    e = 2 * (hd + 8) * 2.0 ** -23 * 13 * hd / 64
    bound = (e + 2.0 ** -19 + n * 2.0 ** -22) * np.abs(want) + n * 2.0 ** -38 * 100 / 64
    assert np.all(np.abs(got - want) <= bound), (np.abs(got - want) / bound).max()


def test_a_marked_block_in_sight_reads_as_nan(hip_ctx):
    for queries in (1, 80):
        rng = np.random.default_rng(2)
        c = oracle.Kv8(2, 200, 64, rng)
        c.scales[1][1, 3] = np.nan
        cache = upload(hip_ctx, [c], 200)
        q = rng.normal(0, 1, (queries, 4, 64)).astype(np.float32)
        out = hip_ctx.empty(q.nbytes)
        hip_ctx.kv8_attention(cache, hip_ctx.buffer(q), out, 4, 0, 60, queries)
        got = out.read().reshape(queries, 4, 64)
        seen = np.arange(60, 60 + queries) >= 96
        assert np.array_equal(np.isnan(got), np.broadcast_to((seen[:, None] & (np.arange(4) >= 2))[..., None], got.shape))


@pytest.mark.parametrize("queries", [1, 9, 200])
def test_same_bits_each_time(hip_ctx, queries):
    cache, q, first = attend(hip_ctx, 32, 8, 128, 3000, queries)
    qb, out = hip_ctx.buffer(q), hip_ctx.empty(q.nbytes)
    other = hip_ctx.empty(q.nbytes)
    hip_ctx.begin()
    for _ in range(5):
        hip_ctx.kv8_attention(cache, qb, other, 32, 0, 1000, queries)
        hip_ctx.kv8_attention(cache, qb, out, 32, 0, 3000, queries)
    hip_ctx.commit()
    assert np.array_equal(out.read().view(np.uint32), first.view(np.uint32))


def held(ctx, c, q, position, window=0):
    queries, heads, hd = q.shape
    cache = upload(ctx, [c], c.scales[0].shape[1] * 32)
    out = ctx.empty(q.nbytes)
    ctx.kv8_attention(cache, ctx.buffer(q), out, heads, 0, position, queries, window=window)
    return out.read().reshape(q.shape)


@pytest.mark.parametrize("garbage", [np.inf, -np.inf, 3e38, -3e38, -1.0, 0.0])
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (2, 1, 256)])
def test_any_scale_out_of_the_window(hip_ctx, heads, kvh, hd, garbage):
    """Scales that were never stored, ahead of the window and behind the queries."""
    for position, queries, window in ((200, 1, 40), (200, 5, 40), (2048 + 97, 70, 65), (290, 140, 33)):
        print("garbage", garbage, heads, hd, position, queries, window, flush=True)
        rng = np.random.default_rng(position)
        n = position + queries
        c = oracle.Kv8(kvh, n + 70, hd, rng)
        for w in range(2):
            c.scales[w][:, :(position + 1 - window) // 32] = garbage
            c.scales[w][:, (n - 1) // 32 + 1:] = garbage
        q = rng.normal(0, 1, (queries, heads, hd)).astype(np.float32)
        want, bound = oracle.kv8_attention(c, q, position, hd ** -0.5, window)
        err = np.abs(held(hip_ctx, c, q, position, window) - want)
        assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (6, 3, 96), (2, 1, 256)])
@pytest.mark.parametrize("position,queries", [(60, 5), (70, 9), (3000, 9), (9, 200), (1500, 150)])
@pytest.mark.parametrize("large", [2.0 ** 26, 2.0 ** 100])
def test_values_of_later_positions_stay_out_of_earlier_rows(hip_ctx, heads, kvh, hd, position, queries, large):
    """V of the last blocks, which the first queries don't see, is far larger than the others'.  (The bound is of
    each row's own largest value; a factor of 2^-32 and more goes another way than 2^-26, whose log2 is held to 2^-19:
    the rows without the large ones are off by another ln 2 times that.)"""
    print("later values", heads, kvh, hd, position, queries, large, flush=True)
    rng = np.random.default_rng(position + hd)
    n = position + queries
    c = oracle.Kv8(kvh, n, hd, rng)
    first = (position + queries // 2) // 32 + 1
    c.scales[1][:, first:] *= np.float32(large)
    q = rng.normal(0, 1, (queries, heads, hd)).astype(np.float32)
    want, bound = oracle.kv8_attention(c, q, position, hd ** -0.5)
    bound = bound * (1 + 2.0 ** -19 / 2.0 ** -20)
    err = np.abs(held(hip_ctx, c, q, position) - want)
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (6, 3, 96), (2, 1, 256)])
@pytest.mark.parametrize("position,queries", [(500, 1), (9000, 1), (500, 9), (2500, 12), (400, 150), (1500, 40)])
def test_large_values_of_no_weight(hip_ctx, heads, kvh, hd, position, queries):
    """A block of values 2^110 times the others', whose keys score hundreds below them, and one of values 2^-100
    times theirs.  Bound: the weights' relative errors (longctx_oracle) times the sum of weight x |value|."""
    print("weightless values", heads, kvh, hd, position, queries, flush=True)
    rng = np.random.default_rng(position + hd)
    n = position + queries
    c = oracle.Kv8(kvh, n, hd, rng)
    q = np.abs(rng.normal(0, 1, (queries, heads, hd))).astype(np.float32) + np.float32(0.5)
    c.codes[0][:, 64:96] = -127
    c.scales[0][:, 2] = 2.0
    c.scales[1][:, 2] *= np.float32(2.0 ** 110)
    c.scales[1][:, 4] *= np.float32(2.0 ** -100)
    c.scales[1][:, 6] = 0
    c.codes[1][:, 192:224] = 0
    want, _ = oracle.kv8_attention(c, q, position, hd ** -0.5)
    got = held(hip_ctx, c, q, position)
    group = heads // kvh
    scale = float(np.float32(hd ** -0.5))
    for h in range(heads):
        k = c.codes[0][h // group].astype(np.float64)[:n]
        ks = np.repeat(c.scales[0][h // group].astype(np.float64), 32)[:n]
        v = np.abs(c.codes[1][h // group].astype(np.float64)[:n] * np.repeat(c.scales[1][h // group].astype(np.float64), 32)[:n, None])
        for i in range(queries):
            p = position + i + 1
            s = (k[:p] @ q[i, h].astype(np.float64)) * ks[:p] * scale
            e = (hd + 8) * 2.0 ** -23 * ((np.abs(k[:p]) @ np.abs(q[i, h]).astype(np.float64)) * ks[:p] * scale)
            # an error counts with the weight of its own position; the most of a weight below 2^-60 of the largest is 0
            w = np.exp(s - s.max())
            live = w > 2.0 ** -60
            bound = (2 * e[live].max() + 2.0 ** -20 + p * 2.0 ** -22) * (w[live] @ v[:p][live]) / w.sum()
            err = np.abs(got[i, h] - want[i, h])
            assert np.all(err <= bound), (h, i, (err / bound).max())


@pytest.mark.parametrize("queries", [1, 9, 80])
@pytest.mark.parametrize("power", [-125, -110, 100])
def test_values_near_the_ends_of_the_range(hip_ctx, queries, power):
    """Scales of 2^power: outputs are scaled by it, to a step, but for what falls below 2^-126 (16 roundings of half
    of 2^-149 at most: a sum and its share by each of four wavefronts, and of four splits)."""
    rng = np.random.default_rng(power + 1000)
    c = oracle.Kv8(2, 300, 64, rng)
    q = rng.normal(0, 1, (queries, 4, 64)).astype(np.float32)
    plain = held(hip_ctx, c, q, 200)
    c.scales[1] *= np.float32(2.0 ** power * 64)
    got = held(hip_ctx, c, q, 200)
    want = plain.astype(np.float64) * 2.0 ** power * 64
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * np.abs(want) + 16 * 2.0 ** -150)


@pytest.mark.parametrize("group", [3, 5, 7, 11, 17, 31, 33, 43, 63, 64])
@pytest.mark.parametrize("queries", [1, 2, 3, 12, 41])
def test_groups_of_any_size(hip_ctx, group, queries):
    """Rows of a kv head that fill a workgroup's tile in part, queries that end inside one."""
    for hd, position, window in ((64, 130, 0), (128, 2000, 77), (256, 40, 0)):
        attend(hip_ctx, group, 1, hd, position, queries, window)


@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (5, 5, 64)])
def test_a_session_of_steps_of_every_length(hip_ctx, heads, kvh, hd):
    """A cache stored and read a few positions at a time, from the first, with the same buffers."""
    rng = np.random.default_rng(1)
    n = 170
    k, v = (rng.normal(0, 1, (n, kvh, hd)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 1, (n, heads, hd)).astype(np.float32)
    near, cache = oracle.Kv8(kvh, n, hd), hip_ctx.kv8_cache(1, kvh, hd, n)
    p = 0
    for step in (1, 1, 2, 3, 5, 8, 13, 21, 34, 31, 32, 1, 17, 1):
        near.store(k[p:p + step], v[p:p + step], p)
        kb, vb, qb = (hip_ctx.buffer(a[p:p + step]) for a in (k, v, q))
        out = hip_ctx.empty(qb.nbytes)
        hip_ctx.begin()
        hip_ctx.kv8_store(cache, kb, vb, 0, p, step)
        hip_ctx.kv8_attention(cache, qb, out, heads, 0, p, step)
        hip_ctx.commit()
        want, bound = oracle.kv8_attention(near, q[p:p + step], p, hd ** -0.5)
        assert np.all(np.abs(out.read().reshape(want.shape) - want) <= bound)
        p += step
    assert p == n
