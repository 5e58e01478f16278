"""Attention over the 8-bit cache where weights and values span many orders of magnitude."""
import time

import numpy as np
import pytest

from tests import longctx_oracle as oracle
from tests.test_gpu_kv8 import upload

pytestmark = pytest.mark.gpu


def unit_scale():
    """A score scale whose binary32 product with log2 e is 1: scores are powers of two of small dyadic numbers."""
    log2e, s = np.float32(1.44269504088896340736), np.float32(0.6931472)
    for _ in range(8):
        s = np.nextafter(s, np.float32(0))
    for _ in range(16):
        if s * log2e == np.float32(1):
            return s
        s = np.nextafter(s, np.float32(1))
    raise AssertionError("no such scale")


def attend(ctx, c, q, position, scale=None, window=0):
    queries, heads, hd = q.shape
    cache = upload(ctx, [c], c.scales[0].shape[1] * 32)
    out = ctx.empty(q.nbytes)
    ctx.kv8_attention(cache, ctx.buffer(q), out, heads, 0, position, queries, window=window, scale=scale)
    return out.read().reshape(q.shape)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("queries", [1, 12, 90])
def test_one_small_weight(hip_ctx, hd, queries):
    """A key of weight 1 whose value is 0, one of weight 2^-18 .. 2^-22 whose value is 100, others of weight 0.  The
    scores are exact, so the weight is off by its exponential (2^-22 of itself) and its pieces (2^-22 of itself or
    2^-37 of the largest weight: 2^-25 left by the first, 2^-12 of that by the second), and the result by the sum,
    the quotient and two products (2^-24 each)."""
    print("one small weight", hd, queries, flush=True)
    heads, n = 8, 2 + queries
    c = oracle.Kv8(1, n, hd)
    c.scales[0][:] = 1
    c.scales[1][:] = 1
    c.codes[0][0, 1, 0] = -1
    c.codes[0][0, 2:, 0] = -127
    c.codes[1][0, 1] = 100
    q = np.zeros((queries, heads, hd), np.float32)
    exponent = 18 + 4 * np.random.default_rng(hd + queries).integers(0, 257, (queries, heads)) / 256
    q[:, :, 0] = exponent
    got = attend(hip_ctx, c, q, 2, unit_scale())
    w = 2.0 ** -exponent[:, :, None]
    err = np.abs(got - 100 * w / (1 + w))
    bound = 100 * (2.0 ** -37 + w * (2 * 2.0 ** -22 + 4 * 2.0 ** -24))
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (6, 3, 96), (2, 1, 256)])
@pytest.mark.parametrize("queries", [1, 9, 80])
def test_any_codes_behind_the_last_row(hip_ctx, heads, kvh, hd, queries):
    """Codes that were never stored, -128 among them, behind the last query's row, in a block whose scale is near the
    largest that a row gives (-128 of them lie past binary32), and beside blocks of far smaller scales."""
    print("codes behind the last row", heads, kvh, hd, queries, flush=True)
    rng = np.random.default_rng(hd + queries)
    n = 101
    c = oracle.Kv8(kvh, n, hd, rng)
    c.scales[1][:, -1] = np.float32(3.4e38) / np.float32(127)
    c.codes[1][:, 96:n] = rng.integers(-9, 10, c.codes[1][:, 96:n].shape)
    c.codes[1][:, n:] = -128
    c.codes[0][:, n:] = -128
    q = rng.normal(0, 1, (queries, heads, hd)).astype(np.float32)
    want, bound = oracle.kv8_attention(c, q, n - queries, hd ** -0.5)
    err = np.abs(attend(hip_ctx, c, q, n - queries, hd ** -0.5) - want)
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("heads,kvh,hd,position,queries", [(32, 8, 128, 4000, 1), (32, 8, 128, 8000, 9), (8, 2, 128, 3000, 300), (8, 8, 64, 2000, 200),
                                                           (4, 2, 256, 1500, 100)])
def test_one_block_of_tiny_values_costs_little(hip_ctx, heads, kvh, hd, position, queries):
    """The first block's values are 2^-40 times the others': within four times the time without it (a row at a time
    would be 6 to 300 times).  Least of several runs of a few passes each."""
    print("tiny first block", heads, kvh, hd, position, queries, flush=True)
    rng = np.random.default_rng(1)
    q = hip_ctx.buffer(rng.normal(0, 1, (queries, heads, hd)).astype(np.float32))
    out = hip_ctx.empty(4 * queries * heads * hd)
    c = oracle.Kv8(kvh, position + queries, hd, rng)
    caches = [upload(hip_ctx, [c], position + queries)]
    c.scales[1][:, 0] *= np.float32(2.0 ** -40)
    caches.append(upload(hip_ctx, [c], position + queries))
    least = [np.inf, np.inf]
    for _ in range(10):
        for i, cache in enumerate(caches):
            t = time.perf_counter()
            hip_ctx.begin()
            for _ in range(5):
                hip_ctx.kv8_attention(cache, q, out, heads, 0, position, queries)
            hip_ctx.commit()
            least[i] = min(least[i], time.perf_counter() - t)
    assert least[1] <= 4 * least[0], least


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (6, 3, 96), (34, 2, 256), (64, 1, 128)])
@pytest.mark.parametrize("position,queries,window", [(150, 1, 0), (150, 9, 0), (3000, 7, 0), (3000, 12, 700), (64, 150, 0), (1500, 90, 77), (10, 300, 33)])
def test_scales_far_apart_everywhere(hip_ctx, heads, kvh, hd, position, queries, window):
    """Every block's V scale at random between 2^-100 and 2^100 and its keys' scores tens apart, blocks of zeros
    among them; the blocks out of every row's sight hold NaN scales and codes of -128.  Bound: the weights' relative
    errors (longctx_oracle) times the sum of weight x |value|, weights below 2^-60 of a row's largest left out."""
    print("far apart", heads, kvh, hd, position, queries, window, flush=True)
    rng = np.random.default_rng(position + hd + queries)
    n = position + queries
    c = oracle.Kv8(kvh, n, hd, rng)
    c.scales[1][:] = 2.0 ** rng.uniform(-100, 100, c.scales[1].shape)
    c.scales[0][:] *= 3
    for b in range(2, c.nb, 5):
        c.codes[1][:, 32 * b:32 * b + 32] = 0
        c.scales[1][:, b] = 0
    first = max(0, position + 1 - window) if window else 0
    for w in range(2):
        c.scales[w][:, :first // 32] = np.nan
        c.scales[w][:, (n - 1) // 32 + 1:] = np.nan
        c.codes[w][:, n:] = -128
    q = rng.normal(0, 1, (queries, heads, hd)).astype(np.float32)
    want, _ = oracle.kv8_attention(c, q, position, hd ** -0.5, window)
    got = attend(hip_ctx, c, q, position, hd ** -0.5, window)
    scale = float(np.float32(hd ** -0.5))
    for h in range(0, heads, max(1, heads // 6)):
        kv = h // (heads // kvh)
        k, ks = c.codes[0][kv].astype(np.float64), np.repeat(c.scales[0][kv].astype(np.float64), 32)
        v = np.abs(c.codes[1][kv].astype(np.float64) * np.repeat(c.scales[1][kv].astype(np.float64), 32)[:, None])
        for i in range(0, queries, max(1, queries // 25)):
            p = position + i + 1
            at = slice(max(0, p - window) if window else 0, p)
            s = (k[at] @ q[i, h].astype(np.float64)) * ks[at] * scale
            e = (hd + 8) * 2.0 ** -23 * ((np.abs(k[at]) @ np.abs(q[i, h]).astype(np.float64)) * ks[at] * scale)
            w = np.exp(s - s.max())
            live = w > 2.0 ** -60
            some = (w[~live] @ v[at][~live]) / w.sum()
            bound = (2 * e.max() + 2.0 ** -20 + p * 2.0 ** -22) * (w[live] @ v[at][live]) / w.sum() + some
            err = np.abs(got[i, h] - want[i, h])
            assert np.all(err <= bound), (h, i, (err / bound).max())


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (6, 3, 96), (2, 1, 256)])
@pytest.mark.parametrize("position,queries", [(60, 1), (60, 9), (5000, 1), (3000, 9), (60, 70), (3000, 70), (2500, 600)])
@pytest.mark.parametrize("far", [False, True])
def test_values_whose_sum_passes_binary32(hip_ctx, heads, kvh, hd, position, queries, far):
    """Values near binary32's end under weights about alike: their mean is a number, their sum is none.  far: with
    blocks of values 2^-60 times theirs among them."""
    print("large values", heads, kvh, hd, position, queries, far, flush=True)
    rng = np.random.default_rng(position + hd)
    n = position + queries
    c = oracle.Kv8(kvh, n, hd, rng)
    c.scales[1][:] = (np.float32(3.39e38) / np.float32(127)) * rng.uniform(0.9, 1, c.scales[1].shape).astype(np.float32)
    c.codes[1][:] = rng.integers(100, 128, c.codes[1].shape)
    if far:
        c.scales[1][:, 1::3] *= np.float32(2.0 ** -60)
    q = rng.normal(0, 0.1, (queries, heads, hd)).astype(np.float32)
    want, bound = oracle.kv8_attention(c, q, position, hd ** -0.5)
    err = np.abs(attend(hip_ctx, c, q, position, hd ** -0.5) - want)
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("position,queries", [(100, 1), (92, 9), (60, 80), (2000, 1), (1990, 100)])
def test_a_marked_block_beside_scales_far_apart(hip_ctx, which, hd, position, queries):
    """A NaN scale of K or V in the block of positions 96 .. 127 of one kv head: NaN in every row that sees it, in no
    other; other rows as without it."""
    print("marked beside far", which, hd, position, queries, flush=True)
    rng = np.random.default_rng(position + hd)
    n = position + queries
    c = oracle.Kv8(2, n, hd, rng)
    c.scales[1][:, ::2] *= np.float32(2.0 ** -50)
    q = rng.normal(0, 1, (queries, 4, hd)).astype(np.float32)
    plain = attend(hip_ctx, c, q, position, hd ** -0.5)
    assert np.isfinite(plain).all()
    c.scales[which][1, 3] = np.nan
    got = attend(hip_ctx, c, q, position, hd ** -0.5)
    seen = np.arange(position, n) >= 96
    marked = np.broadcast_to((seen[:, None] & (np.arange(4) >= 2))[..., None], got.shape)
    assert np.array_equal(np.isnan(got), marked)
    want, bound = oracle.kv8_attention(c, q, position, hd ** -0.5)
    assert np.all(np.abs(got - want)[~marked] <= bound[~marked])
