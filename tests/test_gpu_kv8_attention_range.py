"""Attention over the 8-bit cache where weights and values span many orders of magnitude."""
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
