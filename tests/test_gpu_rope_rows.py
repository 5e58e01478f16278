"""ziggy_hip_rope_rows_f32 against a 64-bit form: both pairings, part of the head, every scaling, factors per
pair, positions far out and in no order, offsets and strides off the vector loads' alignment, in place.

Tolerance: the angle is rounded to 2^-24 of half a turn (2^-24 pi), sine and cosine to 2^-22 (four roundings'
worth of half a step each), their product with the magnitude, the two products and the sum to 2^-24 each:
(pi + 4 + 4) 2^-24 < 12 2^-24 of |x0| + |x1| times the magnitude."""
import numpy as np
import pytest

from tests import longctx_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu

SCALINGS = {"none": {}, "linear": dict(scaling=hip.ROPE_LINEAR, factor=4.0),
            "yarn": dict(scaling=hip.ROPE_YARN, factor=4.0, orig=32768, low=1.0, high=32.0),
            "yarn_short": dict(scaling=hip.ROPE_YARN, factor=8.0, orig=2048, low=1.0, high=32.0),
            "bands": dict(scaling=hip.ROPE_BANDS, factor=8.0, orig=8192, low=1.0, high=4.0)}


def rotate(ctx, rows, heads, hd, rd, style, base=10000.0, first=0, positions=None, factors=None, magnitude=1.0,
           extra=0, off=0, in_place=False, **scaling):
    print("rope", rows, heads, hd, rd, style, scaling, first, extra, off, in_place, flush=True)
    rng = np.random.default_rng(rows * 7 + heads + rd)
    width = heads * hd
    x = rng.normal(0, 1, (rows, width + extra)).astype(np.float32)
    held = np.concatenate([np.full(off, 9, np.float32), x.reshape(-1)])
    desc = hip.RopeDesc(hd, rd, style, base, scaling.get("scaling", 0), scaling.get("factor", 1.0),
                        scaling.get("orig", 0), scaling.get("low", 1.0), scaling.get("high", 32.0), magnitude)
    src = ctx.buffer(held)
    dst = src if in_place else ctx.buffer(np.full(off + rows * (width + extra), 7, np.float32))
    at = np.arange(first, first + rows, dtype=np.uint32) if positions is None else positions.astype(np.uint32)
    ctx.rope_rows(desc, src, dst, rows, heads, positions=None if positions is None else ctx.buffer(at),
                  first_position=first, src_stride=width + extra, dst_stride=width + extra, src_off=4 * off,
                  dst_off=4 * off, freq_factors=None if factors is None else ctx.buffer(factors))
    got = dst.read(np.float32)
    f = oracle.rope_frequencies(rd, base, **scaling)
    if factors is not None:
        f = f / factors.astype(np.float64)
    want, size = oracle.rope(x[:, :width].reshape(rows, heads, hd), at, f, rd, style, magnitude)
    inner = got[off:].reshape(rows, -1)
    assert np.all(got[:off] == (9 if in_place else 7))
    if extra:  # what lies between the rows stays
        assert np.array_equal(inner[:, width:], x[:, width:] if in_place else np.full((rows, extra), 7, np.float32))
    err = np.abs(inner[:, :width].reshape(want.shape) - want)
    assert np.all(err <= 12 * 2.0 ** -24 * size), (err / np.maximum(size, 1e-30)).max()


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("name", list(SCALINGS))
def test_scalings(hip_ctx, style, name):
    rotate(hip_ctx, 5, 40, 128, 128, style, base=500000.0, first=100003, **SCALINGS[name])


@pytest.mark.parametrize("rows,heads,hd,rd,style", [(1, 1, 64, 64, 0), (1, 40, 128, 128, 1), (3, 2, 96, 48, 1),
                                                    (2, 3, 80, 22, 0), (2, 3, 80, 22, 1), (7, 1, 256, 2, 0),
                                                    (7, 5, 256, 250, 1), (4, 2, 512, 512, 0), (4, 2, 512, 6, 1), (3, 7, 2, 2, 0),
                                                    (3, 9, 6, 4, 1), (1100, 40, 128, 128, 0), (2100, 3, 64, 32, 1)])
def test_shapes(hip_ctx, rows, heads, hd, rd, style):
    rotate(hip_ctx, rows, heads, hd, rd, style, first=11)


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("extra,off,in_place", [(0, 0, True), (128, 0, True), (1, 0, False), (3, 1, True), (256, 4, False), (6, 2, False)])
def test_strides_and_offsets(hip_ctx, style, extra, off, in_place):
    rotate(hip_ctx, 9, 5, 64, 64, style, first=3, extra=extra, off=off, in_place=in_place)
    rotate(hip_ctx, 9, 3, 96, 40, style, first=3, extra=extra, off=off, in_place=in_place)


def test_far_positions_in_any_order(hip_ctx):
    at = np.array([0, 1 << 20, 3, 3, (1 << 24) + 1, 999983, 0, 16777215], np.uint32)
    rotate(hip_ctx, at.size, 8, 128, 128, 1, base=1000000.0, positions=at)
    rotate(hip_ctx, at.size, 8, 128, 64, 0, base=10000.0, positions=at, **SCALINGS["yarn"])


@pytest.mark.parametrize("name", ["none", "linear", "bands"])
def test_factors_and_magnitude(hip_ctx, name):
    rd = 48
    factors = np.random.default_rng(5).uniform(1, 8, rd // 2).astype(np.float32)
    rotate(hip_ctx, 6, 4, 96, rd, 1, first=4000, factors=factors, magnitude=1.2079442, **SCALINGS[name])
    rotate(hip_ctx, 6, 4, 96, rd, 0, first=4000, factors=factors, magnitude=-0.5, **SCALINGS[name])


def test_one_position_as_apply_rope(hip_ctx):
    """Without scaling, the rows of the single-position call (whose denominators are 32-bit: 2^-24 of the angle's
    each, so 2 * 2^-24 * position of the pair's size)."""
    heads, hd, at = 4, 64, 1000
    x = np.random.default_rng(1).normal(0, 1, heads * hd).astype(np.float32)
    a, b = hip_ctx.buffer(x), hip_ctx.buffer(x)
    hip_ctx.rope(a, heads, hd, hd, at, 10000.0, 1)
    hip_ctx.rope_rows(hip.RopeDesc(hd, style=1), b, b, 1, heads, first_position=at)
    assert np.max(np.abs(a.read() - b.read())) <= 2 * 2.0 ** -24 * at * 2 * np.abs(x).max()
