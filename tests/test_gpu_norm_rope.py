"""ziggy_hip_norm_rope_rows_f32 against a 64-bit form: query and key heads with their own weights, both pairings, part of
the head, odd shapes, offsets and strides off the vector loads' alignment, in place.

Tolerance: sine and cosine are rounded once from 64 bits, 2^-24, the norm's factor and the weight's sum with the
offset 2^-24 each, their product and the head's with it 2^-24 each, the two products and the sum of the rotation 2^-24
each: 8 2^-24 of (|x0| + |x1|) times the magnitude and the weights, x0 and x1 the normalised values.  The angle is a
product in 64 bits: the position (exact) times a frequency f = base^(-2 i / rd), which the kernel and the form here
each have to (4 + |log2 f|) 2^-53 of itself (the exponent's rounding, 2^-53 of log2 f, the power's own, the two products
with 1 / 2 pi and the position): the pair may be turned by position f (8 + 2 |log2 f|) 2^-53 more, 3 10^-8 at
position 10^7, and 4 10^-6 at 2^32, where a rotation's own angle has no more digits in 64 bits."""
import numpy as np
import pytest

from tests import serving_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu


def turn(ctx, rows, q_heads, k_heads, hd, rd, style, base=10000.0, first=0, positions=None, factors=None, magnitude=1.0,
         q_norm=True, k_norm=True, eps=1e-6, offset=0.0, extra=0, off=0, in_place=False, size=1.0, **scaling):
    print("norm rope", rows, q_heads, k_heads, hd, rd, style, extra, off, in_place, flush=True)
    rng = np.random.default_rng(rows * 7 + q_heads + rd)
    heads = q_heads + k_heads
    width = heads * hd
    x = (size * rng.normal(0, 1, (rows, width + extra))).astype(np.float32)
    held = np.concatenate([np.full(off, 9, np.float32), x.reshape(-1)])
    weights = [rng.normal(1 - offset, 0.2, hd).astype(np.float32) if n else None for n in (q_norm, k_norm)]
    desc = hip.RopeDesc(hd, rd, style, base, scaling.get("scaling", 0), scaling.get("factor", 1.0), scaling.get("orig", 0),
                        scaling.get("low", 1.0), scaling.get("high", 32.0), magnitude)
    heads_desc = hip.Heads(desc, *(ctx.buffer(w) if w is not None else None for w in weights), eps=eps, weight_offset=offset,
                           freq_factors=None if factors is None else ctx.buffer(factors))
    src = ctx.buffer(held)
    dst = src if in_place else ctx.buffer(np.full(off + rows * (width + extra), 7, np.float32))
    at = np.arange(first, first + rows, dtype=np.uint32) if positions is None else positions.astype(np.uint32)
    ctx.norm_rope_rows(heads_desc, src, dst, rows, q_heads, k_heads, positions=None if positions is None else ctx.buffer(at),
                       first_position=first, src_stride=width + extra, dst_stride=width + extra, src_off=4 * off, dst_off=4 * off)
    got = dst.read(np.float32)
    f = oracle.rope_frequencies(rd, base, **scaling)
    if factors is not None:
        f = f / factors.astype(np.float64)
    y = x[:, :width].reshape(rows, heads, hd)
    y = np.concatenate([oracle.norm(y[:, :q_heads], weights[0], eps, offset), oracle.norm(y[:, q_heads:], weights[1], eps, offset)], axis=1)
    want, pair = oracle.rope(y, at, f, rd, style, magnitude)
    pair = np.maximum(pair, np.abs(want))
    inner = got[off:].reshape(rows, -1)
    assert np.all(got[:off] == (9 if in_place else 7))
    if extra:  # what lies between the rows stays
        assert np.array_equal(inner[:, width:], x[:, width:] if in_place else np.full((rows, extra), 7, np.float32))
    inner = inner[:, :width].reshape(want.shape)
    assert np.array_equal(np.isnan(inner), np.isnan(want))
    err = np.abs(inner - want)[~np.isnan(want)]
    angle = at.astype(np.float64)[:, None] * f * (8 + 2 * np.abs(np.log2(f))) * 2.0 ** -53
    bound = ((8 * 2.0 ** -24 + angle.max(axis=1)[:, None, None]) * pair + 2.0 ** -149)[~np.isnan(want)]
    assert np.all(err <= bound), (err / bound).max()


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("rows,q_heads,k_heads,hd,rd", [
    (1, 1, 0, 64, 64), (1, 0, 1, 64, 64), (1, 32, 8, 128, 128), (3, 2, 1, 96, 48), (2, 3, 2, 80, 22), (7, 1, 1, 256, 2), (7, 5, 3, 256, 250),
    (4, 2, 1, 512, 512), (4, 2, 1, 512, 6), (3, 7, 2, 2, 2), (3, 9, 1, 6, 4), (900, 32, 8, 128, 128), (2100, 3, 1, 64, 32), (5, 300, 17, 128, 128)])
def test_shapes(hip_ctx, style, rows, q_heads, k_heads, hd, rd):
    turn(hip_ctx, rows, q_heads, k_heads, hd, rd, style, first=11)


@pytest.mark.parametrize("q_norm,k_norm", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("style", [0, 1])
def test_heads_without_norms(hip_ctx, style, q_norm, k_norm):
    turn(hip_ctx, 5, 6, 2, 128, 128, style, first=100003, base=500000.0, q_norm=q_norm, k_norm=k_norm)


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("extra,off,in_place", [(0, 0, True), (128, 0, True), (1, 0, False), (3, 1, True), (256, 4, False), (6, 2, False)])
def test_strides_and_offsets(hip_ctx, style, extra, off, in_place):
    turn(hip_ctx, 9, 5, 2, 64, 64, style, first=3, extra=extra, off=off, in_place=in_place)
    turn(hip_ctx, 9, 3, 1, 96, 40, style, first=3, extra=extra, off=off, in_place=in_place)


@pytest.mark.parametrize("scaling", [dict(scaling=hip.ROPE_LINEAR, factor=4.0), dict(scaling=hip.ROPE_YARN, factor=4.0, orig=32768),
                                     dict(scaling=hip.ROPE_BANDS, factor=8.0, orig=8192, low=1.0, high=4.0)])
def test_scalings_factors_and_offset(hip_ctx, scaling):
    factors = np.random.default_rng(5).uniform(1, 8, 24).astype(np.float32)
    turn(hip_ctx, 6, 4, 2, 96, 48, 1, first=4000, factors=factors, magnitude=1.2079442, offset=1.0, **scaling)
    turn(hip_ctx, 6, 4, 2, 96, 48, 0, first=4000, factors=factors, magnitude=-0.5, eps=0.3, **scaling)


def test_far_positions_in_any_order(hip_ctx):
    at = np.array([0, 1 << 20, 3, 3, (1 << 24) + 1, 999983, 0, 0xFFFFFFFF], np.uint32)
    turn(hip_ctx, at.size, 8, 2, 128, 128, 1, base=1000000.0, positions=at)


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e18, 1e30])
def test_sizes_whose_squares_pass_binary32(hip_ctx, size):
    turn(hip_ctx, 4, 3, 1, 128, 128, 1, first=9, size=size)
    turn(hip_ctx, 4, 3, 1, 128, 64, 0, first=9, size=size, eps=0.0)


def test_zero_and_bad_heads_stay_their_own(hip_ctx):
    """A head of zeros (eps alone below the root), and heads with an infinity or a NaN, beside ordinary ones."""
    heads, hd = 5, 64
    x = np.random.default_rng(0).normal(0, 1, (2, heads, hd)).astype(np.float32)
    x[0, 1], x[0, 2, 5], x[1, 3, 7] = 0, np.inf, np.nan
    w = np.ones(hd, np.float32)
    d = hip.Heads(hip.RopeDesc(hd, style=1), hip_ctx.buffer(w), hip_ctx.buffer(w))
    a = hip_ctx.buffer(x)
    hip_ctx.norm_rope_rows(d, a, a, 2, 3, 2, first_position=5)
    got = a.read().reshape(x.shape)
    assert np.all(got[0, 1] == 0) and np.isnan(got[1, 3]).all() and np.isnan(got[0, 2]).any()
    fine = np.ones((2, heads), bool)
    fine[0, 1:3] = fine[1, 3] = False
    want, pair = oracle.rope(oracle.norm(x, w), np.array([5, 6]), oracle.rope_frequencies(hd, 10000.0), hd, 1)
    assert np.all(np.abs(got - want)[fine] <= 8 * 2.0 ** -24 * pair[fine])


def test_as_the_two_calls_one_after_the_other(hip_ctx):
    """ziggy_hip_rms_norm_per_head_f32, then ziggy_hip_rope_rows_f32: their roundings (the norm's sum of squares in
    binary32, 128 2^-24 / 2 of the factor at most) beside these."""
    heads, hd = 6, 128
    rng = np.random.default_rng(3)
    x, w = rng.normal(0, 1, (1, heads * hd)).astype(np.float32), rng.normal(1, 0.2, hd).astype(np.float32)
    a, b, wb = hip_ctx.buffer(x), hip_ctx.empty(x.nbytes), hip_ctx.buffer(w)
    rope = hip.RopeDesc(hd, style=1, base=1000000.0)
    hip_ctx.rms_norm_per_head(a, wb, b, heads, hd, 1e-6)
    hip_ctx.rope_rows(rope, b, b, 1, heads, first_position=77)
    hip_ctx.norm_rope_rows(hip.Heads(rope, wb, wb), a, a, 1, 4, 2, first_position=77)
    assert np.max(np.abs(a.read() - b.read())) <= (64 + 24) * 2.0 ** -24 * 2 * np.abs(b.read()).max()
