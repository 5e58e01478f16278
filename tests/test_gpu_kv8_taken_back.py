"""The 8-bit cache where rows are taken back, as a verify pass does with its rejected drafts, and its rows against the
values themselves: what a store leaves off, and what later stores into the same block add to it."""
import numpy as np
import pytest

from tests import longctx_oracle as oracle
from zhip import hip

pytestmark = pytest.mark.gpu

B = oracle.BLOCK


def read(ctx, cache, rows, heads, hd):
    out = [ctx.empty(4 * rows * heads * hd) for _ in range(2)]
    ctx.kv8_load(cache, *out, 0, 0, rows)
    return [o.read().reshape(rows, heads, hd) for o in out]


def scales(cache, heads):
    return [cache.buffers[i].read().reshape(heads, -1) for i in (1, 3)]


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (2, 1, 256)])
@pytest.mark.parametrize("spoil", ["large", "inf", "nan"])
def test_rejected_drafts_leave_nothing(hip_ctx, heads, kvh, hd, spoil):
    """Passes of a token and 8 drafts of which 0 to 8 stay, stored from the open block's first position; the rejected
    ones are 50 times as large or not finite.  Each pass attends, which is checked where all rows are finite.  In the
    end the cache is that of the rows that stayed, stored at once, code for code and scale for scale."""
    print("taken back", heads, kvh, hd, spoil, flush=True)
    rng = np.random.default_rng(hd)
    n, context = 0, 260
    kept = [np.zeros((0, kvh, hd), np.float32) for _ in range(2)]
    cache = hip_ctx.kv8_cache(1, kvh, hd, context)
    out = hip_ctx.empty(4 * 9 * heads * hd)
    while n < 230:
        stay = 1 + int(rng.integers(0, 9))
        new = [rng.normal(0, 1, (9, kvh, hd)).astype(np.float32) for _ in range(2)]
        for x in new:
            x[stay:] *= 50
            if spoil != "large" and stay < 9:
                x[stay + int(rng.integers(0, 9 - stay)), :, 3] = np.float32(spoil)
        first = n // B * B
        rows = [np.concatenate([a[first:], b]) for a, b in zip(kept, new)]
        q = rng.normal(0, 1, (9, heads, hd)).astype(np.float32)
        hip_ctx.begin()
        hip_ctx.kv8_store(cache, hip_ctx.buffer(rows[0]), hip_ctx.buffer(rows[1]), 0, first, rows[0].shape[0])
        hip_ctx.kv8_attention(cache, hip_ctx.buffer(q), out, heads, 0, n, 9)
        hip_ctx.commit()
        if spoil == "large" or stay == 9:
            plain = oracle.Kv8(kvh, n + 9, hd)
            for lo in range(0, first, B):
                plain.store(kept[0][lo:lo + B], kept[1][lo:lo + B], lo)
            plain.store(rows[0], rows[1], first)
            want, bound = oracle.kv8_attention(plain, q, n, hd ** -0.5)
            err = np.abs(out.read().reshape(want.shape) - want)
            assert np.all(err <= bound), (err / bound).max()
        kept = [np.concatenate([a, b[:stay]]) for a, b in zip(kept, new)]
        n += stay
    first = n // B * B
    if first < n:
        hip_ctx.kv8_store(cache, hip_ctx.buffer(kept[0][first:]), hip_ctx.buffer(kept[1][first:]), 0, first, n - first)
    want = oracle.Kv8(kvh, context, hd)
    want.store(kept[0], kept[1], 0)
    blocks = -(-n // B)
    for w, (got, scale, x) in enumerate(zip(read(hip_ctx, cache, n, kvh, hd), scales(cache, kvh), kept)):
        assert np.array_equal(scale[:, :blocks], want.scales[w][:, :blocks])
        assert np.array_equal(got, want.rows(w, 0, n))
        half = np.repeat(scale[:, :blocks], B, axis=1)[:, :n].T[..., None] / 2
        assert np.all(np.abs(got - x) <= half * (1 + 2.0 ** -14))  # 127 roundings of 2^-23 in the largest code's step


@pytest.mark.parametrize("step", [1, 3, 9])
def test_what_growing_scales_leave_off(hip_ctx, step):
    """Rows stored `step` at a time where the cache ends, 3 of them kept: (1 + g) / 2 of the scale after g growths."""
    rng = np.random.default_rng(step)
    heads, hd, context = 2, 128, 200
    cache = hip_ctx.kv8_cache(1, heads, hd, context)
    kept = [np.zeros((context, heads, hd), np.float32) for _ in range(2)]
    growths = [np.zeros((heads, context), int) for _ in range(2)]
    n, stay = 0, min(step, 3)
    before = scales(cache, heads)
    while n + step <= context:
        new = [(rng.normal(0, 1, (step, heads, hd)) * (1 + n % 11)).astype(np.float32) for _ in range(2)]
        hip_ctx.kv8_store(cache, hip_ctx.buffer(new[0]), hip_ctx.buffer(new[1]), 0, n, step)
        after = scales(cache, heads)
        for w in range(2):
            b = n // B
            grew = after[w][:, b] > before[w][:, b]
            growths[w][grew, b * B:n] += 1
            growths[w][:, n:] = 0
            kept[w][n:n + step] = new[w]
        n, before = n + stay, after
    for w, (got, scale) in enumerate(zip(read(hip_ctx, cache, n, heads, hd), before)):
        unit = np.repeat(scale, B, axis=1)[:, :n]
        bound = ((1 + growths[w][:, :n]) / 2 * unit).T[..., None] * (1 + 2.0 ** -14)
        err = np.abs(got - kept[w][:n])
        assert np.all(err <= bound), (err / bound).max()
        assert growths[w].max() >= 2
