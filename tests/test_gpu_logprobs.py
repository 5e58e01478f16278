"""ziggy_hip_token_logprobs_f32 against a 64-bit form.

Tolerance: an exponential of binary32 is off by 2^-21 of itself (its argument's rounding, 2^-24 of at most 8 in powers of
two where it counts, and its own), the sums are 64-bit, so ln of the sum is off by 2^-21, the log probability by that
and its rounding to binary32, 2^-24 of itself.  The entropy is ln S - T / S, T = sum e d: each term off by 2^-21 of
itself and d's rounding 2^-24, so 2^-20 of sum |e d| / S + |ln S| in all, and its rounding."""
import numpy as np
import pytest

from tests import serving_oracle as oracle

pytestmark = pytest.mark.gpu


def check(ctx, x, tokens, top=0, stride=None, entropy=True):
    rows, vocab = x.shape
    print("logprobs", rows, vocab, top, stride, flush=True)
    held = np.full((rows, stride or vocab), np.nan, np.float32)
    held[:, :vocab] = x
    out, h = (ctx.buffer(np.full(rows + 1, 7, np.float32)) for _ in range(2))
    ids, best = (ctx.buffer(np.full(rows * max(top, 1) + 1, 7, t)) for t in (np.uint32, np.float32))
    ctx.token_logprobs(ctx.buffer(held.reshape(-1)[:(rows - 1) * (stride or vocab) + vocab]), ctx.buffer(np.asarray(tokens, np.uint32)), out, rows, vocab,
                       entropy=h if entropy else None, top=top, top_tokens=ids if top else None, top_logprobs=best if top else None,
                       row_stride=stride or 0)
    y, e, ids, best = out.read(), h.read(), ids.read(np.uint32), best.read()
    assert y[-1] == 7 and e[-1] == 7 and ids[-1] == 7 and best[-1] == 7
    eps = 2.0 ** -21
    for r in range(rows):
        want, entropy64, order, logs = oracle.logprobs(x[r], int(tokens[r]), top)
        near(y[r], want, eps + 2.0 ** -24 * abs(want) if np.isfinite(want) else 0)
        if entropy:
            near(e[r], entropy64, 2 * eps * (2 * abs(entropy64) + 2.0 ** -20) + 2.0 ** -24 * abs(entropy64))
        if top:
            assert np.array_equal(ids[r * top:(r + 1) * top], order), (r, ids[r * top:(r + 1) * top], order)
            for a, b in zip(best[r * top:(r + 1) * top], logs):
                near(a, b, eps + 2.0 ** -24 * abs(b) if np.isfinite(b) else 0)
    if not entropy:
        assert np.all(e == 7)
    return y, e, ids, best


def near(got, want, bound):
    if abs(want) > np.finfo(np.float32).max:
        want = np.copysign(np.inf, want)
    if np.isnan(want) or np.isinf(want):
        assert (np.isnan(got) and np.isnan(want)) or got == want, (got, want)
    else:
        assert abs(got - want) <= bound, (got, want, abs(got - want) / bound)


def logits(rng, rows, vocab, spread=2.0):
    x = (spread * rng.normal(0, 1, (rows, vocab))).astype(np.float32)
    x[np.arange(rows), rng.integers(0, vocab, rows)] = 6
    return x


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 2048, 2049, 4096, 4099, 32000, 128256, 151936, 262144])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_vocabularies(hip_ctx, vocab, top):
    rng = np.random.default_rng(vocab + top)
    for rows in (1, 3):
        x = logits(rng, rows, vocab)
        check(hip_ctx, x, rng.integers(0, vocab, rows), min(top, vocab))


@pytest.mark.parametrize("rows", [2, 17, 64, 255, 256, 300, 1100])
def test_rows(hip_ctx, rows):
    rng = np.random.default_rng(rows)
    x = logits(rng, rows, 777)
    check(hip_ctx, x, rng.integers(0, 777, rows), 5)
    check(hip_ctx, x, rng.integers(0, 777, rows), 0, stride=801)
    check(hip_ctx, x, rng.integers(0, 777, rows), 7, stride=780, entropy=False)


@pytest.mark.parametrize("vocab", [5000, 70001])
def test_ties_go_to_the_lower_id(hip_ctx, vocab):
    rng = np.random.default_rng(1)
    x = np.round(rng.normal(0, 1, (4, vocab)) * 2).astype(np.float32) / 2
    x[1] = 0.5
    x[2] = -np.arange(vocab) // 3
    x[3] = np.arange(vocab) // 3
    check(hip_ctx, x, [0, 1, 2, 3], 50)
    z = np.zeros((1, vocab), np.float32)
    z[0, ::2] = -0.0  # the zeros are equal
    check(hip_ctx, z, [5], 20)


@pytest.mark.parametrize("order", ["up", "down", "up in steps", "last"])
@pytest.mark.parametrize("vocab", [3000, 151936])
def test_orders(hip_ctx, order, vocab):
    """The best last, first, each better than all before it in groups, and all in the row's end."""
    x = {"up": np.arange(vocab), "down": -np.arange(vocab), "up in steps": np.arange(vocab) // 100,
         "last": np.where(np.arange(vocab) >= vocab - 70, 5.0 + np.arange(vocab) % 7, 0.0)}[order]
    check(hip_ctx, (x * 1e-4 if order != "last" else x).astype(np.float32)[None], [vocab // 2], 64)


def test_a_sure_token_keeps_its_digits(hip_ctx):
    """Log probabilities near 0 come from the others' sum, not from a difference with 1."""
    x = np.full((3, 1000), -30.0, np.float32)
    x[:, 7] = [0, 5, 20]
    y, e, _, _ = check(hip_ctx, x, [7, 7, 7])
    want = [-np.log1p(999 * np.exp(-30.0 - v)) for v in (0, 5, 20)]
    assert np.all(np.abs(y[:3] / want - 1) < 2.0 ** -20)


def test_what_is_not_finite(hip_ctx):
    rng = np.random.default_rng(2)
    x = logits(rng, 8, 3001)
    x[0, rng.random(3001) < 0.7] = -np.inf
    x[1, :] = -np.inf
    x[2, :] = np.nan
    x[3, 100] = np.inf
    x[4, rng.random(3001) < 0.5] = np.nan
    x[5, :] = -np.inf
    x[5, 2000] = 1.5
    x[6, :] = np.finfo(np.float32).min
    x[7, :2000] = np.finfo(np.float32).min
    check(hip_ctx, x, [int(np.argmin(x[0])), 0, 1, 100, int(np.flatnonzero(np.isnan(x[4]))[0]), 2000, 9, 0], 30)
    check(hip_ctx, x, [5, 0, 1, 3, 2, 5, 9, 2500], 0)
    y = check(hip_ctx, logits(rng, 3, 500), [500, 0xFFFFFFFF, 499])[0]  # no tokens of the vocabulary
    assert np.isnan(y[:2]).all() and np.isfinite(y[2])


def test_large_logits(hip_ctx):
    rng = np.random.default_rng(3)
    for size in (1e3, 1e30, 3e38):
        check(hip_ctx, (size * rng.uniform(-1, 1, (2, 5000))).astype(np.float32), [3, 4999], 10)
    check(hip_ctx, (1e5 + rng.normal(0, 1, (2, 5000))).astype(np.float32), [3, 4999], 10)


def test_beside_the_sampler(hip_ctx):
    """The greedy token of the sampler is the first of the top tokens."""
    from zhip import hip
    rng = np.random.default_rng(4)
    x = logits(rng, 5, 32000, 1.0)
    x[4, 5:9] = 11.0
    lb, out, u, ids, best, y = (hip_ctx.buffer(x), hip_ctx.empty(20), hip_ctx.buffer(np.zeros(5)), hip_ctx.empty(40), hip_ctx.empty(40), hip_ctx.empty(20))
    hip_ctx.begin()
    hip_ctx.sample_rows(lb, out, u, hip.SamplingOptions(temperature=0.0), 5, 32000)
    hip_ctx.token_logprobs(lb, out, y, 5, 32000, top=2, top_tokens=ids, top_logprobs=best)
    hip_ctx.commit()
    assert np.array_equal(out.read(np.uint32), ids.read(np.uint32)[::2]) and np.array_equal(y.read(), best.read()[::2])


@pytest.mark.parametrize("vocab", [200, 1024, 4096, 4097, 8191, 8192, 8193])
@pytest.mark.parametrize("top", [0, 1, 13, 48, 64])
def test_rows_about_the_size_of_a_slice(hip_ctx, vocab, top):
    """Rows that one workgroup answers, and those that two do: ordinary ones, ties by the hundred, few finite logits, none,
    infinities and NaN among them."""
    rng = np.random.default_rng(vocab * 3 + top)
    x = logits(rng, 10, vocab)
    x[1] = np.round(x[1])
    x[2, :] = -2.5
    x[3, rng.permutation(vocab)[:vocab - 20]] = -np.inf
    x[4, rng.permutation(vocab)[:vocab // 2]] = np.nan
    x[5, :] = -np.inf
    x[6, vocab // 3] = np.inf
    x[7, :] = np.nan
    x[8, :vocab // 2] = 3.0  # (a wavefront's list overflows)
    x[9] = np.sort(x[9])
    check(hip_ctx, x, list(rng.integers(0, vocab, 9)) + [vocab], top, stride=vocab + 3)
