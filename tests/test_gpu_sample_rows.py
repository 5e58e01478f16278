"""Sampling on the device against the host sampler on the same logits and against a 64-bit form: token for token.
Draws that fall within 1e-9 of a border between two tokens (2^-44 weights: none by chance) are not in these."""
import numpy as np
import pytest

from tests import longctx_oracle as oracle
from zhip import hip
from zhip.hip import SamplingOptions

pytestmark = pytest.mark.gpu


def draw(ctx, x, u, o, recent=None, stride=None):
    """Tokens of logits x [rows, vocab]."""
    rows, vocab = x.shape
    stride = stride or vocab
    held = np.full(rows * stride, 1e30, np.float32)
    held[np.arange(rows)[:, None] * stride + np.arange(vocab)] = x
    out = ctx.buffer(np.full(rows + 3, 77, np.uint32))
    rec = None if recent is None else np.ascontiguousarray(recent, np.uint32)
    ctx.sample_rows(ctx.buffer(held), out, ctx.buffer(np.ascontiguousarray(u, np.float64)), o, rows, vocab,
                    recent=None if rec is None else ctx.buffer(rec), recent_count=0 if rec is None else rec.shape[1],
                    row_stride=stride)
    got = out.read(np.uint32)
    assert np.all(got[rows:] == 77)
    return got[:rows]


def check(ctx, x, u, kw, recent=None, host=True, stride=None):
    print("sample", x.shape, kw, flush=True)
    o = SamplingOptions(temperature=kw.get("temperature", 1.0), repeat_penalty=kw.get("penalty", 1.0),
                        top_k=kw.get("top_k", 0), top_p=kw.get("top_p", 1.0), min_p=kw.get("min_p", 0.0))
    got = draw(ctx, x, u, o, recent, stride)
    for r in range(x.shape[0]):
        rec = [] if recent is None else [t for t in recent[r] if t < x.shape[1]]
        want = oracle.sample(x[r], u[r], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0),
                             kw.get("min_p", 0.0), kw.get("penalty", 1.0), rec)
        assert got[r] == want, (r, got[r], want)
        if host:
            assert got[r] == hip.sample_logits(x[r], rec, o, float(u[r]))


def logits(rng, rows, vocab, size=3.0):
    return rng.normal(0, size, (rows, vocab)).astype(np.float32)


POLICIES = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_k=40, top_p=0.9), dict(top_p=0.9),
            dict(top_p=0.5, temperature=1.7), dict(min_p=0.1), dict(min_p=0.05, top_p=0.8, top_k=100, temperature=1.3),
            dict(top_k=1024, temperature=2.0), dict(top_k=1000, top_p=0.99, temperature=3.0), dict(top_p=0.0), dict(min_p=1.0),
            dict(temperature=0.0), dict(temperature=-1.0, top_k=5), dict(top_p=0.97, min_p=0.002), dict(temperature=0.01)]


@pytest.mark.parametrize("kw", POLICIES, ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 37, 64, 65, 1000, 4097, 32000])
def test_policies(hip_ctx, kw, vocab):
    rng = np.random.default_rng(vocab)
    check(hip_ctx, logits(rng, 5, vocab), rng.random(5), kw)


@pytest.mark.parametrize("kw", [dict(top_k=40, top_p=0.9, temperature=0.8), dict(top_p=0.95), dict(), dict(min_p=0.02, top_p=0.9), dict(top_k=1024)], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (3, 151936), (2, 262144), (40, 70001)])
def test_large_vocabularies(hip_ctx, kw, rows, vocab):
    rng = np.random.default_rng(rows)
    check(hip_ctx, logits(rng, rows, vocab, 2.0), rng.random(rows), kw, host=rows < 4 or kw.get("top_k", 0) == 0)


@pytest.mark.parametrize("kw", [k for k in POLICIES if k.get("temperature", 1) > 0], ids=str)
def test_repeat_penalty(hip_ctx, kw):
    rng = np.random.default_rng(17)
    rows, vocab = 6, 5000
    x = logits(rng, rows, vocab)
    best = np.argsort(-x, axis=1)
    recent = np.concatenate([best[:, :6], best[:, 10:14], best[:, -3:], rng.integers(0, vocab, (rows, 60)),
                             np.full((rows, 3), 0xFFFFFFFF), np.full((rows, 1), vocab), best[:, :2]], axis=1).astype(np.uint32)
    check(hip_ctx, x, rng.random(rows), dict(kw, penalty=1.3), recent)
    check(hip_ctx, x, rng.random(rows), dict(kw, penalty=0.5), recent)  # at most 1: none, as on the host


@pytest.mark.parametrize("kw", POLICIES, ids=str)
def test_ties(hip_ctx, kw):
    """Rows of few distinct logits, and of one: ties go to the lower token id."""
    rng = np.random.default_rng(23)
    x = rng.integers(-3, 4, (4, 3000)).astype(np.float32)
    x[2] = -1.5
    x[3] = np.where(rng.random(3000) < 0.5, 0.0, -0.0)
    check(hip_ctx, x, np.array([0.013, 0.77, 0.35617, 0.6113]), kw)


@pytest.mark.parametrize("kw", [k for k in POLICIES if k.get("temperature", 1) > 0], ids=str)
def test_thousands_of_equal_or_near_logits(hip_ctx, kw):
    """Rows whose finest bins hold more than a thousand logits: all equal; quarters; thousands of different values
    within a billionth of the range; the same beside higher ones, with equal ones among them."""
    rng = np.random.default_rng(53)
    n = 60000
    x = np.zeros((5, n), np.float32)
    x[0] = 2.5
    x[1] = np.rint(rng.normal(0, 2, n) * 4) / 4
    x[2] = np.where(rng.random(n) < 0.5, 0.01 * (1 + 1e-4 * rng.random(n)), -10)
    x[3] = np.where(rng.random(n) < 0.7, np.rint(rng.random(n) * 40) * 1e-7, -8)
    x[3, rng.integers(0, n, 300)] = 3 + rng.random(300)
    x[4] = np.where(rng.random(n) < 0.3, -1.0, np.where(rng.random(n) < 0.5, 1.0, 1.0 + 2.0 ** -23))
    for u in ([0.02, 0.5, 0.31, 0.77, 0.64], [0.97, 0.11, 0.9, 0.4, 0.05]):
        check(hip_ctx, x, np.array(u), kw)


@pytest.mark.parametrize("kw", POLICIES, ids=str)
def test_masked_logits(hip_ctx, kw):
    """-infinity where a grammar forbids a token: all but one, all but two, half of them."""
    rng = np.random.default_rng(29)
    x = logits(rng, 4, 2000)
    x[0, np.arange(2000) != 1234] = -np.inf
    x[1, (np.arange(2000) != 7) & (np.arange(2000) != 1999)] = -np.inf
    x[2, ::2] = -np.inf
    x[3, :1500] = np.finfo(np.float32).min
    for u in (0.0, 0.3, 1 - 2.0 ** -53):
        check(hip_ctx, x, np.full(4, u), kw, host=u > 0)


@pytest.mark.parametrize("kw", POLICIES, ids=str)
def test_rows_without_a_finite_largest_logit(hip_ctx, kw):
    x = np.zeros((5, 500), np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, [30, 400]] = np.inf
    x[3] = np.nan
    x[3, [40, 60]] = 2.0
    x[4, ::3] = np.nan
    rng = np.random.default_rng(1)
    check(hip_ctx, x, rng.random(5), kw, host=False)
    check(hip_ctx, x[[0, 2]], rng.random(2), kw)


def test_draws_follow_the_softmax(hip_ctx):
    """The tokens of a grid of random numbers: each token's share of the grid is its probability to one step."""
    rng = np.random.default_rng(31)
    x = logits(rng, 1, 50, 1.5)
    rows = 2000
    u = (np.arange(rows) + 0.5) / rows
    got = draw(hip_ctx, np.repeat(x, rows, axis=0), u, SamplingOptions(temperature=1.0))
    p = np.exp(x[0].astype(np.float64) - x.max())
    p /= p.sum()
    share = np.bincount(got, minlength=50) / rows
    assert np.all(np.abs(share - p) <= 1.0 / rows + 1e-9)


def test_random_numbers_out_of_range(hip_ctx):
    rng = np.random.default_rng(37)
    x = logits(rng, 1, 900)
    o = SamplingOptions(temperature=1.0)
    first, last = (draw(hip_ctx, x, [u], o)[0] for u in (0.0, 1 - 2.0 ** -53))
    for u, want in ((-1.0, first), (np.nan, first), (1.0, last), (7.0, last)):
        assert draw(hip_ctx, x, [u], o)[0] == want


def test_strided_rows(hip_ctx):
    rng = np.random.default_rng(41)
    check(hip_ctx, logits(rng, 7, 1003), rng.random(7), dict(top_p=0.9), stride=1010)
    check(hip_ctx, logits(rng, 7, 1003), rng.random(7), dict(top_k=9), stride=1003)


def test_many_rows(hip_ctx):
    """More rows than the workspace holds at a time."""
    rng = np.random.default_rng(43)
    x = logits(rng, 70, 262144, 1.0)
    check(hip_ctx, x, rng.random(70), dict(top_p=0.8), host=False)


def test_same_tokens_each_time(hip_ctx):
    rng = np.random.default_rng(47)
    x, u = logits(rng, 16, 50000, 1.0), rng.random(16)
    o = SamplingOptions(temperature=1.5, top_p=0.98)
    xb, ub, out, other = hip_ctx.buffer(x), hip_ctx.buffer(u), hip_ctx.empty(64), hip_ctx.empty(64)
    want = draw(hip_ctx, x, u, o)
    hip_ctx.begin()
    for _ in range(20):
        hip_ctx.sample_rows(xb, other, ub, SamplingOptions(temperature=0.9, top_k=30), 16, 50000)
        hip_ctx.sample_rows(xb, out, ub, o, 16, 50000)
    hip_ctx.commit()
    assert np.array_equal(out.read(np.uint32), want)


def test_a_penalty_that_leaves_no_finite_logit(hip_ctx):
    """Logits that the penalty takes to -infinity, all of them: the first, as on the host."""
    x = np.full((1, 40), -3e38, np.float32)
    x[0, 7] = -2.9e38
    for kw in (dict(), dict(top_p=0.9), dict(top_k=5), dict(top_k=5, top_p=0.5)):
        check(hip_ctx, x, np.array([0.5]), dict(kw, penalty=2.0), np.arange(40, dtype=np.uint32)[None])


@pytest.mark.parametrize("top_k", [1, 2, 62, 63, 64, 65, 66, 127, 128, 129, 511, 513, 1023])
@pytest.mark.parametrize("vocab", [1025, 1100, 3000, 50000])
def test_counts_of_candidates_about_the_widths_of_sorts(hip_ctx, top_k, vocab):
    rng = np.random.default_rng(top_k + vocab)
    x = logits(rng, 4, vocab)
    x[2] = np.round(x[2] * 8) / 8
    x[3, : vocab // 2] = -np.inf
    recent = np.argsort(-x, axis=1)[:, rng.integers(0, top_k + 3, 90)].astype(np.uint32)
    for kw in (dict(), dict(top_p=0.9, temperature=2.0), dict(top_p=0.8, penalty=1.2), dict(penalty=1.5, temperature=0.6)):
        check(hip_ctx, x, rng.random(4), dict(kw, top_k=top_k), recent)


@pytest.mark.parametrize("equal", [63, 64, 65, 1023, 1024, 1025, 1026, 3000])
def test_counts_of_equal_logits_about_the_widths_of_sorts(hip_ctx, equal):
    """Logits that are equal, or apart by a step of 1, where the nucleus ends and the draw falls."""
    rng = np.random.default_rng(equal)
    vocab = 20000
    x = logits(rng, 3, vocab)
    for r in range(3):
        at = rng.permutation(vocab)[:equal]
        x[r, at] = 14.0
        if r == 1:
            x[r, at] = (np.float32(14).view(np.uint32) + np.arange(equal)).astype(np.uint32).view(np.float32)
    for kw in (dict(top_p=0.5), dict(top_p=0.999), dict(top_p=0.9, min_p=0.3), dict(top_k=1000, top_p=0.7)):
        check(hip_ctx, x, rng.random(3), kw)
