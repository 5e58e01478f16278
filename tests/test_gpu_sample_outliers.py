"""Sampling from rows with logits far from the others: finite masks, and one far above.  Tokens as the host sampler's
and the 64-bit form's (draws at least 1e-9 from a border), in about the time of a row without them."""
import time

import numpy as np
import pytest

from tests.test_gpu_sample_rows import check
from zhip.hip import SamplingOptions

pytestmark = pytest.mark.gpu

ROWS = {"mask -100": (-100.0, None), "mask -1e4": (-1e4, None), "mask -1e9": (-1e9, None), "mask -2e30": (-2e30, None),
        "high 60": (None, 60.0), "high 1e4": (None, 1e4), "high 1e9": (None, 1e9), "both": (-1e9, 1e5), "high 30 masks": (-1e4, 30.0)}
LIMITS = [dict(top_k=40, top_p=0.9, temperature=0.8), dict(top_k=40), dict(top_k=1000, temperature=1.5, min_p=0.01), dict(top_k=1024, top_p=0.99, temperature=8.0),
          dict(top_k=2), dict(top_k=64, min_p=1.0), dict(top_k=50, temperature=0.01), dict(top_k=7, temperature=100.0), dict(top_p=0.9), dict()]


def rows(rng, count, vocab, mask, high, share=0.5):
    x = rng.normal(0, 2, (count, vocab)).astype(np.float32)
    best = rng.integers(0, vocab, (count, 24))
    for r in range(count):
        x[r, best[r]] = 6 + 4 * rng.normal(0, 1, 24)
    if mask is not None:
        x[rng.random(x.shape) < share] = mask
    if high is not None:
        x[:, vocab // 3] = high
    return x


@pytest.mark.parametrize("kw", LIMITS, ids=str)
@pytest.mark.parametrize("name", list(ROWS))
def test_tokens(hip_ctx, name, kw):
    rng = np.random.default_rng(5)
    x = rows(rng, 4, 30011, *ROWS[name])
    x[1, rng.random(x.shape[1]) < 0.998] = ROWS[name][0] or x[1].min()  # few are left of a row
    check(hip_ctx, x, rng.random(4), kw)
    recent = np.concatenate([np.argsort(-x, axis=1)[:, :30], rng.integers(0, x.shape[1], (4, 40))], axis=1).astype(np.uint32)
    for penalty in (1.1, 3.0):
        check(hip_ctx, x, rng.random(4), dict(kw, penalty=penalty), recent)
        check(hip_ctx, -np.abs(x), rng.random(4), dict(kw, penalty=penalty), recent)


def test_the_largest_logit_penalised_below_all_others(hip_ctx):
    """Every logit above the penalised largest one's reach stays a candidate: 90 / 3 lies below the others' 60 and 55."""
    x = np.full((1, 5000), 50.0, np.float32)
    x[0, 17], x[0, 400], x[0, 401:440] = 90.0, 60.0, 55.0
    recent = np.full((1, 3), 17, np.uint32)
    for u in (0.0, 0.3, 0.999, 1 - 2.0 ** -53):
        for kw in (dict(top_k=50), dict(top_k=50, top_p=0.5), dict(top_k=300, temperature=20.0), dict(top_k=1000, min_p=0.2, temperature=9.0)):
            check(hip_ctx, x, np.array([u]), dict(kw, penalty=3.0), recent, host=u > 0)


@pytest.mark.parametrize("kw", [dict(top_p=0.5), dict(top_k=40, top_p=0.6), dict(top_k=900, top_p=0.8, min_p=0.5), dict(top_p=0.9, temperature=3.0)], ids=str)
def test_logits_whose_weights_are_equal(hip_ctx, kw):
    """Logits of 1e-30: every weight is 1 in 64 bits, the nucleus and the draw go by the logits (the host sampler's by
    the ids)."""
    rng = np.random.default_rng(9)
    check(hip_ctx, (rng.normal(0, 1, (5, 5000)) * 1e-30).astype(np.float32), rng.random(5), kw, host=False)


@pytest.mark.parametrize("top_k", [40, 500])
@pytest.mark.parametrize("name", list(ROWS))
def test_time(hip_ctx, name, top_k):
    """Within twice the time of the rows without (before top-k left out what has no weight: up to 13 and 23 times).
    Least of several runs of ten calls each."""
    vocab, o = 128256, SamplingOptions(temperature=0.8, top_k=top_k, top_p=0.9, repeat_penalty=1.1)
    rng = np.random.default_rng(3)
    u, out = hip_ctx.buffer(rng.random(1)), hip_ctx.empty(4)
    recent = hip_ctx.buffer(rng.integers(0, vocab, 512).astype(np.uint32))
    logits = [hip_ctx.buffer(rows(rng, 1, vocab, *ROWS[name])), hip_ctx.buffer(rows(rng, 1, vocab, None, None))]
    least = [np.inf, np.inf]
    for _ in range(12):
        for i, x in enumerate(logits):
            t = time.perf_counter()
            hip_ctx.begin()
            for _ in range(10):
                hip_ctx.sample_rows(x, out, u, o, 1, vocab, recent=recent, recent_count=512)
            hip_ctx.commit()
            least[i] = min(least[i], time.perf_counter() - t)
    assert least[0] <= 2 * least[1], least
