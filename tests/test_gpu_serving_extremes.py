"""The operators that serve several sequences at values and sizes far from a model's ordinary ones."""
import numpy as np
import pytest

from tests import serving_oracle as oracle
from tests.test_gpu_kv4_attention import attend

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
