"""ziggy_hip_token_logprobs_f32 of more rows than its workspace holds at once."""
import numpy as np
import pytest

from tests.test_gpu_logprobs import check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,top", [(62700, 8193, 64), (131000, 100, 64), (70001, 300, 5)])
def test_rows_past_the_workspace(hip_ctx, rows, vocab, top):
    """64 MiB of partial results are 62601 rows of two slices with 64 alternatives each: the rest is another pair of launches.
    1021 rows, checked for themselves, come again and again: a row's answer is theirs, whichever launch it is in."""
    print("rows", rows, vocab, top, flush=True)
    rng = np.random.default_rng(vocab)
    period = 1021
    x = logits(rng, period, vocab)
    tokens = rng.integers(0, vocab, period).astype(np.uint32)
    y, e, ids, best = check(hip_ctx, x, tokens, top)
    at = np.arange(rows) % period
    src, given = hip_ctx.buffer(x[at]), hip_ctx.buffer(tokens[at])
    outs = [hip_ctx.buffer(np.full(n + 1, 7, np.float32)) for n in (rows, rows, rows * top, rows * top)]
    hip_ctx.token_logprobs(src, given, outs[0], rows, vocab, entropy=outs[1], top=top, top_tokens=outs[2], top_logprobs=outs[3])
    for b, want in zip(outs, (y, e, ids, best)):
        got = b.read(want.dtype)
        n = 1 if b in outs[:2] else top
        assert got[-1] == np.float32(7).view(want.dtype) if want.dtype == np.uint32 else got[-1] == 7
        assert np.array_equal(got[:-1].reshape(rows, n), want[:period * n].reshape(period, n)[at])
        b.free()
    src.free()
