"""The long-context operators together, as a decoding loop uses them: rotate, store, attend, project, draw, each
step's calls in one open sequence; and the session's step that draws on the device."""
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import zo
from tests import longctx_oracle as oracle
from zhip import hip, synth
from zhip.hip import SamplingOptions

pytestmark = pytest.mark.gpu

F32 = 0


@pytest.mark.parametrize("heads,kvh,hd,style,scaling", [(8, 2, 128, 1, "yarn"), (4, 4, 64, 0, "bands"), (6, 2, 96, 1, "linear")])
def test_a_prompt_and_decoding_steps(hip_ctx, heads, kvh, hd, style, scaling):
    """A prompt of 75 rows, then 40 tokens, each drawn from the one before.  Every operator's result is checked
    against its 64-bit form on what the device gave it, the cache code for code."""
    rng = np.random.default_rng(hd)
    ctx_len, vocab, prompt, base = 130, 777, 75, 500000.0
    kw = {"yarn": dict(scaling=hip.ROPE_YARN, factor=4.0, orig=64, low=1.0, high=8.0),
          "bands": dict(scaling=hip.ROPE_BANDS, factor=8.0, orig=64, low=1.0, high=4.0),
          "linear": dict(scaling=hip.ROPE_LINEAR, factor=2.0)}[scaling]
    desc = hip.RopeDesc(hd, hd, style, base, kw["scaling"], kw["factor"], kw.get("orig", 0), kw.get("low", 1.0),
                        kw.get("high", 32.0))
    f = oracle.rope_frequencies(hd, base, **kw)
    wq, wk = heads * hd, kvh * hd
    width = wq + 2 * wk
    table = rng.normal(0, 1, (vocab, width)).astype(np.float32)  # a token's q, k and v side by side
    head = (rng.normal(0, 1, (vocab, wq)) / 8).astype(np.float32)
    o = SamplingOptions(temperature=0.9, repeat_penalty=1.2, top_k=50, top_p=0.95, min_p=0.01)
    cache = hip_ctx.kv8_cache(2, kvh, hd, ctx_len)
    plain = [oracle.Kv8(kvh, ctx_len, hd) for _ in range(2)]
    hb = hip_ctx.buffer(head)
    out = hip_ctx.empty(4 * prompt * wq)
    lg, tok, u = hip_ctx.empty(4 * vocab), hip_ctx.empty(4), hip_ctx.empty(8)
    last = hip_ctx.empty(4 * wq)
    tokens = [int(t) for t in rng.integers(0, vocab, prompt)]
    position, rows = 0, prompt
    for step in range(41):
        xs = table[tokens[position:position + rows]]
        x = hip_ctx.buffer(xs)
        draw = float(rng.random())
        u.write(np.array([draw]))
        recent = np.array(tokens[-32:], np.uint32)
        rb = hip_ctx.buffer(recent)
        hip_ctx.begin()
        hip_ctx.rope_rows(desc, x, x, rows, heads + kvh, first_position=position, src_stride=width, dst_stride=width)
        hip_ctx.kv8_store(cache, x, x, 1, position, rows, row_stride=width, k_off=4 * wq, v_off=4 * (wq + wk))
        hip_ctx.kv8_attention(cache, x, out, heads, 1, position, rows, q_stride=width)
        hip_ctx.copy(out, 4 * (rows - 1) * wq, last, 0, 4 * wq)
        hip_ctx.matvec(F32, hb, last, lg, vocab, wq)
        hip_ctx.sample_rows(lg, tok, u, o, 1, vocab, recent=rb, recent_count=recent.size)
        hip_ctx.commit()
        after = x.read().reshape(rows, width)
        assert np.array_equal(after[:, wq + wk:], xs[:, wq + wk:])
        got = after[:, :wq + wk].reshape(rows, heads + kvh, hd)
        want, size = oracle.rope(xs[:, :wq + wk].reshape(rows, heads + kvh, hd), np.arange(position, position + rows), f, hd, style)
        assert np.all(np.abs(got - want) <= 12 * 2.0 ** -24 * size)
        plain[1].store(np.ascontiguousarray(got[:, heads:]), xs[:, wq + wk:].reshape(rows, kvh, hd), position)
        n = position + rows
        for w, at in ((0, "k"), (1, "v")):
            assert np.array_equal(cache.buffers[2 * w + 1].read().reshape(2, kvh, -1)[1][:, :-(-n // 32)],
                                  plain[1].scales[w][:, :-(-n // 32)]), at
        y, bound = oracle.kv8_attention(plain[1], got[:, :heads], position, hd ** -0.5)
        mine = out.read()[:rows * wq].reshape(y.shape)
        assert np.all(np.abs(mine - y) <= bound)
        logits = lg.read()
        assert np.allclose(logits, head.astype(np.float64) @ mine[-1].reshape(-1), rtol=0, atol=1e-4)
        t = int(tok.read(np.uint32)[0])
        assert t == oracle.sample(logits, draw, 0.9, 50, 0.95, 0.01, 1.2, recent)
        assert t == hip.sample_logits(logits, recent, o, draw)
        tokens.append(t)
        position, rows = n, 1
    # the cache's layer 0 was never touched, layer 1 holds what the plain form stored
    kc = cache.buffers[0].read(np.int8).reshape(2, kvh, -1, hd)
    assert not kc[0].any() and np.array_equal(kc[1][:, :position], plain[1].codes[0][:, :position])


STREAMS = [dict(temperature=0.8, top_k=40, top_p=0.9, repeat_penalty=1.1), dict(temperature=1.2, top_p=0.8),
           dict(temperature=1.0, min_p=0.05, repeat_penalty=1.3), dict(temperature=0.9, top_k=500), dict(temperature=0.0)]


@pytest.mark.parametrize("kw", STREAMS, ids=str)
def test_session_step_sample_streams(hip_ctx, kw):
    """24 steps: the tokens that the host sampler draws from the session's own logits, and, of at most 40 candidates,
    those that it draws from the oracle's.  (Not of more: the oracle's logits are up to 1e-4 of their size away, which
    moves the borders between thousands of tokens of like weight by about 1e-4 of the whole, a border lying every
    3e-4 of it: a draw in three or so falls between.)"""
    spec = synth.small_spec(vocab=4000)
    img = synth.build(spec, seed=43)
    prompt = [int(t) for t in synth.prompt_tokens(4, 9, spec.vocab)]
    o = SamplingOptions(**kw)
    draws = np.random.default_rng(2025).random(24)
    few = 0 < o.top_k <= 40 or o.temperature == 0
    ref = zo.Session(zo.Model(img.buf), context=spec.context, kv_f16=True)
    for t in prompt[:-1]:
        ref.step_no_output(t)
    s = hip.Session(hip_ctx, img, context=spec.context)
    s.generate(np.array(prompt[:-1], np.uint32), 0)
    hist, tok = list(prompt), prompt[-1]
    for u in draws:
        got = s.step_sample(tok, hist, o, float(u))
        assert got == hip.sample_logits(s.logits(), hist, o, float(u))
        if few:
            assert got == hip.sample_logits(ref.step(tok), hist, o, float(u))
        tok = got
        hist.append(tok)
    assert s.position == len(hist) - 1
    s.close()


def test_session_step_sample_with_a_long_history(hip_ctx):
    """More recent tokens than the pinned words hold, and a list that grows from call to call."""
    spec = synth.small_spec(vocab=300)
    img = synth.build(spec, seed=11)
    s = hip.Session(hip_ctx, img, context=spec.context)
    o = SamplingOptions(temperature=1.0, repeat_penalty=1.5)
    rng = np.random.default_rng(3)
    tok = 1
    for n in (0, 5, 4097, 64503, 64504, 64505, 100000, 3):
        recent = rng.integers(0, 40, n).astype(np.uint32)
        u = float(rng.random())
        got = s.step_sample(tok, recent, o, u)
        assert got == hip.sample_logits(s.logits(), recent, o, u)
        tok = got
    s.close()


def test_session_step_sample_refusals(hip_ctx):
    spec = synth.small_spec(vocab=3000)
    img = synth.build(spec, seed=11)
    s = hip.Session(hip_ctx, img, context=spec.context)
    good = dict(temperature=1.0)
    for kw, u, token in ((dict(good, top_k=1025), 0.5, 1), (dict(good, top_p=2.0), 0.5, 1), (dict(good, min_p=-1.0), 0.5, 1),
                         (dict(temperature=float("nan")), 0.5, 1), (good, 1.0, 1), (good, -0.1, 1), (good, float("nan"), 1), (good, 0.5, 3000)):
        with pytest.raises(hip.HipError) as e:
            s.step_sample(token, [], SamplingOptions(**kw), u)
        assert e.value.status == 6 and s.position == 0
    assert 0 <= s.step_sample(1, [], SamplingOptions(**good), 0.5) < 3000 and s.position == 1
    s.close()


WRAP = """
import sys
sys.path[:0] = [{repo!r}, {repo!r} + "/ziggy-llm_amd"]
import torch
x = torch.arange(2 * 64, dtype=torch.float32, device="cuda").reshape(2, 64)
y = torch.zeros(3, 64, device="cuda")
torch.cuda.synchronize()
import numpy as np
from tests import longctx_oracle as oracle
from zhip import hip
ctx = hip.Context(0)
a, b = ctx.wrap(x.data_ptr(), x.numel() * 4), ctx.wrap(y[1:].data_ptr(), 2 * 64 * 4)
ctx.rope_rows(hip.RopeDesc(64), a, b, 2, 1)
want, size = oracle.rope(x.cpu().numpy().reshape(2, 1, 64), np.arange(2), oracle.rope_frequencies(64, 10000.0), 64, 0)
assert np.all(np.abs(y[1:].cpu().numpy().reshape(want.shape) - want) <= 12 * 2.0 ** -24 * size)
assert not y[0].any()
assert np.array_equal(a.read(), x.cpu().numpy().reshape(-1))
a.free()
b.free()
assert float(x.sum()) == 128 * 127 / 2
host = torch.zeros(64)
for at, n in ((host.data_ptr(), 256), (0, 16), (x.data_ptr() + 4, 16), (x.data_ptr(), 1 << 40)):
    try:
        ctx.wrap(at, n)
    except hip.HipError as e:
        assert e.status == 6
    else:
        raise AssertionError((at, n))
ctx.close()
print("wrapped ok")
"""


def test_wrapped_device_memory():
    """Operators on torch's tensors; freeing the buffer leaves them alone, host memory and lengths past the allocation
    are refused.  In a process of its own: torch brings its HIP runtime, which has to be the first one loaded."""
    pytest.importorskip("torch")
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", WRAP.format(repo=repo)], capture_output=True, text=True, timeout=100, cwd=repo)
    assert r.returncode == 0 and "wrapped ok" in r.stdout, r.stderr[-2000:]


def test_two_contexts_at_once():
    """Two threads, a context each, the same steps in sequences of their own: the outputs of either are those of a
    context by itself (attention's splits and sampling share a context's workspace, not another's)."""
    import threading
    rng = np.random.default_rng(11)
    heads, kvh, hd, n, vocab = 16, 4, 128, 6000, 40000
    k, v = (rng.normal(0, 1, (n, kvh, hd)).astype(np.float32) for _ in range(2))
    q, x = rng.normal(0, 1, (9, heads, hd)).astype(np.float32), rng.normal(0, 3, (3, vocab)).astype(np.float32)
    u, o = rng.random(3), hip.SamplingOptions(temperature=0.9, top_p=0.9)

    def steps(sign, results, start=None):
        ctx = hip.Context(0)
        c = ctx.kv8_cache(1, kvh, hd, n)
        kb, vb, qb, xb, ub = ctx.buffer(k), ctx.buffer(v * np.float32(sign)), ctx.buffer(q), ctx.buffer(x * np.float32(sign)), ctx.buffer(u)
        out, tokens = [ctx.empty(q.nbytes) for _ in range(2)], ctx.empty(12)
        if start:
            start.wait()
        for _ in range(20):
            ctx.begin()
            ctx.kv8_store(c, kb, vb, 0, 0, n)
            ctx.kv8_attention(c, qb, out[0], heads, 0, n - 1)
            ctx.sample_rows(xb, tokens, ub, o, 3, vocab)
            ctx.kv8_attention(c, qb, out[1], heads, 0, n - 9, 9)
            ctx.commit()
            results.append([out[0].read()[:heads * hd], out[1].read(), tokens.read(np.uint32)])
        ctx.close()

    alone, at_once = {1: [], -1: []}, {1: [], -1: []}
    for sign in alone:
        steps(sign, alone[sign])
    start = threading.Barrier(2)
    threads = [threading.Thread(target=steps, args=(sign, at_once[sign], start)) for sign in at_once]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for sign in alone:
        assert len(at_once[sign]) == 20
        for got in at_once[sign] + alone[sign]:
            for a, b in zip(got, alone[sign][0]):
                assert np.array_equal(a, b)
