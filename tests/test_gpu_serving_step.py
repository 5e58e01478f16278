"""The operators that serve several sequences together, as a serving loop uses them: heads normalised and rotated, K/V
appended to pages, attention, the output head, a draw, its log probabilities, each step's calls in one open sequence."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

from tests import longctx_oracle
from tests import serving_oracle as oracle
from zhip import hip
from zhip.hip import SamplingOptions

pytestmark = pytest.mark.gpu

F32 = 0
NONE = 0xFFFFFFFF


class Pool:
    """A pool's free pages, and whose are whose: tables in the order in which pages come free."""

    def __init__(self, rng, pages, per_sequence):
        self.free, self.per_sequence = list(rng.permutation(pages)), per_sequence

    def grow(self, pages, length):
        while len(pages) * oracle.PAGE < length:
            pages.append(int(self.free.pop()))

    def batch(self, rows, lengths, pages):
        b = oracle.Batch.__new__(oracle.Batch)
        b.rows, b.lengths = list(rows), list(lengths)
        b.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        b.table = np.full((len(rows), self.per_sequence), NONE, np.uint32)
        for i, p in enumerate(pages):
            b.table[i, :len(p)] = p
        b.n = int(b.starts[-1])
        return b


def heads_of(ctx, rng, hd, style, norms, base):
    weights = [rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2)] if norms else [None, None]
    desc = hip.Heads(hip.RopeDesc(hd, hd, style, base), *(None if w is None else ctx.buffer(w) for w in weights))
    f = oracle.rope_frequencies(hd, base)

    def turn(x, at, w):  # (turned heads in 64 bits, what their roundings are relative to)
        y, pair = oracle.rope(oracle.norm(x, weights[w]), at, f, hd, style)
        return y, np.maximum(pair, np.abs(y))
    return desc, turn


def log_probabilities_agree(logits, tokens, out, entropy, ids, best, top):
    for r in range(len(tokens)):
        want, h, order, logs = oracle.logprobs(logits[r], int(tokens[r]), top)
        eps = 2.0 ** -21  # (of the exponentials' sum; then the roundings to binary32)
        assert abs(out[r] - want) <= eps + 2.0 ** -24 * abs(want)
        assert abs(entropy[r] - h) <= 2 * eps * (2 * abs(h) + 2.0 ** -20) + 2.0 ** -24 * abs(h)
        assert np.array_equal(ids[r], order) and np.all(np.abs(best[r] - logs) <= eps + 2.0 ** -24 * np.abs(logs))


@pytest.mark.parametrize("heads,kvh,hd,style,norms", [(8, 2, 128, 1, True), (4, 4, 64, 0, False), (6, 2, 96, 1, True), (2, 1, 256, 0, True)])
def test_prompts_and_decoding_steps(hip_ctx, heads, kvh, hd, style, norms):
    """Four sequences over 14 steps: prompts of their own lengths, two of which share their first page; then tokens, each
    drawn from the one before; one ends, and its pages are another's; one takes tokens in threes and gives some back."""
    rng = np.random.default_rng(hd + heads)
    vocab, top, layers = 700, 6, 2
    wq, wk = heads * hd, kvh * hd
    width = wq + 2 * wk
    desc, turn = heads_of(hip_ctx, rng, hd, style, norms, 500000.0)
    table = rng.normal(0, 1, (layers, vocab, width)).astype(np.float32)  # a token's q, k and v side by side
    head = (rng.normal(0, 1, (vocab, wq)) / 8).astype(np.float32)
    pool = Pool(rng, 14, 5)
    cache = oracle.Kv4(layers, 14, kvh, hd, rng)
    held = oracle.upload(hip_ctx, cache)
    o = SamplingOptions(temperature=0.9, top_k=50, top_p=0.95)
    prompts = [list(rng.integers(0, vocab, n)) for n in (75, 70, 3, 130)]
    prompts[1][:64] = prompts[0][:64]
    tokens, pages = [list(map(int, p)) for p in prompts], [[], [], [], []]
    stored = [0, 64, 0, 0]  # (the second's first page is the first's)
    pool.grow(pages[0], 75)
    pages[1].append(pages[0][0])
    hb = hip_ctx.buffer(head)
    for step in range(14):
        if step == 6:  # the third ends; a new sequence takes its place and pages
            pool.free.extend(pages[2])
            tokens[2], pages[2], stored[2] = [int(t) for t in rng.integers(0, vocab, 66)], [], 0
        waits = {0: 1, 9: 0}.get(step)  # (the shared page has to be stored ahead; the first waits a step)
        if step in (4, 8):  # two guesses behind the fourth's token
            tokens[3] += [int(t) for t in rng.integers(0, vocab, 2)]
        rows = [0 if s == waits else len(tokens[s]) - stored[s] for s in range(4)]
        lengths = [len(tokens[s]) if s != waits else max(stored[s], 1) for s in range(4)]
        for s in range(4):
            pool.grow(pages[s], lengths[s])
        b = pool.batch(rows, lengths, pages)
        on = b.on(hip_ctx, max_rows=max(rows), max_length=max(lengths))
        places = b.positions()
        ids = [tokens[s][p] for _, s, p in places]
        x = [hip_ctx.buffer(table[l][ids]) for l in range(layers)]
        out = [hip_ctx.buffer(np.full((b.n, wq), 7, np.float32)) for _ in range(layers)]
        lasts = [s for s in range(4) if rows[s]]
        last = [hip_ctx.empty(4 * wq) for _ in lasts]
        own = hip_ctx.empty(4 * b.n * wq)
        lg, tok, u = hip_ctx.empty(4 * len(lasts) * vocab), hip_ctx.empty(4 * len(lasts)), hip_ctx.buffer(rng.random(len(lasts)))
        lp, en = hip_ctx.empty(4 * len(lasts)), hip_ctx.empty(4 * len(lasts))
        ti, tl = hip_ctx.empty(4 * top * len(lasts)), hip_ctx.empty(4 * top * len(lasts))
        hip_ctx.begin()
        for l in range(layers):  # layer 0 turns its queries in place, layer 1 into a buffer of their own
            if l == 0:
                hip_ctx.kv4_append(held, l, on, desc, x[l], 4 * wq, 4 * (wq + wk), width, heads, 0, x[l], 0, width)
                q, q_stride = x[l], width
            else:
                q, q_stride = own, wq
                hip_ctx.kv4_append(held, l, on, desc, x[l], 4 * wq, 4 * (wq + wk), width, heads, 0, q)
            hip_ctx.kv4_attention(held, l, on, q, out[l], heads, 100 if l else 0, q_stride=q_stride)
        for i, s in enumerate(lasts):
            hip_ctx.copy(out[1], 4 * (int(b.starts[s + 1]) - 1) * wq, last[i], 0, 4 * wq)
            hip_ctx.matvec(F32, hb, last[i], lg, vocab, wq, y_off=4 * i * vocab)
        hip_ctx.sample_rows(lg, tok, u, o, len(lasts), vocab)
        hip_ctx.token_logprobs(lg, tok, lp, len(lasts), vocab, en, top, ti, tl)
        hip_ctx.commit()
        at = np.array([p for _, _, p in places])
        for l in range(layers):
            xs = table[l][ids].reshape(b.n, heads + 2 * kvh, hd)
            k, _ = turn(xs[:, heads:heads + kvh], at, 1)
            want, pair = turn(xs[:, :heads], at, 0)
            for r, s, p in places:
                cache.put(l, *b.place(s, p), k[r].astype(np.float32), xs[r, heads + kvh:])
            if l == 0:
                after = x[0].read().reshape(xs.shape)
                assert np.array_equal(after[:, heads:], xs[:, heads:])
                got = after[:, :heads]
            else:
                got = q.read().reshape(want.shape)
            assert np.all(np.abs(got - want) <= 8 * 2.0 ** -24 * pair)  # as for norm_rope_rows
            y, bound = oracle.attention(cache, l, b, got, hd ** -0.5, 100 if l else 0)
            assert np.all(np.abs(out[l].read().reshape(y.shape) - y) <= bound), (step, l)
        logits, drawn = lg.read().reshape(-1, vocab), tok.read(np.uint32)
        hidden = np.stack([y.read() for y in last]).astype(np.float64)
        # sums of wq products in binary32 in any order
        assert np.all(np.abs(logits - hidden @ head.T) <= wq * 2.0 ** -23 * (np.abs(hidden) @ np.abs(head.T)))
        for i in range(len(lasts)):
            assert drawn[i] == longctx_oracle.sample(logits[i], float(u.read(np.float64)[i]), 0.9, 50, 0.95, 0.0, 1.0, np.zeros(0, np.uint32))
        log_probabilities_agree(logits, drawn, lp.read(), en.read(), ti.read(np.uint32).reshape(-1, top), tl.read().reshape(-1, top), top)
        for i, s in enumerate(lasts):
            if step in (4, 8) and s == 3:  # a guess is right, the other is not: its position is stored again
                tokens[3] = tokens[3][:-1]
            stored[s] = len(tokens[s])
            tokens[s].append(int(drawn[i]))
    for got, want in zip((b.read(np.uint8) for b in held.buffers), cache.device()):
        assert np.array_equal(got, want)  # the whole pool, byte for byte


def test_rotated_rows_beside_the_append(hip_ctx):
    """Queries that norm_rope_rows turns are the append's to the bit, at the batch's positions."""
    rng = np.random.default_rng(1)
    heads, kvh, hd = 6, 2, 128
    batch = oracle.Batch([2, 0, 30, 1], [900, 5, 64, 1], rng)
    desc, _ = heads_of(hip_ctx, rng, hd, 0, True, 10000.0)
    w, wk = heads * hd, kvh * hd
    x = rng.normal(0, 1, (batch.n, w + 2 * wk)).astype(np.float32)
    cache, src = hip_ctx.kv4_cache(1, kvh, hd, batch.pool), hip_ctx.buffer(x)
    a, b = hip_ctx.empty(4 * batch.n * w), hip_ctx.empty(4 * batch.n * w)
    hip_ctx.kv4_append(cache, 0, batch.on(hip_ctx), desc, src, 4 * w, 4 * (w + wk), w + 2 * wk, heads, 0, a)
    at = hip_ctx.buffer(np.array([p for _, _, p in batch.positions()], np.uint32))
    hip_ctx.norm_rope_rows(desc, src, b, batch.n, heads, positions=at, src_stride=w + 2 * wk)
    assert np.array_equal(a.read(), b.read())


def loop(ctx, seed, steps, results):
    """Decoding steps of one context on inputs of the seed; results gets the outputs' bytes."""
    rng = np.random.default_rng(seed)
    heads, kvh, hd, vocab = 8, 2, 64, 2100
    pool = oracle.Batch([1] * 5, [300 + steps] * 5, rng)
    held = oracle.upload(ctx, oracle.Kv4(1, pool.pool, kvh, hd))
    desc = hip.Heads(hip.RopeDesc(hd, hd, 1, 10000.0))
    w, wk = heads * hd, kvh * hd
    pages = ctx.buffer(pool.table)
    every = []
    for step in range(steps):
        rows = 300 if step == 0 else 1
        n = 5 * rows
        batch = hip.Batch(pages, ctx.buffer(np.arange(6, dtype=np.uint32) * rows), ctx.buffer(np.full(5, 300 + step, np.uint32)), 5, pool.table.shape[1], n, rows, 300 + step)
        x = ctx.buffer(rng.normal(0, 1, (n, w + 2 * wk)).astype(np.float32))
        out, lg = ctx.empty(4 * n * w), ctx.buffer(rng.normal(0, 2, (5, vocab)).astype(np.float32))
        tokens, lp, ti, tl = ctx.buffer(rng.integers(0, vocab, 5).astype(np.uint32)), ctx.empty(20), ctx.empty(4 * 5 * 9), ctx.empty(4 * 5 * 9)
        ctx.begin()
        ctx.kv4_append(held, 0, batch, desc, x, 4 * w, 4 * (w + wk), w + 2 * wk, heads, 0, x, 0, w + 2 * wk)
        ctx.kv4_attention(held, 0, batch, x, out, heads, q_stride=w + 2 * wk)
        ctx.token_logprobs(lg, tokens, lp, 5, vocab, None, 9, ti, tl)
        ctx.commit()
        every += [out.read().tobytes(), lp.read().tobytes(), ti.read(np.uint32).tobytes(), tl.read().tobytes()]
    results[seed] = every + [b.read(np.uint8).tobytes() for b in held.buffers]


def test_two_contexts_at_once(hip_ctx):
    """Two threads with a context each: both get what they get alone."""
    alone, together = {}, {}
    for seed in (1, 2):
        loop(hip_ctx, seed, 6, alone)
    contexts = [hip.Context(0) for _ in range(2)]
    threads = [threading.Thread(target=loop, args=(c, seed, 6, together)) for seed, c in zip((1, 2), contexts)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c in contexts:
        c.close()
    assert alone == together


def test_tables_that_change_between_calls(hip_ctx):
    """The same buffers with other tables in them, call after call in one open sequence after device copies."""
    rng = np.random.default_rng(8)
    heads, hd = 4, 64
    b = [oracle.Batch([3, 2], [200, 90], rng), oracle.Batch([1, 4], [70, 130], rng)]
    for x in b:
        x.table = np.concatenate([x.table, np.full((2, 8 - x.table.shape[1]), NONE, np.uint32)], axis=1)
    cache = oracle.Kv4(1, max(x.pool for x in b), 2, hd, rng)
    held = oracle.upload(hip_ctx, cache)
    q = rng.normal(0, 1, (5, heads, hd)).astype(np.float32)
    source = [[hip_ctx.buffer(np.ascontiguousarray(y, np.uint32)) for y in (x.table, x.starts, x.lengths)] for x in b]
    now = [hip_ctx.empty(s.nbytes) for s in source[0]]
    batch = hip.Batch(*now, 2, 8, 5)
    src = hip_ctx.buffer(q)
    outs = [hip_ctx.empty(q.nbytes) for _ in range(4)]
    hip_ctx.begin()
    for i, out in enumerate(outs):
        for a, z in zip(source[i % 2], now):
            hip_ctx.copy(a, 0, z, 0, a.nbytes)
        hip_ctx.kv4_attention(held, 0, batch, src, out, heads)
    hip_ctx.commit()
    for i, out in enumerate(outs):
        want, bound = oracle.attention(cache, 0, b[i % 2], q, hd ** -0.5)
        assert np.all(np.abs(out.read().reshape(want.shape) - want) <= bound)

WRAPPED = r"""
import sys
import torch
g = torch.Generator(device="cuda").manual_seed(3)
heads, kvh, hd, rows, vocab, pages = 4, 2, 64, 70, 3000, 4
x = torch.randn(rows, (heads + 2 * kvh) * hd, generator=g, device="cuda")
kc, vc = (torch.zeros(kvh * pages * 32 * hd, dtype=torch.uint8, device="cuda") for _ in range(2))
ks, vs = (torch.zeros(kvh * pages * 2 * hd, dtype=torch.uint8, device="cuda") for _ in range(2))
table = torch.tensor([[3, 1], [0, -1]], dtype=torch.int32, device="cuda")
starts = torch.tensor([0, 66, 70], dtype=torch.int32, device="cuda")
lengths = torch.tensor([66, 4], dtype=torch.int32, device="cuda")
out = torch.full((rows, heads * hd), 7.0, device="cuda")
logits = torch.randn(2, vocab, generator=g, device="cuda")
tokens = torch.tensor([5, vocab - 1], dtype=torch.int32, device="cuda")
lp = torch.zeros(2, device="cuda")
other = torch.cuda.Stream()
with torch.cuda.stream(other):  # made on a stream of torch's, which is waited for before the calls
    logits = logits * 2
torch.cuda.synchronize()
sys.path[:0] = sys.argv[1:]
from zhip import hip
ctx = hip.Context(0)
w = lambda t: ctx.wrap(t.data_ptr(), t.numel() * t.element_size())
cache = hip.Kv4Cache(w(kc), w(ks), w(vc), w(vs), 1, kvh, hd, pages)
batch = hip.Batch(w(table), w(starts), w(lengths), 2, 2, rows)
src, width = w(x), (heads + 2 * kvh) * hd
ctx.begin()
ctx.kv4_append(cache, 0, batch, None, src, 4 * heads * hd, 4 * (heads + kvh) * hd, width)
ctx.kv4_attention(cache, 0, batch, src, w(out), heads, q_stride=width)
ctx.token_logprobs(w(logits), w(tokens), w(lp), 2, vocab)
ctx.commit()
want = torch.log_softmax(logits.double(), 1)[torch.arange(2, device="cuda"), tokens.long()]
assert bool(((lp.double() - want).abs() <= 2.0 ** -21 + 2.0 ** -24 * want.abs()).all())
# the same calls on buffers of the context's own
own = hip.Kv4Cache(*(ctx.buffer(t.cpu().numpy() * 0) for t in (kc, ks, vc, vs)), 1, kvh, hd, pages)
y = ctx.empty(4 * out.numel())
b = hip.Batch(*(ctx.buffer(t.cpu().numpy()) for t in (table, starts, lengths)), 2, 2, rows)
s = ctx.buffer(x.cpu().numpy())
ctx.kv4_append(own, 0, b, None, s, 4 * heads * hd, 4 * (heads + kvh) * hd, width)
ctx.kv4_attention(own, 0, b, s, y, heads, q_stride=width)
assert (out.cpu().numpy().reshape(-1) == y.read()).all()
for t, o in zip((kc, ks, vc, vs), own.buffers):
    assert (t.cpu().numpy() == o.read("u1")).all()
ctx.close()
print("wrapped: fine")
"""


def test_torch_memory():
    """The operators on torch's tensors, tables among them.  In a process of its own: torch brings its HIP runtime, which
    has to be the first one loaded."""
    pytest.importorskip("torch")
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", WRAPPED, os.path.join(repo, "ziggy-llm_amd")], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "wrapped: fine" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
