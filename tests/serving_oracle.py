"""Plain 64-bit forms (numpy) of the operators that serve several sequences, written from their definitions."""
import numpy as np

from tests import longctx_oracle

PAGE = 64
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def norm(x, weights, eps=1e-6, offset=0.0):
    """x [..., hd] over its last axis, in 64 bits (weights None: x)."""
    x = x.astype(np.float64)
    if weights is None:
        return x
    w = weights.astype(np.float64) + float(np.float32(offset))
    return x * w / np.sqrt((x * x).mean(axis=-1, keepdims=True) + float(np.float32(eps)))


def in_four_bits(x):
    """(codes, scale bytes) of f32 values [..., hd]: 32 of them share a scale."""
    x = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(x).max(axis=-1).astype(np.float64)
    power = np.full(top.shape, -96)
    for _ in range(92 + 96):
        power = np.where((top > 7 * np.ldexp(1.0, power)) & (power < 92), power + 1, power)
    a = np.abs(x.astype(np.float64)) / np.ldexp(1.0, power)[..., None]
    off = np.abs(np.minimum(a, 6.0)[..., None] - VALUES)
    off[..., 1::2] = np.nextafter(off[..., 1::2], np.inf)  # a tie goes to the even code
    code = off.argmin(axis=-1) + 8 * np.signbit(x)
    return code.astype(np.uint8).reshape(*x.shape[:-2], -1), (power + 127).astype(np.uint8)


def of_four_bits(codes, scales):
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return v * np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, axis=-1)


class Kv4:
    """A cache as rows: per layer, page, position and kv head the codes [hd] and scales [hd / 32] of K and V, and marks."""

    def __init__(self, layers, pages, heads, hd, rng=None):
        self.shape = (layers, pages, PAGE, heads)
        self.hd = hd
        g = hd // 32
        draw = (lambda lo, hi, n: rng.integers(lo, hi, (*self.shape, n)).astype(np.uint8)) if rng else (
            lambda lo, hi, n: np.full((*self.shape, n), lo, np.uint8))
        self.codes = [draw(0, 16, hd) for _ in range(2)]
        self.scales = [draw(124, 130, g) for _ in range(2)]

    def put(self, layer, page, slot, k, v):
        """k, v [heads][hd] f32."""
        bad = ~(np.isfinite(k).all(axis=-1) & np.isfinite(v).all(axis=-1))
        for w, x in enumerate((k, v)):
            c, s = in_four_bits(np.where(bad[:, None], np.float32(0), x))
            s[bad] = 127 if w else 255
            self.codes[w][layer, page, slot], self.scales[w][layer, page, slot] = c, s

    def rows(self, layer, page, slot):
        """(k, v) [heads][hd] in 64 bits."""
        marked = (self.scales[0][layer, page, slot] == 255).any(axis=-1)
        out = []
        for w in range(2):
            s = np.where(marked[..., None], 127, self.scales[w][layer, page, slot])
            v = of_four_bits(self.codes[w][layer, page, slot], s)
            v[marked] = np.nan
            out.append(v)
        return out

    def device(self):
        """(k_codes, k_scales, v_codes, v_scales) in the device's layout, flat."""
        layers, pages, _, heads = self.shape
        g = self.hd // 32
        k = self.codes[0].transpose(0, 1, 3, 2, 4).reshape(layers, pages, heads, PAGE, g, 4, 4, 2)  # .. t, g, byte, half
        k = (k[..., 0] | k[..., 1] << 4).transpose(0, 1, 2, 3, 5, 4, 6)
        v = self.codes[1].transpose(0, 1, 3, 2, 4).reshape(layers, pages, heads, 2, 4, 8, g, 2, 16)  # .. half, g, j, t, high, d
        v = (v[..., 0, :] | v[..., 1, :] << 4).transpose(0, 1, 2, 3, 4, 7, 5, 6)
        scales = [s.transpose(0, 1, 3, 2, 4) for s in self.scales]
        return [np.ascontiguousarray(x).reshape(-1) for x in (k, scales[0], v, scales[1])]


class Batch:
    """Sequences' rows and lengths, and their pages in no order."""

    def __init__(self, rows, lengths, rng, spare=2, extra_pages=1):
        self.rows, self.lengths = list(rows), list(lengths)
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        used = [-(-n // PAGE) for n in lengths]
        self.pool = sum(used) + spare
        free = rng.permutation(self.pool)
        self.table = np.full((len(rows), max(max(used), 1) + extra_pages), 0xFFFFFFFF, np.uint32)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = free[at:at + n]
            at += n
        self.n = int(self.starts[-1])

    def positions(self):
        """(row, sequence, position) of every row."""
        return [(int(self.starts[s]) + i, s, n - r + i) for s, (r, n) in enumerate(zip(self.rows, self.lengths)) for i in range(r)]

    def place(self, s, t):
        return int(self.table[s, t // PAGE]), t % PAGE

    def on(self, ctx, rows=None, max_rows=0, max_length=0):
        from zhip import hip
        return hip.Batch(ctx.buffer(self.table), ctx.buffer(self.starts), ctx.buffer(np.asarray(self.lengths, np.uint32)),
                         len(self.rows), self.table.shape[1], self.n if rows is None else rows, max_rows, max_length)


def upload(ctx, cache):
    from zhip import hip
    layers, pages, _, heads = cache.shape
    return hip.Kv4Cache(*(ctx.buffer(x) for x in cache.device()), layers, heads, cache.hd, pages)


def attention(cache, layer, batch, q, scale, window=0, hidden=()):
    """q [rows, heads, hd]: (outputs in 64 bits, bound of the error).

    The bound, per output.  Keys, values and the queries' pieces are exact, so a score is a sum of 3 hd exact products
    in binary32: off by at most e = (3 hd + 8) 2^-23 sum |q k| scale (the scale's own two roundings among the 8), the
    largest over the row's positions, however the unit orders and rounds its sums to a step each; a weight is then off by
    2 e of itself (its own score and the maximum), its exponential and pieces by 2^-21, and the two sums of 3 n and n terms
    by 3 n 2^-23 and n 2^-24: (2 e + 2^-20 + n 2^-21) max |v| in all."""
    n, heads, hd = q.shape
    kvh = cache.shape[3]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    scale = float(np.float32(scale))
    for r, s, p in batch.positions():
        lo = max(0, p + 1 - window) if window else 0
        at = np.array([t for t in range(lo, p + 1) if (s, t // PAGE) not in hidden], int)
        if at.size == 0:
            continue
        k, v = cache.rows(layer, batch.table[s, at // PAGE].astype(int), at % PAGE)
        for h in range(heads):
            kk, vv = k[:, h // (heads // kvh)], v[:, h // (heads // kvh)]
            x = q[r, h].astype(np.float64)
            z = kk @ x * scale
            e = (3 * hd + 8) * 2.0 ** -23 * (np.abs(kk) @ np.abs(x)).max() * abs(scale)
            w = np.exp(z - z.max())
            out[r, h] = w @ vv / w.sum()
            bound[r, h] = (2 * e + 2.0 ** -20 + at.size * 2.0 ** -21) * np.abs(vv).max()
    return out, bound


def logprobs(x, token, top):
    """(log probability, entropy, top tokens, their log probabilities) of one row of f32 logits in 64 bits."""
    x = np.where(np.isnan(x), np.float32(-np.inf), x).astype(np.float64)
    order = np.argsort(-x, kind="stable")[:top]
    m = x.max()
    if not np.isfinite(m):
        return np.nan, np.nan, order, np.full(top, np.nan)
    w = np.exp(x - m)
    log = x - m - np.log(w.sum())
    seen = w > 0
    return log[token] if token < x.size else np.nan, -(np.exp(log[seen]) * log[seen]).sum(), order, log[order]


rope_frequencies, rope = longctx_oracle.rope_frequencies, longctx_oracle.rope
