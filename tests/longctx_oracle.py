"""Plain 64-bit forms of a long-context step's operators (numpy), written from their definitions."""
import math

import numpy as np

BLOCK = 32


def rope_frequencies(d, base, scaling=0, factor=1.0, orig=0, low=1.0, high=32.0):
    i = np.arange(d // 2, dtype=np.float64)
    f = float(np.float32(base)) ** (-2.0 * i / d)
    factor = float(np.float32(factor))
    if scaling == 0:
        return f
    if scaling == 1:
        return f / factor
    if scaling == 2:
        def c(t):
            return d * math.log(orig / (2 * math.pi * t)) / (2 * math.log(base))
        a, b = max(0, math.floor(c(high))), min(d - 1, math.ceil(c(low)))
        g = 1 - np.clip((i - a) / max(0.001, b - a), 0, 1)
    else:
        g = np.clip((orig * f / (2 * math.pi) - low) / (high - low), 0, 1)
    return f * (g + (1 - g) / factor)


def rope(x, positions, f, rd, style, magnitude=1.0):
    """x [rows, heads, hd]: (rotated rows, |x0| + |x1| of each rotated value's pair, 0 elsewhere)."""
    x = x.astype(np.float64)
    y, size = x.copy(), np.zeros_like(x)
    t = positions.astype(np.float64)[:, None] * f
    m = float(np.float32(magnitude))
    c, s = m * np.cos(t)[:, None], m * np.sin(t)[:, None]
    a, b = (slice(0, rd // 2), slice(rd // 2, rd)) if style else (slice(0, rd, 2), slice(1, rd, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = abs(m) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


class Kv8:
    """One layer of the cache: codes [heads, positions, hd] (K and V alike), scales [heads, blocks] as f32."""

    def __init__(self, heads, positions, hd, rng=None):
        self.nb = -(-positions // BLOCK)
        shape = (heads, self.nb * BLOCK, hd)
        self.codes = [np.zeros(shape, np.int8) if rng is None else rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
        self.scales = [np.zeros((heads, self.nb), np.float32) if rng is None else rng.uniform(0.5, 2, (heads, self.nb)).astype(np.float32) / 64
                       for _ in range(2)]

    def store(self, k, v, position):
        """k, v [rows, heads, hd] f32."""
        rows = k.shape[0]
        for x, codes, scales in ((k, self.codes[0], self.scales[0]), (v, self.codes[1], self.scales[1])):
            for h in range(codes.shape[0]):
                for b in range(position // BLOCK, (position + rows - 1) // BLOCK + 1):
                    lo, hi = max(position, b * BLOCK), min(position + rows, (b + 1) * BLOCK)
                    new = x[lo - position:hi - position, h]
                    was = scales[h, b] if lo > b * BLOCK else np.float32(0)
                    top = np.abs(new).max() if np.isfinite(new).all() else np.float32(np.nan)
                    now = np.maximum(was, np.float32(top) * np.float32(1 / 127))
                    scales[h, b] = now
                    kept = codes[h, b * BLOCK:lo]
                    if np.isnan(now):
                        if not now == was:
                            codes[h, b * BLOCK:hi] = 0
                        continue
                    if now == 0:
                        codes[h, lo:hi] = 0
                        continue
                    if now != was:
                        codes[h, b * BLOCK:lo] = np.rint(kept.astype(np.float64) * float(was) / float(now))
                    codes[h, lo:hi] = np.clip(np.rint(new.astype(np.float64) / float(now)), -127, 127)

    def rows(self, which, position, rows):
        """f32 values [rows, heads, hd]: code * scale in binary32."""
        at = np.arange(position, position + rows)
        return (self.codes[which][:, at].astype(np.float32) * self.scales[which][:, at // BLOCK, None]).transpose(1, 0, 2)


def kv8_device(layers, context):
    """The layers' codes and scales in the device's layout: (k_codes, k_scales, v_codes, v_scales) as flat arrays."""
    kc = np.concatenate([c.codes[0].reshape(-1) for c in layers])
    vc = np.concatenate([c.codes[1].reshape(c.codes[1].shape[0], c.nb, BLOCK, -1).transpose(0, 1, 3, 2).reshape(-1) for c in layers])
    ks, vs = (np.concatenate([c.scales[w].reshape(-1) for c in layers]) for w in range(2))
    return kc, ks, vc, vs


def kv8_attention(cache, q, position, scale, window=0):
    """q [queries, heads, hd]: (outputs in 64 bits, bound of the error that 32-bit sums make).

    The bound, per output.  A score is a sum of hd products of exact codes with a query value known to 2^-22
    (two binary16 pieces): off by at most e = (hd + 8) 2^-23 sum |q c| s scale, the largest over the row's
    positions; a weight is then off by 2 e of itself (its own score and the maximum), its exponential by 2^-21,
    and the two sums of n terms by n 2^-23 each: (2 e + 2^-20 + n 2^-22) max |v| in all.
    """
    queries, heads, hd = q.shape
    group = heads // cache.codes[0].shape[0]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    scale = float(np.float32(scale))
    for h in range(heads):
        kv = h // group
        for i in range(queries):
            p = position + i
            lo = max(0, p + 1 - window) if window else 0
            at = np.arange(lo, p + 1)
            kc = cache.codes[0][kv, at].astype(np.float64)
            ks = cache.scales[0][kv, at // BLOCK].astype(np.float64)
            v = cache.codes[1][kv, at].astype(np.float64) * cache.scales[1][kv, at // BLOCK].astype(np.float64)[:, None]
            x = q[i, h].astype(np.float64)
            s = (kc @ x) * ks * scale
            e = (hd + 8) * 2.0 ** -23 * ((np.abs(kc) @ np.abs(x)) * ks * abs(scale)).max()
            w = np.exp(s - s.max())
            out[i, h] = w @ v / w.sum()
            bound[i, h] = (2 * e + 2.0 ** -20 + at.size * 2.0 ** -22) * np.abs(v).max()
    return out, bound


def sample(x, u, temperature, top_k=0, top_p=1.0, min_p=0.0, penalty=1.0, recent=()):
    """The token of logits x (f32) for the random number u, in 64 bits."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    x = np.where(np.isnan(x), np.float32(-np.inf), x)
    n = x.size
    if temperature <= 0:
        return int(np.argmax(x))
    a = x.copy()
    if penalty > 1:
        ids = np.unique([r for r in recent if r < n]).astype(int)
        p = np.float32(penalty)
        a[ids] = np.where(a[ids] < 0, a[ids] * p, a[ids] / p)
    order = np.arange(n)
    if 0 < top_k < n:
        order = np.argsort(-x.astype(np.float64), kind="stable")[:top_k]
    a = a[order]
    m = a.max()
    if not np.isfinite(m):
        return int(order[np.argmax(a)])
    w = np.exp((a.astype(np.float64) - float(m)) / f(temperature))
    w[w < f(min_p)] = 0
    # the definition's own cut: what rounds to 0 in units of 2^-s (it shows where u is 0: the first weight that is not)
    w[w < 2.0 ** -(63 - math.ceil(math.log2(a.size)))] = 0
    if top_p < 1:
        by = np.argsort(-a.astype(np.float64), kind="stable")
        w, order = w[by], order[by]
        share = np.cumsum(w)
        share /= share[-1]
        w[np.argmax(share >= f(top_p)) + 1:] = 0
    run = np.cumsum(w)  # the total is the running sum's end: numpy's own sum adds in another order
    return int(order[np.argmax((run >= u * run[-1]) & (w > 0))])
