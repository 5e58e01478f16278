"""The 4-bit oracle against its definition's own words, value by value (CPU)."""
import numpy as np

from tests import serving_oracle as oracle


def test_codes_are_the_nearest_and_scales_the_least():
    rng = np.random.default_rng(1)
    for size in (1e-40, 1e-29, 1e-3, 1.0, 6.999999, 7.0, 7.000001, 1e5, 1e28, 1e30):
        x = (np.clip(rng.normal(0, 0.5, (3, 64)), -1, 1) * size).astype(np.float32)
        x[0, 0] = size
        codes, scales = oracle.in_four_bits(x)
        got = oracle.of_four_bits(codes, scales)
        for r in range(3):
            for t in range(2):
                v = x[r, 32 * t:32 * t + 32].astype(np.float64)
                e = int(scales[r, t]) - 127
                top = np.abs(v).max()
                assert -96 <= e <= 92 and (top <= 7 * 2.0 ** e or e == 92) and (e == -96 or top > 7 * 2.0 ** (e - 1))
                grid = np.concatenate([oracle.VALUES, -oracle.VALUES]) * 2.0 ** e
                off = np.abs(np.clip(v, -6 * 2.0 ** e, 6 * 2.0 ** e)[:, None] - grid).min(axis=1)
                assert np.array_equal(np.abs(np.clip(v, -6 * 2.0 ** e, 6 * 2.0 ** e) - got[r, 32 * t:32 * t + 32]), off)


def test_the_layout_keeps_every_code():
    """The device's bytes hold each code once, at the place that the interface says."""
    rng = np.random.default_rng(2)
    c = oracle.Kv4(2, 3, 2, 96, rng)
    k, ks, v, vs = c.device()
    g = 3
    for _ in range(200):
        layer, page, pos, head, d = (int(rng.integers(n)) for n in (2, 3, 64, 2, 96))
        at = ((layer * 3 + page) * 2 + head) * 64
        b = k[at * 48 + pos * 48 + (d % 32 // 8 * g + d // 32) * 4 + d % 8 // 2]
        assert (b >> 4 * (d % 2) & 15) == c.codes[0][layer, page, pos, head, d]
        b = v[at * 48 + ((pos // 8) * 16 + d % 16) * 8 * g + pos % 8 * g + d // 32]
        assert (b >> 4 * (d % 32 // 16) & 15) == c.codes[1][layer, page, pos, head, d]
        assert ks[(at + pos) * g + d // 32] == c.scales[0][layer, page, pos, head, d // 32]
        assert vs[(at + pos) * g + d // 32] == c.scales[1][layer, page, pos, head, d // 32]
