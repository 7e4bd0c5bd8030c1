"""The paged cache's operators in numpy, in 64 bits and without the library:
what the tests compare with."""
import math

import numpy as np


def cache_values(x, f16):
    """What the cache holds of f32 rows (as f64)."""
    x = np.asarray(x, np.float32)
    if f16:
        y = np.clip(x, -65504, 65504).astype(np.float16).astype(np.float64)
    else:
        y = x.astype(np.float64)
    return np.where(np.isfinite(x), y, np.nan)


def norm_turn(x, pos, inv_freq, rot, half, norm=None, eps=1e-5, freq_scale=1.0, magnitude=1.0):
    """x [tokens, heads, hd] at positions pos: RMSNorm by head (with norm), then the rotation of the first rot dims."""
    y = np.asarray(x, np.float64)
    if norm is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + max(np.float32(eps), np.finfo(np.float32).eps)) * np.asarray(norm, np.float64)
    if rot:
        a = np.asarray(pos, np.float64)[:, None] * float(np.float32(freq_scale)) * np.asarray(inv_freq, np.float64)
        z = float(np.float32(magnitude)) * np.exp(1j * a)[:, None, :]
        one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
        z = (y[..., one] + 1j * y[..., two]) * z
        y = y.copy()
        y[..., one], y[..., two] = z.real, z.imag
    return y


def visible(p, n, window, n_sink, there=None):
    """The positions that a query at position p sees, of n."""
    j = np.arange(n)
    see = j <= p
    if window:
        see &= (j > p - window) | (j < n_sink)
    if there is not None:
        see &= there
    return j[see]


def attention(q, seqs, window=0, n_sink=0):
    """q [heads, tokens, hd]; seqs: (new tokens, k [n, kv heads, hd], v, there [n] or None) each.

    -> out [tokens, heads, hd], and what an element of it may be off by:
    a score's error is at most B 2^-18 (B: the sum of |q_i k_i| / sqrt(hd), the largest of the row's; q's split
    2^-23 of it, up to 66 sums of the MFMA that are cut instead of rounded, 2^-23 each at most, the scaling), so a weight's
    is that and 2^-21 of itself (exp2, its split, the sums over it), and 2^-40 of the row's
    largest; each key step adds 2^-22 of the sum so far."""
    q = np.asarray(q, np.float64)
    heads, tokens, hd = q.shape
    out, off = np.zeros((tokens, heads, hd)), np.zeros((tokens, heads, hd))
    t = 0
    for new, k, v, there in seqs:
        n, kv = k.shape[0], k.shape[1]
        for i in range(new):
            see = visible(n - new + i, n, window, n_sink, there)
            for h in range(heads if len(see) else 0):
                kk, vv = k[see, h * kv // heads], v[see, h * kv // heads]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk @ q[h, t] / math.sqrt(hd)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[t, h] = p @ vv
                    big = (np.abs(kk) @ np.abs(q[h, t])).max() / math.sqrt(hd)
                    off[t, h] = (2 * big * 2.0 ** -18 + 2.0 ** -20 + len(see) / 16 * 2.0 ** -22) * (p @ np.abs(vv)) \
                        + 2.0 ** -39 * p.max() * np.abs(vv).sum(0)
            t += 1
    return out, off


def assert_within(got, want, off, what=""):
    got = np.asarray(got, np.float64)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"{what}: NaN in other places"
    far = np.abs(got - want)[~nan] > off[~nan]
    assert not far.any(), f"{what}: {far.sum()} of {far.size} off, the first by {np.abs(got - want)[~nan][far][0]:.3g}, " \
                          f"{off[~nan][far][0]:.3g} allowed"
