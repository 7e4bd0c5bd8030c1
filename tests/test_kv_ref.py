"""The numpy model of the 4-bit KV cache against its definition, spelled out
element by element."""
from fractions import Fraction

import numpy as np
import pytest

from kv_ref import D_MAX, attention, kept, q4_quantize, q4_values


def slow_block(x):
    t = x[0]
    for e in x[1:]:
        if abs(e) > abs(t):
            t = e
    d = float(np.float16(np.float64(t) / -8)) if abs(t) < 8 * 65504 else np.copysign(np.inf, -t)
    d = max(-D_MAX, min(D_MAX, d))
    if d == 0:
        return d, [8] * 32
    codes = []
    for e in x:
        f = Fraction(float(e)) / Fraction(d) + Fraction(17, 2)
        codes.append(max(0, min(15, f.numerator // f.denominator)))
    return d, codes


@pytest.mark.parametrize("scale", [1.0, 1e-6, 3e4, 3e6, 2.0 ** -25, 0.0])
def test_quantizer_is_the_nearest_code(scale):
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((40, 32)) * scale).astype(np.float32)
    # borders and ties of |x|
    x[0] = (np.arange(32) % 16 - 7.5) / 8 * scale
    x[1, ::2], x[1, 1::2] = scale, -scale
    c, d = q4_quantize(x)
    for i in range(len(x)):
        sd, sc = slow_block([np.float32(e) for e in x[i]])
        assert d[i, 0] == sd and list(c[i]) == sc


def test_not_finite_blocks_read_as_nan():
    x = np.ones((3, 64), np.float32)
    x[0, 3], x[1, 40], x[2, 63] = np.nan, np.inf, -np.inf
    v = q4_values(x)
    assert np.isnan(v[0, :32]).all() and np.isfinite(v[0, 32:]).all()
    assert np.isnan(v[1:, 32:]).all() and np.isfinite(v[1:, :32]).all()


def test_values_round_trip():
    x = np.random.default_rng(6).standard_normal((64, 128)).astype(np.float32)
    v = q4_values(x)
    assert np.array_equal(q4_values(v), v)
    # half a step: d / 2 (the block's other end holds 7 of the 8 steps: one whole step there)
    step = np.abs(q4_quantize(x)[1]).repeat(32, 1)
    assert np.all(np.abs(v - x) <= step * (1 + 2.0 ** -10))


def test_attention_rows_and_mass():
    rng = np.random.default_rng(7)
    q, k, v = rng.standard_normal((4, 3, 64)), rng.standard_normal((2, 10, 64)), rng.standard_normal((2, 10, 64))
    out, mass = attention(q, k, v, 7)
    w = np.exp(q[3, 0] @ k[1, :8].T / 8)
    assert np.allclose(out[0, 3], (w / w.sum()) @ v[1, :8], rtol=1e-12)
    assert np.allclose(mass.sum(1), 2 * 3) and np.all(mass[:, 9] > 0)


def test_kept_is_heaviest_then_earliest_then_newest():
    m = np.array([[5, 1, 5, 0, 5, 9, 9], [0, 0, 0, 0, 0, 0, np.nan]], np.float32)
    assert kept(m, 7, 4, 2).tolist() == [[0, 2, 5, 6], [0, 1, 5, 6]]
    assert kept(m, 7, 2, 2).tolist() == [[5, 6], [5, 6]]
    assert kept(m, 7, 9, 1).tolist() == [list(range(7))] * 2
    assert kept(m[:, ::-1], 7, 1, 0).tolist() == [[0], [1]]
