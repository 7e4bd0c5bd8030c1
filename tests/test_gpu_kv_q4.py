"""The KV cache held in 4 bits: what appends leave in it, bit for bit, and
attention over it.

Bars:
  - codes and scales (read back as f32): exact.  The quantizer is defined by
    comparisons that are exact in f32, and a value (code - 8) * d has 15 bits.
  - attention against 64 bits on the rows the cache reads as: a score (in
    log2 units) sums HD products in two parts (three of a query whose elements
    are very uneven).  With S the sum of their
    sizes (about 0.64 * 1.44 * sqrt(HD) = 10 to 15 for normal queries and
    keys), HD roundings or truncations of at most 2^-23 of the partial sum
    add up to sqrt(3 * 32) * 2^-23 * S = 1.7e-5 root mean square over a block's 96
    steps at most, and a weight is off by ln 2 times that; the output, a mean
    of V rows under weights that sum to 1, by twice as much of max |V| at
    most.  The bar is 2e-5 * max |V|, as for the f32 cache.
"""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import attention as A
from kv_ref import attention, q4_values

pytestmark = pytest.mark.gpu
F32 = np.float32


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def inv_freq(hd, base=500000.0):
    return np.array([np.float32(base) ** np.float32(-2.0 * i / hd) for i in range(hd // 2)], dtype=F32)


def rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(F32)


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_kv,parts", [(1, [1]), (2, [1, 1, 5, 1, 8, 3]), (8, [17]), (3, [7, 2, 40, 1])])
def test_append_and_read(be, hd, n_kv, parts):
    total = sum(parts)
    c = A.KVCache(be, total + 3, 2, n_kv, hd, type=B.Q4_0)
    k, v = rows(hd + total, n_kv, total, hd), rows(hd + total + 1, n_kv, total, hd)
    at = 0
    for i, n in enumerate(parts):
        kk, vv = np.ascontiguousarray(k[:, at:at + n]), np.ascontiguousarray(v[:, at:at + n])
        if i % 2:
            c.append(1, kk, vv, n, hd, mem=B.MEM_HOST)
        else:
            c.append(1, dev(kk), dev(vv), n, hd)
        at += n
    assert c.layer_len(1) == total and c.layer_len(0) == 0 and c.size() == 0
    kq, vq = q4_values(k), q4_values(v)
    gk, gv = (t.cpu().numpy() for t in c.read(1, 0, total))
    assert same(gk, kq) and same(gv, vq)
    hk, hv = c.read(1, 0, total, mem=B.MEM_HOST)
    assert same(hk, kq) and same(hv, vq)
    first = total // 3
    gk, gv = (t.cpu().numpy() for t in c.read(1, first, total - first))
    assert same(gk, kq[:, first:]) and same(gv, vq[:, first:])
    assert same(c.get_head(1, n_kv - 1)[1], vq[n_kv - 1])


def test_quantizer_edges(be):
    x = rows(9, 2, 24, 64)
    x[0, 0] = 0
    x[0, 1, :32] = (np.arange(32) % 16 - 7.5) / 8        # borders between codes
    x[0, 2, ::2], x[0, 2, 1::2] = 1, -1                  # equal sizes: the first decides the sign
    x[0, 3] *= 2.0 ** -24                                # f16 subnormal scales
    x[0, 4] *= 2.0 ** -40                                # scales that vanish
    x[0, 5] *= 1e5                                       # values beyond f16: the scale stops
    x[0, 6] *= 1e38
    x[0, 7, 5], x[0, 8, 40], x[0, 9, 0] = np.nan, np.inf, -np.inf
    x[0, 10] = np.float32(-1e-45)
    # one ulp around every border of a scale that is no power of two
    d = F32(np.float16(0.3713))
    b = (np.arange(1, 16) - F32(8.5)) * d
    x[1, 0, :32] = np.concatenate([[F32(-8) * d], b, np.nextafter(b, F32(9)), [0]])
    x[1, 1, :32] = np.concatenate([[F32(-8) * d], b, np.nextafter(b, F32(-9)), [0]])
    x[1, 2] = -x[1, 0]
    x[1, 3] = -x[1, 1]
    c = A.KVCache(be, 24, 1, 2, 64, type=B.Q4_0)
    c.append(0, dev(x), dev(x[:, ::-1]), 24, 64)
    gk, gv = (t.cpu().numpy() for t in c.read(0, 0, 24))
    assert same(gk, q4_values(x)) and same(gv, q4_values(x[:, ::-1]))


@pytest.mark.parametrize("layout", [A.ROPE_INTERLEAVED, A.ROPE_SPLIT_HALF])
@pytest.mark.parametrize("hd,n", [(64, 11), (128, 1), (256, 9)])
def test_append_rope_equals_rope_then_append(be, layout, hd, n):
    n_kv, heads = 2, 6
    f, kp, vp, qp = inv_freq(hd), rows(1, n, n_kv * hd), rows(2, n, n_kv * hd), rows(3, n, heads * hd)
    c = [A.KVCache(be, 40, 2, n_kv, hd, type=B.Q4_0) for _ in range(4)]
    q_out = []
    for at in (5, 5 + n):   # the second call starts inside a tile
        kr = A.apply_rope(be, dev(kp), n, n_kv, hd, at, 0.5, dev(f), layout)
        c[0].append(1, kr, A.transpose_heads(be, dev(vp), n, n_kv, hd), n, hd)
        c[1].append_rope(1, dev(kp), dev(vp), n, at, 0.5, dev(f), layout)
        c[2].append_rope(1, kp, vp, n, at, 0.5, f, layout, mem=B.MEM_HOST)
        q_out = [c[3].append_rope_q(1, dev(qp), heads, dev(kp), dev(vp), n, at, 0.5, dev(f), layout)]
        be.sync()
        want = A.apply_rope(be, dev(qp), n, heads, hd, at, 0.5, dev(f), layout)
        assert (q_out[0] == want).all()
    ref = [t.cpu().numpy() for t in c[0].read(1, 0, 2 * n)]
    for o in c[1:]:
        got = [t.cpu().numpy() for t in o.read(1, 0, 2 * n)]
        assert same(got[0], ref[0]) and same(got[1], ref[1])


CASES = [
    # heads, kv heads, hd, rows, start
    (32, 8, 128, 1, 0), (32, 8, 128, 1, 30), (32, 8, 128, 1, 31), (32, 8, 128, 1, 32), (32, 8, 128, 1, 4095),
    (8, 8, 64, 1, 1000), (4, 1, 256, 1, 700), (16, 16, 256, 5, 300), (32, 8, 64, 70, 33), (6, 2, 128, 33, 0),
    (20, 1, 128, 3, 129), (5, 2, 64, 7, 60), (32, 4, 128, 16, 2000), (14, 2, 256, 40, 0), (32, 8, 128, 1, 20000),
]


@pytest.mark.parametrize("heads,n_kv,hd,n,start", CASES)
def test_attention(be, heads, n_kv, hd, n, start):
    total = start + n
    q, k, v = rows(1, heads, n, hd), rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    k[:, :, ::29] *= 5
    c = A.KVCache(be, total + 9, 1, n_kv, hd, type=B.Q4_0)
    c.append(0, dev(k), dev(v), total, hd)
    # rows behind the call's positions: never looked at
    c.append(0, np.full((n_kv, 9, hd), np.nan, F32), np.full((n_kv, 9, hd), np.nan, F32), 9, hd, mem=B.MEM_HOST)
    ref, _ = attention(q, q4_values(k), q4_values(v), start)
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, start).cpu().numpy()
    assert got.shape == ref.shape
    assert np.max(np.abs(got - ref)) <= 2e-5 * np.max(np.abs(v))
    host = A.compute_attention(be, q, c, 0, heads, n_kv, hd, n, total, start, mem=B.MEM_HOST)
    assert np.array_equal(host, got)
    if heads * hd % 256 == 0:   # the rows as the o projection takes them
        q8 = A.compute_attention_q8k(be, dev(q), c, 0, heads, n_kv, hd, n, total, start)
        assert (q8.flatten() == be.quantize_act(B.Q8_K, dev(got.reshape(n, heads * hd)))).all()


def test_attention_of_less_than_the_cache(be):
    """kv_len below the layer's length, and a start position that shows the rows less still."""
    k, v, q = rows(4, 2, 300, 128), rows(5, 2, 300, 128), rows(6, 8, 4, 128)
    c = A.KVCache(be, 300, 1, 2, 128, type=B.Q4_0)
    c.append(0, dev(k), dev(v), 300, 128)
    for kv_len, start in ((300, 10), (77, 200), (200, 0), (1, 0)):
        ref, _ = attention(q, q4_values(k[:, :kv_len]), q4_values(v[:, :kv_len]), start)
        got = A.compute_attention(be, dev(q), c, 0, 8, 2, 128, 4, kv_len, start).cpu().numpy()
        assert np.max(np.abs(got - ref)) <= 2e-5 * np.max(np.abs(v))


@pytest.mark.parametrize("n", [1, 21])
def test_nan_rows_reach_only_those_that_see_them(be, n):
    k, v, q = rows(7, 2, 200, 64), rows(8, 2, 200, 64), rows(9, 4, n, 64)
    v[0, 190, 3] = np.inf        # one block of kv head 0
    v[1, 40, 50] = np.nan
    k[1, 195, 1] = np.nan        # a whole row of scores
    c = A.KVCache(be, 200, 1, 2, 64, type=B.Q4_0)
    c.append(0, dev(k), dev(v), 200, 64)
    kq, vq = q4_values(k), q4_values(v)
    for start in (200 - n, 180 - n, 41 - n if n < 41 else 0):
        ref, _ = attention(q, kq, vq, start)
        got = A.compute_attention(be, dev(q), c, 0, 4, 2, 64, n, 200, start).cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert np.max(np.abs(np.nan_to_num(got) - np.nan_to_num(ref))) <= 2e-5 * 5


def test_spread_scores_and_values(be):
    """A position that takes nearly all the weight and adds nothing, queries
    and values of very different sizes."""
    hd, n = 128, 500
    k, v, q = rows(10, 1, n, hd), rows(11, 1, n, hd), rows(12, 4, 1, hd)
    v[0, 0] = 0
    k[0, 0] = 4 * q[0, 0]
    q[1] *= 1e-20
    q[2, 0, 5] = 1e20
    k[:, :, 5] = 0
    v[0, 100:, :32] *= 2.0 ** -20
    c = A.KVCache(be, n, 1, 1, hd, type=B.Q4_0)
    c.append(0, dev(k), dev(v), n, hd)
    kq, vq = q4_values(k), q4_values(v)
    ref, _ = attention(q, kq, vq, n - 1)
    got = A.compute_attention(be, dev(q), c, 0, 4, 1, hd, 1, n, n - 1).cpu().numpy()
    # against what the weighted values add up to in size, dim by dim: scores
    # here reach 4 |q|^2 / sqrt(hd) * log2(e) = 65, off by 96 * 2^-24 of it (3.7e-4)
    # at most in log2 units
    for h in range(4):
        s = q[h, 0].astype(np.float64) @ kq[0].T.astype(np.float64) / np.sqrt(hd)
        p = np.exp(s - s.max())
        p /= p.sum()
        size = p @ np.abs(vq[0].astype(np.float64))
        assert np.all(np.abs(got[0, h] - ref[0, h]) <= 4e-4 * size + 1e-30)


@pytest.mark.parametrize("peak", [60, 140, 1000])
def test_weights_down_to_the_least(be, peak):
    """Scores that fall evenly from 0 to -peak (log2) over 64 positions, so
    that weights of every size down to f32's least, and zeros, meet in a step."""
    hd, n = 64, 64
    q = np.zeros((2, 1, hd), F32)
    q[:, 0, 0] = 1
    k, v = np.zeros((1, n, hd), F32), rows(13, 1, n, hd)
    k[0, :, 0] = -np.random.default_rng(1).permutation(n) * peak / n * np.log(2) * np.sqrt(hd)
    v[0, np.argmax(k[0, :, 0])] = 0
    c = A.KVCache(be, n, 1, 1, hd, type=B.Q4_0)
    c.append(0, dev(k), dev(v), n, hd)
    kq, vq = q4_values(k), q4_values(v)
    ref, _ = attention(q, kq, vq, n - 1)
    got = A.compute_attention(be, dev(q), c, 0, 2, 1, hd, 1, n, n - 1).cpu().numpy()
    s = kq[0, :, 0].astype(np.float64) / np.sqrt(hd)
    size = np.exp(s - s.max()) @ np.abs(vq[0].astype(np.float64))
    # one product a score: its three roundings and the exponent's (2^-23 of peak each) and 2^-20 for the rest
    assert np.all(np.abs(got[0] - ref[0]) <= (4 * peak * 2.0 ** -23 + 2.0 ** -20) * size + 1e-37)


def test_refusals(be):
    E = B._lib
    with pytest.raises(B.BarqError) as e:
        A.KVCache(be, 16, 1, 2, 96, type=B.Q4_0)
    assert e.value.code == B.E_UNSUPPORTED
    with pytest.raises(B.BarqError) as e:
        A.KVCache(be, 16, 1, 2, 64, type=B.Q8_0)
    assert e.value.code == B.E_UNSUPPORTED
    with pytest.raises(B.BarqError) as e:
        A.KVCache(be, 2 ** 31 - 1, 2 ** 40, 2 ** 20, 64, type=B.Q4_0)
    assert e.value.code == B.E_DIM
    c = A.KVCache(be, 16, 1, 2, 64, type=B.Q4_0)
    k = rows(1, 2, 16, 64)
    c.append(0, k, k, 16, 64, mem=B.MEM_HOST)
    for args, code in (((0, 0, 17), B.E_DIM), ((0, 16, 1), B.E_DIM), ((1, 0, 1), B.E_INVALID), ((0, 2 ** 63, 2 ** 63), B.E_DIM)):
        with pytest.raises(B.BarqError) as e:
            E.check(be._lib.barq_rocm_kv_cache_read(be.h, c.c, *args, k.ctypes.data, None, B.MEM_HOST))
        assert e.value.code == code
    with pytest.raises(B.BarqError) as e:
        c.head_ptrs(0, 0)
    assert e.value.code == B.E_UNSUPPORTED
    for n in (1, 2 ** 63, 2 ** 64 - 1):
        with pytest.raises(B.BarqError) as e:
            E.check(be._lib.barq_rocm_kv_cache_append(be.h, c.c, 0, k.ctypes.data, k.ctypes.data, n, 64, B.MEM_HOST))
        assert e.value.code == B.E_INVALID
    assert c.layer_len(0) == 16
    E.check(be._lib.barq_rocm_kv_cache_read(be.h, c.c, 0, 16, 0, None, None, B.MEM_HOST))
    assert be._lib.barq_rocm_kv_cache_type(c.c) == B.Q4_0 and be._lib.barq_rocm_kv_cache_type(None) == -1


def test_f32_cache_reads_what_it_holds(be):
    k, v = rows(1, 3, 20, 96), rows(2, 3, 20, 96)
    c = A.KVCache(be, 24, 2, 3, 96)
    c.append(1, dev(k), dev(v), 20, 96)
    gk, gv = (t.cpu().numpy() for t in c.read(1, 4, 11))
    assert np.array_equal(gk, k[:, 4:15]) and np.array_equal(gv, v[:, 4:15])
    assert np.array_equal(c.read(1, 4, 11, mem=B.MEM_HOST)[1], gv)
