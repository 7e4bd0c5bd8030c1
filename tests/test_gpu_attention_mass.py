"""Attention that gathers the positions' weights, over f32 and 4-bit caches.

Bars, against 64 bits on the rows the cache reads as:
  - out: 2e-5 * max |V|, as in the attention tests.
  - mass: a weight is off by ln 2 times its score's error (in log2 units
    1.7e-5 root mean square, the bound of the attention tests) and as much
    again through the row's sum: 2.4e-5 of itself, plus 2^-22 for the exponential
    and the division.  Sums of positive terms keep that, so the bar is 2.5e-5
    of what the call adds to the position, plus the sum's rounding: 2^-23 of the
    total.
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


def rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(F32)


def case(be, type_, heads, n_kv, hd, n, start, extra=0):
    total = start + n
    q, k, v = rows(1, heads, n, hd), rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    k[:, :, ::29] *= 3
    c = A.KVCache(be, total + extra, 1, n_kv, hd, type=type_)
    c.append(0, dev(k), dev(v), total, hd)
    if extra:
        c.append(0, *(np.full((n_kv, extra, hd), np.nan, F32) for _ in "kv"), extra, hd, mem=B.MEM_HOST)
    if type_ == B.Q4_0:
        k, v = q4_values(k), q4_values(v)
    return c, q, k, v


def mass_ok(got, before, added):
    total = before.astype(np.float64) + added
    return np.all(np.abs(got - total) <= 2.5e-5 * added + 2.0 ** -23 * total)


CASES = [(32, 8, 128, 1, 0), (32, 8, 128, 1, 4095), (8, 8, 64, 1, 700), (4, 1, 256, 1, 130), (20, 1, 128, 1, 65),
         (5, 2, 64, 3, 40), (16, 16, 256, 5, 300), (32, 8, 128, 70, 60), (14, 2, 64, 33, 0), (6, 2, 128, 200, 11)]


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("heads,n_kv,hd,n,start", CASES)
def test_out_and_mass(be, type_, heads, n_kv, hd, n, start):
    total = start + n
    c, q, k, v = case(be, type_, heads, n_kv, hd, n, start, extra=5)
    ref, added = attention(q, k, v, start)
    before = np.abs(rows(4, n_kv, total + 9))
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, start, dev(before),
                                         mass_out=dev(np.full_like(before, 7)))
    out, mass = out.cpu().numpy(), mass.cpu().numpy()
    assert np.max(np.abs(out - ref)) <= 2e-5 * np.max(np.abs(v))
    assert mass_ok(mass[:, :total], before[:, :total], added)
    assert np.all(mass[:, total:] == 7)   # columns behind the call's positions
    d = dev(before)
    out2, mass2 = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, start, d)
    assert mass2 is d and np.array_equal(mass2.cpu().numpy()[:, :total], mass[:, :total])
    assert np.array_equal(mass2.cpu().numpy()[:, total:], before[:, total:]) and np.array_equal(out2.cpu().numpy(), out)
    h = before.copy()
    oh, mh = A.compute_attention_mass(be, q, c, 0, heads, n_kv, hd, n, total, start, h, mem=B.MEM_HOST)
    assert np.array_equal(oh, out) and np.array_equal(mh[:, :total], mass[:, :total])
    assert np.array_equal(mh[:, total:], before[:, total:])
    _, m0 = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, start, None)
    assert mass_ok(m0.cpu().numpy(), np.zeros((n_kv, total), F32), added)
    if heads * hd % 256 == 0:
        q8, m1 = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, start, None, out_type=B.Q8_K)
        assert (q8.flatten() == be.quantize_act(B.Q8_K, dev(out.reshape(n, heads * hd)))).all() and (m1 == m0).all()


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
def test_rows_in_chunks(be, type_):
    """300 rows of 32 heads against 2300 positions (88 MB of scores), and against 4300: more than one launch keeps
    (128 MiB), 242 rows of them and 58."""
    for start in (2000, 4000):
        total = start + 300
        c, q, k, v = case(be, type_, 32, 8, 64, 300, start)
        ref, added = attention(q, k, v, start)
        out, mass = A.compute_attention_mass(be, dev(q), c, 0, 32, 8, 64, 300, total, start, None)
        assert np.max(np.abs(out.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
        assert mass_ok(mass.cpu().numpy(), np.zeros((8, total), F32), added)


PROMPTS = [(32, 8, 128, 200, 800), (16, 4, 64, 600, 100), (8, 8, 128, 130, 1000), (6, 2, 128, 257, 1500), (12, 4, 128, 500, 0),
           (20, 1, 64, 33, 3000), (14, 2, 256, 100, 400), (14, 2, 256, 300, 500), (4, 2, 256, 40, 3960), (5, 2, 128, 300, 300)]


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("heads,n_kv,hd,n,start", PROMPTS)
def test_prompts(be, type_, heads, n_kv, hd, n, start):
    total = start + n
    c, q, k, v = case(be, type_, heads, n_kv, hd, n, start)
    ref, added = attention(q, k, v, start)
    before = np.abs(rows(4, n_kv, total + 3))
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, start, dev(before))
    out, mass = out.cpu().numpy(), mass.cpu().numpy()
    assert np.max(np.abs(out - ref)) <= 2e-5 * np.max(np.abs(v))
    assert mass_ok(mass[:, :total], before[:, :total], added) and np.array_equal(mass[:, total:], before[:, total:])
    if heads * hd % 256 == 0:
        q8, m1 = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, start, dev(before), out_type=B.Q8_K)
        assert (q8.flatten() == be.quantize_act(B.Q8_K, dev(out.reshape(n, heads * hd)))).all()
        assert np.array_equal(m1.cpu().numpy(), mass)


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompts_of_uneven_rows(be, type_, hd):
    """Values of very different sizes, rows that see a NaN or an infinity, and rows that do not."""
    heads, n_kv, n, start = 8, 2, 300, 500
    q, k, v = rows(5, heads, n, hd), rows(6, n_kv, start + n, hd), rows(7, n_kv, start + n, hd)
    v[:, ::7] *= F32(2.0 ** -40)
    k[:, ::11] *= 4
    for bad in (False, True):
        if bad:
            k[1, 700, 3], v[0, 650, 2] = np.nan, np.inf
        c = A.KVCache(be, start + n, 1, n_kv, hd, type=type_)
        c.append(0, dev(k), dev(v), start + n, hd)
        kk, vv = (q4_values(k), q4_values(v)) if type_ == B.Q4_0 else (k, v)
        ref, added = attention(q, kk, vv, start)
        out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, start + n, start, None)
        out, mass = out.cpu().numpy(), mass.cpu().numpy()
        assert np.array_equal(np.isfinite(out), np.isfinite(ref)) and np.array_equal(np.isnan(mass), np.isnan(added))
        ok = np.isfinite(ref)
        assert np.max(np.abs(out[ok] - ref[ok])) <= 2e-5 * np.nanmax(np.abs(vv[np.isfinite(vv)]))
        seen = ~np.isnan(added)
        assert np.all(np.abs(mass - added)[seen] <= 2.5e-5 * added[seen] + 2.0 ** -23 * added[seen])


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
def test_less_than_the_cache(be, type_):
    c, q, k, v = case(be, type_, 8, 2, 128, 4, 296)
    for kv_len, start in ((300, 10), (77, 200), (200, 0), (1, 0)):
        ref, added = attention(q, k[:, :kv_len], v[:, :kv_len], start)
        out, mass = A.compute_attention_mass(be, dev(q), c, 0, 8, 2, 128, 4, kv_len, start, None)
        assert np.max(np.abs(out.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
        mass = mass.cpu().numpy()
        assert mass_ok(mass, np.zeros((2, kv_len), F32), added)
        assert not mass[:, start + 4:].any()   # seen by no query


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("hd", [128, 256])
def test_prompts_of_less_than_the_cache(be, type_, hd):
    """Positions that no query sees, and queries far behind the last one: whole tiles, and pieces that a tile lacks."""
    c, q, k, v = case(be, type_, 8, 2, hd, 300, 900)
    for kv_len, start in ((1200, 10), (77, 200), (1000, 0), (1000, 5000), (1, 3)):
        ref, added = attention(q, k[:, :kv_len], v[:, :kv_len], start)
        out, mass = A.compute_attention_mass(be, dev(q), c, 0, 8, 2, hd, 300, kv_len, start, None)
        assert np.max(np.abs(out.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
        mass = mass.cpu().numpy()
        assert mass_ok(mass, np.zeros((2, kv_len), F32), added)
        assert not mass[:, start + 300:].any()   # seen by no query


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("heads,n_kv,n,total", [(16, 16, 1, 20000), (8, 2, 3, 66000)])
def test_few_rows_of_a_long_cache(be, type_, heads, n_kv, n, total):
    """More positions than the workgroups that sum the masses take at a time; one row sees fewer than the others."""
    c, q, k, v = case(be, type_, heads, n_kv, 64, n, total - n, extra=3)
    ref, added = attention(q, k, v, total - n)
    before = np.abs(rows(4, n_kv, total + 2))
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, 64, n, total, total - n, dev(before))
    assert np.max(np.abs(out.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
    mass = mass.cpu().numpy()
    assert mass_ok(mass[:, :total], before[:, :total], added) and np.array_equal(mass[:, total:], before[:, total:])


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
def test_nan_keys_reach_only_rows_that_see_them(be, type_):
    q, k, v = rows(5, 4, 2, 64), rows(6, 2, 60, 64), rows(7, 2, 60, 64)
    k[1, 59, 3], v[0, 59, 2] = np.nan, np.inf
    c = A.KVCache(be, 60, 1, 2, 64, type=type_)
    c.append(0, dev(k), dev(v), 60, 64)
    if type_ == B.Q4_0:
        k, v = q4_values(k), q4_values(v)
    ref, added = attention(q, k, v, 58)
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, 4, 2, 64, 2, 60, 58, None)
    assert np.array_equal(np.isnan(out.cpu().numpy()), np.isnan(ref))
    mass = mass.cpu().numpy()
    assert np.array_equal(np.isnan(mass), np.isnan(added)) and mass_ok(mass[0], np.zeros(60, F32), added[0])


def test_refusals(be):
    c, q, k, v = case(be, B.Q4_0, 8, 2, 64, 1, 39)
    d, m = dev(q), dev(np.zeros((2, 40), F32))
    for kw, code in (({"kv_len": 41}, B.E_DIM), ({"kv_len": 0}, B.E_DIM), ({"layer": 1}, B.E_INVALID), ({"q_len": 0}, B.E_DIM),
                     ({"n_head_kv": 4}, B.E_DIM), ({"head_dim": 128}, B.E_DIM), ({"out_type": B.Q8_0}, B.E_UNSUPPORTED),
                     ({"mass": dev(np.zeros((2, 40), np.float64))}, B.E_INVALID), ({"mass": dev(np.zeros((2, 41), F32))[:, 1:]}, B.E_INVALID),
                     ({"mass": dev(np.zeros((2, 39), F32))}, B.E_DIM), ({"mass": dev(np.zeros((1, 40), F32))}, B.E_DIM),
                     ({"q_len": 65536}, B.E_DIM), ({"start_pos": 2 ** 31 - 1}, B.E_DIM), ({"n_head": 6, "out_type": B.Q8_K}, B.E_DIM)):
        a = {"layer": 0, "n_head": 8, "n_head_kv": 2, "head_dim": 64, "q_len": 1, "kv_len": 40, "start_pos": 39, "mass": m,
             "out_type": B.F32} | kw
        with pytest.raises(B.BarqError) as e:
            A.compute_attention_mass(be, d, c, a["layer"], a["n_head"], a["n_head_kv"], a["head_dim"], a["q_len"], a["kv_len"],
                                     a["start_pos"], a["mass"], out_type=a["out_type"], out=d)
        assert e.value.code == code, kw
    assert not m.cpu().numpy().any()
