"""Eviction from the KV cache by accumulated attention weight: which positions
stay (exact), and the rows, masses and lengths afterwards (bit for bit)."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import attention as A
from kv_ref import kept as kept_ref
from kv_ref import q4_values

pytestmark = pytest.mark.gpu
F32 = np.float32


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def masses(kind, n_kv, n, seed=3):
    rng = np.random.default_rng(seed + n)
    if kind == "spread":
        return np.exp(8 * rng.standard_normal((n_kv, n))).astype(F32)
    if kind == "ties":
        return rng.integers(0, 3, (n_kv, n)).astype(F32)
    if kind == "zero":
        return np.zeros((n_kv, n), F32)
    m = rng.standard_normal((n_kv, n)).astype(F32)   # "odd": signs, zeros of both, NaN, infinities
    m[:, ::7], m[:, 3::11], m[:, 5::13], m[:, 2::17] = 0, -0.0, np.nan, np.inf
    m[:, 1::19] = -np.inf
    return m


def fill(be, type_, n_kv, n, hd, layers=2, room=None):
    rng = np.random.default_rng(n + hd)
    k, v = (rng.standard_normal((n_kv, n, hd)).astype(F32) for _ in "kv")
    c = A.KVCache(be, room or n, layers, n_kv, hd, type=type_)
    c.append(layers - 1, dev(k), dev(v), n, hd)
    return c, (q4_values(k), q4_values(v)) if type_ == B.Q4_0 else (k, v)


def check(c, layer, k, v, kept):
    i = np.arange(len(kept))[:, None]
    assert c.layer_len(layer) == kept.shape[1]
    gk, gv = (t.cpu().numpy() for t in c.read(layer, 0, kept.shape[1]))
    assert np.array_equal(gk, k[i, kept]) and np.array_equal(gv, v[i, kept])


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("kind", ["spread", "ties", "zero", "odd"])
@pytest.mark.parametrize("n,keep,recent", [(1, 1, 0), (9, 4, 0), (100, 37, 5), (64, 64, 3), (50, 70, 60), (200, 13, 13),
                                           (4096, 2000, 100), (4097, 1, 0), (5000, 4999, 1),
                                           (12001, 6000, 77), (16383, 16000, 0), (16384, 3, 2)])
def test_evict_in_place(be, type_, kind, n, keep, recent):
    n_kv, hd = 3, 64
    c, (k, v) = fill(be, type_, n_kv, n, hd)
    mass = masses(kind, n_kv, n + 5)   # more room than positions
    want = kept_ref(mass[:, :n], n, keep, recent)
    new = mass.copy()
    new[:, :n] = 0
    new[:, :want.shape[1]] = np.take_along_axis(mass, want, 1)
    d = dev(mass)
    kept, out = c.evict(1, d, keep, recent)
    assert out is d and np.array_equal(kept.cpu().numpy(), want)
    assert np.array_equal(out.cpu().numpy(), new, equal_nan=True)   # the columns behind the positions as they were
    check(c, 1, k, v, want)
    assert c.layer_len(0) == 0 and c.size() == 0


@pytest.mark.parametrize("n", [16384, 16385, 32768, 70000])
def test_long_heads(be, n):
    c, (k, v) = fill(be, B.Q4_0, 2, n, 64, layers=1)
    mass = masses("spread", 2, n)
    mass[:, : n // 2] = np.round(mass[:, : n // 2], 1)   # many small ones become equal
    keep, recent = n // 3, 777
    want = kept_ref(mass, n, keep, recent)
    to = A.KVCache(be, keep + 3, 1, 2, 64, type=B.Q4_0)
    new = np.zeros_like(mass)
    kept, out = c.evict(0, dev(mass), keep, recent, dst=to, mass_out=dev(np.full_like(mass, np.nan)))
    new[:, :keep] = np.take_along_axis(mass, want, 1)
    assert np.array_equal(kept.cpu().numpy(), want) and np.array_equal(out.cpu().numpy(), new)
    check(to, 0, k, v, want)
    assert to.size() == keep and c.size() == n   # the source stays as it was
    check(c, 0, k, v, np.tile(np.arange(n), (2, 1)))


@pytest.mark.parametrize("type_,hd", [(B.F32, 128), (B.F32, 6), (B.F32, 5), (B.Q4_0, 128), (B.Q4_0, 256)])
def test_into_another_cache_then_append(be, type_, hd):
    n_kv, n, keep = 4, 203, 61
    c, (k, v) = fill(be, type_, n_kv, n, hd)
    to, _ = fill(be, type_, n_kv, 90, hd, layers=3)   # layer 2 full, layer 1 empty
    mass = masses("spread", n_kv, n)
    want = kept_ref(mass, n, keep, 10)
    c.evict(1, dev(mass), keep, 10, dst=to)
    check(to, 1, k, v, want)
    assert to.layer_len(2) == 90
    # the rows appended next go behind the kept ones, in the middle of a tile
    rng = np.random.default_rng(8)
    nk, nv = (rng.standard_normal((n_kv, 7, hd)).astype(F32) for _ in "kv")
    to.append(1, dev(nk), dev(nv), 7, hd)
    gk, gv = (t.cpu().numpy() for t in to.read(1, 0, keep + 7))
    i = np.arange(n_kv)[:, None]
    if type_ == B.Q4_0:
        nk, nv = q4_values(nk), q4_values(nv)
    assert np.array_equal(gk, np.concatenate([k[i, want], nk], 1)) and np.array_equal(gv, np.concatenate([v[i, want], nv], 1))


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
def test_host_buffers_and_nothing_kept(be, type_):
    c, (k, v) = fill(be, type_, 2, 77, 64)
    mass = masses("ties", 2, 80)
    want = kept_ref(mass[:, :77], 77, 20, 4)
    kept, out = c.evict(1, mass.copy(), 20, 4, mem=B.MEM_HOST)
    assert np.array_equal(kept, want) and np.array_equal(out[:, 77:], mass[:, 77:])
    assert np.array_equal(out[:, :20], np.take_along_axis(mass, want, 1)) and not out[:, 20:77].any()
    check(c, 1, k, v, want)
    kept, out = c.evict(1, dev(out), 0, 0)
    assert kept.shape == (2, 0) and c.layer_len(1) == 0 and not out[:, :20].any()
    kept, _ = c.evict(1, out, 5, 2)   # an empty layer
    assert kept.shape == (2, 0)


def test_refusals(be):
    c, _ = fill(be, B.Q4_0, 2, 40, 64)
    mass = dev(masses("ties", 2, 40))
    for args, kw, code in (((1, mass, 5, 6), {}, B.E_DIM), ((2, mass, 5, 1), {}, B.E_INVALID),
                           ((1, mass[:, :39].contiguous(), 5, 1), {}, B.E_DIM), ((1, mass[:1], 5, 1), {}, B.E_DIM),
                           ((1, mass, 20, 1), {"dst": A.KVCache(be, 19, 2, 2, 64, type=B.Q4_0)}, B.E_INVALID),
                           ((1, mass, 20, 1), {"dst": A.KVCache(be, 40, 2, 2, 64)}, B.E_DIM),
                           ((1, mass, 20, 1), {"dst": A.KVCache(be, 40, 1, 2, 64, type=B.Q4_0)}, B.E_INVALID),
                           ((1, mass, 20, 1), {"dst": A.KVCache(be, 40, 2, 2, 128, type=B.Q4_0)}, B.E_DIM)):
        with pytest.raises(B.BarqError) as e:
            c.evict(*args, **kw)
        assert e.value.code == code
    with pytest.raises(B.BarqError) as e:
        B._lib.check(be._lib.barq_rocm_kv_cache_evict(be.h, c.c, c.c, 1, None, None, 40, 5, 1, None, B.MEM_DEVICE))
    assert e.value.code == B.E_INVALID
    assert c.layer_len(1) == 40
