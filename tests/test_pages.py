"""Handing out the pages of a paged cache (barq_rocm.paged.Pages), and the
rotary frequencies for long contexts: host code, no GPU."""
import math
import random

import numpy as np
import pytest

from barq_rocm import _lib as L
from barq_rocm import attention as A
from barq_rocm.paged import Pages, Sequence


def test_growing_and_closing():
    p, a, b = Pages(5, 16), Sequence(), Sequence()
    p.grow(a, 16)
    p.grow(b, 17)
    p.grow(a, 1)
    assert (len(a.pages), len(b.pages), p.free()) == (2, 2, 1)
    with pytest.raises(L.BarqError) as e:
        p.grow(b, 32)
    assert e.value.code == L.E_ALLOC and (b.length, len(b.pages), p.free()) == (17, 2, 1)
    p.grow(b, 15)
    assert p.free() == 1
    p.close(a)
    assert (a.length, a.pages, p.free()) == (0, [], 3)
    p.grow(b, 33)
    assert p.free() == 0 and sorted(b.pages) == list(range(5)) and len(set(b.pages)) == 5


def test_a_fork_shares_whole_pages():
    p, a = Pages(6, 16), Sequence()
    p.grow(a, 40)
    b = p.fork(a)
    assert (b.length, b.pages) == (32, a.pages[:2])
    p.grow(b, 5)
    assert b.pages[2] not in a.pages and p.free() == 2
    p.close(a)
    assert p.free() == 3   # the shared ones stay b's
    p.close(b)
    assert p.free() == 6


@pytest.mark.parametrize("window,n_sink", [(1, 0), (16, 0), (20, 1), (33, 16), (100, 17)])
def test_what_is_behind_the_window_is_given_back(window, n_sink):
    p, s = Pages(20, 16), Sequence()
    for n in (50, 1, 1, 70, 1, 100):
        p.grow(s, n)
        p.drop_behind(s, window, n_sink)
        # the next query is at s.length: it sees s.length - window + 1 .. on, and the first n_sink
        for i, page in enumerate(s.pages):
            seen = (i + 1) * 16 > s.length - window + 1 or i * 16 < n_sink
            assert (page >= 0) == seen
        held = [x for x in s.pages if x >= 0]
        assert len(held) == len(set(held)) and p.free() == 20 - len(held)


def test_back_into_a_shared_page_is_refused():
    p, a = Pages(6, 16), Sequence()
    p.grow(a, 40)
    b = p.fork(a)
    p.shrink(a, 33)   # a page of its own
    with pytest.raises(L.BarqError) as e:
        p.shrink(a, 20)   # what it would add next is b's prefix
    assert e.value.code == L.E_INVALID and (a.length, len(a.pages), p.free()) == (33, 3, 3)
    p.shrink(a, 32)
    p.shrink(a, 16)
    p.shrink(b, 32)
    with pytest.raises(L.BarqError):
        p.shrink(a, 9)
    p.shrink(b, 17)   # the second page is b's alone by now
    p.close(b)
    p.shrink(a, 9)
    assert (a.length, len(a.pages), p.free()) == (9, 1, 5)
    for length in (-1, 10):
        with pytest.raises(L.BarqError) as e:
            p.shrink(a, length)
        assert e.value.code == L.E_DIM and a.length == 9
    with pytest.raises(L.BarqError) as e:
        p.grow(a, -1)
    assert e.value.code == L.E_DIM and a.length == 9


@pytest.mark.parametrize("window,n_sink", [(1, 0), (5, 0), (16, 0), (20, 1), (33, 16), (70, 17)])
def test_back_to_where_the_window_is_gone_is_refused(window, n_sink):
    rng = random.Random(window)
    for _ in range(300):
        p, s = Pages(20, 16), Sequence()
        for n in (rng.randint(0, 120), rng.randint(1, 40)):
            p.grow(s, n)
            if rng.random() < 0.8:
                p.drop_behind(s, window, n_sink)

        def there(length):
            """The query at `length` sees no position that is given back, nor goes to one."""
            return all(s.pages[j // 16] >= 0 for j in range(-(-length // 16) * 16) if j > length - window or j < n_sink)
        for what in (p.shrink, p.fork):
            length = rng.randint(0, s.length) if what == p.shrink else s.length // 16 * 16
            try:
                fine, was = there(length), (s.length, list(s.pages))
                got = what(s, length) if what == p.shrink else what(s)
            except L.BarqError as e:
                # (a window of one position needs nothing before the first of a page: refused all the same)
                assert e.code == L.E_INVALID and (not fine or window == 1) and was == (s.length, s.pages)
                continue
            assert fine
            t = s if what == p.shrink else got
            assert t.length == length
            # what it then grows to and gives back stays consistent
            p.grow(t, 3)
            p.drop_behind(t, window, n_sink)
        p.close(s)
        assert s.gone == (0, 0)


def test_drawn_sessions_lose_no_page():
    rng = random.Random(2)
    p, seqs = Pages(30, 16), []
    for _ in range(2000):
        what = rng.random()
        if what < 0.3 and len(seqs) < 12:
            try:
                seqs.append(p.fork(rng.choice(seqs)) if seqs and rng.random() < 0.5 else Sequence())
            except L.BarqError as e:   # (behind the window)
                assert e.code == L.E_INVALID
        elif seqs and what < 0.8:
            try:
                p.grow(rng.choice(seqs), rng.randint(0, 40))
            except L.BarqError:
                pass
        elif seqs and what < 0.85:
            s = rng.choice(seqs)
            try:
                p.shrink(s, rng.randint(0, s.length))
            except L.BarqError as e:
                assert e.code == L.E_INVALID
        elif seqs and what < 0.9:
            p.drop_behind(rng.choice(seqs), rng.randint(1, 30), rng.choice([0, 4, 20]))
        elif seqs:
            p.close(seqs.pop(rng.randrange(len(seqs))))
        held = {x for s in seqs for x in s.pages if x >= 0}
        assert p.free() == 30 - len(held)
    for s in seqs:
        p.close(s)
    assert p.free() == 30


def frequencies(scaling, rot, base, factor=1.0, trained=0.0, fast=32.0, slow=1.0):
    plain = base ** (-2.0 * np.arange(rot // 2) / rot)
    if scaling == L.ROPE_LINEAR:
        return plain / factor, 1.0
    if scaling == L.ROPE_NTK:
        return (base * factor ** (rot / (rot - 2))) ** (-2.0 * np.arange(rot // 2) / rot), 1.0
    if scaling == L.ROPE_YARN:
        turns = trained * plain / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0, 1)
        return plain * keep + plain / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return plain, 1.0


@pytest.mark.parametrize("scaling,args", [(L.ROPE_PLAIN, ()), (L.ROPE_LINEAR, (4.0,)), (L.ROPE_NTK, (8.0,)), (L.ROPE_YARN, (16.0, 4096.0)),
                                          (L.ROPE_YARN, (1.0, 4096.0)), (L.ROPE_YARN, (40.0, 8192.0, 20.0, 0.0))])
@pytest.mark.parametrize("rot,base", [(128, 10000.0), (64, 500000.0), (22, 1e6), (4, 100.0)])
def test_rope_frequencies(scaling, args, rot, base):
    want, magnitude = frequencies(scaling, rot, base, *args)
    f, m = A.rope_frequencies(scaling, rot, base, *args)
    # computed in 64 bits and rounded once: half a step, and one more of 2^-50 for pow
    assert f.dtype == np.float32 and np.all(np.abs(f - want) <= want * 2.0 ** -24 * (1 + 1e-6))
    assert abs(m - magnitude) <= magnitude * 2.0 ** -24
    if scaling == L.ROPE_NTK:   # the fastest pair stays, the slowest is slowed down by the whole factor
        plain = frequencies(L.ROPE_PLAIN, rot, base)[0]
        assert f[0] == 1 and f[-1] == pytest.approx(plain[-1] / args[0], rel=1e-6)


def test_rope_frequencies_refused():
    for code, args in ((L.E_DIM, (L.ROPE_PLAIN, 3, 1e4)), (L.E_DIM, (L.ROPE_PLAIN, 0, 1e4)), (L.E_UNSUPPORTED, (4, 64, 1e4)),
                       (L.E_UNSUPPORTED, (-1, 64, 1e4)), (L.E_INVALID, (L.ROPE_PLAIN, 64, 0.0)), (L.E_INVALID, (L.ROPE_PLAIN, 64, math.nan)),
                       (L.E_INVALID, (L.ROPE_LINEAR, 64, 1e4, 0.5)), (L.E_INVALID, (L.ROPE_NTK, 64, 1e4, math.inf)), (L.E_DIM, (L.ROPE_NTK, 2, 1e4, 2.0)),
                       (L.E_INVALID, (L.ROPE_YARN, 64, 1e4, 2.0)), (L.E_INVALID, (L.ROPE_YARN, 64, 1e4, 2.0, 4096.0, 1.0, 1.0))):
        with pytest.raises(L.BarqError) as e:
            A.rope_frequencies(*args)
        assert e.value.code == code, args
    lib = L.lib()
    assert lib.barq_rocm_rope_frequencies(0, 64, 1e4, 1.0, 0.0, 32.0, 1.0, None, None) == L.E_INVALID


def test_refusals_before_any_device():
    """What the paged calls refuse without a handle."""
    import ctypes
    lib, out = L.lib(), ctypes.c_void_p()
    create = lib.barq_rocm_paged_cache_create
    assert create(None, 4, 16, 1, 2, 64, L.F16, None) == L.E_INVALID
    assert create(None, 4, 16, 1, 2, 64, L.Q4_0, ctypes.byref(out)) == L.E_UNSUPPORTED
    assert create(None, 4, 16, 1, 2, 80, L.F16, ctypes.byref(out)) == L.E_UNSUPPORTED
    for pages, size in ((4, 8), (4, 48), (4, 1 << 17), (0, 16), (1 << 31, 16)):
        assert create(None, pages, size, 1, 2, 64, L.F16, ctypes.byref(out)) == L.E_DIM
    assert create(None, 4, 16, 1, 2, 64, L.F16, ctypes.byref(out)) == L.E_INVALID   # the null handle
    assert lib.barq_rocm_paged_batch_create(None, None, 4, 1, 1, 1, 0, 0, ctypes.byref(out)) == L.E_INVALID
    assert lib.barq_rocm_paged_batch_set(None, None, 0, None, None, None, 0) == L.E_INVALID
    assert lib.barq_rocm_paged_attention(None, None, 0, None, L.F32, None, L.MEM_DEVICE) == L.E_INVALID
    assert lib.barq_rocm_paged_attention(None, None, 0, None, L.F32, None, 7) == L.E_INVALID
    assert lib.barq_rocm_paged_append(None, None, 0, None, None, None, None, None, None, 0.0, None, L.MEM_DEVICE) == L.E_INVALID
    assert lib.barq_rocm_paged_read(None, None, 0, None, None, L.MEM_DEVICE) == L.E_INVALID
    assert lib.barq_rocm_paged_cache_destroy(None) == L.OK and lib.barq_rocm_paged_batch_destroy(None) == L.OK
    norm = lib.barq_rocm_norm_rope
    assert norm(None, None, 1, 1, 96, 0, None, 0.0, None, None, L.MEM_DEVICE) == L.E_UNSUPPORTED
    assert norm(None, None, 1, 1, 64, 0, None, 0.0, None, None, L.MEM_DEVICE) == L.E_INVALID
    for r, code in ((L.RotaryArg(7, 0, 1.0, 1.0, 16), L.E_DIM), (L.RotaryArg(66, 0, 1.0, 1.0, 16), L.E_DIM),
                    (L.RotaryArg(8, 2, 1.0, 1.0, 16), L.E_INVALID), (L.RotaryArg(8, 0, 1.0, 1.0, None), L.E_INVALID)):
        assert norm(None, 16, 1, 1, 64, 0, None, 0.0, ctypes.byref(r), 16, L.MEM_DEVICE) == code
    assert norm(None, 16, 2, 1, 64, 0x7ffffffe, None, 0.0, None, 16, L.MEM_DEVICE) == L.E_DIM
    assert norm(None, 16, 1 << 24, 1, 64, 0, None, 0.0, None, 16, L.MEM_DEVICE) == L.E_DIM
    assert norm(None, 16, 2, 1 << 40, 64, 0, None, 0.0, None, 16, L.MEM_DEVICE) == L.E_DIM
    assert norm(None, None, 0, 1, 64, 0, None, 0.0, None, None, L.MEM_DEVICE) == L.OK


@pytest.mark.parametrize("length", [0, 1, 15, 16, 31, 40])
@pytest.mark.parametrize("n_sink", [0, 1, 40])
def test_without_a_window_nothing_is_given_back(length, n_sink):
    """A window of 0 is none, as for a batch."""
    p, s = Pages(8, 16), Sequence()
    p.grow(s, length)
    was = list(s.pages)
    p.drop_behind(s, 0, n_sink)
    assert s.pages == was and p.free() == 8 - len(was) and s.gone == (0, 0)
    p.grow(s, 1)
    p.shrink(s, 0)
    assert p.free() == 8


@pytest.mark.parametrize("window,n_sink", [(-1, 0), (-100, 4), (5, -1), (0, -1), (16, -40)])
def test_windows_below_nothing_are_refused(window, n_sink):
    p, s = Pages(8, 16), Sequence()
    p.grow(s, 100)
    was = list(s.pages)
    with pytest.raises(L.BarqError) as e:
        p.drop_behind(s, window, n_sink)
    assert e.value.code == L.E_DIM and s.pages == was and p.free() == 1 and s.gone == (0, 0)
