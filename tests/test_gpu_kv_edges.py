"""Edges of attention over the KV cache and of its masses: rows that see only
NaN in a piece of the cache, queries whose elements differ by many powers of two,
scores up to f32's largest.

Calls that are meant for the matrix prompt kernel of a 4-bit cache are in
PROMPT_CALLS (heads, kv heads, head_dim, rows, positions); test_attention_q4_plan.py
checks on the host that they go there.

Bars, where a test names no other: those of test_gpu_kv_q4.py and
test_gpu_attention_mass.py (2e-5 * max |V| for the output; for a position's mass 2.5e-5 of
what the call adds, and 2^-23 of the total)."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import attention as A
from kv_ref import attention, kept, q4_values

pytestmark = pytest.mark.gpu
F32 = np.float32
PROMPT_CALLS = set()


def prompt_calls(*calls):
    PROMPT_CALLS.update(calls)
    return list(calls)


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(F32)


def cache(be, type_, k, v):
    n_kv, n, hd = k.shape
    c = A.KVCache(be, n, 1, n_kv, hd, type=type_)
    c.append(0, dev(k), dev(v), n, hd)
    return (c, q4_values(k), q4_values(v)) if type_ == B.Q4_0 else (c, k, v)


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("total,bad", [(129, 1), (300, 44), (1000, 1), (4097, 1), (4200, 200)])
@pytest.mark.parametrize("n", [1, 3])
def test_masses_of_rows_that_see_only_nan_in_a_piece(be, type_, total, bad, n):
    """The last `bad` keys of one kv head are NaN: the pieces that hold nothing else have no maximum, but their sum
    is NaN, and so are the weights of every position that the rows see."""
    heads, n_kv, hd = 32, 8, 128
    q, k, v = rows(1, heads, n, hd), rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    k[5, total - bad:, 9] = np.nan
    c, k, v = cache(be, type_, k, v)
    ref, added = attention(q, k, v, total - n)
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n, None)
    out, mass = out.cpu().numpy(), mass.cpu().numpy()
    assert np.isnan(added[5]).all() and np.isfinite(np.delete(added, 5, 0)).all()
    assert np.array_equal(np.isnan(out), np.isnan(ref)) and np.array_equal(np.isnan(mass), np.isnan(added))
    ok, seen = np.isfinite(ref), np.isfinite(added)
    assert np.max(np.abs(out[ok] - ref[ok])) <= 2e-5 * np.max(np.abs(v))
    assert np.all(np.abs(mass - added)[seen] <= (2.5e-5 + 2.0 ** -23) * added[seen])


UNEVEN = [(8, 2, 64, 1, 200), (8, 2, 128, 3, 200), (8, 2, 256, 1, 200), (8, 2, 256, 40, 300)] + prompt_calls(
    (8, 2, 64, 33, 200), (8, 2, 128, 40, 300))


@pytest.mark.parametrize("heads,n_kv,hd,n,total", UNEVEN)
@pytest.mark.parametrize("big", [3e4, 1e9, -1e25, 1e38])
def test_few_small_elements_beside_a_large_one(be, heads, n_kv, hd, n, total, big):
    """Keys that are zero in the large dim: the scores come from the small elements alone."""
    q, k, v = np.zeros((heads, n, hd), F32), 3 * rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    q[:, :, 7] = big
    k[:, :, 7] = 0
    for h in range(heads):   # one of them up to as many as a row of this size may have by chance
        few = [1, 2, 4, hd // 16][h % 4]
        q[h][:, 10:10 + few] = rows(h, n, few) + F32(1 / 3)
    c, k, v = cache(be, B.Q4_0, k, v)
    assert not k[:, :, 7].any()
    ref, added = attention(q, k, v, total - n)
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    assert np.max(np.abs(got - ref)) <= 2e-5 * np.max(np.abs(v))
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n, None)
    assert np.max(np.abs(out.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
    assert np.all(np.abs(mass.cpu().numpy() - added) <= (2.5e-5 + 2.0 ** -23) * added)


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("heads,n_kv,hd,n,total", [(8, 2, 64, 1, 300), (8, 2, 128, 2, 700), (8, 2, 256, 1, 300), (8, 2, 256, 40, 300)] +
                         prompt_calls((8, 2, 64, 40, 300), (8, 2, 128, 64, 500)))
@pytest.mark.parametrize("size,signs", [(2.0 ** 22, 0), (2.0 ** 24, 0), (2.0 ** 26, 0), (2.0 ** 28, 0), (2.0 ** 30, 0), (1e33, 0), (1e36, 0), (1e36, 1), (1e36, -1)])
def test_scores_up_to_the_largest(be, type_, heads, n_kv, hd, n, total, size, signs):
    """Queries so large that a row's weight is all on one position; scores of both signs, or of one.  They come near
    f32's largest (a sum's parts must stay below it).  Rows whose two largest scores agree to 2^-16 are left out: 24
    bits may not tell them apart."""
    q, k, v = rows(1, heads, n, hd) * F32(size), rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    if signs:
        q, k = np.abs(q) * signs, np.abs(k) + F32(0.01)
    c, k, v = cache(be, type_, k, v)
    ref, _ = attention(q, k, v, total - n)
    apart = np.empty((n, heads), bool)
    for h in range(heads):
        s = q[h].astype(np.float64) @ k[h * n_kv // heads].T.astype(np.float64) / np.sqrt(hd)
        assert (np.abs(q[h]).astype(np.float64) @ np.abs(k[h * n_kv // heads]).T.astype(np.float64)).max() < 3e38
        for i in range(n):
            two = np.sort(s[i, :total - n + i + 1])[-2:]
            apart[i, h] = two[1] - two[0] > 2.0 ** -16 * np.abs(s[i]).max()
    assert apart.mean() > 0.9
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n, None)
    for o in (got, out.cpu().numpy()):
        assert np.isfinite(o).all()
        # One weight and one V row.  In steps of 2^-23 of the result: the weight's split into two f16 values 1, the
        # product of both low parts (2^-11 of each) that is left out 2, three products' sums that the matrix unit
        # does not round to nearest 3, the sums into O and of the weights 1/2 each, the division 1.
        assert np.max(np.abs(o - ref)[apart]) <= 8 * 2.0 ** -23 * np.max(np.abs(v))
    mass = mass.cpu().numpy()
    assert np.isfinite(mass).all() and np.allclose(mass.sum(1), n * heads // n_kv, rtol=1e-5)


@pytest.mark.parametrize("heads,n_kv,hd,n,total", prompt_calls((4, 1, 64, 6150, 2 ** 20 + 5000)))
def test_a_million_positions_in_one_piece(be, heads, n_kv, hd, n, total):
    """Enough rows that the positions stay in one piece, of more than 2^20; a few of the rows against 64 bits."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v, q = (torch.randn(*s, device="cuda", generator=g) for s in ((n_kv, total, hd), (n_kv, total, hd), (heads, n, hd)))
    k[:, 2 ** 20:] *= 2   # what lies behind 2^20 counts
    c = A.KVCache(be, total, 1, n_kv, hd, type=B.Q4_0)
    torch.cuda.synchronize()
    c.append(0, k, v, total, hd)
    kq, vq = (t.cpu().numpy().astype(np.float64) for t in c.read(0, 0, total))
    got = A.compute_attention(be, q, c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    q = q.cpu().numpy()
    for i in (0, 3001, n - 1):
        ref, _ = attention(q[:, i:i + 1], kq[:, :total - n + i + 1], vq[:, :total - n + i + 1], total - n + i)
        assert np.max(np.abs(got[i] - ref[0])) <= 2e-5 * np.max(np.abs(vq))
    c.close()


def test_eviction_of_more_rows_than_a_launch_moves():
    """A launch takes fewer than 2^32 threads, and rows of one dim take one each: the heads go in two launches."""
    import torch
    be = B.Backend(0)   # (a workspace of 26 GB goes with it)
    heads, n, keep = 32768, 65540, 65537
    c = A.KVCache(be, n, 1, heads, 1)
    x = torch.randint(0, 1 << 20, (heads, n, 1), device="cuda").float()
    mass = torch.rand(heads, n, device="cuda")
    torch.cuda.synchronize()
    c.append(0, x, x, n, 1)
    be.sync()
    few = [0, 1, 20000, heads - 2, heads - 1]
    before = mass[few].clone()
    want = torch.from_numpy(kept(before.cpu().numpy(), n, keep, 10)).cuda().long()
    c.evict(0, mass, keep, 10, want_kept=False)
    assert c.layer_len(0) == keep
    assert torch.equal(mass[few][:, :keep], torch.gather(before, 1, want)) and not mass[:, keep:].any()
    out = torch.empty((heads, keep), device="cuda")
    for k in (True, False):
        B._lib.check(be._lib.barq_rocm_kv_cache_read(be.h, c.c, 0, 0, keep, out.data_ptr() if k else None,
                                                     None if k else out.data_ptr(), B.MEM_DEVICE))
        be.sync()
        assert torch.equal(out[few], torch.gather(x[few, :, 0], 1, want))
    c.close()
    be.close()
    del x, out, mass
    torch.cuda.empty_cache()


def test_attention_of_more_heads_than_a_launch_has_workgroups_for(be):
    """2^24 workgroups of 256 threads are refused; one head less is done (a single position: its V row)."""
    import torch
    n_kv, hd = 2 ** 24 + 16, 64
    v = torch.randint(-7, 8, (n_kv, 1, hd), device="cuda", dtype=torch.int8).float()
    v[:, :, ::32] = -8   # the blocks' scale is 1, and they hold these values
    q = torch.ones((n_kv, 1, hd), device="cuda")
    out = torch.full((n_kv, hd), 9.0, device="cuda")
    c = A.KVCache(be, 8, 1, n_kv, hd, type=B.Q4_0)
    torch.cuda.synchronize()
    c.append(0, v, v, 1, hd)
    for heads in (2 ** 24, 2 ** 24 - 1):
        args = (be.h, q.data_ptr(), c.c, 0, heads, n_kv, hd, 1, 1, 0, out.data_ptr(), B.MEM_DEVICE)
        if heads == 2 ** 24:
            with pytest.raises(B.BarqError) as e:
                B._lib.check(be._lib.barq_rocm_attention(*args))
            assert e.value.code == B.E_DIM
        else:
            B._lib.check(be._lib.barq_rocm_attention(*args))
        be.sync()
        assert torch.all(out[heads:] == 9)
    at = torch.arange(heads, device="cuda") * n_kv // heads
    # one weight, which is no power of two, and one row: the steps of 2^-23 counted in test_scores_up_to_the_largest
    assert torch.all((out[:heads] - v[at, 0]).abs() <= 8 * 2.0 ** -23 * 8)
    c.close()
    del v, q, out, at
    torch.cuda.empty_cache()


@pytest.mark.parametrize("heads,n_kv,hd,n,total", prompt_calls((8, 2, 64, 33, 233), (8, 2, 64, 70, 270), (8, 2, 128, 33, 233), (8, 2, 128, 70, 270)))
def test_prompt_queries_of_every_size(be, heads, n_kv, hd, n, total):
    """Rows with elements of very different sizes, all tiny, all huge, zero."""
    q, k, v = rows(1, heads, n, hd), rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    q[0] *= 1e-30
    q[1] *= 2.0 ** -np.arange(hd)
    q[2] = 0
    q[3, :, 7] = 1e25
    k[0, :, 7] = 0
    q[4] *= 1e-38
    q[5, :, ::2] = 0
    c, k, v = cache(be, B.Q4_0, k, v)
    ref, _ = attention(q, k, v, total - n)
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    assert np.max(np.abs(got - ref)) <= 2e-5 * np.max(np.abs(v))


@pytest.mark.parametrize("heads,n_kv,hd,n,total", prompt_calls((4, 2, 64, 64, 200), (4, 2, 64, 100, 200), (4, 2, 128, 70, 200)))
def test_prompt_nan_rows_reach_only_those_that_see_them(be, heads, n_kv, hd, n, total):
    k, v, q = rows(7, n_kv, total, hd), rows(8, n_kv, total, hd), rows(9, heads, n, hd)
    v[0, 190, 3] = np.inf        # one block of kv head 0
    v[1, 40, 50] = np.nan
    k[1, 195, 1] = np.nan        # a whole row of scores
    c, k, v = cache(be, B.Q4_0, k, v)
    for start in (total - n, total - 20 - n, 0):
        ref, _ = attention(q, k, v, start)
        got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, start).cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert np.max(np.abs(np.nan_to_num(got) - np.nan_to_num(ref))) <= 2e-5 * np.nanmax(np.abs(v))


def sizes(q, k, v, start):
    """sum of p |V|, per row, head and dim: what a relative error of the weights multiplies."""
    return attention(q, k, np.abs(v), start)[0]


@pytest.mark.parametrize("heads,n_kv,hd,n,total", prompt_calls((4, 1, 64, 40, 500), (4, 1, 128, 70, 500)))
def test_prompt_spread_scores_and_values(be, heads, n_kv, hd, n, total):
    """A position that takes nearly all the weight of some rows and adds nothing, queries and values of very
    different sizes."""
    k, v, q = rows(10, n_kv, total, hd), rows(11, n_kv, total, hd), rows(12, heads, n, hd)
    v[0, 0] = 0
    q[0] = q[0, :1]
    k[0, 0] = 4 * q[0, 0]
    q[1] *= 1e-20
    q[2, :, 5] = 1e20
    k[:, :, 5] = 0
    v[0, 100:, :32] *= 2.0 ** -20
    c, k, v = cache(be, B.Q4_0, k, v)
    ref, _ = attention(q, k, v, total - n)
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    # scores reach 4 |q|^2 / sqrt(hd) * log2(e), about 65 with 128 dims, off by 96 * 2^-24 of it (3.7e-4) at most in log2 units
    assert np.all(np.abs(got - ref) <= 4e-4 * sizes(q, k, v, total - n) + 1e-30)


@pytest.mark.parametrize("heads,n_kv,hd,n,total", prompt_calls((2, 1, 64, 64, 200), (2, 1, 128, 90, 200)))
@pytest.mark.parametrize("peak", [60, 140, 1000])
def test_prompt_weights_down_to_the_least(be, heads, n_kv, hd, n, total, peak):
    """Scores that fall evenly from 0 to -peak (log2) over the positions, shuffled."""
    q = np.zeros((heads, n, hd), F32)
    q[:, :, 0] = 1
    k, v = np.zeros((n_kv, total, hd), F32), rows(13, n_kv, total, hd)
    k[0, :, 0] = -np.random.default_rng(1).permutation(total) * peak / total * np.log(2) * np.sqrt(hd)
    v[0, np.argmax(k[0, :, 0])] = 0
    c, k, v = cache(be, B.Q4_0, k, v)
    ref, _ = attention(q, k, v, total - n)
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    # one product a score: its three roundings and the exponent's (2^-23 of peak each) and 2^-20 for the rest
    assert np.all(np.abs(got - ref) <= (4 * peak * 2.0 ** -23 + 2.0 ** -20) * sizes(q, k, v, total - n) + 1e-37)


@pytest.mark.parametrize("heads,n_kv,hd,n,total", [(4, 2, 64, 1, 1), (4, 2, 128, 1, 300), (4, 2, 256, 30, 200)] +
                         prompt_calls((8, 2, 64, 40, 200), (8, 2, 128, 64, 500)))
def test_values_near_f16s_least(be, heads, n_kv, hd, n, total):
    """V rows of 2^-12 down to 2^-28, some rows of 1.  Beside the weights' errors an output is off by 2^-36 at most:
    three sums of products a step, each cut at 2^-24, under a largest weight of 2^14 to 2^15."""
    q, k, v = rows(1, heads, n, hd), rows(2, n_kv, total, hd), rows(3, n_kv, total, hd)
    v *= np.exp2(np.random.default_rng(4).integers(-28, -12, (n_kv, total, 1))).astype(F32)
    v[:, 7::50] = rows(5, *v[:, 7::50].shape)
    c, k, v = cache(be, B.Q4_0, k, v)
    ref, _ = attention(q, k, v, total - n)
    got = A.compute_attention(be, dev(q), c, 0, heads, n_kv, hd, n, total, total - n).cpu().numpy()
    assert np.all(np.abs(got - ref) <= 2 * 2.4e-5 * sizes(q, k, v, total - n) + 2.0 ** -36)
