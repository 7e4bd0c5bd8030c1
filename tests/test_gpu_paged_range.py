"""Attention over a paged cache at the ends of f32's range: finite values of
every size where no query looks, and averages of values near the largest; and
numbers of heads, pages and positions at the ends of theirs."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import paged as P
from paged_ref import assert_within, attention, cache_values
from test_gpu_paged import Case, dev

pytestmark = pytest.mark.gpu
F32 = np.float32
MOST = np.finfo(F32).max
HUGE = np.array([MOST, -MOST, 3.397e38, -3.397e38, 3.395e38], F32)   # (bf16's largest is 3.3895e38; halfway to infinity: 3.3961e38)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (60, 3)])
@pytest.mark.parametrize("rows", [1, 24, 40, 150])
def test_finite_values_where_no_query_looks(be, type_, hd, window, n_sink, rows):
    """Behind the last position of a page, behind the window, after a query: whatever finite values lie there, in K or in V,
    the results are those of the places that are seen."""
    n, heads, kv, page = 300, 8, 2, 16
    rng = np.random.default_rng(hd + rows)
    k, v = (rng.standard_normal((n, kv, hd)).astype(F32) for _ in "kv")

    def huge(x):
        x[...] = HUGE[np.arange(x.size).reshape(x.shape) % len(HUGE)]
    for x in (k, v):
        if rows > 1:
            huge(x[n - 1])   # seen by the last token alone
        if window:
            huge(x[n_sink])
            huge(x[n - rows - window])   # the last one that no row sees
    c = Case(be, type_, heads, kv, hd, page, [(rows, n)], window, n_sink, k=k, v=v)
    tail = np.empty((304 - n, kv, hd), F32)
    huge(tail)
    behind = P.PagedBatch(c.cache, heads, 1, 4, c.table.shape[1])
    behind.set([304 - n], [304], c.table)
    x = dev(tail)
    behind.append(c.layer, x, x)
    be.sync()
    got = c.batch.attention(c.layer, dev(c.q)).cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        want, off = c.want()
    t = rows if rows == 1 else rows - 1
    assert_within(got[:t], want[:t], off[:t])


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,before", [(1, 0), (1, 63), (1, 5000), (24, 40), (24, 1000), (40, 0), (150, 0), (150, 150), (150, 3000)])
def test_averages_of_values_near_the_largest(be, hd, rows, before):
    """An f32 cache: no sum on the way is larger than the largest value."""
    n = rows + before
    rng = np.random.default_rng(n + hd)
    v = rng.uniform(1e38, 3.38e38, (n, 1, hd)).astype(F32) * np.where(np.arange(hd) % 2, F32(-1), F32(1))
    k = (0.3 * rng.standard_normal((n, 1, hd))).astype(F32)
    c = Case(be, B.F32, 4, 1, hd, 32, [(rows, n)], k=k, v=v)
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("rows", [1, 24, 150])
def test_averages_of_small_values(be, rows):
    """V of about 2^-90.  The weights are multiplied by 2^-10 on the way, and a product below 2^-126 may be lost: 874 of them are less
    than 2^-116, a thousandth of the 2^-20 of 2^-90 that each result may be off by in any case."""
    n = rows + 700
    rng = np.random.default_rng(n)
    k, v = (rng.standard_normal((n, 1, 64)).astype(F32) for _ in "kv")
    c = Case(be, B.F32, 4, 1, 64, 32, [(rows, n)], k=F32(0.1) * k, v=v * F32(2.0 ** -90))
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("heads,kv,hd,page,seqs,window,n_sink", [
    (200, 1, 64, 16, [(1, 500), (2, 90)], 0, 0),          # a token's rows over several tiles, of either kernel
    (256, 2, 128, 32, [(1, 333), (3, 3)], 40, 5),
    (600, 600, 64, 16, [(1, 700), (5, 60)], 0, 0),        # more kv heads than workgroups: nothing is split
    (1100, 550, 64, 16, [(70, 130)], 30, 2),
    (8, 2, 64, 65536, [(1, 700), (90, 200)], 0, 0),       # one page
    (6, 2, 256, 4096, [(1, 4097), (0, 3), (33, 5000)], 1000, 64)])
def test_heads_and_pages_of_every_number(be, type_, heads, kv, hd, page, seqs, window, n_sink):
    c = Case(be, type_, heads, kv, hd, page, seqs, window, n_sink, layers=1)
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
def test_a_pool_beyond_32_bits(be, type_):
    """More than 2^32 bytes of K in a layer, and the second layer behind it: rows at both ends."""
    import torch
    hd, kv, page = 256, 8, 64
    pages = (1 << 32) // (kv * hd * page * (2 if type_ == B.F16 else 4)) + 9
    c = P.PagedCache(be, pages, page, 2, kv, hd, type=type_)
    b = P.PagedBatch(c, kv, 2, 400, 4)
    rng = np.random.default_rng(3)
    table = np.array([[0, pages - 1, 1, pages - 2], [pages - 3, 2, pages - 4, 3]], np.int32)
    k, v = (rng.standard_normal((2, 400, kv, hd)).astype(F32) for _ in "kv")
    b.set([200, 200], [200, 200], table)
    for layer in range(2):
        x, y = dev(k[layer]), dev(v[layer])
        b.append(layer, x, y)
        be.sync()
    for layer in range(2):
        kk, vv = (cache_values(x[layer], type_ == B.F16) for x in (k, v))
        for got, held in zip(b.read(layer), (kk, vv)):
            assert np.array_equal(got.cpu().numpy().astype(np.float64), held)
    for new in (1, 100):
        b.set([new, new], [200, 200], table)
        q = rng.standard_normal((kv, 2 * new, hd)).astype(F32)
        for layer in range(2):
            kk, vv = (cache_values(x[layer], type_ == B.F16) for x in (k, v))
            want, off = attention(q, [(new, kk[:200], vv[:200], None), (new, kk[200:], vv[200:], None)])
            assert_within(b.attention(layer, dev(q)).cpu().numpy(), want, off)
    torch.cuda.synchronize()
