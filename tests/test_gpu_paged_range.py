"""Attention over a paged cache at the ends of f32's range: finite values of
every size where no query looks, and averages of values near the largest."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import paged as P
from paged_ref import assert_within
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
