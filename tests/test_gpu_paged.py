"""The paged KV cache: append with norms and rotation, read, attention with and
without a window, over both types; each call against tests/paged_ref.py.

Tolerances.  Rotated f32 values: the norm's sum of at most 256 squares (a tree of 5 levels on 8 in
line: 13 roundings), division, square root, two products: 2^-20 of a normed value with room; cos and sin
2^-22 (an eighth of a turn in f32, the function's ulps, magnitude), a rotated
value two products and a sum: 2^-20 (|x0| + |x1|) of the pair's normed values in all.  The
cache's f16 adds half a step, 2^-11 of the value (2^-25 below 2^-14)."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import _lib as L
from barq_rocm import attention as A
from barq_rocm import paged as P
from paged_ref import assert_within, attention, cache_values, norm_turn

pytestmark = pytest.mark.gpu
F32 = np.float32


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def freqs(rot, base=10000.0):
    return (base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))).astype(F32)


def tables(rng, page, lens, spare=3):
    """Pages in any order for sequences of these lengths -> [sequences, pages] (-1 behind a sequence's end), pages in all."""
    need = [-(-n // page) for n in lens]
    ids = rng.permutation(sum(need) + spare).astype(np.int32)
    out, at = np.full((len(lens), max(max(need), 1)), -1, np.int32), 0
    for s, n in enumerate(need):
        out[s, :n] = ids[at:at + n]
        at += n
    return out, sum(need) + spare


class Case:
    """A cache filled with rows of sequences of these (new tokens, length), and what it holds of them."""

    def __init__(self, be, type_, heads, kv, hd, page, seqs, window=0, n_sink=0, seed=1, gone=(), k=None, v=None, layers=2):
        rng = np.random.default_rng(seed)
        self.new, self.lens = [q for q, _ in seqs], [n for _, n in seqs]
        self.table, pages = tables(rng, page, self.lens)
        for s, i in gone:
            self.table[s, i] = -1
        self.total, self.heads, self.kv, self.hd, self.window, self.n_sink = sum(self.lens), heads, kv, hd, window, n_sink
        self.k = rng.standard_normal((self.total, kv, hd)).astype(F32) if k is None else k
        self.v = rng.standard_normal((self.total, kv, hd)).astype(F32) if v is None else v
        self.q = rng.standard_normal((heads, sum(self.new), hd)).astype(F32)
        self.cache = P.PagedCache(be, pages, page, layers, kv, hd, type=type_)
        self.fill = P.PagedBatch(self.cache, heads, len(seqs), max(self.total, 1), self.table.shape[1])
        self.fill.set(self.lens, self.lens, self.table)
        # what was in the pool before, and is in the places that nothing fills: NaN
        self.poison(be, page, pages, layers)
        self.layer = layers - 1
        if self.total:
            self.fill.append(self.layer, dev(self.k), dev(self.v))
            be.sync()   # (before torch gives their memory to the next tensor)
        self.batch = P.PagedBatch(self.cache, heads, len(seqs), max(sum(self.new), 1), self.table.shape[1], window, n_sink)
        self.batch.set(self.new, self.lens, self.table)
        f16 = type_ == B.F16
        self.kc, self.vc = cache_values(self.k, f16), cache_values(self.v, f16)
        self.there = [np.repeat(t >= 0, page)[:n] for t, n in zip(self.table, self.lens)]

    def poison(self, be, page, pages, layers):
        import torch
        b = P.PagedBatch(self.cache, self.heads, 1, pages * page, pages)
        b.set([pages * page], [pages * page], np.arange(pages, dtype=np.int32)[None])
        bad = torch.full((pages * page, self.kv, self.hd), float("nan"), device="cuda")
        for layer in range(layers):
            b.append(layer, bad, bad)
        be.sync()

    def seqs(self):
        at = np.cumsum([0] + self.lens)
        return [(n, self.kc[a:b], self.vc[a:b], t) for n, a, b, t in zip(self.new, at, at[1:], self.there)]

    def want(self):
        return attention(self.q, self.seqs(), self.window, self.n_sink)


# ---- norm and rotation, append, read --------------------------------------------------

ROT = [  # hd, rot, half, norm, freq_scale, magnitude, start
    (128, 128, True, True, 1.0, 1.0, 0),
    (128, 128, False, False, 1.0, 1.0, 1000003),
    (64, 64, True, False, 0.25, 1.0, 4095),
    (64, 22, False, True, 1.0, 1.25, 77),
    (128, 50, True, True, 1.0, 0.8, 100000),
    (256, 256, True, True, 0.125, 1.1, 131071),
    (256, 64, False, False, 1.0, 1.0, 9),
    (128, 2, True, True, 1.0, 1.0, 5),
    (64, 0, True, True, 1.0, 1.0, 3),
    # halves that end within a lane's eight dims
    (64, 62, True, True, 1.0, 1.0, 500),
    (128, 126, True, False, 1.0, 1.1, 20000),
    (256, 130, True, True, 0.5, 1.0, 12345),
    (128, 10, True, True, 1.0, 1.0, 70),
    (256, 232, True, False, 1.0, 1.0, 33),
]


def turn_bound(x, norm, eps, rot, half, magnitude):
    y = np.abs(norm_turn(x, np.zeros(len(x)), freqs(0), 0, half, norm, eps))
    pair = y.copy()
    if rot:
        one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
        both = (y[..., one] + y[..., two]) * magnitude
        pair[..., one], pair[..., two] = both, both
    return pair * 2.0 ** -20


@pytest.mark.parametrize("hd,rot,half,norm,scale,magnitude,start", ROT)
@pytest.mark.parametrize("rows,heads", [(1, 32), (3, 1), (70, 5)])
def test_norm_rope(be, hd, rot, half, norm, scale, magnitude, start, rows, heads):
    rng = np.random.default_rng(hd + rot + rows)
    x = rng.standard_normal((rows, heads, hd)).astype(F32)
    w = (1 + 0.3 * rng.standard_normal(hd)).astype(F32) if norm else None
    layout = A.ROPE_SPLIT_HALF if half else A.ROPE_INTERLEAVED
    want = norm_turn(x, np.arange(start, start + rows), freqs(rot), rot, half, w, 1e-5, scale, magnitude).transpose(1, 0, 2)
    off = turn_bound(x, w, 1e-5, rot, half, magnitude).transpose(1, 0, 2)
    for mem, to in ((L.MEM_DEVICE, dev), (L.MEM_HOST, np.ascontiguousarray)):
        r = A.Rotary(to(freqs(rot)), rot, layout, scale, magnitude)
        y = A.norm_rope(be, to(x), rows, heads, hd, start, r, None if w is None else to(w), 1e-5, mem=mem)
        assert_within(y if mem == L.MEM_HOST else y.cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("hd,rot,half,norm,scale,magnitude,start", ROT)
@pytest.mark.parametrize("page,heads,kv,seqs", [
    (16, 8, 2, [(1, 1)]), (16, 32, 8, [(1, 40), (0, 16), (17, 17), (5, 100), (33, 70)]), (128, 5, 5, [(200, 300), (1, 129)])])
def test_append(be, type_, hd, rot, half, norm, scale, magnitude, start, page, heads, kv, seqs):
    rng = np.random.default_rng(hd + rot + page)
    new, lens = [q for q, _ in seqs], [n for _, n in seqs]
    table, pages = tables(rng, page, lens)
    t, f16 = sum(new), type_ == B.F16
    c = P.PagedCache(be, pages, page, 2, kv, hd, type=type_)
    b = P.PagedBatch(c, heads, len(seqs), t, table.shape[1])
    whole = P.PagedBatch(c, heads, 1, pages * page, pages)
    whole.set([pages * page], [pages * page], np.arange(pages, dtype=np.int32)[None])
    old = rng.standard_normal((2, pages * page, kv, hd)).astype(np.float16).astype(F32)
    for layer in range(2):
        whole.append(layer, dev(old[0]), dev(old[1]))
        be.sync()
    b.set(new, lens, table)
    q, k, v = (rng.standard_normal((t, n, hd)).astype(F32) for n in (heads, kv, kv))
    wq, wk = ((1 + 0.3 * rng.standard_normal(hd)).astype(F32) for _ in "qk") if norm else (None, None)
    layout = A.ROPE_SPLIT_HALF if half else A.ROPE_INTERLEAVED
    pos = np.concatenate([np.arange(n - m, n) for m, n in seqs])
    rows = np.concatenate([table[s, np.arange(n - m, n) // page].astype(int) * page + np.arange(n - m, n) % page
                           for s, (m, n) in enumerate(seqs)])
    rest = np.setdiff1d(np.arange(pages * page), rows)
    args = (freqs(rot), rot, half)
    want_q = norm_turn(q, pos, *args, wq, 1e-6, scale, magnitude).transpose(1, 0, 2)
    want_k = norm_turn(k, pos, *args, wk, 1e-6, scale, magnitude)
    off_q = turn_bound(q, wq, 1e-6, rot, half, magnitude).transpose(1, 0, 2)
    off_k = turn_bound(k, wk, 1e-6, rot, half, magnitude)
    if f16:
        off_k = off_k + np.maximum(np.abs(want_k) * 2.0 ** -11 * (1 + 2.0 ** -9), 2.0 ** -25)
    for mem, to in ((L.MEM_DEVICE, dev), (L.MEM_HOST, np.ascontiguousarray)):
        r = A.Rotary(to(freqs(rot)), rot, layout, scale, magnitude)
        qo = b.append(1, to(k), to(v), q=to(q), rotary=r, q_norm=None if wq is None else to(wq),
                      k_norm=None if wk is None else to(wk), eps=1e-6, mem=mem)
        kr, vr = b.read(1, mem=mem)
        if mem == L.MEM_DEVICE:
            qo, kr, vr = (x.cpu().numpy() for x in (qo, kr, vr))
        assert kr.dtype == (np.float16 if f16 else F32)
        assert_within(qo, want_q, off_q, "q")
        assert_within(kr, want_k, off_k, "k")
        assert np.array_equal(vr.astype(np.float64), cache_values(v, f16))
        # nothing else of the pool has changed, in this layer or the other
        for layer, at in ((0, np.arange(pages * page)), (1, rest)):
            for x, o in zip(whole.read(layer), old):
                assert np.array_equal(x.cpu().numpy().astype(F32)[at], o[at])
    # k and v as they are: no norm, no rotation, no q
    b.append(0, dev(k), dev(v))
    kr, vr = b.read(0)
    assert np.array_equal(kr.cpu().numpy().astype(np.float64), cache_values(k, f16))
    assert np.array_equal(vr.cpu().numpy().astype(np.float64), cache_values(v, f16))


@pytest.mark.parametrize("type_", [B.F16, B.F32])
def test_what_the_cache_keeps_of_values_out_of_range(be, type_):
    x = np.ones((16, 1, 64), F32)
    x[0, 0, :12] = [np.inf, -np.inf, np.nan, 65504, 65519, 65520, 1e30, -1e30, 2.0 ** -24, 2.0 ** -25, -0.0, 3e38]
    c = P.PagedCache(be, 1, 16, 1, 1, 64, type=type_)
    b = P.PagedBatch(c, 1, 1, 16, 1)
    b.set([16], [16], [[0]])
    b.append(0, dev(x), dev(x))
    for y in b.read(0):
        assert np.array_equal(y.cpu().numpy().astype(np.float64), cache_values(x, type_ == B.F16), equal_nan=True)


def test_tokens_without_a_page(be):
    """They are not kept and read as zeros; their queries are rotated all the same."""
    rng = np.random.default_rng(2)
    c = P.PagedCache(be, 2, 16, 1, 2, 64)
    b = P.PagedBatch(c, 4, 1, 40, 3)
    k, v, q = (rng.standard_normal((40, n, 64)).astype(F32) for n in (2, 2, 4))
    b.set([40], [40], [[1, -1, 0]])
    r = A.Rotary(dev(freqs(64)), 64)
    qo = b.append(0, dev(k), dev(v), q=dev(q), rotary=r)
    be.sync()
    assert_within(qo.cpu().numpy(), norm_turn(q, np.arange(40), freqs(64), 64, False).transpose(1, 0, 2),
                  turn_bound(q, None, 0, 64, False, 1).transpose(1, 0, 2))
    kr, vr = (x.cpu().numpy() for x in b.read(0))
    there = np.r_[0:16, 32:40]
    assert not kr[16:32].any() and not vr[16:32].any() and kr[there].all()
    assert np.array_equal(vr[there].astype(np.float64), cache_values(v[there], True))


# ---- attention ---------------------------------------------------------------------

LENS = [
    [(1, 1)], [(1, 31)], [(1, 32)], [(1, 33)], [(1, 1000)], [(3, 3)], [(17, 200)], [(33, 33)], [(40, 300)], [(130, 130)],
    [(200, 517)], [(300, 300)], [(1, 5), (1, 400), (1, 64), (1, 129)], [(0, 50), (5, 77), (1, 1), (0, 0), (64, 150), (2, 258)],
]


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 128, 16), (4, 4, 64, 32), (7, 1, 64, 16), (4, 1, 256, 64), (20, 1, 128, 256),
                                              (32, 2, 64, 128)])
@pytest.mark.parametrize("seqs", LENS, ids=lambda s: "+".join(f"{q}of{n}" for q, n in s))
def test_attention(be, type_, heads, kv, hd, page, seqs):
    c = Case(be, type_, heads, kv, hd, page, seqs)
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (16, 0), (40, 4), (100, 50), (64, 33), (1000, 3), (2, 500)])
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 2, 128, 16), (4, 1, 256, 64), (10, 5, 64, 32)])
@pytest.mark.parametrize("seqs", [[(1, 1)], [(1, 700), (1, 90), (0, 3), (2, 40)], [(150, 400)], [(90, 90), (1, 300)]],
                         ids=lambda s: "+".join(f"{q}of{n}" for q, n in s))
def test_window(be, type_, window, n_sink, heads, kv, hd, page, seqs):
    """The pages behind the window are gone (and NaN lies there)."""
    gone = [(s, i) for s, (q, n) in enumerate(seqs) for i in range(-(-n // page))
            if i * page >= n_sink and (i + 1) * page <= n - q - window + 1]
    c = Case(be, type_, heads, kv, hd, page, seqs, window, n_sink, gone=gone)
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("seqs", [[(1, 100)], [(5, 100), (1, 16)], [(100, 100)]])
def test_pages_that_are_not_there(be, type_, seqs):
    """Any of them, all of a row's among them: those rows are zeros."""
    c = Case(be, type_, 8, 2, 64, 16, seqs, gone=[(0, 0), (0, 3), (0, 6)] + ([(1, 0)] if len(seqs) > 1 else []))
    want, off = c.want()
    got = c.batch.attention(c.layer, dev(c.q)).cpu().numpy()
    assert_within(got, want, off)
    if seqs[0][0] == 100:
        assert not got[:16].any() and got[16:].all()
    if len(seqs) > 1:
        assert not got[5].any()


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,before", [(1, 99), (6, 94), (30, 70), (100, 0), (180, 20)])
def test_nan_and_infinity_in_the_cache(be, type_, hd, rows, before):
    """They reach the rows that see them: all of the row from K, the dim from V."""
    n = rows + before
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((n, 2, hd)).astype(F32) for _ in "kv")
    k[n - 2, 0, 3] = np.inf
    v[n // 2, 0, 5] = np.nan
    v[n - 1, 1, 7] = -np.inf
    v[n - 3, 1, 9] = np.inf
    c = Case(be, type_, 8, 2, hd, 16, [(rows, n)], k=k, v=v)
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)
    # a query of NaN and one of infinities: their rows, no other
    q = c.q.copy()
    q[0, 0, 0], q[5, rows - 1, 1] = np.nan, np.inf
    got = c.batch.attention(c.layer, dev(q)).cpu().numpy()
    assert np.isnan(got[0, 0]).all() and np.isnan(got[rows - 1, 5]).all()
    got[0, 0], got[rows - 1, 5], want[0, 0], want[rows - 1, 5] = 0, 0, 0, 0
    assert_within(got, want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (17, 2), (64, 16), (90, 70)])
@pytest.mark.parametrize("rows,before", [(1, 299), (7, 200), (200, 150)])
def test_nan_and_infinity_beside_a_window(be, type_, hd, window, n_sink, rows, before):
    n = rows + before
    rng = np.random.default_rng(rows + hd)
    k, v = (rng.standard_normal((n, 2, hd)).astype(F32) for _ in "kv")
    for x in (k, v):
        for value in (np.nan, np.inf, -np.inf):
            for head in range(2):
                x[rng.integers(n), head, rng.integers(hd)] = value
    c = Case(be, type_, 8, 2, hd, 32, [(rows, n)], window, n_sink, k=k, v=v, gone=[(0, 2)])
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("rows", [1, 24, 150])
def test_windows_longer_than_everything(be, type_, rows):
    c = Case(be, type_, 8, 2, 64, 16, [(rows, rows + 333), (0, 5), (1, 1)])
    want = c.batch.attention(c.layer, dev(c.q)).cpu().numpy()
    for window, n_sink in ((rows + 333, 0), (1000, 1000), (2 ** 31 - 4096, 0), (2 ** 31 - 4095, 7), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1)):
        b = P.PagedBatch(c.cache, 8, 3, rows + 1, c.table.shape[1], window, n_sink)
        b.set(c.new, c.lens, c.table)
        assert np.array_equal(b.attention(c.layer, dev(c.q)).cpu().numpy(), want), (window, n_sink)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("rows", [1, 24, 150])
@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-30, 1, 1), (1e4, 1, 1), (1, 300, 1), (30, 30, 6e4), (1, 1e-6, 1e-6), (0, 1, 1),
                                                  (1e30, 1e-20, 1)])
def test_sizes_of_the_values(be, type_, rows, q_size, k_size, v_size):
    rng = np.random.default_rng(4)
    n = rows + 300
    k, v = (rng.standard_normal((n, 2, 128)).astype(F32) * F32(s) for s in (k_size, min(v_size, 1e4)))
    c = Case(be, type_, 4, 2, 128, 32, [(rows, n)], k=k, v=v)
    c.q *= F32(q_size)
    if k_size == 1:   # a few dims far larger than the others, in the queries; none of them counts where k is small
        c.q[..., :3] *= F32(2.0 ** 20)
        k[..., :3] *= F32(2.0 ** -20)
        c = Case(be, type_, 4, 2, 128, 32, [(rows, n)], k=k, v=v)
        c.q *= F32(q_size)
        c.q[..., :3] *= F32(2.0 ** 20)
    want, off = c.want()
    # f16 products below 2^-14 and f32 ones below 2^-126 lose bits: of v's own size here, or of nothing that counts
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off + (2.0 ** -36 if type_ == B.F16 else 1e-38))


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("rows", [1, 24, 150])
@pytest.mark.parametrize("log_size", [10, 19, 21, 23, 25, 30, 60])
def test_scores_of_every_size(be, type_, rows, log_size):
    """Scores of about 2^log_size, the largest one three times: those positions share all of the weight."""
    n, hd, rng = 200 + rows, 64, np.random.default_rng(log_size)
    k, v = np.zeros((n, 1, hd), F32), rng.standard_normal((n, 1, hd)).astype(F32)
    k[:, 0, 0] = rng.choice([0.5, 0.25, -1.0, 0.0], n)
    top = [3, 77, 190]
    k[top, 0, 0] = 1
    c = Case(be, type_, 2, 1, hd, 16, [(rows, n)], k=k, v=v)
    c.q[:] = 0
    c.q[..., 0] = F32(1.37 * 2.0 ** log_size)
    want = np.broadcast_to(c.vc[top].mean(0), (rows, 2, hd))   # (the others' weight: e^(-2^log_size / 16) at most)
    got = c.batch.attention(c.layer, dev(c.q)).cpu().numpy()
    # three equal weights, each f16 part of them exact or off by 2^-23; sums and division 2^-21
    assert_within(got, want, 2.0 ** -20 * np.abs(c.vc[top]).mean(0) + np.zeros_like(want) + 2.0 ** -36 + (np.exp(-2.0 ** log_size / 16) * 4))


@pytest.mark.parametrize("type_", [B.F16, B.F32])
def test_rows_in_q8_k_blocks(be, type_):
    import torch
    for seqs in ([(1, 300)], [(70, 200), (1, 40), (3, 3)]):
        c = Case(be, type_, 8, 2, 64, 16, seqs)
        q = dev(c.q)
        rows = c.batch.attention(c.layer, q)
        blocks = c.batch.attention(c.layer, q, out_type=B.Q8_K)
        want = torch.empty_like(blocks)
        be.quantize_act_raw(B.Q8_K, rows, rows.shape[0], 512, want, B.MEM_DEVICE)
        be.sync()
        assert torch.equal(blocks, want)
        host = c.batch.attention(c.layer, c.q, mem=L.MEM_HOST), c.batch.attention(c.layer, c.q, out_type=B.Q8_K, mem=L.MEM_HOST)
        assert np.array_equal(host[0], rows.cpu().numpy()) and np.array_equal(host[1], want.cpu().numpy())


# 64 kv heads leave 4 to 12 workgroups a head, fewer than these lengths fill evenly: some end one sequence and begin the next
UNEVEN = [[(1, n) for n in (700, 650, 600, 720, 690)], [(1, 40), (1, 900), (2, 33), (0, 300), (1, 1), (1, 820), (1, 760)],
          [(1, 900 + 17 * i) for i in range(8)], [(1, 1500), (1, 1500), (1, 1500)]]


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("hd,window,n_sink", [(64, 0, 0), (128, 0, 0), (256, 0, 0), (128, 500, 40)])
@pytest.mark.parametrize("seqs", UNEVEN, ids=lambda s: "+".join(f"{q}of{n}" for q, n in s))
def test_workgroups_that_go_on_with_another_sequence(be, type_, hd, window, n_sink, seqs):
    c = Case(be, type_, 64, 64, hd, 32, seqs, window, n_sink, layers=1)
    want, off = c.want()
    assert_within(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_more_than_the_caches_keep(be, type_, hd):
    """Over 160 MB of K and V, which are then read past the caches."""
    n = (200 << 20) // (64 * hd * (4 if type_ == B.F16 else 8)) // 3
    c = Case(be, type_, 64, 64, hd, 64, [(1, n), (1, n - 77), (0, 9), (1, n + 30)], layers=1)
    got = c.batch.attention(c.layer, dev(c.q)).cpu().numpy()
    want, off = c.want()
    assert_within(got, want, off)


def test_replays_with_other_workgroups(be):
    """A captured call goes round whatever shares the latest set() made."""
    import torch
    c = Case(be, B.F16, 64, 64, 64, 32, UNEVEN[2], layers=1)
    q = dev(c.q)
    tables = [(c.new, c.lens), ([1] + [0] * 7, [300] * 8), ([1] * 8, [30] * 7 + [1019]), ([0] * 8, c.lens), ([1, 1, 1] + [0] * 5, [300] * 8)]
    out = torch.empty(8 * 64 * 64, device="cuda")

    def call():
        L.check(be._lib.barq_rocm_paged_attention(be.h, c.batch.b, 0, q.data_ptr(), L.F32, out.data_ptr(), L.MEM_DEVICE))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.set_stream(stream)
    be.set_stream(stream.cuda_stream)
    try:
        want = []
        for new, lens in tables:
            c.batch.set(new, lens, c.table)
            out.fill_(-7.0)
            call()
            torch.cuda.synchronize()
            want.append(out.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
        other = torch.randn(1 << 20, device="cuda")
        for i in (0, 1, 2, 0, 3, 4, 0, 2):
            c.batch.set(*tables[i], c.table)
            out.fill_(-7.0)
            other.mul_(1.0001)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]), i
    finally:
        torch.cuda.set_stream(torch.cuda.default_stream())
        be.set_stream(None)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
def test_a_long_cache(be, type_):
    """100000 positions, a few of which matter."""
    import torch
    n, hd = 100000, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(n, 1, hd, device="cuda", generator=g) for _ in "kv")
    c = P.PagedCache(be, -(-n // 64), 64, 1, 1, hd, type=type_)
    b = P.PagedBatch(c, 2, 1, n, c.n_pages)
    table = np.random.default_rng(1).permutation(c.n_pages).astype(np.int32)[None]
    b.set([n], [n], table)
    torch.cuda.synchronize()
    b.append(0, k, v)
    for rows in (1, 3, 140):
        q = torch.randn(2, rows, hd, device="cuda", generator=g)
        torch.cuda.synchronize()
        b.set([rows], [n], table)
        got = b.attention(0, q).double()
        kk, vv = ((x.half() if type_ == B.F16 else x).double()[:, 0] for x in (k, v))
        at = torch.arange(n, device="cuda")
        hidden = at > torch.arange(n - rows, n, device="cuda")[:, None]
        for h in range(2):
            p = torch.softmax((q[h].double() @ kk.T / 8).masked_fill(hidden, -np.inf), -1)
            # scores of a few sums of 64 products, 2 * B 2^-18 of |v|'s mean weight each (paged_ref), most of it far from its bound
            assert ((got[:, h] - p @ vv).abs() <= 2e-4 * (p @ vv.abs())).all()
            assert (got[:, h] - p @ vv).norm() <= 1e-5 * (p @ vv).norm()


# ---- as a server runs them ------------------------------------------------------------

@pytest.mark.parametrize("type_", [B.F16, B.F32])
def test_a_server_grows_its_sequences(be, type_):
    """Chunks and single tokens of three sequences, step after step, pages handed out as they grow; each step's attention
    is over all that has been appended, with norms and rotation on the way."""
    rng = np.random.default_rng(6)
    heads, kv, hd, page, rot = 8, 4, 128, 16, 64
    c = P.PagedCache(be, 40, page, 1, kv, hd, type=type_)
    b, w = P.PagedBatch(c, heads, 3, 100, 12), P.PagedBatch(c, heads, 3, 100, 12, window=20, n_sink=2)
    wq, wk = ((1 + 0.2 * rng.standard_normal(hd)).astype(F32) for _ in "qk")
    r = A.Rotary(dev(freqs(rot)), rot, A.ROPE_SPLIT_HALF)
    free, own, lens = list(rng.permutation(40)), [[], [], []], [0, 0, 0]
    held = [[], [], []]
    for new in ([30, 1, 0], [1, 17, 5], [1, 1, 1], [0, 60, 1], [1, 1, 40]):
        for s in range(3):
            lens[s] += new[s]
            while len(own[s]) * page < lens[s]:
                own[s].append(int(free.pop()))
        b.set(new, lens, own)
        w.set(new, lens, own)
        t = sum(new)
        q, k, v = (rng.standard_normal((t, n, hd)).astype(F32) for n in (heads, kv, kv))
        qo = b.append(0, dev(k), dev(v), q=dev(q), rotary=r, q_norm=dev(wq), k_norm=dev(wk))
        kr, vr = (x.cpu().numpy().astype(np.float64) for x in b.read(0))
        at = np.cumsum([0] + new)
        for s in range(3):
            held[s].append((kr[at[s]:at[s + 1]], vr[at[s]:at[s + 1]]))
        pos = np.concatenate([np.arange(n - m, n) for m, n in zip(new, lens)])
        assert_within(qo.cpu().numpy(), norm_turn(q, pos, freqs(rot), rot, True, wq).transpose(1, 0, 2),
                      turn_bound(q, wq, 1e-5, rot, True, 1).transpose(1, 0, 2))
        seqs = [(m, *(np.concatenate([x[i] for x in held[s]]) for i in (0, 1)), None) for s, m in enumerate(new)]
        for batch, args in ((b, ()), (w, (20, 2))):
            want, off = attention(qo.cpu().numpy(), seqs, *args)
            assert_within(batch.attention(0, qo).cpu().numpy(), want, off)


def test_a_shared_prefix(be):
    """Two sequences over the same first pages."""
    rng = np.random.default_rng(9)
    c = P.PagedCache(be, 6, 16, 1, 1, 64, type=B.F32)
    b = P.PagedBatch(c, 2, 2, 64, 4)
    k, v = (rng.standard_normal((32, 1, 64)).astype(F32) for _ in "kv")
    b.set([32], [32], [[5, 2]])
    b.append(0, dev(k), dev(v))
    be.sync()
    k2, v2 = (rng.standard_normal((9, 1, 64)).astype(F32) for _ in "kv")
    b.set([4, 5], [36, 37], [[5, 2, 0], [5, 2, 3]])
    b.append(0, dev(k2), dev(v2))
    be.sync()
    q = rng.standard_normal((2, 9, 64)).astype(F32)
    seqs = [(m, np.concatenate([k, k2[a:a + m]]).astype(np.float64), np.concatenate([v, v2[a:a + m]]).astype(np.float64), None)
            for m, a in ((4, 0), (5, 4))]
    want, off = attention(q, seqs)
    assert_within(b.attention(0, dev(q)).cpu().numpy(), want, off)


@pytest.mark.parametrize("type_", [B.F16, B.F32])
def test_a_captured_step_replays_with_other_lengths(be, type_):
    """Fewer and more tokens, other pages; rows behind the last token stay as they were."""
    import torch
    rng = np.random.default_rng(7)
    heads, kv, hd, page, most = 8, 2, 64, 16, 80
    c = P.PagedCache(be, 64, page, 1, kv, hd, type=type_)
    b = P.PagedBatch(c, heads, 4, most, 40, window=300, n_sink=3)
    fill = P.PagedBatch(c, heads, 1, 64 * page, 64)
    fill.set([64 * page], [64 * page], np.arange(64, dtype=np.int32)[None])
    k0, v0 = (dev(rng.standard_normal((64 * page, kv, hd)).astype(F32)) for _ in "kv")
    q, k, v = (dev(rng.standard_normal((most, n * hd)).astype(F32)) for n in (heads, kv, kv))
    r = A.Rotary(dev(freqs(hd)), hd)
    qo = torch.empty(heads * most * hd, device="cuda")
    out = torch.empty(most * heads * hd, device="cuda")
    out8 = torch.empty(most * (heads * hd // 256 * 292), dtype=torch.uint8, device="cuda")
    ids = rng.permutation(64)
    steps = [([1, 1, 0, 1], [200, 30, 16, 1]), ([1, 1, 1, 1], [201, 31, 17, 2]), ([70, 1, 1, 1], [300, 64, 80, 90]),
             ([0, 0, 0, 0], [0, 0, 0, 0]), ([1, 5, 20, 1], [500, 200, 20, 100])]
    table = np.full((4, 32), -1, np.int32)
    for s in range(4):
        table[s, :16] = ids[16 * s:16 * s + 16]
    table[0, 16:32] = ids[48:64]   # (the first sequence's later pages are the last one's: read only)

    def call():
        L.check(be._lib.barq_rocm_paged_append(be.h, b.b, 0, q.data_ptr(), qo.data_ptr(), k.data_ptr(), v.data_ptr(), 0, 0, 1e-5,
                                               r.arg, L.MEM_DEVICE))
        L.check(be._lib.barq_rocm_paged_attention(be.h, b.b, 0, qo.data_ptr(), L.F32, out.data_ptr(), L.MEM_DEVICE))
        L.check(be._lib.barq_rocm_paged_attention(be.h, b.b, 0, qo.data_ptr(), L.Q8_K, out8.data_ptr(), L.MEM_DEVICE))

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.set_stream(stream)
    be.set_stream(stream.cuda_stream)
    try:
        want = []
        for new, lens in steps:
            fill.append(0, k0, v0)
            b.set(new, lens, table)
            for x in (qo, out):
                x.fill_(-7.0)
            out8.fill_(9)
            call()
            torch.cuda.synchronize()
            want.append([x.clone() for x in (qo, out, out8)])
        assert (want[3][1] == -7).all()
        b.set(*steps[0], table)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
            with pytest.raises(B.BarqError) as e:
                b.set(*steps[0], table)
            assert e.value.code == L.E_UNSUPPORTED
        other = torch.randn(1 << 20, device="cuda")
        for i in (0, 2, 1, 4, 3, 2, 0):
            fill.append(0, k0, v0)
            b.set(*steps[i], table)
            for x in (qo, out):
                x.fill_(-7.0)
            out8.fill_(9)
            other.mul_(1.0001)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip((qo, out, out8), want[i])), i
    finally:
        torch.cuda.set_stream(torch.cuda.default_stream())
        be.set_stream(None)


def test_batches_on_streams_of_their_own(be):
    """Two handles on two streams, each with a batch on the same cache, in turns without waiting."""
    import torch
    cases = [Case(be, B.F16, 8, 2, 128, 16, [(1, 900), (1, 300)]), Case(be, B.F16, 8, 2, 128, 16, [(90, 400)], seed=5)]
    other = B.Backend(0)
    want = [c.batch.attention(c.layer, dev(c.q)) for c in cases]
    q = [dev(c.q) for c in cases]
    out = [[torch.empty_like(w) for _ in range(20)] for w in want]
    arrays = [(np.array(c.new, np.int32), np.array(c.lens, np.int32)) for c in cases]
    torch.cuda.synchronize()
    for i in range(20):
        for h, c, (new, lens), x, o in zip((be, other), cases, arrays, q, out):
            L.check(be._lib.barq_rocm_paged_batch_set(h.h, c.batch.b, len(new), new.ctypes.data, lens.ctypes.data, c.table.ctypes.data,
                                                      c.table.shape[1]))
            L.check(be._lib.barq_rocm_paged_attention(h.h, c.batch.b, c.layer, x.data_ptr(), L.F32, o[i].data_ptr(), L.MEM_DEVICE))
    be.sync()
    other.sync()
    assert all(torch.equal(y, w) for w, o in zip(want, out) for y in o)
    other.close()


def test_buffers_where_they_are_allowed_to_be(be):
    import torch
    c = Case(be, B.F32, 4, 2, 64, 16, [(3, 40)])
    want = c.batch.attention(c.layer, dev(c.q))
    out = torch.full((3 * 4 * 64 + 9,), -3.0, device="cuda")
    L.check(be._lib.barq_rocm_paged_attention(be.h, c.batch.b, c.layer, dev(c.q).data_ptr(), L.F32, out[5:].data_ptr(), L.MEM_DEVICE))
    be.sync()
    assert torch.equal(out[5:-4].reshape(want.shape), want) and (out[:5] == -3).all() and (out[-4:] == -3).all()


def test_memory_outlives_the_cache_for_its_batches(be):
    c = Case(be, B.F16, 4, 2, 64, 16, [(3, 40)])
    want = c.batch.attention(c.layer, dev(c.q))
    c.cache.close()
    assert np.array_equal(c.batch.attention(c.layer, dev(c.q)).cpu().numpy(), want.cpu().numpy())


def test_an_empty_batch(be):
    c = Case(be, B.F16, 4, 2, 64, 16, [(0, 40), (0, 0)])
    assert c.batch.attention(c.layer, dev(np.zeros((4, 0, 64), F32))).shape == (0, 4, 64)
    assert c.batch.append(0, dev(np.zeros((0, 2, 64), F32)), dev(np.zeros((0, 2, 64), F32))) is None
    c.batch.set([], [], [])
    assert c.batch.read(0)[0].shape == (0, 2, 64)


# ---- refusals ------------------------------------------------------------------------

def refused(code, f, *a, **k):
    with pytest.raises(B.BarqError) as e:
        f(*a, **k)
    assert e.value.code == code, e.value


def test_refusals(be):
    for args, code in (((4, 16, 1, 2, 64, B.Q4_0), L.E_UNSUPPORTED), ((4, 16, 1, 2, 96, B.F16), L.E_UNSUPPORTED),
                       ((4, 24, 1, 2, 64, B.F16), L.E_DIM), ((4, 8, 1, 2, 64, B.F16), L.E_DIM), ((0, 16, 1, 2, 64, B.F16), L.E_DIM),
                       ((4, 16, 0, 2, 64, B.F16), L.E_DIM), ((1 << 28, 16, 1, 2, 64, B.F16), L.E_DIM),
                       ((1 << 20, 16, 1 << 30, 60000, 64, B.F16), L.E_DIM)):
        refused(code, P.PagedCache, be, *args[:5], type=args[5])
    c = P.PagedCache(be, 4, 16, 2, 2, 64)
    for args, code in (((3, 1, 8, 4), L.E_DIM), ((0, 1, 8, 4), L.E_DIM), ((4, 0, 8, 4), L.E_DIM), ((4, 1, 0, 4), L.E_DIM), ((4, 1, 8, 0), L.E_DIM),
                       ((4, 1, 1 << 40, 4), L.E_DIM), ((4, 1 << 20, 8, 1 << 20), L.E_DIM),
                       ((4, 1 << 22, 8, 1), L.E_DIM), ((4, 1, 1 << 26, 1), L.E_DIM)):
        refused(code, P.PagedBatch, c, *args)
    b = P.PagedBatch(c, 4, 2, 8, 3)
    b.set([2], [20], [[1, 3]])
    for q, kv, pages, code in (([9], [9], [[0]], L.E_DIM), ([1], [17], [[0]], L.E_DIM), ([1], [17], [[0, 4]], L.E_INVALID),
                               ([1, 1, 1], [1, 1, 1], [[0], [1], [2]], L.E_DIM), ([2, 1], [2, 1], [[2], [2]], L.E_INVALID),
                               ([3], [2], [[0]], L.E_DIM), ([1], [60], [[0, 1, 2, 3]], L.E_DIM)):
        refused(code, b.set, q, kv, pages)
    refused(L.E_DIM, b.set, [1, 1], [1], [[0], [1]])
    # none of them has changed the batch
    import torch
    k, q = torch.randn(2, 2, 64, device="cuda"), torch.randn(4, 2, 64, device="cuda")
    torch.cuda.synchronize()
    b.append(1, k, k)
    assert torch.equal(b.read(1)[0], k.half())
    refused(L.E_INVALID, b.append, 2, k, k)
    refused(L.E_INVALID, b.append, 0, None, k)
    refused(L.E_DIM, b.append, 0, k[:1], k)
    refused(L.E_INVALID, b.append, 0, k.transpose(0, 1), k)
    refused(L.E_INVALID, b.append, 0, k.half(), k)
    refused(L.E_INVALID, b.attention, 2, q)
    refused(L.E_DIM, b.attention, 0, q[:2])
    refused(L.E_UNSUPPORTED, b.attention, 0, q, out_type=B.Q8_0, out=torch.empty(2 * 292, dtype=torch.uint8, device="cuda"))
    refused(L.E_DIM, b.attention, 0, q, out=q[:2])
    refused(L.E_DIM, b.attention, 0, q, out_type=B.Q8_K, out=q)
    refused(L.E_DIM, b.append, 0, k, k, q=q, q_out=q[:3])
    refused(L.E_DIM, b.append, 0, k, k, k_norm=k[0, 0, :63])
    refused(L.E_DIM, A.norm_rope, be, k, 3, 2, 64, 0)
    refused(L.E_DIM, A.norm_rope, be, k, 2, 2, 64, 0, norm=k[0, 0, :32])
    refused(L.E_DIM, P.PagedBatch(P.PagedCache(be, 1, 16, 1, 1, 64), 2, 1, 1, 1).attention, 0, q[:2, :0], out_type=B.Q8_K)
    for rot, code in ((3, L.E_DIM), (66, L.E_DIM)):
        r = A.Rotary(dev(freqs(rot)), rot)
        refused(code, b.append, 0, k, k, rotary=r)
        refused(code, A.norm_rope, be, k, 2, 2, 64, 0, r)
    refused(L.E_INVALID, b.append, 0, k, k, rotary=A.Rotary(dev(freqs(64)), 64, layout=2))
    refused(L.E_DIM, A.Rotary, dev(freqs(64)), 32)
    refused(L.E_UNSUPPORTED, A.norm_rope, be, k[..., :32].contiguous(), 2, 2, 32, 0)
    refused(L.E_DIM, A.norm_rope, be, k, 2, 2, 64, 0x7fffffff)
    x = torch.zeros(300, device="cuda")[1:257]
    refused(L.E_INVALID, A.norm_rope, be, x, 2, 2, 64, 0)
    refused(L.E_INVALID, b.append, 0, x, k.reshape(-1))
