"""The 4-bit cache, attention mass and eviction as a program runs them: captured
in HIP graphs and replayed with other work in between, on two handles at once,
into buffers at odd addresses, on a stream of the program's."""
import threading

import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import attention as A
from kv_ref import attention, kept, q4_values

pytestmark = pytest.mark.gpu
F32 = np.float32


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(F32)


def inv_freq(hd):
    return np.array([np.float32(500000.0) ** np.float32(-2.0 * i / hd) for i in range(hd // 2)], dtype=F32)


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_a_step_in_a_graph(be, type_, n):
    """append with RoPE, attention with its mass, eviction into another cache."""
    import torch
    heads, n_kv, hd, before = 8, 2, 128, 500
    c, to = (A.KVCache(be, 700, 1, n_kv, hd, type=type_) for _ in range(2))
    k, v = dev(rows(1, n_kv, before, hd)), dev(rows(2, n_kv, before, hd))
    qp, kp, vp = dev(rows(3, n, heads * hd)), dev(rows(4, n, n_kv * hd)), dev(rows(5, n, n_kv * hd))
    f, mass0 = dev(inv_freq(hd)), dev(np.abs(rows(6, n_kv, 700)))
    mass, new = torch.empty_like(mass0), torch.empty_like(mass0)
    q = torch.empty((heads, n, hd), device="cuda")
    out = torch.empty((n, heads, hd), device="cuda")
    out8 = torch.empty((n, heads * hd // 256 * 292), dtype=torch.uint8, device="cuda")
    total = before + n

    def step():
        c.clear()
        c.append(0, k, v, before, hd)
        c.append_rope_q(0, qp, heads, kp, vp, n, before, 1.0, f, A.ROPE_INTERLEAVED, q_out=q)
        A.compute_attention_mass(be, q, c, 0, heads, n_kv, hd, n, total, before, mass0, mass_out=mass, sync=False, out=out)
        A.compute_attention_q8k(be, q, c, 0, heads, n_kv, hd, n, total, before, sync=False, out=out8)
        c.evict(0, mass, 100, 20, dst=to, mass_out=new, sync=False, want_kept=False)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.set_stream(stream)
    be.set_stream(stream.cuda_stream)
    try:
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (q, out, out8, mass[:, :total], new[:, :total])] + list(to.read(0, 0, 100))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step()
        other = torch.randn(1 << 20, device="cuda")
        for _ in range(3):
            for t in (q, out, mass, new):
                t.fill_(float("nan"))
            out8.zero_()
            other.mul_(1.0001)
            A.compute_attention(be, q, to, 0, heads, n_kv, hd, 1, 50, 49)   # the workspace in between
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = [q, out, out8, mass[:, :total], new[:, :total]] + list(to.read(0, 0, 100))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        torch.cuda.set_stream(torch.cuda.default_stream())
        be.set_stream(None)


def test_two_handles_at_once():
    errors = []

    def work(seed):
        try:
            import torch
            be = B.Backend(0)
            for r in range(6):
                n = 100 + 50 * r + seed
                k, v, q = rows(seed + r, 2, n, 64), rows(seed + r + 9, 2, n, 64), rows(seed + r + 17, 4, 3, 64)
                c = A.KVCache(be, n, 1, 2, 64, type=B.Q4_0)
                dk, dv, dq = dev(k), dev(v), dev(q)
                torch.cuda.current_stream().synchronize()
                c.append(0, dk, dv, n, 64)
                out, mass = A.compute_attention_mass(be, dq, c, 0, 4, 2, 64, 3, n, n - 3, None)
                ref, added = attention(q, q4_values(k), q4_values(v), n - 3)
                assert np.max(np.abs(out.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
                m = mass.cpu().numpy()
                assert np.allclose(m, added, rtol=2.6e-5, atol=1e-7)
                got, _ = c.evict(0, mass, n // 2, 5)
                assert np.array_equal(got.cpu().numpy(), kept(m, n, n // 2, 5))
                be.sync()
                c.close()
            be.close()
        except BaseException as e:   # noqa: BLE001 (handed to the test's thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (0, 1000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
@pytest.mark.parametrize("n", [1, 70])
def test_buffers_at_odd_addresses(be, type_, n):
    """Rows, outputs and masses that start 4 bytes behind a 16-byte boundary (q needs 16)."""
    import torch

    def odd(*shape):
        return torch.empty(int(np.prod(shape)) + 1, device="cuda")[1:].view(*shape)
    heads, n_kv, hd, total = 4, 2, 64, 90 + n
    k, v, q = rows(1, n_kv, total, hd), rows(2, n_kv, total, hd), dev(rows(3, heads, n, hd))
    ok, ov = odd(n_kv, total, hd).copy_(dev(k)), odd(n_kv, total, hd).copy_(dev(v))
    torch.cuda.synchronize()
    c = A.KVCache(be, total, 1, n_kv, hd, type=type_)
    c.append(0, ok, ov, total, hd)
    rk, rv = odd(n_kv, total, hd), odd(n_kv, total, hd)
    B._lib.check(be._lib.barq_rocm_kv_cache_read(be.h, c.c, 0, 0, total, rk.data_ptr(), rv.data_ptr(), B.MEM_DEVICE))
    out, mass = odd(n, heads, hd), odd(n_kv, total + 1)
    A.compute_attention_mass(be, q, c, 0, heads, n_kv, hd, n, total, total - n, None, mass_out=mass, out=out)
    plain, m = A.compute_attention_mass(be, q, c, 0, heads, n_kv, hd, n, total, total - n, None)
    assert torch.equal(out, plain) and torch.equal(mass[:, :total], m)
    if type_ == B.Q4_0:
        k, v = q4_values(k), q4_values(v)
    assert np.array_equal(rk.cpu().numpy(), k) and np.array_equal(rv.cpu().numpy(), v)
    att = odd(n, heads, hd)
    B._lib.check(be._lib.barq_rocm_attention(be.h, q.data_ptr(), c.c, 0, heads, n_kv, hd, n, total, total - n, att.data_ptr(),
                                             B.MEM_DEVICE))
    be.sync()
    ref, _ = attention(q.cpu().numpy(), k, v, total - n)
    assert np.max(np.abs(att.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
    want = kept(m.cpu().numpy(), total, 33, 4)
    got, _ = c.evict(0, mass, 33, 4)
    assert np.array_equal(got.cpu().numpy(), want)


def test_rows_shared_by_many_heads(be):
    """One kv head for 20 query heads and a prompt: tiles whose first and last row are of different queries."""
    heads, hd, n, start = 20, 128, 37, 91
    q, k, v = rows(1, heads, n, hd), rows(2, 1, start + n, hd), rows(3, 1, start + n, hd)
    c = A.KVCache(be, start + n, 1, 1, hd, type=B.Q4_0)
    c.append(0, dev(k), dev(v), start + n, hd)
    ref, added = attention(q, q4_values(k), q4_values(v), start)
    out, mass = A.compute_attention_mass(be, dev(q), c, 0, heads, 1, hd, n, start + n, start, None)
    got = A.compute_attention(be, dev(q), c, 0, heads, 1, hd, n, start + n, start)
    for o in (out, got):
        assert np.max(np.abs(o.cpu().numpy() - ref)) <= 2e-5 * np.max(np.abs(v))
    assert np.allclose(mass.cpu().numpy(), added, rtol=2.6e-5, atol=0)


@pytest.mark.parametrize("n", [1, 30])
def test_queries_of_every_size(be, n):
    """Rows with elements of very different sizes, all tiny, all huge, zero: the
    scores come from f32 whatever the split of the row is."""
    heads, hd, total = 8, 64, 200 + n
    q, k, v = rows(1, heads, n, hd), rows(2, 2, total, hd), rows(3, 2, total, hd)
    q[0] *= 1e-30
    q[1] *= 2.0 ** -np.arange(hd)
    q[2] = 0
    q[3, :, 7] = 1e25
    k[0, :, 7] = 0
    q[4] *= 1e-38
    q[5, :, ::2] = 0
    c = A.KVCache(be, total, 1, 2, hd, type=B.Q4_0)
    c.append(0, dev(k), dev(v), total, hd)
    ref, _ = attention(q, q4_values(k), q4_values(v), total - n)
    got = A.compute_attention(be, dev(q), c, 0, heads, 2, hd, n, total, total - n).cpu().numpy()
    assert np.max(np.abs(got - ref)) <= 2e-5 * np.max(np.abs(v))
