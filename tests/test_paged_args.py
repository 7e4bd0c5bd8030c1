"""What the Python side of the paged cache and norm_rope refuses before the
library is called: host code, no GPU."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from barq_rocm import _lib as L
from barq_rocm import attention as A
from barq_rocm.paged import PagedBatch


class NoCalls:
    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was called")
        return call


BE = SimpleNamespace(h=None, device=0, _lib=NoCalls(), sync=lambda: None)


def batch(n_tokens=3, n_head=4, n_head_kv=2, head_dim=64):
    b = PagedBatch.__new__(PagedBatch)
    b.be, b.b, b.n_head, b.n_tokens = BE, None, n_head, n_tokens
    b.cache = SimpleNamespace(n_head_kv=n_head_kv, head_dim=head_dim, type=L.F16)
    return b


def refused(code, f, *a, **k):
    with pytest.raises(L.BarqError) as e:
        f(*a, **k)
    assert e.value.code == code, e.value


HOST = [lambda *s: np.zeros(s, np.float32), lambda *s: torch.zeros(s)]


@pytest.mark.parametrize("host", HOST, ids=["numpy", "torch"])
def test_host_memory_in_device_calls(host):
    """16 stands for an address on the device, which is taken as it is."""
    b, kv, q, hd = batch(), host(3, 2, 64), host(3, 4, 64), host(64)
    for args in (dict(k=kv, v=16), dict(k=16, v=kv), dict(k=16, v=16, q=q, q_out=16), dict(k=16, v=16, q=16, q_out=q),
                 dict(k=16, v=16, q=16, q_out=16, q_norm=hd), dict(k=16, v=16, k_norm=hd),
                 dict(k=16, v=16, rotary=A.Rotary(host(32), 64))):
        refused(L.E_INVALID, b.append, 0, **args)
    refused(L.E_INVALID, b.attention, 0, q)
    refused(L.E_INVALID, b.attention, 0, 16, out=q)
    for out in (np.zeros((3, 292), np.uint8), torch.zeros((3, 292), dtype=torch.uint8)):
        refused(L.E_INVALID, b.attention, 0, 16, out_type=L.Q8_K, out=out)
    for args in (dict(x=q, out=16), dict(x=16, out=q), dict(x=16, out=16, norm=hd), dict(x=16, out=16, rotary=A.Rotary(host(32), 64))):
        x = args.pop("x")
        refused(L.E_INVALID, A.norm_rope, BE, x, 3, 4, 64, 0, **args)


@pytest.mark.parametrize("host", HOST, ids=["numpy", "torch"])
def test_host_memory_in_host_calls(host):
    """It gets as far as the library."""
    b, kv, q, hd, r = batch(), host(3, 2, 64), host(3, 4, 64), host(64), A.Rotary(host(32), 64)
    for f in (lambda: b.append(0, kv, kv, q=q, q_out=host(4, 3, 64), rotary=r, q_norm=hd, k_norm=hd, mem=L.MEM_HOST),
              lambda: b.attention(0, q, out=host(3, 4, 64), mem=L.MEM_HOST),
              lambda: A.norm_rope(BE, q, 3, 4, 64, 0, r, hd, mem=L.MEM_HOST, out=host(4, 3, 64))):
        with pytest.raises(AssertionError, match="was called"):
            f()


@pytest.mark.gpu
def test_device_memory_in_host_calls_and_on_other_devices():
    b, kv, q, hd = batch(), torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 4, 64, device="cuda"), torch.zeros(64, device="cuda")
    h, r = np.zeros(1000, np.float32), A.Rotary(torch.zeros(32, device="cuda"), 64)
    other = SimpleNamespace(h=None, device=1, _lib=NoCalls(), sync=lambda: None)
    for be, mem, at in ((BE, L.MEM_HOST, h.ctypes.data), (other, L.MEM_DEVICE, 16)):
        b.be = be
        for args in (dict(k=kv, v=at), dict(k=at, v=kv), dict(k=at, v=at, q=q, q_out=at), dict(k=at, v=at, q=at, q_out=q),
                     dict(k=at, v=at, k_norm=hd), dict(k=at, v=at, rotary=r)):
            refused(L.E_INVALID, b.append, 0, mem=mem, **args)
        refused(L.E_INVALID, b.attention, 0, q, mem=mem)
        refused(L.E_INVALID, b.attention, 0, at, out=q, mem=mem)
        refused(L.E_INVALID, A.norm_rope, be, q, 3, 4, 64, 0, mem=mem)
        refused(L.E_INVALID, A.norm_rope, be, at, 3, 4, 64, 0, rotary=r, out=at, mem=mem)


def test_outputs_that_are_not_side_by_side():
    """Their bytes are as many as the call writes, in more memory or in less."""
    b = batch()
    b.be = SimpleNamespace(h=None, device=-1, _lib=NoCalls(), sync=lambda: None)   # (so that memory here is what the call wants)
    for out in (torch.zeros((3, 584), dtype=torch.uint8)[:, ::2], torch.zeros((1, 292), dtype=torch.uint8).expand(3, 292),
                np.zeros((3, 584), np.uint8)[:, ::2], np.broadcast_to(np.zeros((1, 292), np.uint8), (3, 292))):
        for mem in (L.MEM_DEVICE, L.MEM_HOST):
            refused(L.E_INVALID, b.attention, 0, 16, out_type=L.Q8_K, out=out, mem=mem)


@pytest.mark.parametrize("host", HOST, ids=["numpy", "torch"])
def test_outputs_of_transpose_heads(host):
    for out, code in ((host(4, 3, 63), L.E_DIM), (host(5, 3, 64), L.E_DIM), (host(4, 3, 128)[..., ::2], L.E_INVALID),
                      (host(4, 3, 64).astype("float64") if isinstance(host(1), np.ndarray) else host(4, 3, 64).double(), L.E_INVALID)):
        refused(code, A.transpose_heads, BE, host(3, 4, 64), 3, 4, 64, mem=L.MEM_HOST, out=out)
    refused(L.E_INVALID, A.transpose_heads, BE, 16, 3, 4, 64, out=host(4, 3, 64))
    with pytest.raises(AssertionError, match="was called"):
        A.transpose_heads(BE, host(3, 4, 64), 3, 4, 64, mem=L.MEM_HOST, out=host(4, 3, 64))


@pytest.mark.parametrize("arrays", [
    (np.array([2 ** 32 + 1]), [20], [[1, 2]]), ([1], np.array([2 ** 32 + 20]), [[1, 2]]), ([1], [20], np.array([[1, 2 ** 32 + 2]])),
    ([1], [20], [np.array([1, 2 ** 32 + 2])]), ([1], [20], [[1, 2 ** 32 + 2]]), ([1], [20], [[1, 2 ** 64]]), ([2 ** 31], [20], [[1, 2]]), ([1], [20], np.array([[1, 2 ** 31]], np.uint32)),
    ([1.5], [20], [[1, 2]]), ([1], [20], np.array([[1, 2.25]])), ([1], [float("nan")], [[1, 2]]), ([1], [20], [[1, 2.5]])])
def test_numbers_that_are_no_int32(arrays):
    """They were taken for others: 2^32 + 2 for 2, 1.5 for 1."""
    b = batch()
    refused(L.E_INVALID, b.set, *arrays)
    assert b.n_tokens == 3


def test_numbers_of_other_types():
    """What is an int32 in value gets as far as the library, as that."""
    b, got = batch(), []

    class Takes:
        @staticmethod
        def barq_rocm_paged_batch_set(h, batch, n, q, kv, pages, stride):
            at = [np.ctypeslib.as_array((ctypes.c_int32 * k).from_address(p)).tolist() for p, k in ((q, n), (kv, n), (pages, n * stride)) if k]
            got.append((n, stride, at))
            return 0
    b.be = SimpleNamespace(h=None, device=0, _lib=Takes, sync=lambda: None)
    for t in (np.int32, np.int64, np.uint8, np.float64):
        b.set(np.array([1, 3], t), np.array([4, 20], t), np.array([[5, 7], [9, 3]], t))
        assert got.pop() == (2, 2, [[1, 3], [4, 20], [5, 7, 9, 3]]) and b.n_tokens == 4
    b.set([1, 3], (4, 20), [[5], np.array([9, -1])])
    assert got.pop() == (2, 2, [[1, 3], [4, 20], [5, -1, 9, -1]])
    b.set([], [], [])
    assert got.pop() == (0, 0, []) and b.n_tokens == 0


def test_token_ids_that_are_no_int32():
    """A step fails with them, and its sequences are as before."""
    from barq_rocm.llama import PagedLlama
    from barq_rocm.paged import Pages, Sequence
    m, s = PagedLlama.__new__(PagedLlama), Sequence()
    m.be, m.cfg, m.pages = BE, SimpleNamespace(window=0, n_sink=0), Pages(4, 16)
    m.batch = SimpleNamespace(set=lambda *a: None)
    for ids in (np.array([5, 2 ** 32 + 5]), [1.5], np.array([2 ** 31]), [2 ** 32 + 5]):
        refused(L.E_INVALID, m.step, [(s, [1, 2]), (s, ids)])
        assert s.length == 0 and m.pages.free() == 4
