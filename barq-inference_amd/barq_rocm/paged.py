"""The paged KV cache over the C ABI: a pool of pages, a step's batch of
sequences, append with norm and rotation, attention.

Device buffers are torch tensors, host buffers numpy arrays (``mem=MEM_HOST``).
"""
from __future__ import annotations

import ctypes
from array import array

import numpy as np

from . import _lib as L
from .attention import _check_place, _empty, _f32_at, _place
from .backend import Backend, _ptr


def _int32(who, what, a):
    """Numbers as int32, side by side; refused where that would make others of them."""
    if a.__class__ is list and a:
        try:
            return np.frombuffer(array("i", a), np.int32)   # (a third of the time; no number out of range, no fraction passes)
        except (TypeError, OverflowError):
            pass
    x = np.asarray(a)
    if x.dtype == np.int32:
        return np.ascontiguousarray(x)
    if x.dtype.kind in "iub":
        y = np.ascontiguousarray(x, dtype=np.int32)
    else:
        try:
            with np.errstate(invalid="ignore"):
                y = np.ascontiguousarray(x, dtype=np.int32)
        except OverflowError:
            y = None
    if y is None or np.count_nonzero(x != y):
        raise L.BarqError(L.E_INVALID, f"{who}: {what} must be whole numbers of 32 bits")
    return y


class PagedCache:
    """n_pages pages of page_size positions for each layer and kv head; type
    F16 or F32."""

    def __init__(self, be: Backend, n_pages: int, page_size: int, n_layers: int, n_head_kv: int, head_dim: int,
                 type: int = L.F16):
        self.be, self.c = be, None
        c = ctypes.c_void_p()
        L.check(be._lib.barq_rocm_paged_cache_create(be.h, n_pages, page_size, n_layers, n_head_kv, head_dim, type,
                                                     ctypes.byref(c)))
        self.c = c
        self.n_pages, self.page_size, self.n_layers, self.n_head_kv, self.head_dim, self.type = (
            n_pages, page_size, n_layers, n_head_kv, head_dim, type)
        self._like = None

    def like(self):
        """A torch tensor of the cache's type on its device."""
        if self._like is None:
            import torch
            self._like = torch.empty(0, dtype=torch.float16 if self.type == L.F16 else torch.float32, device=f"cuda:{self.be.device}")
        return self._like

    def close(self):
        if self.c:
            self.be._lib.barq_rocm_paged_cache_destroy(self.c)
            self.c = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedBatch:
    """The sequences of one step (see barq_rocm_paged_batch_set) and the calls
    on their new tokens.  window, n_sink: a query sees its last `window`
    positions (0: all before it) and the first n_sink."""

    def __init__(self, cache: PagedCache, n_head: int, max_seqs: int, max_tokens: int, max_pages: int, window: int = 0,
                 n_sink: int = 0):
        self.be, self.cache, self.b = cache.be, cache, None
        b = ctypes.c_void_p()
        L.check(self.be._lib.barq_rocm_paged_batch_create(self.be.h, cache.c, n_head, max_seqs, max_tokens, max_pages, window,
                                                          n_sink, ctypes.byref(b)))
        self.b = b
        self.n_head, self.max_seqs, self.max_tokens, self.max_pages = n_head, max_seqs, max_tokens, max_pages
        self.n_tokens = 0

    def close(self):
        if self.b:
            self.be._lib.barq_rocm_paged_batch_destroy(self.b)
            self.b = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set(self, q_lens, kv_lens, pages):
        """q_lens, kv_lens: one number a sequence; pages: [sequences, pages]
        int32 (or a list of lists of ids), -1 where there is none."""
        who = "paged_batch_set"
        q, kv = _int32(who, "q_lens", q_lens), _int32(who, "kv_lens", kv_lens)
        if not isinstance(pages, np.ndarray):
            lens = [len(p) for p in pages]
            width, flat = max(lens, default=0), []
            for p, n in zip(pages, lens):
                flat += p.tolist() if isinstance(p, np.ndarray) else p
                flat += [-1] * (width - n)
            pages = _int32(who, "pages", flat).reshape(len(lens), width)
        else:
            pages = _int32(who, "pages", pages)
        if q.ndim != 1 or q.shape != kv.shape or pages.ndim != 2 or len(pages) != len(q):
            raise L.BarqError(L.E_DIM, f"paged_batch_set: q_lens {q.shape}, kv_lens {kv.shape}, pages {pages.shape}")
        L.check(self.be._lib.barq_rocm_paged_batch_set(self.be.h, self.b, len(q), _ptr(q), _ptr(kv), _ptr(pages), pages.shape[1]))
        self.n_tokens = int(q.sum())

    def append(self, layer, k, v, q=None, rotary=None, q_norm=None, k_norm=None, eps=1e-5, q_out=None, mem=L.MEM_DEVICE):
        """k, v [n_tokens, n_head_kv*head_dim] into the layer's pages, k normed by
        head (with k_norm) and rotated (with rotary); returns q [n_tokens,
        n_head*head_dim] likewise, as [n_head, n_tokens, head_dim], or None.  Enqueued on
        the backend's stream and not waited for."""
        c, t = self.cache, self.n_tokens
        hd = c.head_dim
        nq, nk, who, place = t * self.n_head * hd, t * c.n_head_kv * hd, "paged_append", _place(self.be, mem)
        if q is not None and q_out is None:
            q_out = _empty((self.n_head, t, hd), q, mem)
        rc = self.be._lib.barq_rocm_paged_append(
            self.be.h, self.b, layer, _f32_at(who, "q", q, nq, place), _f32_at(who, "q_out", q_out, nq, place),
            _f32_at(who, "k", k, nk, place), _f32_at(who, "v", v, nk, place), _f32_at(who, "q_norm", q_norm, hd, place),
            _f32_at(who, "k_norm", k_norm, hd, place), eps, None if rotary is None else rotary.ref_in(who, place), mem)
        if rc:
            L.check(rc)
        return q_out

    def read(self, layer, mem=L.MEM_DEVICE, sync=True):
        """The tokens' rows as the cache holds them: (k, v), each [n_tokens,
        n_head_kv, head_dim] float16 or float32."""
        c = self.cache
        shape = self.n_tokens, c.n_head_kv, c.head_dim
        if mem == L.MEM_HOST:
            dtype = "float16" if c.type == L.F16 else "float32"
            k, v = np.empty(shape, dtype), np.empty(shape, dtype)
            rc = self.be._lib.barq_rocm_paged_read(self.be.h, self.b, layer, _ptr(k), _ptr(v), mem)
        else:
            like = c.like()
            k, v = like.new_empty(shape), like.new_empty(shape)
            rc = self.be._lib.barq_rocm_paged_read(self.be.h, self.b, layer, k.data_ptr(), v.data_ptr(), mem)
        if rc:
            L.check(rc)
        if sync and mem == L.MEM_DEVICE:
            self.be.sync()
        return k, v

    def attention(self, layer, q, out_type=L.F32, mem=L.MEM_DEVICE, sync=True, out=None):
        """q [n_head, n_tokens, head_dim] -> [n_tokens, n_head, head_dim], or with
        out_type Q8_K the rows' blocks, uint8 [n_tokens, n_head*head_dim/256 * 292]."""
        c, t = self.cache, self.n_tokens
        width, place = self.n_head * c.head_dim, _place(self.be, mem)
        at = _f32_at("paged_attention", "q", q, t * width, place)
        if out is not None and not isinstance(out, int):
            if out_type == L.F32:
                _f32_at("paged_attention", "out", out, t * width, place)
            elif (out.nbytes if isinstance(out, np.ndarray) else out.numel() * out.element_size()) != t * (width // 256 * 292):
                raise L.BarqError(L.E_DIM, f"paged_attention: out must have {t} rows of {width // 256 * 292} bytes")
            elif not (out.flags.c_contiguous if isinstance(out, np.ndarray) else out.is_contiguous()):
                raise L.BarqError(L.E_INVALID, "paged_attention: out must be contiguous")
            else:
                _check_place("paged_attention", "out", out, place)
        if out is None:
            out = (_empty((t, self.n_head, c.head_dim), q, mem) if out_type == L.F32
                   else _empty((t, width // 256 * 292), q, mem, dtype="uint8"))
        rc = self.be._lib.barq_rocm_paged_attention(self.be.h, self.b, layer, at, out_type, _ptr(out), mem)
        if rc:
            L.check(rc)
        if sync and mem == L.MEM_DEVICE:
            self.be.sync()
        return out


class Sequence:
    """A sequence of a paged cache: its length and its page ids (-1: given back).
    gone: between these two lengths the next query would miss positions that were given back."""

    def __init__(self):
        self.length, self.pages, self.gone = 0, [], (0, 0)


class Pages:
    """Which pages of a cache are free, and how many sequences have each.  A page that
    is not full belongs to one sequence."""

    def __init__(self, n_pages: int, page_size: int):
        self.page_size = page_size
        self._free = list(range(n_pages - 1, -1, -1))
        self._users = [0] * n_pages

    def free(self) -> int:
        return len(self._free)

    def grow(self, seq: Sequence, n_tokens: int):
        """n_tokens more positions.  Fails without changing anything when the pages run out."""
        if n_tokens < 0:
            raise L.BarqError(L.E_DIM, f"pages: {n_tokens} tokens")
        need = -(-(seq.length + n_tokens) // self.page_size) - len(seq.pages)
        if need > len(self._free):
            raise L.BarqError(L.E_ALLOC, f"pages: {need} more are needed, {len(self._free)} are free")
        for _ in range(need):
            p = self._free.pop()
            self._users[p] = 1
            seq.pages.append(p)
        seq.length += n_tokens

    def shrink(self, seq: Sequence, length: int):
        """Back to `length` positions (drafted tokens that were not taken).  Refused where the next token would go to a page
        that other sequences have, or would miss positions that were given back."""
        if not 0 <= length <= seq.length:
            raise L.BarqError(L.E_DIM, f"pages: from {seq.length} back to {length} positions")
        self._check_window(seq, length)
        n = -(-length // self.page_size)
        if length % self.page_size and length < seq.length and self._users[seq.pages[n - 1]] > 1:
            raise L.BarqError(L.E_INVALID, f"pages: position {length} is on a page that other sequences have")
        while len(seq.pages) > n:
            self._release(seq.pages.pop())
        seq.length = length
        if length <= seq.gone[0]:
            seq.gone = (0, 0)

    def fork(self, seq: Sequence) -> Sequence:
        """A sequence over the same whole pages: its length is theirs, and what it adds goes to pages of its own."""
        new = Sequence()
        n = seq.length // self.page_size
        self._check_window(seq, n * self.page_size)
        new.length, new.pages = n * self.page_size, seq.pages[:n]
        if new.length > seq.gone[0]:
            new.gone = seq.gone
        for p in new.pages:
            if p >= 0:
                self._users[p] += 1
        return new

    def drop_behind(self, seq: Sequence, window: int, n_sink: int = 0):
        """Give back the pages that no query to come sees (window and n_sink as a batch has them; without a window, 0, none)."""
        if window < 0 or n_sink < 0:
            raise L.BarqError(L.E_DIM, f"pages: a window of {window} positions, {n_sink} first ones")
        if window == 0:
            return
        first = -(-n_sink // self.page_size)
        for i in range(first, max(seq.length - window + 1, 0) // self.page_size):
            if seq.pages[i] >= 0:
                self._release(seq.pages[i])
                seq.pages[i] = -1
                start, end = seq.gone
                seq.gone = (min(start, i * self.page_size) if end else i * self.page_size,
                            max(end, (i + 1) * self.page_size + window - 1))

    def close(self, seq: Sequence):
        """The end of the sequence: its pages are free again."""
        self.shrink(seq, 0)

    def _check_window(self, seq: Sequence, length: int):
        if seq.gone[0] < length < seq.gone[1]:
            raise L.BarqError(L.E_INVALID, f"pages: a query at position {length} would miss positions that were given back (one at "
                                           f"{seq.gone[1]} does not)")

    def _release(self, p: int):
        if p < 0:
            return
        self._users[p] -= 1
        if self._users[p] == 0:
            self._free.append(p)
