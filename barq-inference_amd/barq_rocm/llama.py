"""LlamaTransformer::forward (models/src/transformer.rs:81-94) on the device,
integer path: every projection takes Q8_K activation rows written by the
fused residual-add + RMSNorm quantizer, as a deployment runs it.

    get_embeddings (:96-119)              -> barq_rocm_get_rows
    forward_layer (:123-144), per layer:
      rms_norm(attn_norm) (:148-172)      -> barq_rocm_add_rms_norm_quantize
                                             (the previous layer's closing
                                             residual add fused in)
      q / k / v proj (:212-220) + biases  -> barq_rocm_qkv_append_rope (one
        (:206-220), RoPE (:222-240),         token, no biases) or matmul x3
        KV append (:243-245)                 [+ add_bias] + kv_cache_append_rope_q
      compute_attention (:301-374)        -> barq_rocm_attention_q8k (rows
                                             quantized for the o projection)
      o proj (:247-251)                   -> barq_rocm_matmul
      residual add + ffn_norm (:136-139)  -> barq_rocm_add_rms_norm_quantize
      feed_forward (:378-408)             -> barq_rocm_ffn
    final_output (:468-498): output_norm of the last row, the LM head
      (output.weight, else the tied token_embd.weight), output.bias when its
      length is the vocabulary's           -> add_rms_norm_quantize, matmul,
                                             barq_rocm_add_bias

The KV cache may hold f32 rows or 4-bit blocks (attention.KVCache's type).
With a KVBudget the chain gathers each position's attention weight
(barq_rocm_attention_mass in place of _q8k) and drops the lightest ones when a
layer has outgrown the budget (barq_rocm_kv_cache_evict).

Models with norms of their query and key heads (blk.N.attn_q_norm.weight,
attn_k_norm.weight), or whose rotation covers part of a head or is stretched
for long contexts, rotate with barq_rocm_norm_rope.  PagedLlama runs the same
chain for the new tokens of many sequences at once over a paged cache
(barq_rocm_paged_append, barq_rocm_paged_attention), with a window of positions
if the model has one.

Weights come from a lookup name -> (type, n_rows, k, device pointer) or
None: a WeightCache of a GGUF file (WeightCache.find) or any mapping with
the GGUF tensor names.  Every compute step is a libbarq_rocm call on the
backend's stream; torch only allocates the activation buffers.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

from . import _lib as L
from . import attention as A
from . import paged as P
from .backend import Backend


@dataclass
class LlamaConfig:
    n_layer: int
    n_embd: int
    n_head: int
    n_head_kv: int
    head_dim: int
    n_ff: int
    rope_freq_base: float = 500000.0
    rope_freq_scale: float = 1.0
    rms_norm_eps: float = 1e-5
    rope_layout: int = A.ROPE_INTERLEAVED
    rot_dim: int = 0                    # dims of a head that are rotated (0: all)
    rope_scaling: int = L.ROPE_PLAIN    # rope_frequencies' scaling, for contexts
    rope_factor: float = 1.0            # rope_factor times the
    rope_trained: float = 0.0           # rope_trained positions (YARN)
    window: int = 0                     # positions that a query sees (0: all; PagedLlama)
    n_sink: int = 0                     # and the first ones that stay visible

    def whole_head_rope(self) -> bool:
        """Whether barq_rocm_rope's rotation is the model's."""
        return self.rot_dim in (0, self.head_dim) and self.rope_scaling == L.ROPE_PLAIN

    def rotary(self) -> A.Rotary:
        import torch
        if self.whole_head_rope():
            f, m, rot = self.inv_freq(), 1.0, self.head_dim
        else:
            rot = self.rot_dim or self.head_dim
            f, m = A.rope_frequencies(self.rope_scaling, rot, self.rope_freq_base, self.rope_factor, self.rope_trained)
        return A.Rotary(torch.from_numpy(f).cuda(), rot, self.rope_layout, self.rope_freq_scale, m)

    def inv_freq(self) -> np.ndarray:
        """rope_inv_freq (transformer.rs:48-52): base^(-2i/head_dim) in f32."""
        hd = self.head_dim
        return np.array([np.float32(self.rope_freq_base) ** np.float32(-2.0 * i / hd) for i in range(hd // 2)],
                        dtype=np.float32)


@dataclass
class KVBudget:
    """How many positions a layer keeps: once it holds more than keep + slack
    after a forward's attention, the newest `recent` and the heaviest others
    stay, keep in all.  slack spreads the cost of an eviction over that many
    tokens."""
    keep: int
    recent: int
    slack: int = 0


class DeviceLlama:
    """forward(tokens, start_pos) -> logits of the last token, on the device.

    get(name) returns (type, n_rows, k, device pointer) or None.  The KV
    cache is the caller's (attention.KVCache with cfg.n_layer layers); clear()
    it for a new session.  budget: see KVBudget."""

    def __init__(self, be: Backend, cfg: LlamaConfig, get, kv: A.KVCache, budget: KVBudget | None = None):
        import torch
        if budget is not None and not (0 <= budget.recent <= budget.keep and budget.keep > 0 and budget.slack >= 0):
            raise ValueError(f"{budget}: recent may be at most keep, and neither keep 0 nor anything negative")
        self.budget = budget
        # the weight each cached position has gathered, per layer
        self.mass = (None if budget is None else
                     [torch.zeros((cfg.n_head_kv, kv.max_size), dtype=torch.float32, device="cuda") for _ in range(cfg.n_layer)])
        self.be, self.cfg, self.get, self.kv = be, cfg, get, kv
        if kv is not None and cfg.window:
            raise NotImplementedError("a session over its own cache sees all of its positions: windows are PagedLlama's")
        self.inv_freq = torch.from_numpy(cfg.inv_freq()).cuda()
        self.rotary = cfg.rotary()
        head = get("output.weight") or get("token_embd.weight")
        if head is None:
            raise KeyError("No output or token embedding weight found")
        self.head = head
        self.n_vocab = head[1]
        bias = get("output.bias")
        self.out_bias = bias if bias is not None and bias[2] * bias[1] == self.n_vocab else None
        # (asked once: two lookups a layer are 6 % of a small model's token, 95 us of 1600 for 32 layers)
        self.has_head_norms = any(get(f"blk.{il}.attn_{m}_norm.weight") is not None for il in range(cfg.n_layer) for m in "qk")
        self._bufs = {}

    def _need(self, name):
        w = self.get(name)
        if w is None:
            raise KeyError(f"{name} not found in cache")
        return w

    def _norm(self, name):
        w = self.get(name)
        if w is None:
            # rms_norm returns its input unchanged without a weight (:153-156);
            # the fused quantizer always normalises, so that form is not offered
            raise NotImplementedError(f"{name} absent: the integer path needs every norm weight")
        return w[3]

    def _buf(self, key, shape, dtype="float32"):
        """Activation buffers reused across calls (so a captured graph replays
        on the same addresses)."""
        import torch
        b = self._bufs.get(key)
        if b is None or tuple(b.shape) != tuple(shape):
            b = torch.empty(shape, dtype=getattr(torch, dtype), device="cuda")
            self._bufs[key] = b
        return b

    def embed(self, tokens):
        """get_embeddings: tokens (device int32 [seq]) -> [seq, n_embd] f32."""
        t, n_rows, k, p = self._need("token_embd.weight")
        out = self._buf(("emb", len(tokens)), (len(tokens), k))
        return self.be.get_rows(t, p, n_rows, k, tokens, sync=False, out=out)

    def forward(self, tokens, start_pos: int, trace=None):
        """Logits [n_vocab] (device f32) of the last of the tokens at
        positions start_pos .. start_pos + len(tokens) - 1."""
        return self.forward_hidden(self.embed(tokens), start_pos, trace)

    def forward_hidden(self, hidden, start_pos: int, trace=None):
        import torch
        """trace: a list that receives, per layer, device copies of the
        layer's input rows, its attention output (after the o projection) and
        the two addends of its output (residual, FFN output); the output sum
        itself is formed inside the next layer's norm."""
        be, c = self.be, self.cfg
        seq = int(hidden.shape[0])
        nbq = c.n_embd // 256 * 292
        q_rows = c.n_head * c.head_dim
        xq = self._buf(("xq", seq), (seq, nbq), "uint8")
        xq2 = self._buf(("xq2", seq), (seq, nbq), "uint8")
        aq = self._buf(("aq", seq), (seq, q_rows // 256 * 292), "uint8")
        qr = self._buf(("qr", seq), (c.n_head, seq, c.head_dim))
        o = self._buf(("o", seq), (seq, c.n_embd))
        res = [self._buf(("res0", seq), (seq, c.n_embd)), self._buf(("res1", seq), (seq, c.n_embd))]
        ff = self._buf(("ff", seq), (seq, c.n_embd))
        x, prev = hidden, None
        r_mid = res[1]
        for il in range(c.n_layer):
            pre = f"blk.{il}."
            r_in = res[0]
            # x + previous FFN output (the closing add of the last layer), normed
            be.add_rms_norm_quantize(L.Q8_K, x, prev, self._norm(pre + "attn_norm.weight"), c.rms_norm_eps,
                                     sum_out=r_in if prev is not None else None, out=xq, sync=False)
            if prev is None:
                r_in = x
            self._attend(il, xq, seq, start_pos, qr, aq)
            wo = self._need(pre + "attn_output.weight")
            be.matmul_raw(wo[0], wo[3], wo[1], wo[2], L.Q8_K, aq, seq, o, L.MEM_DEVICE)
            be.add_rms_norm_quantize(L.Q8_K, r_in, o, self._norm(pre + "ffn_norm.weight"), c.rms_norm_eps,
                                     sum_out=r_mid, out=xq2, sync=False)
            g, u, d = (self._need(pre + f"ffn_{m}.weight") for m in ("gate", "up", "down"))
            be.ffn(g[0], g[3], u[0], u[3], d[0], d[3], c.n_embd, c.n_ff, L.Q8_K, xq2, seq, sync=False, out=ff)
            if trace is not None:
                be.sync()   # the copies run on torch's stream, the layer on the backend's
                trace.append((r_in.clone(), o.clone(), r_mid.clone(), ff.clone()))
                torch.cuda.synchronize()
            # the next layer sums x + ff into res[0] (x is res[1]: no buffer aliases another)
            x, prev = r_mid, ff
        return self._final(x, prev)

    def _final(self, res, ff):
        """Logits of the rows res + ff that are asked for: the last one."""
        n = int(res.shape[0])
        return self.final_output(res[n - 1:n], ff[n - 1:n])

    def _project(self, il, xq, seq):
        """q, k and v of the layer's normed rows, with their biases."""
        be, outs = self.be, []
        for m in "qkv":
            w, b = self._need(f"blk.{il}.attn_{m}.weight"), self.get(f"blk.{il}.attn_{m}.bias")
            y = self._buf((m, seq), (seq, w[1]))
            be.matmul_raw(w[0], w[3], w[1], w[2], L.Q8_K, xq, seq, y, L.MEM_DEVICE)
            if b is not None and b[1] * b[2] == w[1]:
                be.add_bias(y, b[3], seq, w[1], sync=False)
            outs.append(y)
        return outs

    def _head_norms(self, il):
        """The weights of the norms of query and key heads (None: the model has none)."""
        if not self.has_head_norms:
            return [None, None]
        out = []
        for m in "qk":
            w = self.get(f"blk.{il}.attn_{m}_norm.weight")
            if w is not None and (w[0] != L.F32 or w[1] * w[2] != self.cfg.head_dim):
                raise NotImplementedError(f"blk.{il}.attn_{m}_norm.weight: {w[1] * w[2]} values of type {w[0]}, not an f32 one for each dim "
                                          "of a head")
            out.append(None if w is None else w[3])
        return out

    def _attend(self, il, xq, seq, start_pos, qr, aq):
        """The layer's attention of the rows at start_pos .. on, their keys and
        values appended: Q8_K rows in aq (qr: room for the rotated queries)."""
        c, kv, be = self.cfg, self.kv, self.be
        norms = self._head_norms(il)
        if c.whole_head_rope() and norms == [None, None]:
            ws = [self._need(f"blk.{il}.attn_{m}.weight") for m in "qkv"]
            if seq == 1 and all(self.get(f"blk.{il}.attn_{m}.bias") is None for m in "qkv"):
                kv.qkv_append_rope(il, [w[0] for w in ws], [w[3] for w in ws], c.n_head, c.n_embd, L.Q8_K, xq, start_pos,
                                   c.rope_freq_scale, self.inv_freq, c.rope_layout, q_out=qr)
            else:
                q, k, v = self._project(il, xq, seq)
                kv.append_rope_q(il, q, c.n_head, k, v, seq, start_pos, c.rope_freq_scale, self.inv_freq, c.rope_layout,
                                 q_out=qr)
        else:
            q, k, v = self._project(il, xq, seq)
            kr, vt = (self._buf((n, seq), (c.n_head_kv, seq, c.head_dim)) for n in ("kr", "vt"))
            for x, heads, norm, out in ((q, c.n_head, norms[0], qr), (k, c.n_head_kv, norms[1], kr)):
                A.norm_rope(be, x, seq, heads, c.head_dim, start_pos, self.rotary, norm, c.rms_norm_eps, sync=False, out=out)
            A.transpose_heads(be, v, seq, c.n_head_kv, c.head_dim, sync=False, out=vt)
            kv.append(il, kr, vt, seq, c.head_dim)
        if self.budget is None:
            A.compute_attention_q8k(be, qr, kv, il, c.n_head, c.n_head_kv, c.head_dim, seq, start_pos + seq, start_pos,
                                    sync=False, out=aq)
        else:
            self._attend_and_evict(il, qr, seq, aq)

    def _attend_and_evict(self, il, qr, seq, aq):
        """The layer's attention over all its cached rows (the last seq are
        this call's), their masses, and an eviction when they are too many."""
        import torch
        be, c, kv, n = self.be, self.cfg, self.kv, self.kv.layer_len(il)
        if n == seq:   # the layer was empty: a new session
            with torch.cuda.stream(torch.cuda.ExternalStream(be.stream())):
                self.mass[il].zero_()
        A.compute_attention_mass(be, qr, kv, il, c.n_head, c.n_head_kv, c.head_dim, seq, n, n - seq, self.mass[il],
                                 out_type=L.Q8_K, sync=False, out=aq)
        if n > self.budget.keep + self.budget.slack:
            kv.evict(il, self.mass[il], self.budget.keep, self.budget.recent, sync=False, want_kept=False)

    def final_output(self, res_last, ff_last):
        """final_output of the last row: output_norm(res + ff) as Q8_K, the
        LM head, output.bias."""
        return self._logits(res_last, ff_last)[0]

    def _logits(self, res_last, ff_last):
        be, c, m = self.be, self.cfg, int(res_last.shape[0])
        xq = self._buf("xq_out" if m == 1 else ("xq_out", m), (m, c.n_embd // 256 * 292), "uint8")
        be.add_rms_norm_quantize(L.Q8_K, res_last, ff_last, self._norm("output_norm.weight"), c.rms_norm_eps,
                                 out=xq, sync=False)
        t, n, k, p = self.head
        logits = self._buf("logits" if m == 1 else ("logits", m), (m, n))
        be.matmul_raw(t, p, n, k, L.Q8_K, xq, m, logits, L.MEM_DEVICE)
        if self.out_bias is not None:
            be.add_bias(logits, self.out_bias[3], m, n, sync=False)
        return logits


class PagedLlama(DeviceLlama):
    """The new tokens of up to max_seqs sequences in one call, over a paged
    cache: prompts' chunks and single tokens side by side.

    pages hands out the cache's pages (paged.Pages; by default one over the
    whole cache); step() keeps the sequences' page lists."""

    def __init__(self, be: Backend, cfg: LlamaConfig, get, cache: P.PagedCache, max_seqs: int, max_tokens: int, max_pages: int,
                 pages: P.Pages | None = None):
        if (cache.n_layers, cache.n_head_kv, cache.head_dim) != (cfg.n_layer, cfg.n_head_kv, cfg.head_dim):
            raise L.BarqError(L.E_DIM, f"PagedLlama: a cache of {cache.n_layers} layers, {cache.n_head_kv} kv heads of {cache.head_dim} "
                                       f"dims, the model has {cfg.n_layer}, {cfg.n_head_kv}, {cfg.head_dim}")
        super().__init__(be, cfg, get, None)
        self.cache = cache
        self.pages = P.Pages(cache.n_pages, cache.page_size) if pages is None else pages
        self.batch = P.PagedBatch(cache, cfg.n_head, max_seqs, max_tokens, max_pages, cfg.window, cfg.n_sink)

    def step(self, news, trace=None):
        """news: (paged.Sequence, its new tokens: a list or array of ids) for each sequence.
        -> logits [sequences with new tokens, n_vocab] (device f32) of their last tokens.  The
        sequences grow by their tokens (a step that fails leaves them as they were); pages behind the
        window are given back.  The logits' buffer is the next step's too."""
        import torch
        c = self.cfg
        q_lens = [len(t) for _, t in news]
        before = [(seq, seq.length) for seq, _ in news]
        try:
            for seq, t in news:
                self.pages.grow(seq, len(t))
            self.batch.set(q_lens, [s.length for s, _ in news], [s.pages for s, _ in news])
            ids = P._int32("PagedLlama.step", "token ids", np.concatenate([np.asarray(t) for _, t in news]) if news else [])
            if len(ids) == 0:
                return torch.empty((0, self.n_vocab), dtype=torch.float32, device="cuda")
            last = np.cumsum(q_lens)[np.asarray(q_lens) > 0].astype(np.int32) - 1
            with torch.cuda.stream(torch.cuda.ExternalStream(self.be.stream())):
                both = torch.from_numpy(np.concatenate([ids, last])).cuda()
            self.last = None if len(last) == len(ids) else both[len(ids):]
            logits = self.forward_hidden(self.embed(both[:len(ids)]), 0, trace)
        except Exception:
            for seq, length in before:   # (what a layer has written lies behind their ends)
                self.pages.shrink(seq, length)
            raise
        if c.window:
            for seq, _ in news:
                self.pages.drop_behind(seq, c.window, c.n_sink)
        return logits

    def _buf(self, key, shape, dtype="float32"):
        """A part of one buffer for each use, of a step's most rows: steps have any number of them."""
        import torch
        name, n = key if isinstance(key, tuple) else (key, 1)
        size = math.prod(shape)
        if name not in self._bufs:
            most = self.batch.max_seqs if name in ("xq_out", "logits", "last_res", "last_ff") else self.batch.max_tokens
            self._bufs[name] = torch.empty(size // n * most, dtype=getattr(torch, dtype), device="cuda")
        return self._bufs[name][:size].view(shape)

    def _attend(self, il, xq, seq, start_pos, qr, aq):
        q, k, v = self._project(il, xq, seq)
        q_norm, k_norm = self._head_norms(il)
        self.batch.append(il, k, v, q=q, rotary=self.rotary, q_norm=q_norm, k_norm=k_norm, eps=self.cfg.rms_norm_eps, q_out=qr)
        self.batch.attention(il, qr, out_type=L.Q8_K, sync=False, out=aq)

    def _final(self, res, ff):
        if self.last is None:   # every row is its sequence's last
            return self._logits(res, ff)
        n, m, k = int(res.shape[0]), len(self.last), self.cfg.n_embd
        rows = [self.be.get_rows(L.F32, x, n, k, self.last, sync=False, out=self._buf((name, m), (m, k)))
                for name, x in (("last_res", res), ("last_ff", ff))]
        return self._logits(*rows)
