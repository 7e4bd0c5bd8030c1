"""PagedLlama: many sequences' steps over a paged cache, with norms of the
heads, part of a head rotated for a long context, and windows; and the norms
and that rotation in DeviceLlama's sessions.

Bar for a layer's attention output after the o projection: teacher-forced, as
in test_gpu_llama_kv.py: the formulas in 64 bits over the rows the cache reads
as, with the queries of the traced layer input, through the library's Q8_K
quantizer and projection; both sides quantize rows that agree to 2e-5, so now
and then an element moves by one Q8 step: relative L2 1e-3."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import _lib as L
from barq_rocm import attention as A
from barq_rocm import paged as P
from barq_rocm import synth
from barq_rocm.llama import DeviceLlama, LlamaConfig, PagedLlama
from conftest import rel_err
from paged_ref import attention, norm_turn

pytestmark = pytest.mark.gpu
SHAPE = dict(n_layer=2, n_embd=512, n_head=8, n_head_kv=2, head_dim=64, n_ff=512)
N_VOCAB = 256
CONFIGS = {
    "plain": LlamaConfig(**SHAPE),
    "norms": LlamaConfig(**SHAPE, rope_layout=A.ROPE_SPLIT_HALF),
    "part": LlamaConfig(**SHAPE, rot_dim=24, rope_scaling=L.ROPE_YARN, rope_factor=4.0, rope_trained=256.0),
    "window": LlamaConfig(**SHAPE, rot_dim=32, window=20, n_sink=3),
}


@pytest.fixture(scope="module")
def weights():
    import torch
    w, kv = {}, SHAPE["n_head_kv"] * SHAPE["head_dim"]

    def put(name, t, n, k, data):
        w[name] = (t, n, k, torch.from_numpy(data).cuda())
    for il in range(2):
        for i, (sfx, n) in enumerate((("attn_q", 512), ("attn_k", kv), ("attn_v", kv), ("attn_output", 512), ("ffn_gate", 512),
                                      ("ffn_up", 512), ("ffn_down", 512))):
            put(f"blk.{il}.{sfx}.weight", B.Q4_K, n, 512, synth.gen_weights(B.Q4_K, n, 512, 40 + 16 * il + i))
        for j, nm in enumerate(("attn_norm", "ffn_norm")):
            put(f"blk.{il}.{nm}.weight", B.F32, 1, 512, (0.05 * (1 + 0.1 * synth.gen_f32(512, 90 + 2 * il + j))).astype(np.float32))
        for j, nm in enumerate(("attn_q_norm", "attn_k_norm")):
            put(f"blk.{il}.{nm}.weight", B.F32, 1, 64, (1 + 0.2 * synth.gen_f32(64, 110 + 2 * il + j)).astype(np.float32))
    put("token_embd.weight", B.Q4_K, N_VOCAB, 512, synth.gen_weights(B.Q4_K, N_VOCAB, 512, 98))
    put("output_norm.weight", B.F32, 1, 512, (0.05 * (1 + 0.1 * synth.gen_f32(512, 99))).astype(np.float32))
    return w


def table(weights, name):
    return {k: (t, n, kk, d.data_ptr()) for k, (t, n, kk, d) in weights.items() if name == "norms" or "q_norm" not in k and "k_norm" not in k}.get


def ids(n, seed):
    return np.random.default_rng(seed).integers(0, N_VOCAB, n).astype(np.int32)


def mm(be, w, xq, seq):
    import torch
    y = torch.empty((seq, w[1]), dtype=torch.float32, device="cuda")
    be.matmul_raw(w[0], w[3], w[1], w[2], B.Q8_K, xq, seq, y, B.MEM_DEVICE)
    be.sync()
    return y


def wanted(be, m, weights, il, r_in, pos, seqs):
    """The layer's attention of the rows r_in at pos after the o projection, and their queries."""
    import torch
    c, t = m.cfg, r_in.shape[0]
    xq = be.add_rms_norm_quantize(B.Q8_K, r_in, None, m.get(f"blk.{il}.attn_norm.weight")[3], c.rms_norm_eps)
    q = mm(be, m.get(f"blk.{il}.attn_q.weight"), xq, t).cpu().numpy().reshape(t, c.n_head, c.head_dim)
    norm = weights[f"blk.{il}.attn_q_norm.weight"][3].cpu().numpy() if m.get(f"blk.{il}.attn_q_norm.weight") else None
    r = m.rotary
    q = norm_turn(q, pos, r.inv_freq.cpu().numpy(), r.arg.rot_dim, c.rope_layout == A.ROPE_SPLIT_HALF, norm, c.rms_norm_eps,
                  c.rope_freq_scale, r.arg.magnitude)
    out, _ = attention(q.transpose(1, 0, 2), seqs, c.window, c.n_sink)
    aq = be.quantize_act(B.Q8_K, torch.from_numpy(out.reshape(t, -1).astype(np.float32)).cuda())
    return mm(be, m.get(f"blk.{il}.attn_output.weight"), aq, t).cpu().numpy()


@pytest.mark.parametrize("type_", [B.F16, B.F32])
@pytest.mark.parametrize("name", CONFIGS)
def test_steps_of_many_sequences(be, weights, type_, name):
    c = CONFIGS[name]
    cache = P.PagedCache(be, 24, 16, 2, c.n_head_kv, c.head_dim, type=type_)
    m = PagedLlama(be, c, table(weights, name), cache, 4, 100, 16)
    reader = P.PagedBatch(cache, c.n_head, 1, 256, 16)
    seqs = [P.Sequence() for _ in range(4)]
    for step, new in enumerate(([30, 1, 0, 5], [1, 1, 40, 1], [1, 1, 1, 1], [0, 60, 1, 0], [1, 1, 1, 1])):
        toks = [ids(n, 10 * step + s) for s, n in enumerate(new)]
        trace = []
        logits = m.step(list(zip(seqs, toks)), trace)
        be.sync()
        assert logits.shape == (sum(n > 0 for n in new), N_VOCAB) and np.isfinite(logits.cpu().numpy()).all()
        pos = np.concatenate([np.arange(s.length - n, s.length) for s, n in zip(seqs, new)])
        for il, (r_in, o, _, _) in enumerate(trace):
            held = []
            for s, n in zip(seqs, new):
                there = np.repeat(np.array(s.pages + [-1]) >= 0, 16)[:s.length]
                reader.set([s.length], [s.length], [s.pages])
                k, v = (x.cpu().numpy().astype(np.float64) for x in reader.read(il))
                held.append((n, k, v, None))
                assert c.window or there.all()
            if c.window:
                # pages given back after the step were there during it, but no row of it that is checked here needs them:
                # the last `window` positions and the first ones of each sequence's last row
                rows = np.cumsum(new)[np.array(new) > 0] - 1
                want = wanted(be, m, weights, il, r_in[rows], pos[rows], [(1, k, v, None) for n, k, v, _ in held if n])
                assert rel_err(o.cpu().numpy()[rows], want) <= 1e-3
            else:
                assert rel_err(o.cpu().numpy(), wanted(be, m, weights, il, r_in, pos, held)) <= 1e-3
    if c.window:
        assert m.pages.free() > 24 - sum(-(-s.length // 16) for s in seqs)
    for s in seqs:
        m.pages.close(s)
    assert m.pages.free() == 24


@pytest.mark.parametrize("name", ["plain", "norms", "part"])
def test_sessions_of_their_own(be, weights, name):
    """DeviceLlama over a contiguous f32 cache: the same formulas."""
    c = CONFIGS[name]
    kv = A.KVCache(be, 64, 2, c.n_head_kv, c.head_dim)
    m = DeviceLlama(be, c, table(weights, name), kv)
    import torch
    for n, start in ((23, 0), (1, 23), (4, 24)):
        trace = []
        m.forward(torch.from_numpy(ids(n, start)).cuda(), start, trace)
        be.sync()
        for il, (r_in, o, _, _) in enumerate(trace):
            k, v = (x.cpu().numpy().astype(np.float64).transpose(1, 0, 2) for x in kv.read(il, 0, start + n))
            want = wanted(be, m, weights, il, r_in, np.arange(start, start + n), [(n, k, v, None)])
            assert rel_err(o.cpu().numpy(), want) <= 1e-3


def test_a_step_that_does_not_fit_changes_nothing(be, weights):
    c = CONFIGS["plain"]
    m = PagedLlama(be, c, table(weights, "plain"), P.PagedCache(be, 4, 16, 2, c.n_head_kv, c.head_dim), 2, 24, 4)
    a, b = P.Sequence(), P.Sequence()
    m.step([(a, ids(20, 1)), (b, ids(3, 2))])
    was = [(s.length, list(s.pages)) for s in (a, b)] + [m.pages.free()]
    for news in ([(a, ids(10, 3)), (b, ids(40, 4))], [(a, ids(12, 3)), (b, ids(13, 4))],   # pages run out; too many tokens
                 [(a, ids(2, 3)), (a, ids(2, 4))]):                                # a sequence twice
        with pytest.raises(B.BarqError):
            m.step(news)
        assert [(s.length, s.pages) for s in (a, b)] + [m.pages.free()] == was
    assert m.step([]).shape == (0, N_VOCAB) and m.step([(a, [])]).shape == (0, N_VOCAB)


def test_a_step_that_fails_on_its_way_changes_nothing(be, weights):
    c, there = CONFIGS["plain"], table(weights, "plain")
    full = PagedLlama(be, c, there, P.PagedCache(be, 6, 16, 2, c.n_head_kv, c.head_dim), 2, 40, 4)
    lame = PagedLlama(be, c, lambda name: None if name == "blk.1.ffn_up.weight" else there(name), full.cache, 2, 40, 4, pages=full.pages)
    a, b = P.Sequence(), P.Sequence()
    news = [(a, ids(20, 1)), (b, ids(3, 2))], [(a, ids(13, 3)), (b, ids(14, 4))]
    full.step(news[0])
    was = [(s.length, list(s.pages)) for s in (a, b)] + [full.pages.free()]
    with pytest.raises(KeyError):
        lame.step(news[1])
    assert [(s.length, s.pages) for s in (a, b)] + [full.pages.free()] == was

    def logits(step):
        x = full.step(step)
        be.sync()
        return x.cpu().numpy()
    got = logits(news[1])
    again = [P.Sequence(), P.Sequence()]
    full.pages.close(a)
    full.pages.close(b)
    for new in news:
        want = logits([(s, t) for s, (_, t) in zip(again, new)])
    assert np.array_equal(got, want)   # what the failed step has written is overwritten


def test_buffers_do_not_grow_with_the_steps(be, weights):
    c = CONFIGS["plain"]
    m = PagedLlama(be, c, table(weights, "plain"), P.PagedCache(be, 24, 16, 2, c.n_head_kv, c.head_dim), 4, 40, 16)
    seqs, where = [P.Sequence() for _ in range(4)], None
    for n in (1, 2, 3, 7, 1, 8, 9, 4):
        m.step([(s, ids(n, i)) for i, s in enumerate(seqs)])
        m.step([(seqs[0], ids(1, 9))])
        now = {k: (b.data_ptr(), b.numel()) for k, b in m._bufs.items()}
        assert where is None or {k: now[k] for k in where} == where
        where = now
    assert len(where) <= 16


def test_windows_are_for_pages(be, weights):
    c = CONFIGS["window"]
    with pytest.raises(NotImplementedError):
        DeviceLlama(be, c, table(weights, "window"), A.KVCache(be, 64, 2, c.n_head_kv, c.head_dim))
    with pytest.raises(B.BarqError):
        PagedLlama(be, c, table(weights, "window"), P.PagedCache(be, 4, 16, 3, c.n_head_kv, c.head_dim), 1, 8, 4)


def test_a_model_without_head_norms_is_not_asked_for_them_again(be, weights):
    """A lookup in every layer of every token costs the host more than a launch saves."""
    import torch
    for name, asked in (("plain", 0), ("norms", 4)):
        c, names, find = CONFIGS[name], [], table(weights, name)

        def get(n):
            names.append(n)
            return find(n)
        m = DeviceLlama(be, c, get, A.KVCache(be, 8, 2, c.n_head_kv, c.head_dim))
        names.clear()
        for pos in range(2):
            m.forward(torch.tensor([pos], dtype=torch.int32, device="cuda"), pos)
        be.sync()
        assert sum("_norm.weight" in n and ".attn_q" in n or ".attn_k_norm" in n for n in names) == 2 * asked
