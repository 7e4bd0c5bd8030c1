"""DeviceLlama over a 4-bit KV cache and under a KV budget: append, attention,
masses and eviction as a session runs them (a prompt, then token by token).

Bar for a layer's attention output after the o projection: teacher-forced,
i.e. numpy attention over the rows the cache reads as, with the queries the
library's own projection and RoPE of the traced layer input give, through the
library's Q8_K quantizer and projection.  Both sides quantize rows that agree
to 2e-5, so now and then an element moves by one Q8 step: relative L2 1e-3
(conftest.assert_close_1e3's bar for one projection)."""
import numpy as np
import pytest

import barq_rocm as B
from barq_rocm import attention as A
from barq_rocm import synth
from barq_rocm.llama import DeviceLlama, KVBudget, LlamaConfig
from conftest import rel_err
from kv_ref import attention, kept

pytestmark = pytest.mark.gpu
CFG = LlamaConfig(n_layer=2, n_embd=1024, n_head=8, n_head_kv=2, head_dim=128, n_ff=1024)
N_VOCAB = 512


@pytest.fixture(scope="module")
def weights():
    import torch
    w = {}

    def put(name, t, n, k, data):
        w[name] = (t, n, k, torch.from_numpy(data).cuda())
    kv = CFG.n_head_kv * CFG.head_dim
    for il in range(CFG.n_layer):
        for i, (sfx, n, k) in enumerate((("attn_q", 1024, 1024), ("attn_k", kv, 1024), ("attn_v", kv, 1024),
                                         ("attn_output", 1024, 1024), ("ffn_gate", 1024, 1024), ("ffn_up", 1024, 1024),
                                         ("ffn_down", 1024, 1024))):
            put(f"blk.{il}.{sfx}.weight", B.Q4_K, n, k, synth.gen_weights(B.Q4_K, n, k, 60 + 16 * il + i))
        for j, nm in enumerate(("attn_norm", "ffn_norm")):
            put(f"blk.{il}.{nm}.weight", B.F32, 1, 1024, (0.02 * (1 + 0.1 * synth.gen_f32(1024, 90 + 2 * il + j))).astype(np.float32))
    put("token_embd.weight", B.Q4_K, N_VOCAB, 1024, synth.gen_weights(B.Q4_K, N_VOCAB, 1024, 98))
    put("output_norm.weight", B.F32, 1, 1024, (0.02 * (1 + 0.1 * synth.gen_f32(1024, 99))).astype(np.float32))
    return w


def model(be, weights, room, type_, budget=None):
    table = {k: (t, n, kk, d.data_ptr()) for k, (t, n, kk, d) in weights.items()}
    return DeviceLlama(be, CFG, table.get, A.KVCache(be, room, CFG.n_layer, CFG.n_head_kv, CFG.head_dim, type=type_), budget)


def tokens(n, seed):
    import torch
    return torch.from_numpy(np.random.default_rng(seed).integers(0, N_VOCAB, n).astype(np.int32)).cuda()


def mm(be, w, xq, seq):
    import torch
    y = torch.empty((seq, w[1]), dtype=torch.float32, device="cuda")
    be.matmul_raw(w[0], w[3], w[1], w[2], B.Q8_K, xq, seq, y, B.MEM_DEVICE)
    be.sync()
    return y


def layer_attention(be, m, il, r_in, pos):
    """The layer's attention (after the o projection) of the last rows of the
    cache, and what it adds to the masses, the long way."""
    import torch
    seq = r_in.shape[0]
    xq = be.add_rms_norm_quantize(B.Q8_K, r_in, None, m.get(f"blk.{il}.attn_norm.weight")[3], CFG.rms_norm_eps)
    q = A.apply_rope(be, mm(be, m.get(f"blk.{il}.attn_q.weight"), xq, seq), seq, CFG.n_head, CFG.head_dim, pos, 1.0,
                     m.inv_freq, CFG.rope_layout).cpu().numpy()
    n = m.kv.layer_len(il)
    k, v = (t.cpu().numpy() for t in m.kv.read(il, 0, n))
    out, mass = attention(q, k, v, n - seq)
    aq = be.quantize_act(B.Q8_K, torch.from_numpy(out.reshape(seq, -1).astype(np.float32)).cuda())
    return mm(be, m.get(f"blk.{il}.attn_output.weight"), aq, seq).cpu().numpy(), mass


def check_layers(be, m, trace, pos, masses=None):
    for il, (r_in, o, _, _) in enumerate(trace):
        want, mass = layer_attention(be, m, il, r_in, pos)
        assert rel_err(o.cpu().numpy(), want) <= 1e-3
        if masses is not None:
            n = mass.shape[1]
            got = m.mass[il].cpu().numpy()
            # 2.5e-5 for the weights (the mass tests' bar) and 1e-4 for the
            # queries, which two launches of different summation order give
            assert np.allclose(got[:, :n] - masses[il][:, :n], mass, rtol=2e-4, atol=1e-6 * seq_of(r_in))
            assert not got[:, n:].any()


def seq_of(r):
    return r.shape[0]


def test_session_on_a_4_bit_cache(be, weights):
    m = model(be, weights, 64, B.Q4_0)
    for seq, pos in ((23, 0), (1, 23), (1, 24), (5, 25)):
        trace = []
        logits = m.forward(tokens(seq, pos), pos, trace)
        be.sync()
        assert np.isfinite(logits.cpu().numpy()).all()
        assert m.kv.size() == m.kv.layer_len(1) == pos + seq
        check_layers(be, m, trace, pos)


@pytest.mark.parametrize("type_", [B.F32, B.Q4_0])
def test_session_under_a_budget(be, weights, type_):
    keep, recent, slack = 24, 6, 4
    m = model(be, weights, 64, type_, KVBudget(keep, recent, slack))
    for session in range(2):   # the second one starts from cleared rows and masses
        m.kv.clear()
        pos, length = 0, 0
        for seq in (20, 1, 1, 3, 1, 1, 1, 1, 1, 6, 1):
            before = [t.cpu().numpy() for t in m.mass]
            if length == 0:
                before = [np.zeros_like(b) for b in before]
            trace = []
            m.forward(tokens(seq, pos + session), pos, trace)
            be.sync()
            pos += seq
            length += seq
            if length > keep + slack:
                length = keep
            else:   # (an evicting call's rows are gone)
                check_layers(be, m, trace, pos - seq, before)
            assert [m.kv.layer_len(il) for il in range(2)] == [length] * 2
        assert length < pos


def test_budget_is_checked(be, weights):
    for b in (KVBudget(4, 5), KVBudget(0, 0), KVBudget(4, 1, -1)):
        with pytest.raises(ValueError):
            model(be, weights, 16, B.F32, b)


def test_evicting_a_layer_keeps_the_heaviest(be, weights):
    """What the budget run dropped, against the masses just before."""
    m = model(be, weights, 64, B.Q4_0, KVBudget(30, 8, 30))
    m.forward(tokens(40, 1), 0)
    be.sync()
    mass = m.mass[1].cpu().numpy().copy()
    k, v = (t.cpu().numpy() for t in m.kv.read(1, 0, 40))
    want = kept(mass[:, :40], 40, 30, 8)
    got, _ = m.kv.evict(1, m.mass[1], 30, 8)
    assert np.array_equal(got.cpu().numpy(), want)
    gk, gv = (t.cpu().numpy() for t in m.kv.read(1, 0, 30))
    i = np.arange(2)[:, None]
    assert np.array_equal(gk, k[i, want]) and np.array_equal(gv, v[i, want])
