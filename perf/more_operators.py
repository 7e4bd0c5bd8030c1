"""Performance cases of a server's step over a paged KV cache.

A server that answers many sequences at once keeps their K and V rows in pages
of a pool, hands the pages out as the sequences grow, and in one step computes
a few new tokens of every sequence: a chunk of one's prompt, the single next
token of another.  Three kinds of case:

  append     the new tokens' projections: RMSNorm of each head of q and k
             (where the model has it), rotation by the positions, K and V into
             the pages; q rotated, and the rows that the cache then holds
  rotate     the same norm and rotation of the queries of a session whose cache
             is not paged
  attention  the causal grouped-query attention of the new tokens over their
             sequence's pages, or of the last `window` positions of it and the
             first `sinks`

Positions on a page that a sequence has no longer (-1 in its table: behind the
window) are seen by no query.

The rotation: pair i of a row at position p turns by the angle p * inv_freq[i];
pairs are neighbours ("interleaved") or i and i + rot / 2 ("half") of the first
`rot` dims, the other dims stay.  For contexts longer than the model was
trained on, the slow pairs are slowed down by `stretch` and cos and sin
multiplied by 0.1 ln(stretch) + 1.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
BASE = 500000.0


# ---- the cases -----------------------------------------------------------------

def listed():
    def append(name, cache, heads, kv_heads, dim, rot, layout, norm, stretch, seqs, chunks, rows, past_lo, past, page):
        return {"name": name, "kind": "append", "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
                "layout": layout, "norm": norm, "stretch": stretch, "seqs": seqs, "chunks": chunks, "rows": rows,
                "past_lo": past_lo, "past": past, "page": page, "window": 0, "sinks": 0}

    def rotate(name, heads, dim, rot, layout, norm, stretch, rows, past):
        return {"name": name, "kind": "rotate", "heads": heads, "dim": dim, "rot": rot, "layout": layout, "norm": norm,
                "stretch": stretch, "rows": rows, "past": past}

    def attention(name, cache, heads, kv_heads, dim, seqs, chunks, rows, past_lo, past, page, window=0, sinks=0):
        return {"name": name, "kind": "attention", "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "seqs": seqs, "chunks": chunks, "rows": rows, "past_lo": past_lo, "past": past, "page": page,
                "window": window, "sinks": sinks}

    return [
        # the smallest call: the next token of one sequence of an 8B model's layer, with norms of its heads
        append("append_token", "f16", 32, 8, 128, 128, "half", True, 1.0, 1, 0, 1, 4095, 4095, 16),
        # 64 sequences' next tokens, half of each head rotated, far beyond the trained context
        append("append_batch", "f16", 32, 8, 128, 64, "interleaved", False, 4.0, 64, 0, 1, 300, 60000, 16),
        # a chunk of 2048 tokens late in a document
        append("append_prompt", "f16", 32, 8, 128, 128, "half", True, 8.0, 1, 1, 2048, 30000, 30000, 64),
        # a session of its own: one token's queries, and those of a ragged prompt chunk with heads of 256 dims
        rotate("rotate_token", 32, 128, 128, "interleaved", True, 1.0, 1, 5000),
        rotate("rotate_prompt", 16, 256, 64, "half", True, 8.0, 1000, 100000),
        # one sequence's next token against 4096 positions
        attention("attention_token", "f16", 32, 8, 128, 1, 0, 1, 4095, 4095, 16),
        # 32 sequences' next tokens, as long as they happen to be
        attention("attention_batch", "f16", 32, 8, 128, 32, 0, 1, 200, 8000, 16),
        # five drafted tokens of each of four sequences checked at once, f32 rows, seven heads to a kv head
        attention("attention_drafted", "f32", 14, 2, 64, 4, 4, 5, 700, 3001, 32),
        # a long document's next 2048 tokens
        attention("attention_chunk", "f16", 32, 8, 128, 1, 1, 2048, 6000, 6000, 64),
        # two prompts' chunks among ten sequences that decode, heads of 256 dims
        attention("attention_mixed", "f16", 16, 4, 256, 12, 2, 300, 50, 3000, 16),
        # 16 long sequences that see their last 4096 positions and the first four
        attention("window_batch", "f16", 32, 8, 128, 16, 0, 1, 1000, 15000, 32, 4096, 4),
        # a prompt of 4000 tokens that sees 1024 back, 64-element heads
        attention("window_prompt", "f16", 32, 8, 64, 1, 1, 4000, 0, 0, 128, 1024, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "rotate", "attention", "attention", "attention", "window", "window"])
    dim = rng.choice([64, 128, 128, 256])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 4), (32, 32), (24, 8), (16, 8), (14, 2), (20, 1)])
    rot = {"rot": rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]), "layout": rng.choice(["half", "interleaved"]),
           "norm": rng.random() < 0.6, "stretch": rng.choice([1.0, 1.0, 4.0, 8.0, 32.0])}
    if kind == "rotate":
        return {"kind": kind, "heads": heads, "dim": dim, **rot, "rows": rng.choice([1, _log(rng, 2, 64), _log(rng, 65, 4000)]),
                "past": rng.choice([0, _log(rng, 10, 100000), _log(rng, 100000, 1000000)])}
    rows = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 65, 2000)])
    seqs = rng.choice([1, _log(rng, 2, 48)]) if rows <= 64 else rng.choice([1, 1, 2, 3])
    chunks = 0 if rows == 1 else rng.randint(1, seqs)
    past = rng.choice([0, _log(rng, 16, 2000), _log(rng, 2000, 16000)])
    case = {"kind": "attention" if kind == "window" else kind, "cache": rng.choice(["f16", "f16", "f16", "f32"]), "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "seqs": seqs, "chunks": chunks, "rows": rows, "past_lo": rng.randint(0, past),
            "past": past, "page": rng.choice([16, 16, 32, 64, 128, 256])}
    case["window"], case["sinks"] = (_log(rng, 1, 4096), rng.choice([0, 4, rng.randint(1, 200)])) if kind == "window" else (0, 0)
    if kind == "append":
        case["past"] *= rng.choice([1, 60])
        return {**case, **rot}
    # what the plain form has in memory, and both compute, stays below the largest listed case's
    while seqs * (rows if chunks else 1) * heads * (case["past"] + rows) > 5e8 or work(case)["flops"] > 1.8e11 \
            or seqs * kv_heads * dim * (case["past"] + rows) > 2.5e8:
        if case["past"] > 16:
            case["past"] //= 2
            case["past_lo"] = min(case["past_lo"], case["past"])
        else:
            seqs = case["seqs"] = max(1, seqs // 2)
            chunks = case["chunks"] = min(chunks, seqs)
            rows = case["rows"] = max(1, rows * 3 // 4)
    return case


def _lengths(case):
    """New tokens and positions before them, of each sequence: the first is the longest."""
    n, c, lo, hi = case["seqs"], case["chunks"], case["past_lo"], case["past"]
    new = [case["rows"] - case["rows"] * i // (2 * c) if i < c else 1 for i in range(n)]
    past = [hi if i == 0 else lo + int((hi - lo) * (i * 0.6180339887498949 % 1)) for i in range(n)]
    return new, past


# ---- inputs ----------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + 31)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _keys(g, n, kv_heads, dim):
    """Normal rows with a few dims several times as large as the others, the same for all positions of a head."""
    loud = 1 + 4 * (torch.rand(1, kv_heads, dim, device="cuda", generator=g) < 0.03)
    return _normal(g, n, kv_heads, dim) * loud


def _frequencies(case):
    """inv_freq of the rotary pairs (f32) and what cos and sin are multiplied by."""
    rot, s = case["rot"], case["stretch"]
    f = BASE ** (-2.0 * np.arange(rot // 2) / rot)
    if s != 1:   # pairs that turn less than once in 8192 positions: all of the stretch; more than 32 times: none
        keep = np.clip((8192 * f / (2 * math.pi) - 1) / 31, 0, 1)
        f = f * keep + f / s * (1 - keep)
    return f.astype(np.float32), (0.1 * math.log(s) + 1 if s != 1 else 1.0)


def _inputs(case, seed):
    g, kind, d = _gen(seed), case["kind"], case["dim"]
    if kind == "rotate":
        i = {"q": _normal(g, case["rows"], case["heads"], d)}
    else:
        new, past = _lengths(case)
        t = sum(new) if kind == "append" else sum(new) + sum(past)
        i = {"k": _keys(g, t, case["kv_heads"], d), "v": _normal(g, t, case["kv_heads"], d)}
        i["q"] = _normal(g, sum(new), case["heads"], d) if kind == "append" else _normal(g, case["heads"], sum(new), d)
    if kind != "attention" and case["norm"]:
        i["q_norm"], i["k_norm"] = 1 + 0.2 * _normal(g, d), 1 + 0.2 * _normal(g, d)
    return i


def _table(case, seed):
    """The page table [sequences, pages], in any order, -1 where a sequence has no page: behind the window, and (of an
    append, which reads none of them) before the new tokens.  -> table, pages of the pool"""
    new, past = _lengths(case)
    page, w = case["page"], case["window"]
    rng = np.random.default_rng(seed)
    table = np.full((len(new), max(-(-(n + p) // page) for n, p in zip(new, past))), -1, np.int32)
    for s, (n, p) in enumerate(zip(new, past)):
        at = np.arange(-(-(n + p) // page))
        if case["kind"] == "append":
            at = at[at >= p // page]
        elif w:
            at = at[(at * page < case["sinks"]) | ((at + 1) * page > p - w + 1)]
        table[s, at] = 0
    n = int((table >= 0).sum())
    table[table >= 0] = rng.permutation(n)
    return table, n


def _rows(case, table, first, lengths):
    """The pool's row of each of the positions first .. first + length of the sequences (-1: none), sequence after sequence."""
    page = case["page"]
    at = [table[s, np.arange(f, f + n) // page].astype(np.int64) * page + np.arange(f, f + n) % page
          for s, (f, n) in enumerate(zip(first, lengths))]
    gone = [table[s, np.arange(f, f + n) // page] < 0 for s, (f, n) in enumerate(zip(first, lengths))]
    return torch.from_numpy(np.where(np.concatenate(gone), -1, np.concatenate(at))).cuda()


_be = None


def _backend():
    """The program's one handle; the program's torch work runs on the same stream."""
    global _be
    if _be is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "barq-inference_amd"))
        import barq_rocm as B
        _be = B.Backend(0)
        torch.cuda.set_stream(torch.cuda.Stream())
        _be.set_stream(torch.cuda.current_stream().cuda_stream)
    return _be


def _rotary(case):
    from barq_rocm import attention as A
    freq, magnitude = _frequencies(case)
    layout = A.ROPE_SPLIT_HALF if case["layout"] == "half" else A.ROPE_INTERLEAVED
    return A.Rotary(torch.from_numpy(freq).cuda(), case["rot"], layout, magnitude=magnitude)


def prepare(case, seed):
    if own:
        _backend()
    i, kind = _inputs(case, seed), case["kind"]
    s = {"case": case, "q_norm": i.get("q_norm"), "k_norm": i.get("k_norm"), "q": i["q"]}
    if kind == "rotate":
        if own:
            s["rotary"] = _rotary(case)
        else:
            s["pos"] = torch.arange(case["past"], case["past"] + case["rows"], device="cuda")
            s["freq"], s["magnitude"] = torch.from_numpy(_frequencies(case)[0]).cuda(), _frequencies(case)[1]
        torch.cuda.synchronize()
        return s
    new, past = _lengths(case)
    total = [n + p for n, p in zip(new, past)]
    table, pages = _table(case, seed)
    dtype = torch.float16 if case["cache"] == "f16" else torch.float32
    if own:
        import barq_rocm as B
        from barq_rocm import paged as P
        cache = P.PagedCache(_backend(), pages, case["page"], 1, case["kv_heads"], case["dim"],
                             type=B.F16 if case["cache"] == "f16" else B.F32)
        s["batch"] = P.PagedBatch(cache, case["heads"], case["seqs"], sum(new), table.shape[1], window=case["window"],
                                  n_sink=case["sinks"])
        if kind == "attention":
            fill = P.PagedBatch(cache, case["heads"], case["seqs"], sum(total), table.shape[1])
            fill.set(total, total, table)
            fill.append(0, i["k"], i["v"])
        s["batch"].set(new, total, table)
    if kind == "append":
        s["k"], s["v"] = i["k"], i["v"]
        if own:
            s["rotary"] = _rotary(case)
        else:
            s["at"] = _rows(case, table, past, new)
            s["pool"] = [torch.zeros(pages * case["page"], case["kv_heads"], case["dim"], device="cuda", dtype=dtype) for _ in "kv"]
            s["pos"] = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in zip(new, past)])
            s["freq"], s["magnitude"] = torch.from_numpy(_frequencies(case)[0]).cuda(), _frequencies(case)[1]
    elif not own:
        at = _rows(case, table, [0] * len(new), total)
        s["pool"] = [torch.zeros(pages * case["page"], case["kv_heads"], case["dim"], device="cuda", dtype=dtype) for _ in "kv"]
        for pool, x in zip(s["pool"], (i["k"], i["v"])):
            pool[at[at >= 0]] = x[at >= 0].to(dtype)
        # of each sequence padded to the longest: the pool's rows, the new tokens and their positions
        n, r = max(total), max(new)
        s["rows"] = torch.full((len(new), n), -1, device="cuda", dtype=torch.int64)
        s["pos"] = torch.full((len(new), r), -1, device="cuda", dtype=torch.int64)
        s["token"] = torch.zeros((len(new), r), device="cuda", dtype=torch.int64)
        starts, ends = np.cumsum([0] + total), np.cumsum([0] + new)
        for j in range(len(new)):
            s["rows"][j, :total[j]] = at[starts[j]:starts[j + 1]]
            s["pos"][j, :new[j]] = torch.arange(past[j], total[j], device="cuda")
            s["token"][j, :new[j]] = torch.arange(int(ends[j]), int(ends[j + 1]), device="cuda")
        s["taken"] = (s["pos"] >= 0).nonzero(as_tuple=True)
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------

def _turned(state, x, norm):
    """x [tokens, heads, dim], normed by head and rotated."""
    case, rot = state["case"], state["case"]["rot"]
    if norm is not None:
        x = x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * norm
    angle = state["pos"].double()[:, None, None] * state["freq"].double()
    c, s = (torch.cos(angle) * state["magnitude"]).float(), (torch.sin(angle) * state["magnitude"]).float()
    x0, x1 = (x[..., :rot // 2], x[..., rot // 2:rot]) if case["layout"] == "half" else (x[..., :rot:2], x[..., 1:rot:2])
    y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
    y = torch.cat([y0, y1], -1) if case["layout"] == "half" else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _attend(state):
    case, q = state["case"], state["q"]
    kv, d, w = case["kv_heads"], case["dim"], case["window"]
    rows, pos, token = state["rows"], state["pos"], state["token"]
    (seqs, n), r, g = rows.shape, pos.shape[1], case["heads"] // kv
    # [sequences, kv heads, positions, dim]
    k, v = (pool[rows.clamp(min=0)].float().transpose(1, 2) for pool in state["pool"])
    qs = q[:, token].permute(1, 0, 2, 3).reshape(seqs, kv, g * r, d)
    s = torch.matmul(qs, k.transpose(2, 3).contiguous()).reshape(seqs, kv, g, r, n) / math.sqrt(d)
    at = torch.arange(n, device="cuda")
    seen = (at <= pos[:, :, None]) & (rows >= 0)[:, None, :]
    if w:
        seen &= (at > pos[:, :, None] - w) | (at < case["sinks"])
    seen = seen[:, None, None]
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p.reshape(seqs, kv, g * r, n), v.contiguous()).reshape(seqs, kv * g, r, d)
    return o.transpose(1, 2)[state["taken"]]


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "attention":
            return _attend(state)
        q = _turned(state, state["q"], state["q_norm"]).transpose(0, 1).contiguous()
        if kind == "rotate":
            return q
        for pool, x in zip(state["pool"], (_turned(state, state["k"], state["k_norm"]), state["v"])):
            pool[state["at"]] = x.to(pool.dtype)
        return {"q": q, "k": state["pool"][0][state["at"]], "v": state["pool"][1][state["at"]]}
    if kind == "rotate":
        from barq_rocm import attention as A
        return A.norm_rope(_backend(), state["q"], case["rows"], case["heads"], case["dim"], case["past"], state["rotary"],
                           norm=state["q_norm"], eps=EPS, sync=False)
    batch = state["batch"]
    if kind == "attention":
        return batch.attention(0, state["q"], sync=False)
    q = batch.append(0, state["k"], state["v"], q=state["q"], rotary=state["rotary"], q_norm=state["q_norm"],
                     k_norm=state["k_norm"], eps=EPS)
    k, v = batch.read(0, sync=False)
    return {"q": q, "k": k, "v": v}


# ---- what a pass cannot do without ---------------------------------------------------

def _pairs(new, past, window, sinks):
    """How many positions the new tokens of a sequence see, all together, and how many of its positions are seen at all."""
    p = np.arange(past, past + new, dtype=np.int64)
    if not window:
        return int((p + 1).sum()), past + new
    low = np.maximum(p - window + 1, 0)
    return int((p - low + 1 + np.minimum(low, sinks)).sum()), int(past + new - low[0] + min(low[0], sinks))


def work(case):
    kind, d = case["kind"], case["dim"]
    if kind == "rotate":
        n = case["rows"] * case["heads"] * d
        return {"bytes": 8 * n, "flops": (7 if case["norm"] else 3) * n}
    size = 2 if case["cache"] == "f16" else 4
    new, past = _lengths(case)
    h, kv, t = case["heads"], case["kv_heads"], sum(new)
    if kind == "append":   # q read and written; K and V read, written into the pages, read there and written once more
        return {"bytes": t * d * (8 * h + 2 * kv * (4 + 3 * size)), "flops": t * d * ((7 if case["norm"] else 3) * (h + kv) + kv)}
    seen = [_pairs(n, p, case["window"], case["sinks"]) for n, p in zip(new, past)]
    return {"bytes": 2 * kv * d * size * sum(s for _, s in seen) + 8 * t * h * d, "flops": 4 * h * d * sum(n for n, _ in seen)}


# ---- the same in 64 bits -------------------------------------------------------------

def _exact_turn(case, x, norm, pos):
    """By complex numbers: pair i of a row is x0 + i x1, times magnitude * e^(i angle)."""
    freq, magnitude = _frequencies(case)
    rot = case["rot"]
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
    turn = torch.polar(torch.full((), magnitude, dtype=torch.float64, device="cuda"),
                       torch.outer(pos.double(), torch.from_numpy(freq.astype(np.float64)).cuda()))
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn[:, None, :]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    i, kind = _inputs(case, seed), case["kind"]
    if kind == "rotate":
        pos = torch.arange(case["past"], case["past"] + case["rows"], device="cuda")
        return _exact_turn(case, i["q"], i.get("q_norm"), pos).transpose(0, 1).contiguous()
    new, past = _lengths(case)
    if kind == "append":
        pos = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in zip(new, past)])
        return {"q": _exact_turn(case, i["q"], i.get("q_norm"), pos).transpose(0, 1).contiguous(),
                "k": _exact_turn(case, i["k"], i.get("k_norm"), pos), "v": i["v"].double()}
    if case["cache"] == "f16":
        i["k"], i["v"] = i["k"].half(), i["v"].half()
    out, t, c, g = [], 0, 0, case["heads"] // case["kv_heads"]
    for n, p in zip(new, past):
        at, row = torch.arange(p + n, device="cuda"), torch.arange(p, p + n, device="cuda")[:, None]
        hidden = at > row
        if case["window"]:
            hidden |= (row - at >= case["window"]) & (at >= case["sinks"])
        heads = []
        for h in range(case["heads"]):
            k, v = i["k"][c:c + p + n, h // g].double(), i["v"][c:c + p + n, h // g].double()
            s = (i["q"][h, t:t + n].double() @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
            heads.append(torch.softmax(s, -1) @ v)
        out.append(torch.stack(heads, 1))
        t, c = t + n, c + p + n
    return torch.cat(out)
