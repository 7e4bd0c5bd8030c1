"""Performance cases of the KV cache held in 4 bits and of its eviction.

A program that answers long prompts keeps the cache small in two ways: it
holds K and V as Q4_0 blocks (32 elements, one f16 scale d, element =
(code - 8) * d with a 4-bit code), and it drops the positions that the queries
have given little attention weight so far.  Four kinds of case:

  append     K and V rows of new positions into the cache, and the rows that
             the cache then stands for
  attention  one layer's causal grouped-query attention over a Q4_0 cache
  mass       the same (over a Q4_0 or an f32 cache) that also adds, for every
             kv head and position, the softmax weights of all the queries and
             query heads to the mass that the position has gathered so far
  evict      of every kv head the newest `recent` positions stay, and of the
             older ones those with the largest mass, `keep` in all (of equal
             ones the earlier), in the order of their positions

A block's scale is its largest element (the first of the largest |x|) over -8,
rounded to f16 and at most 8188 in size; an element's code is the nearest one
under that scale (a border belongs to the larger code).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
D_MAX = 8188.0


# ---- the cases -----------------------------------------------------------------

def listed():
    def append(name, kv_heads, dim, rows):
        return {"name": name, "kind": "append", "kv_heads": kv_heads, "dim": dim, "rows": rows}

    def attention(name, heads, kv_heads, dim, rows, start):
        return {"name": name, "kind": "attention", "cache": "q4_0", "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rows": rows, "start": start}

    def mass(name, cache, heads, kv_heads, dim, rows, start):
        return {"name": name, "kind": "mass", "cache": cache, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rows": rows, "start": start}

    def evict(name, cache, kv_heads, dim, n, keep, recent):
        return {"name": name, "kind": "evict", "cache": cache, "kv_heads": kv_heads, "dim": dim, "n": n, "keep": keep,
                "recent": recent}

    return [
        # the smallest call: one decoded token's rows of an 8B model's layer
        append("append_token", 8, 128, 1),
        # a 2048-token prompt of that layer
        append("append_prompt", 8, 128, 2048),
        # one decoded token of an 8B model against 4096 cached positions
        attention("attention_token", 32, 8, 128, 1, 4095),
        # the same at the end of a long document
        attention("attention_token_long", 32, 8, 128, 1, 65535),
        # five drafted tokens checked at once, heads of 256 dims that share nothing
        attention("attention_drafted", 16, 16, 256, 5, 2998),
        # a 1B model (64-element heads): a later chunk of a prompt, a ragged one
        attention("attention_chunk", 32, 8, 64, 200, 800),
        # a 2048-token prompt
        attention("attention_prompt", 32, 8, 128, 2048, 0),
        # a decoded token that keeps account of the positions' weights, on either cache
        mass("mass_token", "q4_0", 32, 8, 128, 1, 4095),
        mass("mass_token_f32", "f32", 32, 8, 128, 1, 4095),
        # the last 512 tokens of a 2048-token prompt decide what is kept of it
        mass("mass_prompt", "q4_0", 32, 8, 128, 512, 1536),
        # a long prompt cut to a quarter, its newest 512 positions among them
        evict("evict_q4_0", "q4_0", 8, 128, 16384, 4096, 512),
        # the f32 cache one position over twice its budget
        evict("evict_f32", "f32", 8, 128, 4097, 2048, 256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "mass", "mass", "evict"])
    if kind == "append":
        return {"kind": kind, "kv_heads": rng.choice([1, 2, 4, 8, 16]), "dim": rng.choice([64, 128, 256]),
                "rows": rng.choice([1, _log(rng, 2, 64), _log(rng, 65, 4096)])}
    if kind == "evict":
        n = _log(rng, 64, 32768)
        keep = rng.randint(1, n)
        return {"kind": kind, "cache": rng.choice(["q4_0", "q4_0", "f32"]), "kv_heads": rng.choice([1, 2, 4, 8]),
                "dim": rng.choice([64, 128]), "n": n, "keep": keep, "recent": rng.randint(0, keep)}
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 4), (32, 32), (24, 8), (16, 8), (14, 2), (20, 1)])
    rows = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 65, 1000)])
    start = rng.choice([0, _log(rng, 16, 6000), _log(rng, 16, 50000)]) if rows <= 64 else rng.choice([0, _log(rng, 16, 1500)])
    return {"kind": kind, "cache": "q4_0" if kind == "attention" else rng.choice(["q4_0", "q4_0", "f32"]),
            "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128, 256]), "rows": rows, "start": start}


# ---- inputs ----------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)


def _keys(g, kv_heads, n, dim):
    """Normal rows with a few dims several times as large as the others, the same for all positions of a head."""
    loud = 1 + 4 * (torch.rand(kv_heads, 1, dim, device="cuda", generator=g) < 0.03)
    return torch.randn(kv_heads, n, dim, device="cuda", generator=g) * loud


def _mass(g, kv_heads, n):
    """What positions gather: a few take most of it, some nothing at all."""
    m = torch.exp(2 * torch.randn(kv_heads, n, device="cuda", generator=g))
    return torch.where(torch.rand(kv_heads, n, device="cuda", generator=g) < 0.1, torch.zeros_like(m), m)


def _inputs(case, seed):
    g, kind, kv, d = _gen(seed), case["kind"], case["kv_heads"], case["dim"]
    n = {"append": lambda: case["rows"], "evict": lambda: case["n"]}.get(kind, lambda: case["start"] + case["rows"])()
    i = {"k": _keys(g, kv, n, d), "v": torch.randn(kv, n, d, device="cuda", generator=g)}
    if kind in ("attention", "mass"):
        i["q"] = torch.randn(case["heads"], case["rows"], d, device="cuda", generator=g)
    if kind in ("mass", "evict"):
        i["mass"] = _mass(g, kv, n)
    if kind == "mass":   # about what four decoded tokens have left there
        i["mass"] *= 4 * case["heads"] / kv / (math.exp(2) * n)
    return i


def _quantize(x):
    """f32 rows -> codes (uint8) and scales (f16, one for each 32 elements)."""
    b = x.reshape(-1, BLOCK)
    a = b.abs()
    at = torch.arange(BLOCK, device=x.device).expand_as(b)
    first = torch.where(a == a.amax(1, keepdim=True), at, BLOCK).amin(1, keepdim=True)
    d = (torch.gather(b, 1, first) / -8).half().clamp(-D_MAX, D_MAX)
    s = torch.where(d == 0, torch.ones_like(d), d)
    # quotients in 64 bits: no f32 element then rounds onto a border it is not on
    c = torch.floor(b.double() / s.double() + 8.5).clamp(0, 15)
    c = torch.where(d == 0, torch.full_like(c, 8), c).to(torch.uint8)
    return c.reshape(x.shape), d.reshape(*x.shape[:-1], x.shape[-1] // BLOCK)


def _values(c, d):
    """codes and scales -> f32 rows (exact: 4 bits times 11)."""
    b = (c.reshape(-1, BLOCK).float() - 8) * d.reshape(-1, 1).float()
    return b.reshape(c.shape)


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


def _cache(case, i, n, room):
    """The program's cache of one layer, with the first n rows of k and v in it."""
    be = _backend()
    import barq_rocm as B
    from barq_rocm import attention as A
    kind = B.Q4_0 if case.get("cache", "q4_0") == "q4_0" else B.F32
    kv = A.KVCache(be, max(room, 1), 1, case["kv_heads"], case["dim"], type=kind)
    if n:
        kv.append(0, i["k"], i["v"], n, case["dim"])
    return kv


def prepare(case, seed):
    if own:
        _backend()
    i, kind = _inputs(case, seed), case["kind"]
    n = i["k"].shape[1]
    s = {"case": case, "mass": i.get("mass"), "q": i.get("q")}
    if kind == "append":
        s["k"], s["v"] = i["k"], i["v"]
        if own:
            s["kv"] = _cache(case, i, 0, n)
    else:
        if own:
            s["kv"] = _cache(case, i, n, n)
            if kind == "evict":
                s["to"] = _cache(case, i, 0, case["keep"])
        elif case["cache"] == "q4_0":
            s["kq"], s["vq"] = _quantize(i["k"]), _quantize(i["v"])
        else:
            s["k"], s["v"] = i["k"], i["v"]
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------

def _rows(state):
    """The cached rows as f32."""
    if state["case"]["cache"] == "q4_0":
        return _values(*state["kq"]), _values(*state["vq"])
    return state["k"], state["v"]


def _attend(state):
    """-> outputs [rows, heads, dim] and weights [kv heads, heads per kv head, rows, positions]."""
    case, q = state["case"], state["q"]
    k, v = _rows(state)
    kv, d, rows, n = case["kv_heads"], case["dim"], case["rows"], k.shape[1]
    g = case["heads"] // kv
    s = torch.matmul(q.reshape(kv, g * rows, d), k.transpose(1, 2)).reshape(kv, g, rows, n) / math.sqrt(d)
    seen = torch.arange(n, device="cuda")[None, :] <= case["start"] + torch.arange(rows, device="cuda")[:, None]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(kv, g * rows, n), v).reshape(kv * g, rows, d)
    return o.transpose(0, 1).contiguous(), p


def _evict(state):
    case, mass = state["case"], state["mass"]
    n, keep, recent = case["n"], case["keep"], case["recent"]
    old = n - recent
    if keep < n:
        order = torch.sort(mass[:, :old], dim=1, descending=True, stable=True).indices[:, :keep - recent]
        newest = torch.arange(old, n, device="cuda").expand(mass.shape[0], recent)
        kept = torch.cat([torch.sort(order, dim=1).values, newest], 1)
    else:
        kept = torch.arange(n, device="cuda").repeat(mass.shape[0], 1)
    new = torch.zeros_like(mass)
    new[:, :kept.shape[1]] = torch.gather(mass, 1, kept)

    def take(t):
        return torch.gather(t, 1, kept[:, :, None].expand(-1, -1, t.shape[2]))
    if case["cache"] == "q4_0":
        k, v = (_values(take(c), take(d)) for c, d in (state["kq"], state["vq"]))
    else:
        k, v = take(state["k"]), take(state["v"])
    return {"kept": kept.to(torch.int32), "mass": new, "k": k, "v": v}


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "append":
            return {"k": _values(*_quantize(state["k"])), "v": _values(*_quantize(state["v"]))}
        if kind == "evict":
            return _evict(state)
        out, p = _attend(state)
        return {"out": out, "mass": state["mass"] + p.sum((1, 2))} if kind == "mass" else out
    from barq_rocm import attention as A
    be, kv = _backend(), state["kv"]
    if kind == "append":
        kv.clear()   # the cache's next prompt, or the token of another one
        kv.append(0, state["k"], state["v"], case["rows"], case["dim"])
        k, v = kv.read(0, 0, case["rows"], sync=False)
        return {"k": k, "v": v}
    if kind == "evict":
        to = state["to"]
        kept, mass = kv.evict(0, state["mass"], case["keep"], case["recent"], dst=to, mass_out=torch.empty_like(state["mass"]),
                              sync=False)
        k, v = to.read(0, 0, to.layer_len(0), sync=False)
        return {"kept": kept, "mass": mass, "k": k, "v": v}
    shape = (be, state["q"], kv, 0, case["heads"], case["kv_heads"], case["dim"], case["rows"], case["start"] + case["rows"],
             case["start"])
    if kind == "mass":
        out, mass = A.compute_attention_mass(*shape, state["mass"], mass_out=torch.empty_like(state["mass"]), sync=False)
        return {"out": out, "mass": mass}
    return A.compute_attention(*shape, sync=False)


# ---- what a pass cannot do without ---------------------------------------------------

def _row_bytes(case):
    """One cached row of K or V of one kv head."""
    d = case["dim"]
    return d // 2 + d // BLOCK * 2 if case.get("cache", "q4_0") == "q4_0" else 4 * d


def work(case):
    kind, kv, d = case["kind"], case["kv_heads"], case["dim"]
    if kind == "append":   # read, written as blocks, read again as f32
        n = 2 * kv * case["rows"]
        return {"bytes": n * (8 * d + 2 * _row_bytes(case)), "flops": 4 * n * d}
    if kind == "evict":
        n, m = case["n"], min(case["n"], case["keep"])
        # the mass read and written; the kept rows moved, and read again as f32
        return {"bytes": kv * (8 * n + 4 * m) + 2 * kv * m * (3 * _row_bytes(case) + 4 * d), "flops": 2 * kv * m * d + kv * n}
    r, s, h = case["rows"], case["start"], case["heads"]
    pairs = r * s + r * (r + 1) // 2
    mass = kind == "mass"
    return {"bytes": 2 * kv * (s + r) * _row_bytes(case) + 8 * r * h * d + (8 * kv * (s + r) if mass else 0),
            "flops": 4 * h * d * pairs + (h * pairs if mass else 0)}


# ---- the same in 64 bits -------------------------------------------------------------

def _q4_0(x):
    """What the Q4_0 blocks of the rows stand for, in numpy's 64 bits."""
    b = x.cpu().numpy().reshape(-1, BLOCK)
    top = b[np.arange(len(b)), np.abs(b).argmax(1)].astype(np.float64)   # argmax: the first
    d = np.clip((top / -8).astype(np.float16).astype(np.float64), -D_MAX, D_MAX)[:, None]
    y = b.astype(np.float64) / np.where(d == 0, 1, d)
    low = np.floor(y)
    code = np.clip(low + (y - low >= 0.5), -8, 7)
    return torch.from_numpy((code * d).reshape(x.shape)).cuda()


def exact(case, seed):
    i, kind = _inputs(case, seed), case["kind"]
    if kind == "append":
        return {"k": _q4_0(i["k"]), "v": _q4_0(i["v"])}
    if case["cache"] == "q4_0":
        # (beyond some 30 million elements the host's pass over them takes too long)
        if i["k"].numel() > 40_000_000:
            c = [_quantize(t) for t in (i["k"], i["v"])]
            k, v = ((a.double() - 8) * b.double().repeat_interleave(BLOCK, -1) for a, b in c)
        else:
            k, v = _q4_0(i["k"]), _q4_0(i["v"])
    else:
        k, v = i["k"].double(), i["v"].double()
    if kind == "evict":
        n, recent, m = case["n"], case["recent"], min(case["n"], case["keep"])
        mass = i["mass"].double().cpu().numpy()
        kept = np.empty((len(mass), m), np.int64)
        for h, w in enumerate(mass):
            # lexsort: by mass downwards, then by position
            old = np.lexsort((np.arange(n - recent), -w[:n - recent]))[:max(m - recent, 0)] if m < n else np.arange(n - recent)
            kept[h] = np.sort(np.concatenate([old, np.arange(n - recent, n)]))
        new = np.zeros_like(mass)
        new[:, :m] = np.take_along_axis(mass, kept, 1)
        heads, at = torch.arange(len(mass), device="cuda")[:, None], torch.from_numpy(kept).cuda()
        return {"kept": at.to(torch.int32), "mass": torch.from_numpy(new).cuda(), "k": k[heads, at], "v": v[heads, at]}
    heads, rows = case["heads"], case["rows"]
    vis = torch.arange(k.shape[1], device="cuda")[None, :] - torch.arange(rows, device="cuda")[:, None] <= case["start"]
    out, mass = [], i["mass"].double() if kind == "mass" else None
    for h in range(heads):
        j = h * case["kv_heads"] // heads
        w = torch.softmax((i["q"][h].double() @ k[j].T / math.sqrt(case["dim"])).masked_fill(~vis, -math.inf), -1)
        out.append(w @ v[j])
        if kind == "mass":
            mass[j] += w.sum(0)
    out = torch.stack(out, 1)
    return {"out": out, "mass": mass} if kind == "mass" else out
