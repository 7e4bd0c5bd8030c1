"""The 4-bit KV cache, attention, attention mass and eviction in numpy, in 64
bits and without the library: what the GPU tests compare with."""
import numpy as np

D_MAX = 8188.0


def q4_quantize(x):
    """f32 rows [..., hd] -> (codes uint8 [..., hd], scales f32 (f16 values) [..., hd / 32])."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    b = x.reshape(-1, 32)
    a = np.abs(b)
    bad = ~np.isfinite(b).all(1)
    top = b[np.arange(len(b)), np.where(np.isnan(a), -1, a).argmax(1)].astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        d = np.clip((top / -8).astype(np.float16).astype(np.float64), -D_MAX, D_MAX)
        d[bad] = np.nan
        y = b.astype(np.float64) / np.where((d == 0) | bad, 1, d)[:, None]
        c = np.clip(np.floor(np.nan_to_num(y, nan=0.0, posinf=0.0, neginf=0.0) + 8.5), 0, 15)
    c[(d == 0) | bad] = 8
    return c.astype(np.uint8).reshape(x.shape), d.astype(np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32)


def q4_values(x):
    """What the blocks of the rows read as (f32, exact)."""
    c, d = q4_quantize(x)
    v = (c.reshape(-1, 32).astype(np.float32) - 8) * d.reshape(-1, 1)
    return v.reshape(c.shape).astype(np.float32)


def attention(q, k, v, start):
    """q [heads, rows, hd], k and v [kv heads, n, hd] -> (out [rows, heads, hd], mass [kv heads, n]) in f64."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    heads, rows, hd = q.shape
    n_kv, n = k.shape[:2]
    out, mass = np.empty((rows, heads, hd)), np.zeros((n_kv, n))
    seen = np.arange(n)[None, :] <= start + np.arange(rows)[:, None]
    for h in range(heads):
        j = h * n_kv // heads
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(seen, q[h] @ k[j].T / np.sqrt(hd), -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
        if np.isfinite(v[j]).all():
            out[:, h] = p @ v[j]
        else:
            for i in range(rows):
                out[i, h] = p[i, seen[i]] @ v[j][seen[i]]
        mass[j] += p.sum(0)
    return out, mass


def kept(mass, n, keep, recent):
    """Positions each kv head keeps of its n, ascending: [kv heads, min(keep, n)]."""
    m = min(keep, n)
    if m == n:
        return np.tile(np.arange(n, dtype=np.int32), (len(mass), 1))
    old = n - recent
    out = np.empty((len(mass), m), np.int32)
    for h, w in enumerate(np.asarray(mass, np.float64)):
        w = np.where(np.isnan(w[:old]), -np.inf, w[:old])
        out[h] = np.sort(np.concatenate([np.lexsort((np.arange(old), -w))[:m - recent], np.arange(old, n)]))
    return out
