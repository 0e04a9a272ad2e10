"""Plain 64-bit results of the operators over paged caches (include/xqhip.h): what a page holds, attention over a
sequence's positions, log probabilities."""
import numpy as np


def to_pages_k(x, e):
    """[pages][nkv][page][hd] -> the pool's [pages][nkv][hd / e][page][e]."""
    n, nkv, page, hd = x.shape
    return np.ascontiguousarray(x.reshape(n, nkv, page, hd // e, e).transpose(0, 1, 3, 2, 4))


def to_pages_v(x, e):
    """[pages][nkv][page][hd] -> the pool's [pages][nkv][page / e][hd][e]."""
    n, nkv, page, hd = x.shape
    return np.ascontiguousarray(x.reshape(n, nkv, page // e, e, hd).transpose(0, 1, 2, 4, 3))


def from_pages_k(x):
    n, nkv, b, page, e = x.shape
    return np.ascontiguousarray(x.transpose(0, 1, 3, 2, 4)).reshape(n, nkv, page, b * e)


def from_pages_v(x):
    n, nkv, b, hd, e = x.shape
    return np.ascontiguousarray(x.transpose(0, 1, 2, 4, 3)).reshape(n, nkv, b * e, hd)


def codes(x16):
    """Codes and scale of one page and head's fp16 values [positions][hd]."""
    x = x16.astype(np.float64)
    mx = np.abs(x).max() if x.size else 0.0
    c = np.rint(x * 127 / mx) if mx > 0 else np.zeros_like(x)
    return c.astype(np.int8), np.float32(mx / 127)


def held(x):
    """The fp16 values that 8-bit pages are taken of."""
    x = np.asarray(x, np.float32)
    return np.where(np.isnan(x), 0, np.clip(x, -65504, 65504)).astype(np.float16)


def prepared(x, w, cs, eps):
    """x [.., hd] normalised and turned by cs [.., pairs][2], in 64 bits, rounded to fp32."""
    x, w, cs = x.astype(np.float64), w.astype(np.float64), cs.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float32(eps).astype(np.float64)) * w
    half = cs.shape[-2]
    a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
    y[..., :half] = a * cs[..., 0] - b * cs[..., 1]
    y[..., half:2 * half] = b * cs[..., 0] + a * cs[..., 1]
    return y.astype(np.float32)


def attend(q, k, v, see):
    """q [nq][hd] over k, v [positions][nkv][hd] (64 bits); see [positions]; 0 where nothing is seen."""
    nq, hd = q.shape
    g = nq // k.shape[1]
    out = np.zeros((nq, hd))
    at = np.flatnonzero(see)
    for h in range(nq):
        z = k[at, h // g].astype(np.float64) @ q[h].astype(np.float64) / np.sqrt(hd)
        z = z[z > -np.inf] if len(z) and not np.isnan(z).any() else z
        if not len(z):
            continue
        keep = at[k[at, h // g].astype(np.float64) @ q[h].astype(np.float64) / np.sqrt(hd) > -np.inf] if not np.isnan(z).any() else at
        e = np.exp(z - z.max())
        out[h] = e @ v[keep, h // g].astype(np.float64) / e.sum()
    return out


def sigmoid(x):
    return 1 / (1 + np.exp(-np.asarray(x, np.float64)))


def logprobs(x, t, inv_t, top):
    """One row of logits: log probability of t, entropy, rank, top ids, their log probabilities."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    order = np.lexsort((np.arange(len(x)), -x))
    has = 0 <= t < len(x)
    rank = int(np.flatnonzero(order == t)[0]) if has else -1
    ids, lps = np.full(top, -1), np.full(top, -np.inf)
    if m == -np.inf:
        return -np.inf, 0.0, rank, ids, lps
    with np.errstate(invalid="ignore"):
        d = np.where(x == m, 0.0, (x - m) * np.float64(np.float32(inv_t)))
    e = np.exp(d)
    rest = np.delete(e, np.argmax(x)).sum()
    lp = d - np.log1p(rest)
    with np.errstate(invalid="ignore"):
        ent = -np.where(e > 0, e / (1 + rest) * lp, 0.0).sum()
    first = order[:top]
    first = first[x[first] > -np.inf]
    ids[:len(first)], lps[:len(first)] = first, lp[first]
    return (lp[t] if has else -np.inf), ent, rank, ids, lps
