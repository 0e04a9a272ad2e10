"""Plain 64-bit results of the operators of a decode step over a tree of drafted
tokens, row by row from their definitions (include/xqhip.h)."""
import numpy as np


def random_tree(rng, n, reach=6):
    return [-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, n)]


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def path_masks(parents):
    m = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def quantise(x):
    """Codes and scales of 8-bit rows, in the float32 steps of the definition."""
    x = np.asarray(x, np.float32)
    scale = (np.abs(x).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        codes = np.clip(np.rint(x / np.where(scale > 0, scale, np.float32(1))), -127, 127)
        return np.where((scale > 0) & np.isfinite(scale), codes, 0).astype(np.int8), scale[..., 0]


def prepared(x, w, cs, eps):
    """RMSNorm and partial RoPE of heads x [..., hd]; cs [..., pairs, 2]."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    n = cs.shape[-2]
    c, s = cs[..., 0].astype(np.float64), cs[..., 1].astype(np.float64)
    a, b = y[..., :n].copy(), y[..., n:2 * n].copy()
    y[..., :n], y[..., n:2 * n] = a * c - b * s, b * c + a * s
    return y


def attention(q, gate, k, v, pos0, see):
    """q, gate [T][nq][hd]; k, v [positions][nkv][hd]; see [T][T]: drafted rows each row reads."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    T, nq, hd = q.shape
    group = nq // k.shape[1]
    out = np.zeros_like(q)
    for t in range(T):
        rows = np.concatenate([np.arange(pos0), pos0 + np.flatnonzero(see[t])]).astype(int)
        if not len(rows):
            continue
        for h in range(nq):
            s = k[rows, h // group] @ q[t, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            out[t, h] = p @ v[rows, h // group] / p.sum()
    return out if gate is None else out / (1 + np.exp(-gate.astype(np.float64)))


def linear(mixed, a, b, hist, conv_w, a_log, dt, state, lk, lv, parents):
    """Per row: output, state and convolution window after it.  hist [conv_dim][ksize - 1]."""
    mixed, a, b, hist, conv_w, a_log, dt, state = (np.asarray(x, np.float64) for x in
                                                   (mixed, a, b, hist, conv_w, a_log, dt, state))
    _, dk, dv = state.shape
    outs, states, wins = [], [], []
    for i, par in enumerate(parents):
        win = np.concatenate([(wins[par][:, 1:] if par >= 0 else hist), mixed[i][:, None]], 1)
        y = (win * conv_w).sum(1)
        y = y / (1 + np.exp(-y))
        q, k = y[:lk * dk].reshape(lk, dk), y[lk * dk:2 * lk * dk].reshape(lk, dk)
        q, k = (np.repeat(z / np.sqrt((z * z).sum(1, keepdims=True) + 1e-6), lv // lk, 0) for z in (q, k))
        v = y[2 * lk * dk:].reshape(lv, dv)
        g = np.exp(-np.exp(a_log) * np.logaddexp(0, a[i] + dt))
        S = (states[par] if par >= 0 else state) * g[:, None, None]
        delta = (v - np.einsum("hi,hij->hj", k, S)) / (1 + np.exp(-b[i]))[:, None]
        S = S + k[:, :, None] * delta[:, None, :]
        outs.append(np.einsum("hi,hij->hj", q, S).ravel() / np.sqrt(dk))
        states.append(S)
        wins.append(win)
    return np.array(outs), states, wins


def verify(logits, parents, tokens, draft, inv_t, u_accept, u_sample):
    """(kept rows, new tokens)."""
    n, vocab = logits.shape
    logits = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    at, path, out = 0, [0], []
    while True:
        row, kids = logits[at], [j for j in range(1, n) if parents[j] == at]
        top = row.max()
        if top == -np.inf:
            return path, out + [-1]
        if inv_t == 0:
            best = int(row.argmax())
            nxt = next((j for j in kids if tokens[j] == best), None)
            if nxt is None:
                return path, out + [best]
        else:
            with np.errstate(invalid="ignore"):
                e = np.where(row == top, 1.0, np.exp((row - top) * inv_t))
            whole = p = e  # weights: their sum is the whole, so that equal ones stay exact
            q = None if draft is None else draft[at].astype(np.float64)
            nxt = None
            for j in kids:
                x = tokens[j]
                if p.sum() > 0 and 0 <= x < vocab and u_accept[j] * (1.0 if q is None else q[x]) < p[x] / p.sum():
                    nxt = j
                    break
                p = p.copy()
                if q is None:
                    if 0 <= x < vocab:
                        p[x] = 0
                elif p.sum() > 0:
                    p = np.maximum(p / p.sum() - q, 0)
            if nxt is None:
                if p.sum() == 0:
                    p = whole
                cum = np.cumsum(p)
                i = int(np.searchsorted(cum, u_sample * cum[-1], side="right"))
                return path, out + [i if i < vocab else int(np.flatnonzero(p)[-1])]
        path.append(nxt)
        out.append(int(tokens[nxt]))
        at = nxt
