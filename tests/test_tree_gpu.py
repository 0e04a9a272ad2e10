"""The operators of a decode step over a tree of drafted tokens against plain
64-bit results (tree_oracle), and a whole step of them together.

Bounds.  fp32 results of sums over n terms are off by at most n 2^-24 of the sum
of magnitudes; what each test allows is written beside it.
Attention: q and the weights carry 22 bits or more, so a score of |q||k| /
sqrt(hd) <= 16 is off by at most 16 x 2^-22 and a weight by 4e-6 of itself; the
output, a convex combination of |v| <= 6, by 3e-5."""
import ctypes
import math

import numpy as np
import pytest

import tree_oracle as to
import xqbind as xb

pytestmark = pytest.mark.gpu
EPS = 1e-6


_held = []  # a test's buffers, alive until it ends: calls take bare addresses


def dev(a):
    _held.append(xb.DeviceBuffer.from_array(np.ascontiguousarray(a)))
    return _held[-1]


@pytest.fixture(autouse=True)
def _release():
    yield
    xb.ck(xb.hip().xqhip_device_synchronize())
    _held.clear()


def i32(*v):
    return dev(np.array(v, np.int32))


class Cache:
    """A cache of either type; rows that no test writes hold NaN (fp16) or a NaN scale."""

    def __init__(self, kind, nkv, hd, cap, k=None, v=None):
        self.kind, self.shape, n = kind, (cap, nkv, hd), 0 if k is None else len(k)
        held = np.full((2, *self.shape), 99 if kind == xb.KV_I8 else np.nan, np.int8 if kind == xb.KV_I8 else np.float16)
        scales = np.full((2, cap, nkv), np.nan, np.float32)
        for i, x in enumerate((k, v)):
            if x is None:
                continue
            if kind == xb.KV_I8:
                held[i, :n], scales[i, :n] = to.quantise(x)
            else:
                held[i, :n] = x
        self.buf = [dev(held[0]), dev(held[1]), dev(scales[0]), dev(scales[1])]
        self.kv = xb.Kv(kind, nkv, hd, cap, *(b.ptr for b in self.buf))
        if kind == xb.KV_F16:
            self.kv.k_scale = self.kv.v_scale = None
        self.ref = ctypes.byref(self.kv)

    def raw(self):
        n, t = math.prod(self.shape), np.int8 if self.kind == xb.KV_I8 else np.float16
        out = [b.download(t, n).reshape(self.shape) for b in self.buf[:2]]
        return out + [b.download(np.float32, n // self.shape[2]).reshape(self.shape[:2]) for b in self.buf[2:]]

    def values(self):
        """k and v, as float64."""
        k, v, ks, vs = self.raw()
        if self.kind == xb.KV_F16:
            return k.astype(np.float64), v.astype(np.float64)
        return k * ks[..., None].astype(np.float64), v * vs[..., None].astype(np.float64)


def rope(rotary, cap):
    t = np.empty((cap, rotary // 2, 2), np.float32)
    xb.ck(xb.hip().xqhip_rope_table(1e4, rotary, cap, xb.ptr(t)))
    return t


# ---- the cache ------------------------------------------------------------------
def prep(rng, cache, nq, rotary, pos0, T, parents=None, gated=1, pad=0, x=None):
    """Runs xqhip_attn_prep_kv on [T][row] projections; returns (projections, q, gate, norms, rope)."""
    cap, nkv, hd = cache.shape
    wq = nq * hd * (2 if gated else 1)
    row = wq + 2 * nkv * hd + pad
    x = rng.normal(0, 1, (T, row)).astype(np.float32) if x is None else x
    qn, kn = (rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2))
    cs = rope(rotary, cap) if rotary else np.zeros((cap, 0, 2), np.float32)
    src, out = dev(x), nq * hd + 3
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    qo, go = dev(np.full((T, out), 7, np.float32)), dev(np.full((T, out), 7, np.float32))
    tree = ctypes.byref(xb.tree(parents)) if parents else None
    xb.ck(xb.hip().xqhip_attn_prep_kv(at(0), at(wq), at(wq + nkv * hd), gated, nq, rotary, dev(qn).ptr, dev(kn).ptr,
                                      EPS, dev(cs).ptr if rotary else None, i32(pos0).ptr, tree, T, row, out, qo.ptr,
                                      go.ptr if gated else None, cache.ref, None))
    q, g = (b.download(np.float32, T * out).reshape(T, out) for b in (qo, go))
    assert (q[:, nq * hd:] == 7).all() and (g[:, nq * hd:] == 7).all()
    return x, q[:, :nq * hd].reshape(T, nq, hd), g[:, :nq * hd].reshape(T, nq, hd), qn, kn, cs


@pytest.mark.parametrize("kind", [xb.KV_F16, xb.KV_I8])
@pytest.mark.parametrize("nq,nkv,hd,rotary,pos0,T,tree,gated,pad", [
    (32, 8, 128, 32, 0, 1, True, 1, 0), (32, 8, 128, 32, 300, 17, True, 1, 0), (16, 4, 256, 64, 5, 64, True, 1, 4),
    (16, 4, 256, 256, 9, 130, False, 1, 1), (4, 4, 64, 16, 0, 3, False, 0, 0), (6, 2, 80, 20, 2, 9, True, 1, 0),
    (2, 1, 1024, 0, 1, 2, False, 1, 0), (5, 5, 33, 32, 3, 5, True, 0, 3)])
def test_prep_writes_the_cache(kind, nq, nkv, hd, rotary, pos0, T, tree, gated, pad):
    """A normalised value: sum, square root, division, two products and the turn's two products and sum, 16 roundings of
    2^-24 on magnitudes up to sqrt(2) of the head's largest."""
    rng = np.random.default_rng(hd + T)
    cap = pos0 + T + 2
    cache = Cache(kind, nkv, hd, cap)
    before = cache.raw()
    par = to.random_tree(rng, T) if tree else None
    x, q, gate, qn, kn, cs = prep(rng, cache, nq, rotary, pos0, T, par, gated, pad)
    pos = pos0 + np.array(to.depths(par) if tree else np.arange(T))
    wq = nq * hd * (2 if gated else 1)
    qx = x[:, :wq].reshape(T, nq, -1)
    want = to.prepared(qx[..., :hd], qn, cs[pos][:, None], EPS)
    tol = 16 * 2**-24 * 1.5
    assert (np.abs(q - want) <= tol * np.abs(want).max(-1, keepdims=True)).all()
    if gated:
        assert np.array_equal(gate, qx[..., hd:])
    k = to.prepared(x[:, wq:wq + nkv * hd].reshape(T, nkv, hd), kn, cs[pos][:, None], EPS)
    v = x[:, wq + nkv * hd:wq + 2 * nkv * hd].reshape(T, nkv, hd)
    raw, at = cache.raw(), slice(pos0, pos0 + T)
    for i in range(4):  # rows outside the step are untouched
        keep = np.ones(cap, bool)
        keep[at] = False
        assert np.array_equal(raw[i][keep], before[i][keep], equal_nan=i > 1 or kind == xb.KV_F16)
    if kind == xb.KV_F16:
        assert np.array_equal(raw[1][at], v.astype(np.float16))
        assert (np.abs(raw[0][at] - k) <= 2**-11 * np.abs(k) + 2**-25 + tol * np.abs(k).max(-1, keepdims=True)).all()
        return
    codes, scales = to.quantise(v)
    assert np.array_equal(raw[1][at], codes) and np.array_equal(raw[3][at], scales)
    top = np.abs(k).max(-1, keepdims=True)
    assert (np.abs(raw[2][at][..., None] * 127.0 - top) <= (tol + 2**-23) * top).all()
    # half a step, and the value's own error (half a step is top / 254)
    assert (np.abs(cache.values()[0][at] - k) <= top / 254 + 2 * (tol + 2**-22) * top).all()


@pytest.mark.parametrize("hd", [128, 256, 80])
def test_prep_rows_of_extremes(hd):
    """Rows of zeros, of one value, of the smallest magnitudes, of fp32's largest and with values that are not finite."""
    rng = np.random.default_rng(1)
    rows = rng.normal(0, 1, (7, 1, hd)).astype(np.float32)
    rows[0] = 0
    rows[1] = 0
    rows[1, 0, 3] = -2.5
    rows[2] *= np.float32(1e-42)
    rows[3] *= np.float32(1e37)
    rows[4, 0, 5] = np.inf
    rows[5, 0, hd - 1] = np.nan
    cache = Cache(xb.KV_I8, 1, hd, 7)
    x = np.concatenate([rng.normal(0, 1, (7, 2 * hd)).astype(np.float32), rows[:, 0]], 1)
    prep(rng, cache, 1, 0, 0, 7, gated=0, x=x)
    k, v, ks, vs = cache.raw()
    codes, scales = to.quantise(rows)
    good = [0, 1, 2, 3, 6]
    assert np.array_equal(v[good], codes[good]) and np.array_equal(vs[good], scales[good])
    assert np.isnan(vs[[4, 5]]).all() and (v[[4, 5]] == 0).all()
    for t in (xb.F32, xb.F16):
        out = dev(np.zeros((7, hd), np.float32 if t == xb.F32 else np.float16))
        xb.ck(xb.hip().xqhip_kv_read(cache.ref, 0, 7, t, None, out.ptr, None))
        got = out.download(np.float32 if t == xb.F32 else np.float16, 7 * hd).reshape(7, hd)
        with np.errstate(over="ignore"):
            want = (codes[:, 0].astype(np.float32) * scales).astype(got.dtype)
        assert np.array_equal(got[good], want[good]) and np.isnan(got[[4, 5]]).all()


def test_prep_past_the_capacity_writes_nothing():
    rng = np.random.default_rng(3)
    cache = Cache(xb.KV_I8, 2, 128, 8)
    before = cache.raw()
    _, q, gate, *_ = prep(rng, cache, 4, 32, 6, 4, [-1, 0, 1, 0])
    raw = cache.raw()
    assert not np.array_equal(raw[0][6:], before[0][6:]) and np.array_equal(raw[0][:6], before[0][:6])
    assert np.isfinite(q[:2]).all() and np.isnan(q[2:]).all() and np.isfinite(gate).all()
    for pos0 in (-1, -2147483648, 2147483647, 8):
        cache = Cache(xb.KV_I8, 2, 128, 8)
        _, q, *_ = prep(rng, cache, 4, 32, pos0, 1)
        assert np.isnan(q).all() and all(np.array_equal(a, b, equal_nan=True) for a, b in zip(cache.raw(), before))


@pytest.mark.parametrize("t", [xb.F32, xb.F16])
@pytest.mark.parametrize("nkv,hd,first,count", [(8, 128, 0, 1), (4, 256, 3, 77), (1, 16, 0, 40), (3, 33, 1, 9),
                                               (8, 128, 100, 1000), (2, 72, 5, 301)])
def test_read_back(nkv, hd, first, count, t):
    rng = np.random.default_rng(count)
    cap = first + count + 3
    k, v = (rng.normal(0, 1, (cap, nkv, hd)) for _ in range(2))
    cache, dt = Cache(xb.KV_I8, nkv, hd, cap, k, v), np.float32 if t == xb.F32 else np.float16
    raw = cache.raw()
    n = count * nkv * hd
    outs = [dev(np.full(n + 8, 3, dt)) for _ in range(2)]
    xb.ck(xb.hip().xqhip_kv_read(cache.ref, first, count, t, outs[0].ptr, outs[1].ptr, None))
    for i in range(2):
        got = outs[i].download(dt, n + 8)
        want = raw[i][first:first + count].astype(np.float32) * raw[2 + i][first:first + count, :, None]
        assert np.array_equal(got[:n].reshape(want.shape), want.astype(dt)) and (got[n:] == 3).all()
    xb.ck(xb.hip().xqhip_kv_read(cache.ref, first, count, t, None, outs[0].ptr, None))  # v alone
    assert np.array_equal(outs[0].download(dt, n).reshape(want.shape), want.astype(dt))


@pytest.mark.parametrize("path,count", [([0], 1), ([0, 1, 2], 3), ([0, 2, 5, 9], 4), ([3, 4, 5, 6], 4),
                                        (list(range(0, 64, 2)), 32), ([0, 5, 9, 2, 7], 5), ([0, 4, 4, 8], 4),
                                        ([1, 3, 200, 5], 4), ([-1, 2], 2), ([0, 3, 6], 2), ([0, 3, 6], 0)])
def test_keep(path, count):
    """Buffers of several widths and alignments, one behind a position; paths that stop increasing, or leave the buffer,
    are followed up to there."""
    rng = np.random.default_rng(len(path))
    widths = [16, 32768, 12, 1, 4096 + 8, 65536]
    bufs = [rng.integers(0, 255, (70, w), dtype=np.uint8) for w in widths]
    firsts = [0, 6, 0, 6, 6, 0]
    d, pos = [dev(b) for b in bufs], i32(6)
    sets = xb.rows([(x.ptr, w, 70, pos.ptr if f else None) for x, w, f in zip(d, widths, firsts)])
    xb.ck(xb.hip().xqhip_tree_keep(sets, len(sets), i32(*path).ptr, i32(count).ptr, max(len(path), 1), None))
    for x, b, w, f in zip(d, bufs, widths, firsts):
        want, last = b.copy(), -1
        for j, at in enumerate(path[:count]):
            if at <= last or f + at >= 70:
                break
            want[f + j], last = b[f + at], at
        assert np.array_equal(x.download(np.uint8, b.size).reshape(b.shape), want)


def test_keep_of_many_buffers():
    rng = np.random.default_rng(2)
    bufs = [rng.integers(0, 255, (9, 48), dtype=np.uint8) for _ in range(131)]
    d = [dev(b) for b in bufs]
    sets = xb.rows([(x.ptr, 48, 9, None) for x in d])
    xb.ck(xb.hip().xqhip_tree_keep(sets, len(sets), i32(0, 4, 8).ptr, i32(3).ptr, 3, None))
    for x, b in zip(d, bufs):
        assert np.array_equal(x.download(np.uint8, b.size).reshape(b.shape)[:3], b[[0, 4, 8]])


# ---- attention ------------------------------------------------------------------
def attend(cache, q, gate, pos0, parents=None, masks=None, stream=None, pad=4, ws=None):
    T, nq, hd = q.shape
    cap, nkv, _ = cache.shape
    n, stride = nq * hd, nq * hd + pad
    row = lambda a: dev(np.concatenate([a.reshape(T, n), np.full((T, pad), np.nan, np.float32)], 1))  # noqa: E731
    out = dev(np.full((T, stride), 7.0, np.float32))
    tree = xb.tree(parents) if parents else None
    for i, m in enumerate(masks if masks is not None else []):
        tree.mask[i] = sum(1 << int(j) for j in np.flatnonzero(m))
    size = xb.hip().xqhip_tree_attention_workspace_bytes(nq, nkv, hd, T)
    ws = dev(np.full(size, 0xff, np.uint8))
    dq, dg, dp = row(q), row(gate) if gate is not None else None, i32(pos0)
    xb.ck(xb.hip().xqhip_tree_attention(dq.ptr, dg.ptr if dg else None, cache.ref, nq,
                                        ctypes.byref(tree) if tree else None, T, stride, dp.ptr, out.ptr, stride,
                                        ws.ptr, size, stream))
    if stream is not None:
        xb.ck(xb.hip().xqhip_stream_synchronize(stream))
    got = out.download(np.float32, T * stride).reshape(T, stride)
    assert (got[:, n:] == 7.0).all()
    return got[:, :n].reshape(q.shape)


def attention_case(rng, kind, nq, nkv, hd, T, pos0, spare=70):
    k, v = (rng.normal(0, 1, (pos0 + T, nkv, hd)) for _ in range(2))
    cache = Cache(kind, nkv, hd, pos0 + T + spare, k, v)
    q, gate = (rng.normal(0, 1, (T, nq, hd)).astype(np.float32) for _ in range(2))
    return cache, q, gate


KINDS = pytest.mark.parametrize("kind", [xb.KV_F16, xb.KV_I8])
SHAPES = pytest.mark.parametrize("nq,nkv,hd,T,pos0", [
    (32, 8, 128, 1, 0), (32, 8, 128, 1, 1), (32, 8, 128, 1, 31), (32, 8, 128, 2, 63), (32, 8, 128, 5, 64),
    (32, 8, 128, 8, 540), (32, 8, 128, 21, 127), (32, 8, 128, 64, 1000), (32, 8, 128, 64, 0), (32, 8, 128, 33, 4099),
    (16, 4, 256, 1, 700), (16, 4, 256, 7, 33), (16, 4, 256, 64, 515), (8, 8, 128, 9, 100), (16, 2, 128, 40, 65),
    (14, 2, 128, 11, 300), (3, 1, 128, 64, 31), (10, 2, 256, 13, 255), (4, 2, 64, 6, 200), (6, 2, 80, 17, 90),
    (8, 1, 33, 3, 5)])


@KINDS
@SHAPES
def test_tree_attention(kind, nq, nkv, hd, T, pos0):
    rng = np.random.default_rng(T * 7 + pos0 + hd)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    par = to.random_tree(rng, T)
    k, v = cache.values()
    want = to.attention(q, gate, k, v, pos0, to.path_masks(par))
    got = attend(cache, q, gate, pos0, par)
    assert np.abs(got - want).max() <= 3e-5, np.abs(got - want).max()
    assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T,pos0", [(16, 2, 990, 5, 70), (14, 2, 1024, 3, 64), (2, 2, 1024, 9, 63), (3, 1, 1, 6, 65)])
def test_attention_of_the_largest_and_smallest_heads(kind, nq, nkv, hd, T, pos0):
    """A score, an fp32 sum of up to 1024 terms, is off by 1024 2^-24 sum |q_i k_i| / sqrt(hd) <= 1024 2^-24 0.64 sqrt(1024) =
    1.3e-3 at most, and an output, an average of |v| <= 6, by 2 x 6 times that.  Roundings of either sign add up to sqrt(1024)
    2^-24 of partial sums of sqrt(1024), 2e-6 of a score; for the norm ten times that is allowed."""
    rng = np.random.default_rng(hd + T)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    par = to.random_tree(rng, T)
    k, v = cache.values()
    want = to.attention(q, gate, k, v, pos0, to.path_masks(par))
    got = attend(cache, q, gate, pos0, par)
    assert np.abs(got - want).max() <= 1.6e-2 and np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T,pos0", [(32, 8, 128, 1, 5), (32, 8, 128, 3, 40), (32, 8, 128, 8, 300), (16, 4, 256, 2, 31),
                                              (32, 8, 128, 65, 0), (32, 8, 128, 130, 70),
                                              (32, 8, 128, 1030, 21), (16, 4, 256, 100, 3), (16, 4, 256, 300, 513), (6, 3, 64, 70, 9)])
def test_chunk_attention(kind, nq, nkv, hd, T, pos0):
    rng = np.random.default_rng(T + pos0)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    k, v = cache.values()
    want = to.attention(q, gate, k, v, pos0, np.tril(np.ones((T, T), bool)))
    got = attend(cache, q, gate, pos0)
    assert np.abs(got - want).max() <= 3e-5, np.abs(got - want).max()


@KINDS
@pytest.mark.parametrize("hd", [128, 256, 64])
@pytest.mark.parametrize("pos0", [0, 37])
def test_masks_of_the_callers_own(kind, hd, pos0):
    """Masks that leave a row nothing (0, or the context alone), skip the row itself, or reach later rows."""
    rng = np.random.default_rng(hd + pos0)
    T, nq, nkv = 24, 8, 2
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    see = rng.random((T, T)) < 0.3
    see[[0, 5, 23]] = False
    k, v = cache.values()
    got = attend(cache, q, gate, pos0, [-1] * T, see)
    want = to.attention(q, gate, k, v, pos0, see)
    assert np.abs(got - want).max() <= 3e-5
    if pos0 == 0:
        assert (got[[0, 5, 23]] == 0).all()


@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (8, 2, 256), (4, 2, 64)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@KINDS
def test_what_a_row_does_not_see_never_reaches_it(kind, nq, nkv, hd, what):
    """One drafted row's key and value are not finite: rows that read it have outputs that are not, the others are as
    without it."""
    rng = np.random.default_rng(7)
    T, pos0, bad = 20, 45, 6
    k, v = (rng.normal(0, 1, (pos0 + T, nkv, hd)) for _ in range(2))
    q, gate = (rng.normal(0, 1, (T, nq, hd)).astype(np.float32) for _ in range(2))
    par = to.random_tree(rng, T, 9)
    see = to.path_masks(par)
    clean = Cache(kind, nkv, hd, pos0 + T, k, v)
    want = to.attention(q, gate, *clean.values(), pos0, see)
    k[pos0 + bad, :, 3], v[pos0 + bad, :, 5] = what, what
    cache = Cache(kind, nkv, hd, pos0 + T, k, v)
    if kind == xb.KV_I8:  # as the cache's own write leaves such rows
        raw = cache.raw()
        for i in (0, 1):
            raw[i][pos0 + bad], raw[2 + i][pos0 + bad] = 0, np.nan
            cache.buf[i].upload(raw[i])
            cache.buf[2 + i].upload(raw[2 + i])
    got = attend(cache, q, gate, pos0, par)
    hit = see[:, bad]
    assert hit.any() and not hit.all()
    assert np.abs(got[~hit] - want[~hit]).max() <= 3e-5
    if kind == xb.KV_I8 or np.isnan(what):
        assert np.isnan(got[hit]).any(axis=-1).all()


@KINDS
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 60.0, 3e4])
def test_scores_of_every_size(kind, hd, scale):
    """q from tiny to so large that one key takes all the weight.  A score s is off by 2^-22 of |q||k| / sqrt(hd), so
    for large ones the outputs of near-tied keys are not determined to 3e-5: the bound grows with the score."""
    rng = np.random.default_rng(hd)
    nq, nkv, T, pos0 = 8, 2, 10, 333
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    q = (q * np.float32(scale)).astype(np.float32)
    par = to.random_tree(rng, T)
    k, v = cache.values()
    want = to.attention(q, gate, k, v, pos0, to.path_masks(par))
    got = attend(cache, q, gate, pos0, par)
    reach = np.abs(q).max() * math.sqrt(hd) * 4.5  # |q||k| / sqrt(hd) <= max|q| |k|
    assert np.abs(got - want).max() <= 3e-5 + min(12.0, 12 * reach * 2**-21 if scale > 1 else 0.0)
    if scale > 1000:  # the outputs are single values of v
        assert np.abs(got - want).max() <= 1e-3 or (np.abs(got - want).max(-1) <= 1e-3).mean() > 0.9


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T", [(8, 2, 128, 3), (8, 2, 128, 10), (8, 2, 256, 10), (8, 2, 128, 40), (4, 2, 64, 10)])
@pytest.mark.parametrize("scale", [1e3, 3e4])
def test_scores_that_single_out_a_key(kind, nq, nkv, hd, T, scale):
    """Every output of scores so large that a row's best key takes all its weight.  A score is off by E = (hd 2^-24 sum
    |q_i k_i| + 2^-23 max|q| sum |k_i|) / sqrt(hd) at most (an fp32 sum of hd terms, q's 22 bits).  Where the best
    leads by 2 E + 20 the others have 400 e^-20 = 1e-6 of the weight between them and the output is the best key's
    value; elsewhere it lies between the values of the keys that are as near."""
    rng = np.random.default_rng(hd + T)
    pos0 = 333
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    q = (q * np.float32(scale)).astype(np.float32)
    par = to.random_tree(rng, T)
    see = to.path_masks(par)
    k, v = cache.values()
    got = attend(cache, q, gate, pos0, par) * (1 + np.exp(-gate.astype(np.float64)))
    alone = 0
    for t in range(T):
        rows = np.concatenate([np.arange(pos0), pos0 + np.flatnonzero(see[t])])
        for h in range(nq):
            kh, qh = k[rows, h // (nq // nkv)], q[t, h].astype(np.float64)
            vh, s = v[rows, h // (nq // nkv)], kh @ qh / math.sqrt(hd)
            off = (hd * 2**-24 * (np.abs(kh) @ np.abs(qh)).max() + 2**-23 * np.abs(qh).max() * np.abs(kh).sum(1).max()) / math.sqrt(hd)
            near = vh[s >= s.max() - 2 * off - 20]
            alone += len(near) == 1
            tol = 3e-5 * (1 + np.exp(-gate[t, h].astype(np.float64)))
            assert (got[t, h] >= near.min(0) - tol).all() and (got[t, h] <= near.max(0) + tol).all(), (t, h)
    assert alone >= 0.7 * T * nq


@KINDS
def test_attention_without_a_gate_and_unaligned_rows(kind):
    rng = np.random.default_rng(11)
    cache, q, _ = attention_case(rng, kind, 8, 2, 128, 6, 77)
    par = to.random_tree(rng, 6)
    k, v = cache.values()
    want = to.attention(q, None, k, v, 77, to.path_masks(par))
    for pad in (0, 1, 3, 4):
        assert np.abs(attend(cache, q, None, 77, par, pad=pad) - want).max() <= 3e-5


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T,pos0", [
    (8, 8, 128, 16, 20000), (8, 8, 128, 20, 20001), (8, 8, 128, 40, 20031), (4, 4, 256, 3, 20000), (4, 4, 256, 17, 19999),
    (4, 4, 256, 64, 9000), (8, 1, 128, 2, 70000)])
def test_attention_of_several_chunks_per_wave(kind, nq, nkv, hd, T, pos0):
    """Every wave of a split takes several tiles: the loads ahead, the moves of the running maximum."""
    rng = np.random.default_rng(T + hd)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0, spare=3)
    par = to.random_tree(rng, T)
    k, v = cache.values()
    want = to.attention(q, gate, k, v, pos0, to.path_masks(par))
    got = attend(cache, q, gate, pos0, par)
    assert np.abs(got - want).max() <= 3e-5, np.abs(got - want).max()
    assert np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)


@KINDS
@pytest.mark.parametrize("nq,nkv,T,pos0,tree", [(8, 2, 64, 3000, True), (8, 2, 33, 4097, True), (16, 2, 16, 900, True),
                                                (2, 2, 130, 50, False), (32, 8, 600, 65, False), (3, 1, 50, 6000, True)])
def test_attention_over_a_cache_that_can_get_long(kind, nq, nkv, T, pos0, tree):
    """Caches of 40000 positions; the last of the rows' values infinite in one dim, for those that see it."""
    rng = np.random.default_rng(T + pos0)
    k, v = (rng.normal(0, 1, (pos0 + T, nkv, 128)) for _ in range(2))
    q, gate = (rng.normal(0, 1, (T, nq, 128)).astype(np.float32) for _ in range(2))
    par = to.random_tree(rng, T) if tree else None
    see = to.path_masks(par) if tree else np.tril(np.ones((T, T), bool))
    cache = Cache(kind, nkv, 128, 40000, k, v)
    want = to.attention(q, gate, *(x[:pos0 + T] for x in cache.values()), pos0, see)
    assert np.abs(attend(cache, q, gate, pos0, par) - want).max() <= 3e-5
    if kind == xb.KV_F16:
        v[pos0 + T - 1, :, 9] = np.inf
        got = attend(Cache(kind, nkv, 128, 40000, k, v), q, gate, pos0, par)
        assert np.abs(got[:-1] - want[:-1]).max() <= 3e-5 and not np.isfinite(got[-1, :, 9]).any()


@KINDS
@pytest.mark.parametrize("hd,nkv,edge", [(128, 8, 256), (256, 4, 128)])
@pytest.mark.parametrize("T", [1, 4, 6])
def test_attention_around_a_split_of_its_own(kind, hd, nkv, edge, T):
    """The lengths at which a call's keys go from one split to several, and their neighbours."""
    rng = np.random.default_rng(edge + T)
    for n in (edge - 1, edge, edge + 1, edge + 31, edge + 32, edge + 33, 2 * edge + 1):
        cache, q, gate = attention_case(rng, kind, 4 * nkv, nkv, hd, T, n - T, spare=0)
        par = to.random_tree(rng, T)
        want = to.attention(q, gate, *cache.values(), n - T, to.path_masks(par))
        assert np.abs(attend(cache, q, gate, n - T, par) - want).max() <= 3e-5, n


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T,pos0,tree", [
    (64, 64, 128, 5, 200, True), (128, 64, 128, 3, 500, True), (96, 32, 128, 9, 333, True), (300, 300, 128, 2, 70, True),
    (40, 40, 256, 7, 150, True), (64, 64, 128, 40, 90, True), (128, 128, 256, 20, 50, True), (64, 64, 128, 150, 40, False)])
def test_attention_of_many_heads(kind, nq, nkv, hd, T, pos0, tree):
    """So many kv heads that few splits, or one, are left to each."""
    rng = np.random.default_rng(nq + T)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0, spare=0)
    par = to.random_tree(rng, T) if tree else None
    see = to.path_masks(par) if tree else np.tril(np.ones((T, T), bool))
    want = to.attention(q, gate, *cache.values(), pos0, see)
    got = attend(cache, q, gate, pos0, par)
    assert np.abs(got - want).max() <= 3e-5 and np.linalg.norm(got - want) <= 5e-6 * np.linalg.norm(want)


@KINDS
@pytest.mark.parametrize("off", [2, 4, 8, 12])
@pytest.mark.parametrize("hd,T", [(128, 2), (128, 7), (128, 30), (256, 3), (256, 30)])
def test_caches_at_any_address(kind, off, hd, T):
    """Caches that begin `off` bytes behind a 16-byte border: attention, the write, the read-back."""
    rng = np.random.default_rng(off + T)
    nq, nkv, pos0, rotary = 8, 2, 100, 32
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0, spare=T)
    par = to.random_tree(rng, T)
    want = to.attention(q, gate, *cache.values(), pos0, to.path_masks(par))
    size = 1 if kind == xb.KV_I8 else 2
    raw = cache.raw()

    class Moved(Cache):
        def __init__(self):
            self.kind, self.shape = kind, cache.shape
            held = [np.concatenate([np.zeros(off, np.uint8), x.view(np.uint8).ravel()]) for x in raw[:2]]
            self.buf = [dev(held[0]), dev(held[1]), dev(raw[2]), dev(raw[3])]
            self.kv = xb.Kv(kind, nkv, hd, cache.shape[0], *(ctypes.c_void_p(b.ptr.value + off) for b in self.buf[:2]),
                            *(b.ptr if kind == xb.KV_I8 else None for b in self.buf[2:]))
            self.ref = ctypes.byref(self.kv)

        def codes(self, i):
            b = self.buf[i].download(np.uint8, self.buf[i].nbytes)[off:]
            return b.view(np.int8 if size == 1 else np.float16).reshape(self.shape)

    moved = Moved()
    assert np.abs(attend(moved, q, gate, pos0, par) - want).max() <= 3e-5
    x = rng.normal(0, 1, (T, 2 * nq * hd + 2 * nkv * hd)).astype(np.float32)
    prep(np.random.default_rng(1), cache, nq, rotary, pos0 + T, T, par, x=x)
    prep(np.random.default_rng(1), moved, nq, rotary, pos0 + T, T, par, x=x)
    raw = cache.raw()
    for i in (0, 1):
        assert np.array_equal(moved.codes(i), raw[i])
    if kind == xb.KV_I8:
        n = 2 * T * nkv * hd
        for t, dt in ((xb.F32, np.float32), (xb.F16, np.float16)):
            outs = [dev(np.zeros(n, dt)) for _ in range(2)]
            xb.ck(xb.hip().xqhip_kv_read(cache.ref, pos0, 2 * T, t, None, outs[0].ptr, None))
            xb.ck(xb.hip().xqhip_kv_read(moved.ref, pos0, 2 * T, t, None, outs[1].ptr, None))
            a, b = (o.download(dt, n) for o in outs)
            assert a.any() and np.array_equal(a, b)


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T,pos0", [(8, 2, 128, 4, 0), (8, 2, 128, 4, 900), (8, 2, 128, 30, 900), (8, 2, 128, 130, 5),
                                              (8, 2, 256, 6, 300), (4, 2, 64, 6, 50)])
def test_rows_that_are_not_numbers_stay_alone(kind, nq, nkv, hd, T, pos0):
    """NaN in one row's q, and in one gate of another row: the other outputs are those without them."""
    rng = np.random.default_rng(T + hd)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    want = to.attention(q, gate, *cache.values(), pos0, np.tril(np.ones((T, T), bool)))
    q[1, 3, 7] = np.nan
    gate[2, 1, 5] = np.nan
    got = attend(cache, q, gate, pos0)
    clean = np.ones(want.shape, bool)
    clean[1, 3], clean[2, 1, 5] = False, False
    assert np.isnan(got[~clean]).all() and np.abs(got - want)[clean].max() <= 3e-5


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T", [(8, 2, 128, 3), (8, 2, 128, 40), (8, 2, 256, 20), (4, 2, 64, 9)])
def test_chunk_past_the_capacity(kind, nq, nkv, hd, T):
    """A prompt chunk that the cache cannot hold: its rows see the slots that are there."""
    rng = np.random.default_rng(T)
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, 50, spare=0)
    k, v = cache.values()
    for pos0 in (50 + T // 2, 50 + T - 1, 50 + T, 50 + T + 9):
        held = max(0, 50 + T - pos0)
        see = np.tril(np.ones((T, T), bool))
        see[:, held:] = False
        want = to.attention(q, gate, k, v, min(pos0, 50 + T), see)
        assert np.abs(attend(cache, q, gate, pos0) - want).max() <= 3e-5


@pytest.mark.parametrize("T", [1000, 5000])
def test_attention_of_a_long_chunk(T):
    """Many row tiles, so that few splits are left, and a row of infinities in the middle of them."""
    rng = np.random.default_rng(T)
    nq, nkv, hd = 1, 1, 128
    k, v = (rng.normal(0, 1, (T, nkv, hd)) for _ in range(2))
    q, gate = (rng.normal(0, 1, (T, nq, hd)).astype(np.float32) for _ in range(2))
    see = np.tril(np.ones((T, T), bool))
    clean = Cache(xb.KV_F16, nkv, hd, T, k, v)
    want = to.attention(q, gate, *clean.values(), 0, see)
    assert np.abs(attend(clean, q, gate, 0) - want).max() <= 3e-5
    bad = T - 30
    v[bad, :, 7] = np.inf
    got = attend(Cache(xb.KV_F16, nkv, hd, T, k, v), q, gate, 0)
    assert np.abs(got[:bad] - want[:bad]).max() <= 3e-5 and not np.isfinite(got[bad:, 0, 7]).any()
    others = np.arange(hd) != 7
    assert np.abs(got[bad:][..., others] - want[bad:][..., others]).max() <= 3e-5


@KINDS
@pytest.mark.parametrize("nq,nkv,hd,T", [(8, 2, 128, 3), (8, 2, 128, 8), (8, 2, 128, 20), (8, 2, 256, 4), (8, 2, 256, 8),
                                         (8, 2, 256, 30)])
def test_values_of_every_size(kind, nq, nkv, hd, T):
    """A value row that is far larger than the others, in a row that is not seen and under a weight so small that it
    adds as much as they do.  A weight and its value's scale together are off by 2^-22 of the largest such product, so
    the bound is that of ordinary values for each of the two parts; and values that are all tiny."""
    rng = np.random.default_rng(T + hd)
    pos0, far = 100, 2.0**(15 if kind == xb.KV_F16 else 20)
    k, v = (rng.normal(0, 1, (pos0 + T, nkv, hd)) for _ in range(2))
    q, gate = (rng.normal(0, 1, (T, nq, hd)).astype(np.float32) for _ in range(2))
    q[..., 0] = 8
    weight = 4 - math.log(far)  # the key's score
    k[41], k[41, :, 0] = 0, weight * math.sqrt(hd) / 8
    v[41] *= far / 6
    par = [-1] + [0] * (T - 1)  # siblings: row 1's values do not reach the others
    v[pos0 + 1] *= (1 if kind == xb.KV_F16 else 2.0**30) * far / 6
    see = to.path_masks(par)
    cache = Cache(kind, nkv, hd, pos0 + T, k, v)
    ck, cv = cache.values()
    want = to.attention(q, gate, ck, cv, pos0, see)
    plain = cv.copy()
    plain[41] = 0
    other = np.arange(T) != 1
    part = np.abs(want - to.attention(q, gate, ck, plain, pos0, see))[other].max()
    got = attend(cache, q, gate, pos0, par)
    assert part > 0.01 and np.abs(got - want)[other].max() <= 3e-5 * (1 + part)
    reach = np.abs(want[1]).max()
    assert np.abs(got - want)[1].max() <= 3e-5 * reach
    if kind == xb.KV_I8:
        tiny = Cache(kind, nkv, hd, pos0 + T, k, rng.normal(0, 1, v.shape) * 2.0**-80)
        want = to.attention(q, gate, *tiny.values(), pos0, see)
        assert np.abs(attend(tiny, q, gate, pos0, par) - want).max() <= 3e-5 * 2.0**-80


@KINDS
def test_attention_past_the_capacity(kind):
    """Slots past the cache's end are not read: the rows see what lies before it."""
    rng = np.random.default_rng(12)
    nq, nkv, hd, T = 8, 2, 128, 12
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, 40, spare=0)
    k, v = cache.values()
    par = to.random_tree(rng, T)
    see = to.path_masks(par)
    see[:, 52 - 46:] = False
    want = to.attention(q, gate, k, v, 46, see)
    assert np.abs(attend(cache, q, gate, 46, par) - want).max() <= 3e-5
    everything = to.attention(q, gate, k, v, 52, np.zeros((T, T), bool))
    for pos0 in (52, 53, 2147483647):
        assert np.abs(attend(cache, q, gate, pos0, par) - everything).max() <= 3e-5
    see = to.path_masks(par)  # a position below zero counts as zero
    assert np.abs(attend(cache, q, gate, -5, par) - to.attention(q, gate, k, v, 0, see)).max() <= 3e-5


def test_attention_offsets_past_32_bits():
    """A cache of 2^20 positions, 4.3 GB a side: the last rows of it, and a step behind them."""
    L, nq, nkv, hd, cap, T = xb.hip(), 8, 8, 256, 1 << 20, 3
    rng = np.random.default_rng(13)
    bufs = [xb.DeviceBuffer(cap * nkv * hd * 2) for _ in range(2)]
    for b in bufs:
        b.zero()
    tail = 40
    k, v = (rng.normal(0, 1, (tail + T, nkv, hd)).astype(np.float16) for _ in range(2))
    first = cap - tail - T
    for b, x in zip(bufs, (k, v)):
        at = ctypes.c_void_p(b.ptr.value + first * nkv * hd * 2)
        xb.ck(L.xqhip_memcpy_h2d(at, xb.ptr(x), x.nbytes, None))
    cache = xb.Kv(xb.KV_F16, nkv, hd, cap, bufs[0].ptr, bufs[1].ptr, None, None)
    q = (rng.normal(0, 1, (T, nq, hd)) * 8).astype(np.float32)
    size = L.xqhip_tree_attention_workspace_bytes(nq, nkv, hd, T)
    ws, out, par = xb.DeviceBuffer(size), xb.DeviceBuffer(q.nbytes), [-1, 0, 0]
    xb.ck(L.xqhip_tree_attention(dev(q).ptr, None, ctypes.byref(cache), nq, ctypes.byref(xb.tree(par)), T, nq * hd,
                                 i32(cap - T).ptr, out.ptr, nq * hd, ws.ptr, size, None))
    got = out.download(np.float32, q.size).reshape(q.shape).astype(np.float64)
    see = to.path_masks(par)
    for t in range(T):
        rows = np.concatenate([np.arange(tail), tail + np.flatnonzero(see[t])])
        for h in range(nq):
            s = k[rows, h].astype(np.float64) @ q[t, h] / math.sqrt(hd)
            m = max(s.max(), 0.0)
            p = np.exp(s - m)
            want = p @ v[rows, h].astype(np.float64) / (p.sum() + first * math.exp(-m))  # the zero keys before them
            assert np.abs(got[t, h] - want).max() <= 1e-4  # scores up to 8 times those of the other tests
    for b in bufs:
        b.free()


def test_cache_offsets_past_32_bits():
    """The last rows of an 8-bit cache of 5.4 GB a side: written, read back, moved together."""
    L, nq, nkv, hd, cap = xb.hip(), 20, 20, 256, 1 << 20
    rng = np.random.default_rng(15)
    bufs = [xb.DeviceBuffer(cap * nkv * hd) for _ in range(2)] + [xb.DeviceBuffer(cap * nkv * 4) for _ in range(2)]
    kv = xb.Kv(xb.KV_I8, nkv, hd, cap, *(b.ptr for b in bufs))
    x = rng.normal(0, 1, (3, (nq + 2 * nkv) * hd)).astype(np.float32)
    src, q, norm = dev(x), xb.DeviceBuffer(3 * nq * hd * 4), dev(np.ones(hd, np.float32))
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    pos = i32(cap - 3)
    xb.ck(L.xqhip_attn_prep_kv(at(0), at(nq * hd), at((nq + nkv) * hd), 0, nq, 0, norm.ptr, norm.ptr, EPS, None, pos.ptr,
                               ctypes.byref(xb.tree([-1, 0, 0])), 3, x.shape[1], nq * hd, q.ptr, None, ctypes.byref(kv), None))
    codes, scales = to.quantise(x[:, (nq + nkv) * hd:].reshape(3, nkv, hd))
    want = codes.astype(np.float32) * scales[..., None]

    def back():
        out = dev(np.zeros((3, nkv, hd), np.float32))
        xb.ck(L.xqhip_kv_read(ctypes.byref(kv), cap - 3, 3, xb.F32, None, out.ptr, None))
        return out.download(np.float32, want.size).reshape(want.shape)

    assert np.array_equal(back(), want)
    sets = xb.rows([(b.ptr, w, cap, pos.ptr) for b, w in zip(bufs, (nkv * hd, nkv * hd, nkv * 4, nkv * 4))])
    xb.ck(L.xqhip_tree_keep(sets, 4, i32(0, 2).ptr, i32(2).ptr, 2, None))
    assert np.array_equal(back(), want[[0, 2, 2]])
    for b in bufs:
        b.free()


@KINDS
def test_attention_on_two_streams_at_once(kind):
    """Calls in flight together, each with its own workspace: the outputs of calls one after the other."""
    L, rng = xb.hip(), np.random.default_rng(16)
    nq, nkv, hd, n = 32, 8, 128, 32 * 128
    cases = []
    for T, pos0 in ((1, 9000), (64, 5000)):
        cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
        par = to.random_tree(rng, T)
        want = attend(cache, q, gate, pos0, par, pad=0)
        size, s = L.xqhip_tree_attention_workspace_bytes(nq, nkv, hd, T), ctypes.c_void_p()
        xb.ck(L.xqhip_stream_create(ctypes.byref(s)))
        cases.append((cache, dev(q), dev(gate), xb.tree(par), T, i32(pos0), dev(np.zeros((T, n), np.float32)), dev(np.zeros(size, np.uint8)),
                      size, s, want))
    xb.ck(L.xqhip_device_synchronize())
    for _ in range(20):
        for cache, q, gate, tree, T, pos, out, ws, size, s, _want in cases:
            xb.ck(L.xqhip_tree_attention(q.ptr, gate.ptr, cache.ref, nq, ctypes.byref(tree), T, n, pos.ptr, out.ptr, n, ws.ptr, size, s))
    for _cache, _q, _gate, _tree, T, _pos, out, _ws, _size, s, want in cases:
        xb.ck(L.xqhip_stream_synchronize(s))
        assert np.array_equal(out.download(np.float32, T * n).reshape(want.shape), want)
        xb.ck(L.xqhip_stream_destroy(s))


@KINDS
def test_attention_on_another_stream_and_in_a_graph(kind):
    L = xb.hip()
    rng = np.random.default_rng(14)
    nq, nkv, hd, T, pos0 = 32, 8, 128, 9, 700
    cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
    par = to.random_tree(rng, T)
    tree = xb.tree(par)
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    xb.ck(L.xqhip_stream_create(ctypes.byref(s)))
    eager = attend(cache, q, gate, pos0, par, stream=s)
    n = nq * hd
    size = L.xqhip_tree_attention_workspace_bytes(nq, nkv, hd, T)
    ws, out, pos = xb.DeviceBuffer(size), xb.DeviceBuffer(T * n * 4), i32(pos0)
    dq, dg = dev(q), dev(gate)
    xb.ck(L.xqhip_graph_begin(s))
    xb.ck(L.xqhip_tree_attention(dq.ptr, dg.ptr, cache.ref, nq, ctypes.byref(tree), T, n, pos.ptr, out.ptr, n, ws.ptr,
                                 size, s))
    xb.ck(L.xqhip_graph_end(s, ctypes.byref(g)))
    for i in (0, 1, 1, 2):  # the position moves between replays
        pos.upload(np.array([pos0 - 100 * i], np.int32))
        out.zero()
        xb.ck(L.xqhip_device_synchronize())
        xb.ck(L.xqhip_graph_launch(g, s))
        xb.ck(L.xqhip_stream_synchronize(s))
        got = out.download(np.float32, T * n).reshape(q.shape)
        assert np.array_equal(got, eager if i == 0 else attend(cache, q, gate, pos0 - 100 * i, par))
    xb.ck(L.xqhip_graph_destroy(g))
    xb.ck(L.xqhip_stream_destroy(s))


# ---- linear attention -----------------------------------------------------------
def linear_case(rng, lk, dk, lv, dv, ks, n):
    cd = 2 * lk * dk + lv * dv
    return dict(mixed=rng.normal(0, 1, (n, cd)), a=rng.normal(0, 1, (n, lv)), b=rng.normal(0, 1, (n, lv)),
                hist=rng.normal(0, 1, (2, cd, ks - 1)), w=rng.normal(0, 0.3, (cd, ks)), a_log=rng.normal(0, 0.5, lv),
                dt=rng.normal(0, 0.5, lv), S=rng.normal(0, 0.1, (lv, dk, dv)))


def run_linear(c, lk, dk, lv, dv, ks, pos0, par, stream=None):
    c = {m: np.ascontiguousarray(x, np.float32) for m, x in c.items()}
    n, cd = c["mixed"].shape
    row, out_row = cd + 2 * lv + 5, lv * dv + 3
    x = np.full((n, row), np.nan, np.float32)
    x[:, :cd], x[:, cd:cd + lv], x[:, cd + lv:cd + 2 * lv] = c["mixed"], c["a"], c["b"]
    src, hist, S, out = dev(x), dev(c["hist"]), dev(c["S"]), dev(np.full((n, out_row), 7, np.float32))
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    size = xb.hip().xqhip_linear_attn_tree_workspace_bytes(n, lk, dk, lv, dv)
    ws, keep = dev(np.full(max(size, 16), 0xff, np.uint8)), [dev(c[m]) for m in ("w", "a_log", "dt")]
    xb.ck(xb.hip().xqhip_linear_attn_tree(at(0), at(cd), at(cd + lv), row, hist.ptr, i32(pos0).ptr, keep[0].ptr,
                                          keep[1].ptr, keep[2].ptr, S.ptr, lk, dk, lv, dv, ks,
                                          ctypes.byref(xb.tree(par)), out.ptr, out_row, ws.ptr, size, stream))
    got = out.download(np.float32, n * out_row).reshape(n, out_row)
    assert (got[:, lv * dv:] == 7).all()
    assert np.array_equal(S.download(np.float32, c["S"].size).reshape(c["S"].shape), c["S"])  # read only
    assert np.array_equal(hist.download(np.float32, c["hist"].size).reshape(c["hist"].shape), c["hist"])
    return got[:, :lv * dv], c


@pytest.mark.parametrize("lk,dk,lv,dv,ks,n,pos0", [
    (16, 128, 32, 128, 4, 1, 0), (16, 128, 32, 128, 4, 6, 541), (16, 128, 32, 128, 4, 64, 8), (8, 128, 16, 128, 4, 33, 3),
    (2, 128, 2, 128, 4, 16, 1), (2, 128, 6, 128, 4, 17, 0), (1, 64, 2, 64, 4, 40, 5), (2, 256, 4, 256, 4, 64, 2),
    (2, 48, 2, 80, 3, 9, 1), (1, 16, 3, 7, 1, 5, 0), (2, 128, 4, 128, 2, 10, 1), (1, 32, 1, 96, 8, 20, 3)])
@pytest.mark.parametrize("shape", ["tree", "chain", "star", "roots"])
def test_linear_tree(lk, dk, lv, dv, ks, n, pos0, shape):
    """Products over dk terms of unit keys with state columns of norm 0.1 sqrt(dk) are off by dk 2^-24 of that at most
    (1e-5 at 128 and 256 dims), each row's update adds another, damped by its beta and decay, and the outputs are
    divided by sqrt(dk): 2e-5."""
    rng = np.random.default_rng(n + dk + pos0)
    par = {"tree": to.random_tree(rng, n), "chain": list(range(-1, n - 1)), "star": [-1] + [0] * (n - 1),
           "roots": [-1] * n}[shape]
    got, c = run_linear(linear_case(rng, lk, dk, lv, dv, ks, n), lk, dk, lv, dv, ks, pos0, par)
    want, _, _ = to.linear(c["mixed"], c["a"], c["b"], c["hist"][pos0 & 1], c["w"], c["a_log"], c["dt"], c["S"], lk, lv,
                           par)
    assert np.abs(got - want).max() <= 2e-5, np.abs(got - want).max()
    assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


def test_linear_decays_of_every_size():
    """Gates from none to a complete reset in the middle of a path, and of a whole path."""
    rng = np.random.default_rng(3)
    lk, dk, lv, dv, ks, n = 2, 128, 4, 128, 4, 40
    c = linear_case(rng, lk, dk, lv, dv, ks, n)
    c["a"][:, 0] = -100.0  # no decay
    c["a"][::7, 1] = 1e6   # resets
    c["a"][:, 2] = 1e30    # always
    c["a"][5, 3] = np.inf
    par = list(range(-1, n - 1))
    got, c = run_linear(c, lk, dk, lv, dv, ks, 0, par)
    with np.errstate(over="ignore"):
        want, _, _ = to.linear(c["mixed"], c["a"], c["b"], c["hist"][0], c["w"], c["a_log"], c["dt"], c["S"], lk, lv, par)
    assert np.isfinite(want).all() and np.abs(got - want).max() <= 2e-5


def test_linear_rows_that_are_not_finite_stay_on_their_paths():
    rng = np.random.default_rng(4)
    lk, dk, lv, dv, ks, n = 2, 128, 4, 128, 4, 30
    c = linear_case(rng, lk, dk, lv, dv, ks, n)
    par = to.random_tree(rng, n, 12)
    clean, _ = run_linear(c, lk, dk, lv, dv, ks, 1, par)
    c["mixed"][9] = np.nan
    got, _ = run_linear(c, lk, dk, lv, dv, ks, 1, par)
    hit = to.path_masks(par)[:, 9]
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("what", ["a", "b"])
@pytest.mark.parametrize("dk,n", [(128, 9), (128, 30), (64, 20)])
def test_linear_gates_that_are_not_numbers_stay_on_their_paths(dk, n, what):
    """A row's NaN decay or beta of one head reaches the row and those below it in that head, as it does in a scan, and
    nothing else."""
    rng = np.random.default_rng(n)
    lk, lv, ks, row, head = 2, 4, 4, 4, 2
    c = linear_case(rng, lk, dk, lv, dk, ks, n)
    par = to.random_tree(rng, n, 5)
    clean, _ = run_linear(c, lk, dk, lv, dk, ks, 1, par)
    c[what][row, head] = np.nan
    got, _ = run_linear(c, lk, dk, lv, dk, ks, 1, par)
    hit = np.zeros((n, lv, dk), bool)
    hit[to.path_masks(par)[:, row], head] = True
    hit = hit.reshape(n, -1)
    assert hit.any() and np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


# ---- verification ---------------------------------------------------------------
def run_verify(logits, par, tokens, draft, inv_t, ua, us, ld=None, stream=None):
    n, vocab = logits.shape
    ld = ld or vocab
    pad = lambda a: None if a is None else dev(np.concatenate([a, np.full((n, ld - vocab), 1e9)], 1).astype(np.float32))  # noqa: E731
    dl, dd = pad(logits), pad(draft)
    size = xb.hip().xqhip_spec_verify_workspace_bytes(n, vocab)
    ws = dev(np.full(size, 0xff, np.uint8))
    count, path, out = i32(-7), dev(np.full(n, -7, np.int32)), dev(np.full(n, -7, np.int32))
    bufs = [dev(np.asarray(tokens, np.int32)), dev(np.asarray(ua, np.float32)), dev(np.asarray([us], np.float32))]
    for _ in range(2):  # the workspace as the call before left it
        xb.ck(xb.hip().xqhip_spec_verify(dl.ptr, ld, vocab, ctypes.byref(xb.tree(par)), bufs[0].ptr,
                                         dd.ptr if dd else None, ld, inv_t, bufs[1].ptr, bufs[2].ptr, count.ptr,
                                         path.ptr, out.ptr, ws.ptr, size, stream))
    c = int(count.download(np.int32, 1)[0])
    path, out = path.download(np.int32, n).tolist(), out.download(np.int32, n).tolist()
    assert path[c:] == [-1] * (n - c) and out[c:] == [-1] * (n - c)
    return path[:c], out[:c]


@pytest.mark.parametrize("inv_t", [0.0, 1.0, 0.75, 4.0])
@pytest.mark.parametrize("mode", ["point", "probs"])
@pytest.mark.parametrize("vocab,n,reach,ld", [(1, 1, 1, 0), (5, 4, 2, 0), (1000, 17, 3, 0), (8192, 9, 1, 0), (8193, 64, 4, 8195),
                                             (248320, 6, 1, 0), (300001, 5, 2, 0), (50001, 40, 5, 50004), (20000, 64, 64, 0)])
def test_verify(vocab, n, reach, ld, mode, inv_t):
    """Equal, token by token: all decisions are taken in 64 bits."""
    rng = np.random.default_rng(vocab + n)
    for trial in range(6 if vocab < 100000 else 3):
        par = to.random_tree(rng, n, reach)
        logits = rng.normal(0, 2.5, (n, vocab)).astype(np.float32)
        near = logits * (inv_t or 1.0) + rng.normal(0, 0.7, logits.shape)
        draft = np.exp(near - near.max(1, keepdims=True))
        draft = (draft / draft.sum(1, keepdims=True)).astype(np.float32)
        tokens = [0] + [int(np.searchsorted(np.cumsum(draft[p].astype(np.float64)), rng.random() * 0.9999)) for p in par[1:]]
        if trial % 2:  # the likeliest, so that paths get long
            tokens = [0] + [int(np.argsort(-logits[p])[min(vocab - 1, int(rng.integers(0, 3)))]) for p in par[1:]]
        ua, us = rng.random(n).astype(np.float32), np.float32(rng.random())
        if trial % 3 == 0:
            ua *= np.float32(0.3)
        got = run_verify(logits, par, tokens, draft if mode == "probs" else None, inv_t, ua, us, ld)
        assert got == to.verify(logits, par, tokens, draft if mode == "probs" else None, inv_t, ua, us), trial


@pytest.mark.parametrize("mode", ["point", "probs"])
@pytest.mark.parametrize("vocab,n,shape", [(1100003, 3, "chain"), (1 << 24, 1, "chain"), (4096, 64, "star"), (9001, 64, "star"),
                                           (5000, 64, "chain"), (300, 33, "pairs")])
def test_verify_of_long_rows_and_wide_trees(vocab, n, shape, mode):
    """More than 64 pieces of a row; 63 children of one row; a path of 64; drafts that are mostly rejected."""
    rng = np.random.default_rng(vocab % 1000 + n)
    par = {"chain": list(range(-1, n - 1)), "star": [-1] + [0] * (n - 1), "pairs": [-1] + [(i - 1) // 2 for i in range(1, n)]}[shape]
    for trial in range(1 if vocab > 100000 else 5):
        logits = rng.normal(0, 2.5, (n, vocab)).astype(np.float32)
        draft = np.exp(np.minimum(logits + rng.normal(0, 1.5, logits.shape), 12)).astype(np.float32)
        draft = (draft / draft.sum(1, keepdims=True, dtype=np.float64)).astype(np.float32)
        tokens = [0] + [int(np.argmax(logits[p])) if rng.random() < (0.5 if trial % 2 else 0.02) else int(rng.integers(vocab)) for p in par[1:]]
        ua, us = (rng.random(n) * 0.3 + 0.7 * (trial > 2)).astype(np.float32), np.float32(rng.random())
        args = (logits, par, tokens, draft if mode == "probs" else None, 1.0, ua, us)
        assert run_verify(*args) == to.verify(*args), trial


@pytest.mark.parametrize("mode", ["point", "probs"])
def test_verify_of_rows_at_their_limits(mode):
    """Rows of minus infinity, NaN, plus infinity, ties; drafts outside the vocabulary, drafted twice; a draft equal to
    the target; random numbers of 0 and just below 1."""
    vocab, par, n = 300, [-1, 0, 0, 0, 1, 2, 3], 7
    rng = np.random.default_rng(9)
    base = rng.normal(0, 2, (n, vocab)).astype(np.float32)
    cases = []
    for name in ("minf", "nan", "inf", "tie", "one"):
        x = base.copy()
        if name == "minf":
            x[0] = -np.inf
        elif name == "nan":
            x[0, ::3] = np.nan
            x[1] = np.nan
        elif name == "inf":
            x[0, [7, 9]] = np.inf
        elif name == "tie":
            x[:] = 1.0
        else:
            x[0] = -np.inf
            x[0, 44] = -3e38
        cases.append(x)
    top = np.float32(1) - np.float32(2**-24)
    for x in cases:
        with np.errstate(all="ignore"):
            e = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
            e = np.exp(e - e.max(1, keepdims=True))
        draft = np.where(np.isfinite(e), e, 0)
        draft = (draft / np.maximum(draft.sum(1, keepdims=True), 1e-30)).astype(np.float32)
        for tokens in ([0, 7, 9, 44, 3, 4, 5], [0, -1, 300, 44, 3, 4, 5], [0, 12, 12, 12, 3, 4, 5]):
            for ua, us in ((0.0, 0.0), (top, top), (0.5, 0.5)):
                for inv_t in (1.0, 0.0):
                    args = (x, par, tokens, draft if mode == "probs" else None, inv_t, np.full(n, ua, np.float32), np.float32(us))
                    assert run_verify(*args) == to.verify(*args), (tokens, ua, us, inv_t)


@pytest.mark.parametrize("mode", ["point", "probs"])
@pytest.mark.parametrize("inv_t,top", [
    (1e3, 20), (1e4, 20), (1e5, 20), (1e6, 20), (1e7, 20), (1e8, 20), (3e8, 20), (1e12, 20), (3e38, 20), (1e6, 300), (1e7, 300),
    (1e6, 2000), (1.0, 2.0**24), (100.0, 2.0**24), (0.25, 3e9), (1.0, 3e9), (1.0, 3e38), (1e8, -20), (1e-37, 20), (1e-37, 3e9),
    (2e-36, 20), (1e-44, 20)])
def test_verify_temperatures_and_logits_of_every_size(inv_t, top, mode):
    """The maximum behind the first 4096 tokens, a tie or a close second beside it, others at minus infinity, and a
    vocabulary that fills no whole number of 4096s."""
    rng = np.random.default_rng(int(abs(top)) % 1000 + len(mode))
    inv_t, vocab, par = float(np.float32(inv_t)), 12001, [-1, 0, 0, 1, 1, 3]
    n = len(par)
    for trial in range(8):
        logits = (rng.normal(0, 2.5, (n, vocab)) * max(1.0, abs(top) / 64)).astype(np.float32)
        logits = np.minimum(logits - logits.max(), 0).astype(np.float32) * np.float32(0.5) + np.float32(top - abs(top) / 4)
        if trial % 2:
            logits[:, rng.random(vocab) < 0.3] = -np.inf
        best, second, other = (rng.permutation(3800)[:n] + at for at in (4100, 8200, 0))
        rows = np.arange(n)
        logits[rows, best] = top
        logits[rows, second] = np.float32(top - float(rng.random()) * min(2 / inv_t, abs(top) / 8)) if trial % 3 else top
        draft = np.zeros((n, vocab), np.float32)
        draft[rows, best], draft[rows, second], draft[rows, other] = 0.4375, 0.3125, 0.25
        tokens = [0] + [int((best, second, other)[int(rng.integers(3))][p]) for p in par[1:]]
        ua = (rng.random(n) * (0.4 if trial < 4 else 1.0)).astype(np.float32)
        args = (logits, par, tokens, draft if mode == "probs" else None, inv_t, ua, np.float32(rng.random()))
        assert run_verify(*args) == to.verify(*args), trial


@pytest.mark.parametrize("kids", [1, 2, 16, 30])
@pytest.mark.parametrize("first", [0, 4097])
def test_verify_where_rejections_leave_next_to_nothing(kids, first):
    """Two tokens of probabilities 0.6 and 0.4 against a draft of one half each, all children the second: one after the
    other rejected, they leave the first token with 0.1 x 2^-(kids - 1) of the row's distribution, up to 2 10^-10, and the
    second with nothing."""
    vocab, n = first + 2, kids + 1
    logits = np.full((n, vocab), -np.inf, np.float32)
    logits[:, first], logits[:, first + 1] = np.log(0.6), np.log(0.4)
    draft = np.zeros((n, vocab), np.float32)
    draft[:, first:] = 0.5
    top = np.float32(1) - np.float32(2**-24)
    for us in (0.0, 0.5, 0.7, top):
        got = run_verify(logits, [-1] + [0] * kids, [0] + [first + 1] * kids, draft, 1.0, np.full(n, top), np.float32(us))
        assert got == ([0], [first])


@pytest.mark.parametrize("inv_t", [0.0, 1.0])
@pytest.mark.parametrize("mode", ["point", "probs"])
def test_verify_of_a_padded_tree(mode, inv_t):
    """Rows of token -1 below the leaves, their draft rows zeros: the outcome of the tree without them."""
    rng = np.random.default_rng(17)
    vocab, par = 5000, [-1, 0, 0, 1, 1, 2]
    n, padded = len(par), par + [3, 4, 5, 6, 3, 9]
    for trial in range(20):
        logits = rng.normal(0, 2.5, (len(padded), vocab)).astype(np.float32)
        draft = np.exp(logits + rng.normal(0, 0.7, logits.shape))
        draft = (draft / draft.sum(1, keepdims=True)).astype(np.float32)
        draft[3:] = 0
        if trial % 2:
            tokens = [0] + [int(np.argsort(-logits[p])[int(rng.integers(0, 3))]) for p in par[1:]]
        else:
            tokens = [0] + [int(rng.choice(vocab, p=draft[p].astype(np.float64) / draft[p].sum(dtype=np.float64))) for p in par[1:]]
        ua, us = (rng.random(len(padded)) * 0.5).astype(np.float32), np.float32(rng.random())
        ua[n:] = 0
        probs = draft if mode == "probs" else None
        want = to.verify(logits[:n], par, tokens, None if probs is None else probs[:n], inv_t, ua[:n], us)
        assert run_verify(logits, padded, tokens + [-1] * (len(padded) - n), probs, inv_t, ua, us) == want, trial


def test_verify_in_a_graph():
    L = xb.hip()
    rng = np.random.default_rng(10)
    n, vocab = 12, 30000
    par = to.random_tree(rng, n, 3)
    logits = rng.normal(0, 2, (n, vocab)).astype(np.float32)
    tokens = [0] + [int(np.argsort(-logits[p])[int(rng.integers(0, 3))]) for p in par[1:]]
    dl, dt, du, ds = dev(logits), dev(np.array(tokens, np.int32)), dev(np.zeros(n, np.float32)), dev(np.zeros(1, np.float32))
    size = L.xqhip_spec_verify_workspace_bytes(n, vocab)
    ws, count, path, out = xb.DeviceBuffer(size), i32(0), dev(np.zeros(n, np.int32)), dev(np.zeros(n, np.int32))
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    xb.ck(L.xqhip_stream_create(ctypes.byref(s)))
    xb.ck(L.xqhip_graph_begin(s))
    xb.ck(L.xqhip_spec_verify(dl.ptr, vocab, vocab, ctypes.byref(xb.tree(par)), dt.ptr, None, 0, 1.0, du.ptr, ds.ptr,
                              count.ptr, path.ptr, out.ptr, ws.ptr, size, s))
    xb.ck(L.xqhip_graph_end(s, ctypes.byref(g)))
    for _ in range(4):
        ua, us = rng.random(n).astype(np.float32) * np.float32(0.5), np.float32(rng.random())
        du.upload(ua)
        ds.upload(np.array([us], np.float32))
        xb.ck(L.xqhip_device_synchronize())
        xb.ck(L.xqhip_graph_launch(g, s))
        xb.ck(L.xqhip_stream_synchronize(s))
        c = int(count.download(np.int32, 1)[0])
        got = path.download(np.int32, n)[:c].tolist(), out.download(np.int32, n)[:c].tolist()
        assert got == to.verify(logits, par, tokens, None, 1.0, ua, us)
    xb.ck(L.xqhip_graph_destroy(g))
    xb.ck(L.xqhip_stream_destroy(s))


# ---- LDS ------------------------------------------------------------------------
def filled():
    xb.ck(xb.hip().xqhip_lds_fill(math.nan, None))


@KINDS
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_reads_no_lds_that_it_has_not_written(kind, hd):
    rng = np.random.default_rng(hd)
    for nq, nkv, T, pos0 in ((8, 2, 1, 0), (8, 2, 3, 300), (6, 2, 7, 90), (8, 2, 21, 700), (8, 1, 64, 40)):
        cache, q, gate = attention_case(rng, kind, nq, nkv, hd, T, pos0)
        par = to.random_tree(rng, T)
        want = attend(cache, q, gate, pos0, par)
        filled()
        assert np.array_equal(attend(cache, q, gate, pos0, par), want)


@pytest.mark.parametrize("dk", [64, 128])
def test_linear_tree_reads_no_lds_that_it_has_not_written(dk):
    rng = np.random.default_rng(dk)
    for n in (1, 2, 7, 16, 17, 50):
        c, par = linear_case(rng, 2, dk, 4, dk, 4, n), to.random_tree(rng, n)
        want, _ = run_linear(c, 2, dk, 4, dk, 4, 1, par)
        filled()
        assert np.array_equal(run_linear(c, 2, dk, 4, dk, 4, 1, par)[0], want)


@pytest.mark.parametrize("mode", ["point", "probs"])
@pytest.mark.parametrize("inv_t", [0.0, 1.0])
def test_verify_reads_no_lds_that_it_has_not_written(mode, inv_t):
    rng = np.random.default_rng(5)
    for n, vocab in ((1, 50), (9, 5000), (33, 9000)):
        par = to.random_tree(rng, n, 3)
        logits = rng.normal(0, 2, (n, vocab)).astype(np.float32)
        draft = np.full((n, vocab), 1.0 / vocab, np.float32) if mode == "probs" else None
        args = (logits, par, rng.integers(0, vocab, n).tolist(), draft, inv_t, rng.random(n) * 0.5, 0.7)
        want = run_verify(*args)
        filled()
        assert run_verify(*args) == want


# ---- a step of them together ----------------------------------------------------
@KINDS
def test_a_step_over_a_tree(kind):
    """One full-attention and one linear-attention layer over a tree, verification, the kept rows moved together and the
    linear state advanced over them; then the same tokens one at a time through the decode entry points.  Both ways
    leave the same cache (8-bit codes: the single steps' rows are quantised by the same call), state and outputs."""
    L = xb.hip()
    rng = np.random.default_rng(20)
    nq, nkv, hd, rotary, lk, lv, ks, pos0, n, vocab = 8, 2, 128, 32, 2, 4, 4, 37, 14, 500
    cd = 128 * (2 * lk + lv)
    par = [-1, 0, 0, 1, 2, 2, 3, 5, 5, 8, 4, 8, 9, 11]
    k, v = (rng.normal(0, 1, (pos0, nkv, hd)) for _ in range(2))
    cap = pos0 + n
    cache, alone = Cache(kind, nkv, hd, cap, k, v), Cache(kind, nkv, hd, cap, k, v)
    norms = [dev(rng.normal(1, 0.1, hd).astype(np.float32)) for _ in range(2)]
    cs, pos = dev(rope(rotary, cap)), i32(pos0)
    row = 2 * nq * hd + 2 * nkv * hd
    proj = rng.normal(0, 1, (n, row)).astype(np.float32)
    tree = xb.tree(par)
    tr = ctypes.byref(tree)

    def full(cache, x, pos, tree, T):
        src, q, gate, out = dev(x), xb.DeviceBuffer(T * nq * hd * 4), xb.DeviceBuffer(T * nq * hd * 4), xb.DeviceBuffer(T * nq * hd * 4)
        at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
        xb.ck(L.xqhip_attn_prep_kv(at(0), at(2 * nq * hd), at((2 * nq + nkv) * hd), 1, nq, rotary, norms[0].ptr,
                                   norms[1].ptr, EPS, cs.ptr, pos.ptr, tree, T, row, nq * hd, q.ptr, gate.ptr,
                                   cache.ref, None))
        size = L.xqhip_tree_attention_workspace_bytes(nq, nkv, hd, T)
        ws = xb.DeviceBuffer(size)
        xb.ck(L.xqhip_tree_attention(q.ptr, gate.ptr, cache.ref, nq, tree, T, nq * hd, pos.ptr, out.ptr, nq * hd,
                                     ws.ptr, size, None))
        return out.download(np.float32, T * nq * hd).reshape(T, -1)

    tree_out = full(cache, proj, pos, tr, n)
    # the linear layer
    c = {m: np.ascontiguousarray(x, np.float32) for m, x in linear_case(rng, lk, 128, lv, 128, ks, n).items()}
    lrow = cd + 2 * lv
    lin = dev(np.concatenate([c["mixed"], c["a"], c["b"]], 1))
    hist, S, keep = dev(c["hist"]), dev(c["S"]), [dev(c[m]) for m in ("w", "a_log", "dt")]
    at = lambda b, f: ctypes.c_void_p(b.ptr.value + 4 * f)  # noqa: E731
    size = L.xqhip_linear_attn_tree_workspace_bytes(n, lk, 128, lv, 128)
    ws, lout = xb.DeviceBuffer(max(size, 16)), xb.DeviceBuffer(n * lv * 128 * 4)
    xb.ck(L.xqhip_linear_attn_tree(lin.ptr, at(lin, cd), at(lin, cd + lv), lrow, hist.ptr, pos.ptr, keep[0].ptr,
                                   keep[1].ptr, keep[2].ptr, S.ptr, lk, 128, lv, 128, ks, tr, lout.ptr, lv * 128,
                                   ws.ptr, size, None))
    lin_out = lout.download(np.float32, n * lv * 128).reshape(n, -1)
    # verification: logits that favour some drafts
    logits = rng.normal(0, 1, (n, vocab)).astype(np.float32)
    tokens = rng.integers(0, vocab, n).astype(np.int32)
    for i in (2, 5, 8, 11):
        logits[par[i], tokens[i]] += 9
    size = L.xqhip_spec_verify_workspace_bytes(n, vocab)
    vws, count, path, new = xb.DeviceBuffer(size), i32(0), dev(np.zeros(n, np.int32)), dev(np.zeros(n, np.int32))
    dl, ua, us = dev(logits), np.full(n, 0.4, np.float32), np.float32(0.3)
    bufs = [dev(tokens), dev(ua), dev(np.array([us], np.float32))]
    xb.ck(L.xqhip_spec_verify(dl.ptr, vocab, vocab, tr, bufs[0].ptr, None, 0, 1.0, bufs[1].ptr, bufs[2].ptr, count.ptr,
                              path.ptr, new.ptr, vws.ptr, size, None))
    want_path, want_new = to.verify(logits, par, tokens, None, 1.0, ua, us)
    m = int(count.download(np.int32, 1)[0])
    assert path.download(np.int32, n)[:m].tolist() == want_path and new.download(np.int32, n)[:m].tolist() == want_new
    assert want_path[:5] == [0, 2, 5, 8, 11]
    # kept rows together; the state over them
    sets = [(b.ptr, w, cap, pos.ptr) for b, w in zip(cache.buf, 2 * [nkv * hd * (1 if kind == xb.KV_I8 else 2)] + 2 * [nkv * 4])]
    sets = sets[:4 if kind == xb.KV_I8 else 2] + [(lin.ptr, lrow * 4, n, None)]
    xb.ck(L.xqhip_tree_keep(xb.rows(sets), len(sets), path.ptr, count.ptr, n, None))
    step_hist, step_S = dev(c["hist"]), dev(c["S"])
    one = xb.DeviceBuffer(lv * 128 * 4)
    rows = np.concatenate([c["mixed"], c["a"], c["b"]], 1)[want_path]
    assert np.array_equal(lin.download(np.float32, n * lrow).reshape(n, lrow)[:m], rows)
    scan_out = xb.DeviceBuffer(m * lv * 128 * 4)
    xb.ck(L.xqhip_linear_attn_scan(lin.ptr, at(lin, cd), at(lin, cd + lv), lrow, hist.ptr, pos0, keep[0].ptr,
                                   keep[1].ptr, keep[2].ptr, S.ptr, lk, 128, lv, 128, ks, m, scan_out.ptr, lv * 128, None))
    for j, i in enumerate(want_path):
        x, p = dev(rows[j]), i32(pos0 + j)
        xb.ck(L.xqhip_linear_attn_step(x.ptr, step_hist.ptr, keep[0].ptr, at(x, cd), at(x, cd + lv), keep[1].ptr,
                                       keep[2].ptr, step_S.ptr, lk, 128, lv, 128, ks, p.ptr, one.ptr, None))
        assert np.abs(one.download(np.float32, lv * 128) - lin_out[i]).max() <= 2e-5
        got = full(alone, proj[i:i + 1], p, None, 1)
        assert np.abs(got[0] - tree_out[i]).max() <= 3e-5
    for a, b in zip(cache.raw(), alone.raw()):
        assert np.array_equal(a[:pos0 + m], b[:pos0 + m], equal_nan=True)
    a, b = S.download(np.float32, c["S"].size), step_S.download(np.float32, c["S"].size)
    assert np.abs(a - b).max() <= 2e-5
    if kind == xb.KV_F16:  # and as the framework's own decode step does it
        x, out = dev(proj[0]), xb.DeviceBuffer(nq * hd * 4)
        other = Cache(kind, nkv, hd, cap, k, v)
        ws = xb.DeviceBuffer(L.xqhip_gqa_workspace_bytes(nq, nkv, hd))
        xb.ck(L.xqhip_attn_decode(x.ptr, at(x, 2 * nq * hd), at(x, (2 * nq + nkv) * hd), 1, nq, nkv, hd, rotary,
                                  norms[0].ptr, norms[1].ptr, EPS, cs.ptr, i32(pos0).ptr, other.buf[0].ptr,
                                  other.buf[1].ptr, cap, out.ptr, ws.ptr, None))
        assert np.abs(out.download(np.float32, nq * hd) - tree_out[0]).max() <= 3e-5


@KINDS
def test_a_step_in_graphs_that_share_a_workspace(kind):
    """The step's calls captured twice, over trees of 5 and 40 rows with one workspace between them, and replayed in turn
    with eager work in between: each replay leaves what the eager calls leave."""
    L = xb.hip()
    rng = np.random.default_rng(21)
    nq, nkv, hd, rotary, lk, lv, ks, pos0, vocab, cap = 8, 2, 128, 32, 2, 4, 4, 600, 9000, 700
    cd, n = 128 * (2 * lk + lv), 40
    row, lrow = 2 * nq * hd + 2 * nkv * hd, cd + 2 * lv
    k, v = (rng.normal(0, 1, (pos0, nkv, hd)) for _ in range(2))
    fresh = Cache(kind, nkv, hd, cap, k, v)
    held = [b.download(np.uint8, b.nbytes) for b in fresh.buf]
    norms = [dev(rng.normal(1, 0.1, hd).astype(np.float32)) for _ in range(2)]
    cs, pos, proj = dev(rope(rotary, cap)), i32(pos0), dev(rng.normal(0, 1, (n, row)).astype(np.float32))
    c = {m: np.ascontiguousarray(x, np.float32) for m, x in linear_case(rng, lk, 128, lv, 128, ks, n).items()}
    lin, hist, S = dev(np.concatenate([c["mixed"], c["a"], c["b"]], 1)), dev(c["hist"]), dev(c["S"])
    keep = [dev(c[m]) for m in ("w", "a_log", "dt")]
    logits, us = dev(rng.normal(0, 2, (n, vocab)).astype(np.float32)), dev(np.array([0.6], np.float32))
    tokens, ua = dev(rng.integers(0, vocab, n).astype(np.int32)), dev(np.full(n, 1e-6, np.float32))
    sizes = [f(n) for f in (lambda t: L.xqhip_tree_attention_workspace_bytes(nq, nkv, hd, t),
                            lambda t: L.xqhip_linear_attn_tree_workspace_bytes(t, lk, 128, lv, 128),
                            lambda t: L.xqhip_spec_verify_workspace_bytes(t, vocab))]
    size = max([*sizes, L.xqhip_tree_attention_workspace_bytes(nq, nkv, hd, 5)])
    ws = dev(np.full(size, 0xff, np.uint8))
    q, gate, out = (xb.DeviceBuffer(n * nq * hd * 4) for _ in range(3))
    lout, count, path, new = xb.DeviceBuffer(n * lv * 128 * 4), i32(0), dev(np.zeros(n, np.int32)), dev(np.zeros(n, np.int32))
    at = lambda b, f: ctypes.c_void_p(b.ptr.value + 4 * f)  # noqa: E731
    widths = 2 * [nkv * hd * (1 if kind == xb.KV_I8 else 2)] + (2 * [nkv * 4] if kind == xb.KV_I8 else [])
    sets = xb.rows([(b.ptr, w, cap, pos.ptr) for b, w in zip(fresh.buf, widths)])

    def step(par, s):
        T, tr = len(par), ctypes.byref(xb.tree(par))
        xb.ck(L.xqhip_attn_prep_kv(proj.ptr, at(proj, 2 * nq * hd), at(proj, (2 * nq + nkv) * hd), 1, nq, rotary,
                                   norms[0].ptr, norms[1].ptr, EPS, cs.ptr, pos.ptr, tr, T, row, nq * hd, q.ptr, gate.ptr,
                                   fresh.ref, s))
        xb.ck(L.xqhip_tree_attention(q.ptr, gate.ptr, fresh.ref, nq, tr, T, nq * hd, pos.ptr, out.ptr, nq * hd, ws.ptr,
                                     size, s))
        xb.ck(L.xqhip_linear_attn_tree(lin.ptr, at(lin, cd), at(lin, cd + lv), lrow, hist.ptr, pos.ptr, keep[0].ptr,
                                       keep[1].ptr, keep[2].ptr, S.ptr, lk, 128, lv, 128, ks, tr, lout.ptr, lv * 128,
                                       ws.ptr, size, s))
        xb.ck(L.xqhip_spec_verify(logits.ptr, vocab, vocab, tr, tokens.ptr, None, 0, 1.0, ua.ptr, us.ptr, count.ptr,
                                  path.ptr, new.ptr, ws.ptr, size, s))
        xb.ck(L.xqhip_tree_keep(sets, len(sets), path.ptr, count.ptr, T, s))

    def reset():
        for b, x in zip(fresh.buf, held):
            b.upload(x)
        for b in (out, lout, path, new):
            b.zero()
        xb.ck(L.xqhip_device_synchronize())

    def left(s):
        xb.ck(L.xqhip_stream_synchronize(s) if s else L.xqhip_device_synchronize())
        return [b.download(np.uint8, b.nbytes) for b in (*fresh.buf[:len(widths)], out, lout, count, path, new)]

    trees = [to.random_tree(rng, 5), to.random_tree(rng, 40)]
    want = []
    for par in trees:
        reset()
        step(par, None)
        want.append(left(None))
    s, graphs = ctypes.c_void_p(), [ctypes.c_void_p(), ctypes.c_void_p()]
    xb.ck(L.xqhip_stream_create(ctypes.byref(s)))
    for par, g in zip(trees, graphs):
        xb.ck(L.xqhip_graph_begin(s))
        step(par, s)
        xb.ck(L.xqhip_graph_end(s, ctypes.byref(g)))
    for i in (0, 1, 1, 0, 1):
        reset()
        step(trees[1 - i], None)  # eager work of the other tree
        reset()
        xb.ck(L.xqhip_graph_launch(graphs[i], s))
        for a, b in zip(left(s), want[i]):
            assert np.array_equal(a, b)
    for g in graphs:
        xb.ck(L.xqhip_graph_destroy(g))
    xb.ck(L.xqhip_stream_destroy(s))
