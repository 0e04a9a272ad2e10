"""The operators of a step over several sequences in paged caches against plain 64-bit results (paged_oracle), and whole
steps of them together.

Bounds.  Cached keys are computed in 64 bits and rounded to fp32, then to fp16: the oracle's are the same numbers (a
difference of 2^-50 moves an fp32 rounding once in 2^26 values and then an fp16 one once in 2^13).
q: one rounding to fp32, 2^-24 of the value, beside the 64-bit result's.
Attention: q and the weights carry 22 bits or more, so a score of |q||k| / sqrt(hd) <= 16 is off by at most 16 x 2^-22 and
a weight by 4e-6 of itself; the output, a convex combination of |v| <= 6, by 3e-5.
Log probabilities: see the tests."""
import ctypes
import math

import numpy as np
import pytest

import paged_oracle as po
import xqbind as xb

pytestmark = pytest.mark.gpu
EPS = 1e-6
F16, I8 = xb.PAGES_F16, xb.PAGES_I8
_held = []  # a test's buffers, alive until it ends: calls take bare addresses


def dev(a):
    _held.append(xb.DeviceBuffer.from_array(np.ascontiguousarray(a)))
    return _held[-1]


@pytest.fixture(autouse=True)
def _release():
    yield
    xb.ck(xb.hip().xqhip_device_synchronize())
    _held.clear()


def i32(v):
    return dev(np.array(v, np.int32))


class Pool:
    """A pool of pages, every page NaN (fp16) or codes 99 with NaN scales; open pages NaN."""

    def __init__(self, kind, nkv, hd, page, pages, opens=1, k=None, v=None):
        self.kind, self.nkv, self.hd, self.page, self.pages, self.opens = kind, nkv, hd, page, pages, opens
        self.e = 16 if kind == I8 else 8
        t = np.int8 if kind == I8 else np.float16
        fill = 99 if kind == I8 else np.nan
        x = [np.full((pages, nkv, page, hd), fill, t) for _ in range(2)]
        sc = np.full((2, pages, nkv), np.nan, np.float32)
        for i, given in enumerate((k, v)):  # fp16 values [pages][nkv][page][hd]; NaN: not filled
            if given is None:
                continue
            if kind == F16:
                x[i][:] = given
            else:
                for p in range(pages):
                    for h in range(nkv):
                        on = ~np.isnan(given[p, h].astype(np.float32)).any(-1)
                        if on.any():
                            x[i][p, h, on], sc[i, p, h] = po.codes(given[p, h][on])
        self.bk, self.bv = dev(po.to_pages_k(x[0], self.e)), dev(po.to_pages_v(x[1], self.e))
        self.scale = [dev(sc[0]), dev(sc[1])]
        self.open = [dev(np.full((opens, nkv, page, hd), np.nan, np.float16)) for _ in range(2)]
        self.c = xb.Pages(kind, nkv, hd, page, pages, opens, self.bk.ptr, self.bv.ptr,
                          *([b.ptr for b in self.scale + self.open] if kind == I8 else [None] * 4))
        self.ref = ctypes.byref(self.c)

    def raw(self):
        """k, v as [pages][nkv][page][hd], their scales, the open pages."""
        t, n = np.int8 if self.kind == I8 else np.float16, self.pages * self.nkv * self.page * self.hd
        k = self.bk.download(t, n).reshape(self.pages, self.nkv, self.hd // self.e, self.page, self.e)
        v = self.bv.download(t, n).reshape(self.pages, self.nkv, self.page // self.e, self.hd, self.e)
        sc = [b.download(np.float32, self.pages * self.nkv).reshape(self.pages, self.nkv) for b in self.scale]
        op = [b.download(np.float16, self.opens * self.nkv * self.page * self.hd).reshape(self.opens, self.nkv, self.page, self.hd)
              for b in self.open]
        return [po.from_pages_k(k), po.from_pages_v(v)] + sc + op

    def values(self):
        k, v, ks, vs = self.raw()[:4]
        if self.kind == F16:
            return k.astype(np.float64), v.astype(np.float64)
        return k * ks[..., None, None].astype(np.float64), v * vs[..., None, None].astype(np.float64)


class Plan:
    """The step's sequences: positions before, rows, tables of pages taken in random order."""

    def __init__(self, rng, page, past, rows, pad=0, max_rows=None, spare=2, extra=0):
        self.past, self.rows, self.page = list(past), list(rows), page
        self.n = sum(rows)
        need = [(p + r + page - 1) // page for p, r in zip(past, rows)]
        self.most = max(need + [1]) + extra
        self.pages = sum(need) + spare
        order = list(rng.permutation(self.pages))
        self.table = np.full((len(past), self.most), -1, np.int32)
        for s, m in enumerate(need):
            self.table[s, :m] = [order.pop() for _ in range(m)]
        self.open = rng.permutation(len(past)).astype(np.int32)
        self.row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.total = self.n + pad
        self.max_rows = max_rows or max(max(rows), 1)
        self.upload()

    def upload(self):
        self.bufs = [i32(self.row0), i32(self.past), i32(self.table), i32(self.open)]
        self.c = xb.Step(len(self.past), self.total, self.max_rows, self.most, *(b.ptr for b in self.bufs))
        self.ref = ctypes.byref(self.c)

    def each(self):
        """(sequence, index in it, row, position)"""
        for s, (p, m) in enumerate(zip(self.past, self.rows)):
            for j in range(m):
                yield s, j, int(self.row0[s]) + j, p + j

    def seq_values(self, pool_values, s, n):
        """[n positions][nkv][hd] of a sequence, from [pages][nkv][page][hd]."""
        pg = self.table[s, :(n + self.page - 1) // self.page]
        x = pool_values[pg].transpose(0, 2, 1, 3)
        return x.reshape(-1, *x.shape[2:])[:n]


def rope(rotary, cap, theta=1e4):
    t = np.empty((cap, rotary // 2, 2), np.float32)
    xb.ck(xb.hip().xqhip_rope_table(theta, rotary, cap, xb.ptr(t)))
    return t


# ---- the append -----------------------------------------------------------------
def prep(rng, pool, plan, nq, rotary, sections=None, inter=False, axes=None, gated=1, pad=0, x=None, norms=None, cap=None, table=None):
    """Runs xqhip_attn_prep_paged; returns (projections, q, gate, norms, cos/sin of every row)."""
    nkv, hd, T = pool.nkv, pool.hd, plan.total
    wq = nq * hd * (2 if gated else 1)
    row = wq + 2 * nkv * hd + pad
    x = rng.normal(0, 1, (T, row)).astype(np.float32) if x is None else x
    qn, kn = norms or (rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2))
    cap = cap or max(p + m for p, m in zip(plan.past, plan.rows)) + 1
    cs = rope(rotary, cap) if rotary else np.zeros((cap, 0, 2), np.float32)
    rot, angles = None, np.zeros((T, 0, 2), np.float32)
    if rotary:
        sections = sections or [rotary // 2]
        r = xb.rotary(dev(cs).ptr, cap, rotary, sections, inter, i32(axes).ptr if axes is not None else None)
        rot, of = ctypes.byref(r), np.array(list(r.axis)[:rotary // 2])
        angles = np.zeros((T, rotary // 2, 2), np.float32)
        for s, j, i, p in plan.each():
            at = axes[of, i] if axes is not None else np.full(rotary // 2, p)
            ok = (at >= 0) & (at < cap)
            angles[i] = np.where(ok[:, None], cs[np.where(ok, at, 0), np.arange(rotary // 2)], np.nan)
    src, out = dev(x), nq * hd + (3 if pad % 4 else 4)
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    qo, go = dev(np.full((T, out), 7, np.float32)), dev(np.full((T, out), 7, np.float32))
    xb.ck(xb.hip().xqhip_attn_prep_paged(at(0), at(wq), at(wq + nkv * hd), gated, nq, dev(qn).ptr, dev(kn).ptr, EPS, rot, plan.ref,
                                         row, out, qo.ptr, go.ptr if gated else None, pool.ref, None))
    q, g = (b.download(np.float32, T * out).reshape(T, out) for b in (qo, go))
    assert (q[:, nq * hd:] == 7).all() and (g[:, nq * hd:] == 7).all()
    return x, q[:, :nq * hd].reshape(T, nq, hd), g[:, :nq * hd].reshape(T, nq, hd), (qn, kn), angles


def split_heads(x, nq, nkv, hd, gated):
    """q, gate, k, v [rows][heads][hd] of projections."""
    wq = nq * hd * (2 if gated else 1)
    q = x[:, :wq].reshape(len(x), nq, -1)
    return (q[..., :hd], q[..., hd:] if gated else None, x[:, wq: wq + nkv * hd].reshape(len(x), nkv, hd),
            x[:, wq + nkv * hd: wq + 2 * nkv * hd].reshape(len(x), nkv, hd))


def appended(pool_raw, plan, kind, k, v, bad=()):
    """What pool_raw (Pool.raw) holds after rows k, v [rows][nkv][hd] (fp32) were appended; bad: rows that are not held."""
    new = [a.copy() for a in pool_raw]
    for i, x in enumerate((k, v)):
        for s, m in enumerate(plan.rows):
            touched = {}
            for j in range(m):
                row, pos = int(plan.row0[s]) + j, plan.past[s] + j
                pg = plan.table[s, pos // plan.page] if pos // plan.page < plan.most else -1
                if row in bad or pg < 0 or pg >= len(new[0]):
                    continue
                if kind == F16:
                    new[i][pg, :, pos % plan.page] = x[row].astype(np.float16)
                else:
                    touched.setdefault(pos // plan.page, []).append((pos % plan.page, row))
            if kind == F16:
                continue
            last = (plan.past[s] + m - 1) // plan.page
            for at, rows in touched.items():
                pg, lead = plan.table[s, at], max(0, plan.past[s] - at * plan.page)
                vals = po.held(x[[r for _, r in rows]])
                offs = [o for o, _ in rows]
                for h in range(vals.shape[1]):
                    was = np.float16(np.float32(new[2 + i][pg, h] * np.float32(127))) if lead else np.float16(0)
                    mx = np.abs(vals[:, h]).max()
                    kept = pool_raw[4 + i][plan.open[s], h, :lead]
                    leaves = lead and at != last  # the step goes on into another page
                    if leaves:
                        mx = max(mx, np.abs(kept).max())
                    grew, mx = mx > was, max(mx, was)
                    new[2 + i][pg, h] = np.float32(mx.astype(np.float64) / 127)
                    if grew or leaves:
                        new[i][pg, h, :lead] = np.clip(np.rint(kept.astype(np.float64) * 127 / mx.astype(np.float64)), -127, 127)
                    new[i][pg, h, offs] = np.rint(vals[:, h].astype(np.float64) * 127 / float(mx)) if mx > 0 else 0
                if at == last:
                    new[4 + i][plan.open[s]][:, offs] = vals.transpose(1, 0, 2)
    return new


def same(a, b):
    return all(np.array_equal(x, y, equal_nan=x.dtype.kind == "f") for x, y in zip(a, b))


SHAPES = [
    # nq, nkv, hd, rotary, sections, interleaved, page, past, rows, gated, pad, extra rows
    (32, 8, 128, 32, None, False, 64, [0], [1], 1, 0, 0),
    (32, 8, 128, 32, [6, 5, 5], True, 64, [63, 64, 65, 0, 700], [1, 1, 1, 1, 1], 1, 0, 3),
    (16, 4, 256, 64, [12, 10, 10], False, 32, [31, 5, 40], [130, 0, 7], 1, 4, 1),
    (16, 4, 256, 256, None, False, 128, [250], [9], 1, 1, 0),
    (4, 4, 64, 16, [3, 5], False, 32, [0, 31, 32], [33, 1, 2], 0, 0, 2),
    (6, 2, 80, 20, [4, 2, 2, 2], True, 64, [2, 60], [70, 5], 1, 0, 0),
    (5, 5, 48, 48, None, False, 32, [3, 0, 0], [100, 0, 32], 0, 3, 5),
    (2, 1, 16, 0, None, False, 32, [30], [3], 1, 0, 0),
    (4, 1, 112, 2, None, False, 128, [100] * 70, [1] * 70, 1, 0, 0),
    (16, 4, 256, 64, [12, 10, 10], True, 128, [23, 0, 200], [139, 70, 1], 1, 0, 2), (16, 4, 256, 64, None, False, 64, [63, 0], [200, 1], 1, 1, 0),
    (8, 2, 128, 32, None, False, 128, [100, 7], [400, 130], 1, 4, 1), (6, 2, 80, 20, [4, 2, 2, 2], True, 128, [127], [140], 0, 0, 0),
    (8, 2, 128, 32, None, False, 64, [5] * 9, [1, 30, 1, 0, 1, 2, 1, 64, 1], 1, 0, 4),
]


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}_{s[1]}x{s[2]}_{s[6]}_{s[7][0]}_{s[8][0]}" for s in SHAPES])
def test_prep_writes_the_pages(kind, shape):
    """q: 2^-24 of the value for its rounding."""
    nq, nkv, hd, rotary, sections, inter, page, past, rows, gated, pad, behind = shape
    rng = np.random.default_rng(hd + page + len(past))
    plan = Plan(rng, page, past, rows, pad=behind)
    pool = Pool(kind, nkv, hd, page, plan.pages, len(past))
    if kind == I8:  # what was appended before: each sequence's page so far
        before = Plan(rng, page, [p // page * page for p in past], [p % page for p in past])
        if before.n:
            before.table, before.most, before.open = plan.table, plan.most, plan.open
            before.upload()
            prep(rng, pool, before, nq, rotary, gated=gated, cap=4000)
    was = pool.raw()
    cap = max(past) + max(rows) + 40
    axes = rng.integers(0, cap, (len(sections), plan.total)).astype(np.int32) if sections else None
    x, q, g, (qn, kn), cs = prep(rng, pool, plan, nq, rotary, sections, inter, axes, gated, pad, cap=cap)
    qx, gx, kx, vx = split_heads(x, nq, nkv, hd, gated)
    want = po.prepared(qx, qn, cs[:, None], EPS)
    live = plan.n
    assert (np.abs(q[:live] - want[:live]) <= 2**-23 * np.abs(want[:live])).all()
    assert (g[:live] == (gx[:live] if gated else 7)).all() if gated else (g == 7).all()
    assert (q[live:] == 7).all() and (g[live:] == 7).all()
    k = po.prepared(kx, kn, cs[:, None], EPS)
    assert same(pool.raw(), appended(was, plan, kind, k, vx))


def test_prep_takes_gate_zero():
    rng = np.random.default_rng(3)
    plan = Plan(rng, 32, [4], [2])
    pool = Pool(F16, 2, 64, 32, plan.pages)
    x = rng.normal(0, 1, (2, 4 * 64 + 2 * 128)).astype(np.float32)
    src, g = dev(x), dev(np.full((2, 256), 7, np.float32))
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    n = dev(np.ones(64, np.float32))
    xb.ck(xb.hip().xqhip_attn_prep_paged(at(0), at(256), at(384), 0, 4, n.ptr, n.ptr, EPS, None, plan.ref, 512, 256, dev(x[:, :256]).ptr,
                                         g.ptr, pool.ref, None))
    assert (g.download(np.float32, 512) == 0).all()


@pytest.mark.parametrize("hd,page,steps", [(128, 64, [1] * 70), (256, 32, [3, 1, 40, 30, 1, 1, 20]), (64, 128, [100, 1, 1, 60]), (128, 32, [32, 1, 31, 64])])
def test_codes_do_not_depend_on_the_steps(hd, page, steps):
    """8-bit pages of one sequence, appended in parts, are those of one append: codes and scales bit for bit."""
    rng = np.random.default_rng(hd)
    n, nq, nkv = sum(steps), 2, 2
    x = (rng.normal(0, 1, (n, (nq + 2 * nkv) * hd)) * rng.uniform(0.01, 3, (n, 1))).astype(np.float32)
    norms = [rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2)]
    raws = []
    for parts in (steps, [n]):
        whole = Plan(np.random.default_rng(1), page, [0], [n])
        pool, done = Pool(I8, nkv, hd, page, whole.pages), 0
        for m in parts:
            plan = Plan(np.random.default_rng(1), page, [done], [m])
            plan.table, plan.most = whole.table, whole.most
            plan.upload()
            prep(rng, pool, plan, nq, 16, gated=0, x=x[done: done + m], norms=norms, cap=n)
            done += m
        raws.append(pool.raw())
    left = n % page or page  # rows of the open page that both have
    raws = [r[:4] + [r[4][:, :, :left], r[5][:, :, :left]] for r in raws]
    assert same(*raws)


def test_a_sequence_goes_back_within_its_open_page():
    """Positions appended anew after a step back: the new rows' codes, the scale of what was there, earlier rows as they are."""
    rng = np.random.default_rng(8)
    plan = Plan(rng, 64, [0], [40])
    pool = Pool(I8, 1, 128, 64, plan.pages)
    prep(rng, pool, plan, 2, 32, cap=99)
    back = Plan(rng, 64, [30], [5])
    back.table, back.most, back.open = plan.table, plan.most, plan.open
    back.upload()
    was = pool.raw()
    for size in (0.01, 50.0):
        x = rng.normal(0, size, (5, 2 * 256 + 256)).astype(np.float32)
        x, _, _, (_, kn), cs = prep(rng, pool, back, 2, 32, x=x, cap=99)
        _, _, kx, vx = split_heads(x, 2, 1, 128, 1)
        was = appended(was, back, I8, po.prepared(kx, kn, cs[:, None], EPS), vx)
        assert same(pool.raw(), was)


@pytest.mark.parametrize("kind", [F16, I8])
def test_rows_without_a_place(kind):
    """Pages outside the pool, positions past the table, open pages and rotary positions that are none: no cache row, NaN as q,
    everything else as it was."""
    rng = np.random.default_rng(5)
    plan = Plan(rng, 32, [0, 20, 64, 10, 31, 5, 7], [40, 20, 5, 3, 1, 2, 4])
    plan.table[0, 1] = plan.pages          # positions 32 .. of sequence 0
    plan.table[1, 0] = -5                  # 20 .. 31 of sequence 1
    plan.past[2] = 32 * plan.most - 2      # runs past the table after two rows
    plan.table[2, plan.most - 1] = plan.table[2, 0]
    plan.past[5] = -1
    nan = set()
    if kind == I8:
        plan.open[3] = len(plan.past)
    plan.upload()
    pool = Pool(kind, 2, 128, 32, plan.pages, len(plan.past), k=rng.normal(0, 1, (plan.pages, 2, 32, 128)).astype(np.float16),
                v=rng.normal(0, 1, (plan.pages, 2, 32, 128)).astype(np.float16))
    for b in pool.open:
        xb.ck(xb.hip().xqhip_fill_u8(b.ptr, 0, len(plan.past) * 2 * 32 * 128 * 2, None))
    axes = rng.integers(0, 50, (3, plan.total)).astype(np.int32)
    last = int(plan.row0[6])
    axes[1, last], axes[2, last + 2] = -1, 50
    for s, j, row, pos in plan.each():
        pg = plan.table[s, pos // 32] if 0 <= pos < 32 * plan.most else -1
        if not 0 <= pg < plan.pages or plan.past[s] < 0 or (kind == I8 and s == 3) or row in (last, last + 2):
            nan.add(row)
    was = pool.raw()
    x, q, g, (qn, kn), cs = prep(rng, pool, plan, 8, 32, [6, 5, 5], True, axes, cap=50)
    for row in range(plan.n):
        assert np.isnan(q[row]).all() if row in nan else np.isfinite(q[row]).all(), row
    _, gx, kx, vx = split_heads(x, 8, 2, 128, 1)
    assert (g == gx).all()
    assert same(pool.raw(), appended(was, plan, kind, po.prepared(kx, kn, cs[:, None], EPS), vx, nan))


def test_values_that_8_bits_do_not_have():
    """Infinities and values past fp16's range are held as its largest, NaN as 0; fp16 pages keep them."""
    rng = np.random.default_rng(6)
    for kind in (F16, I8):
        plan = Plan(rng, 32, [0], [6])
        pool = Pool(kind, 1, 128, 32, plan.pages)
        x = rng.normal(0, 1, (6, 128 + 256)).astype(np.float32)
        x[1, 256 + 5], x[2, 256 + 6], x[3, 256 + 7], x[4, 256 + 8] = np.inf, -np.inf, np.nan, 1e6
        x, _, _, (_, kn), cs = prep(rng, pool, plan, 1, 0, gated=0, x=x)
        _, _, kx, vx = split_heads(x, 1, 1, 128, 0)
        with np.errstate(over="ignore"):
            k = po.prepared(kx, kn, cs[:, None], EPS)
            want = appended(Pool(kind, 1, 128, 32, plan.pages).raw(), plan, kind, k, vx)
        assert same(pool.raw(), want)


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("nkv,hd,page,past,rows", [(8, 128, 64, [60, 0, 5], [9, 0, 130]), (3, 80, 32, [31], [2]), (4, 256, 128, [0] * 40, [3] * 40)])
@pytest.mark.parametrize("out", [xb.F32, xb.F16])
def test_read(kind, nkv, hd, page, past, rows, out):
    rng = np.random.default_rng(hd)
    plan = Plan(rng, page, past, rows, pad=2)
    pool = Pool(kind, nkv, hd, page, plan.pages, 1, *(rng.normal(0, 2, (plan.pages, nkv, page, hd)).astype(np.float16) for _ in "kv"))
    plan.table[0, past[0] // page] = -1
    plan.upload()
    t = np.float32 if out == xb.F32 else np.float16
    n = plan.total * nkv * hd
    bufs = [dev(np.full(n, 7, t)) for _ in "kv"]
    xb.ck(xb.hip().xqhip_paged_read(pool.ref, plan.ref, out, bufs[0].ptr, bufs[1].ptr, None))
    alone = dev(np.full(n, 7, t))
    xb.ck(xb.hip().xqhip_paged_read(pool.ref, plan.ref, out, None, alone.ptr, None))
    k, v, ks, vs = pool.raw()[:4]
    for x, sc, b in ((k, ks, bufs[0]), (v, vs, bufs[1])):
        got = b.download(t, n).reshape(plan.total, nkv, hd)
        vals = x.astype(np.float32) * (sc[..., None, None] if kind == I8 else np.float32(1))
        for s, j, row, pos in plan.each():
            pg = plan.table[s, pos // page]
            want = vals[pg, :, pos % page].astype(t) if pg >= 0 else np.zeros((nkv, hd), t)
            assert (got[row] == want).all(), (s, j)
        assert (got[plan.n:] == 7).all()
    assert (alone.download(t, n) == bufs[1].download(t, n)).all()


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("out", [xb.F32, xb.F16])
def test_read_to_any_address(kind, out):
    """Outputs at addresses that are multiples of their values' size only."""
    rng = np.random.default_rng(34)
    plan = Plan(rng, 64, [50, 3], [40, 70])
    pool = Pool(kind, 3, 80, 64, plan.pages, 1, *(rng.normal(0, 2, (plan.pages, 3, 64, 80)).astype(np.float16) for _ in "kv"))
    t, n = (np.float32 if out == xb.F32 else np.float16), plan.total * 3 * 80
    got = []
    for shift in (0, 1, 3):
        bufs = [dev(np.full(n + 8, 7, t)) for _ in "kv"]
        xb.ck(xb.hip().xqhip_paged_read(pool.ref, plan.ref, out, *(ctypes.c_void_p(b.ptr.value + shift * t().itemsize) for b in bufs), None))
        x = [b.download(t, n + 8) for b in bufs]
        assert all((y[:shift] == 7).all() and (y[shift + n:] == 7).all() for y in x)
        got.append([y[shift: shift + n] for y in x])
    assert all((a == b).all() for g in got[1:] for a, b in zip(g, got[0]))
    k, v = pool.values()
    want = [np.concatenate([plan.seq_values(x, s, p + m)[p:] for s, (p, m) in enumerate(zip(plan.past, plan.rows))]) for x in (k, v)]
    for g, w in zip(got[0], want):  # a rounding of code * scale to fp32 and one to the output
        assert (np.abs(g.reshape(w.shape) - w) <= (2**-10 if out == xb.F16 else 2**-23) * np.abs(w)).all()


# ---- attention ------------------------------------------------------------------
def attention(pool, plan, nq, q, gate, q_stride=None, out_stride=None, shift=0, stream=None, ws=None):
    L, width = xb.hip(), nq * pool.hd
    qs, os_ = q_stride or width, out_stride or width
    need = L.xqhip_paged_attention_workspace_bytes(nq, pool.nkv, pool.hd)
    ws = ws or dev(np.full(need, 0xff, np.uint8))

    def spread(x):
        y = np.full(plan.total * qs + shift, np.nan, np.float32)
        y[shift:].reshape(plan.total, qs)[:, :width] = x
        return ctypes.c_void_p(dev(y).ptr.value + 4 * shift)

    out = dev(np.full(plan.total * os_ + shift, 7, np.float32))
    xb.ck(L.xqhip_paged_attention(spread(q), spread(gate) if gate is not None else None, pool.ref, nq, plan.ref, qs,
                                  ctypes.c_void_p(out.ptr.value + 4 * shift), os_, ws.ptr, need, stream))
    xb.ck(L.xqhip_stream_synchronize(stream))
    y = out.download(np.float32, plan.total * os_ + shift)[shift:].reshape(plan.total, os_)
    assert (y[:, width:] == 7).all()
    return y[:, :width].reshape(plan.total, nq, pool.hd)


def attend_oracle(pool, plan, nq, q, gate, rows=None):
    k, v = pool.values()
    cap = plan.most * plan.page
    out = {}
    for s, j, row, pos in plan.each():
        if rows is not None and row not in rows or j >= plan.max_rows:
            continue
        n = min(pos + 1, cap)
        pg = plan.table[s, np.arange(n) // plan.page]
        see = (pg >= 0) & (pg < plan.pages)
        at = np.where(see, pg, 0)
        kk, vv = k[at, :, np.arange(n) % plan.page], v[at, :, np.arange(n) % plan.page]
        o = po.attend(q[row].reshape(nq, -1), kk, vv, see)
        out[row] = o * (po.sigmoid(gate[row].reshape(nq, -1)) if gate is not None else 1)
    return out


def filled(rng, kind, nkv, hd, page, plan, scale=1.0):
    """A pool whose sequences' positions hold values, all else NaN."""
    k, v = (np.full((plan.pages, nkv, page, hd), np.nan, np.float16) for _ in range(2))
    for s, (p, m) in enumerate(zip(plan.past, plan.rows)):
        for i in range((p + m + page - 1) // page):
            n = min(page, p + m - i * page)
            for x in (k, v):
                x[plan.table[s, i], :, :n] = rng.normal(0, scale, (nkv, n, hd)) * rng.uniform(0.2, 1.0)
    return Pool(kind, nkv, hd, page, plan.pages, 1, k, v)


def check(got, want, tol=3e-5):
    for row, w in want.items():
        err = np.abs(got[row] - w).max()
        assert err <= tol, (row, err)


ATTEND = [
    # nq, nkv, hd, page, past, rows
    (32, 8, 128, 64, [0], [1]), (32, 8, 128, 64, [0, 1, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 300], [1] * 13),
    (32, 8, 128, 32, [700], [1]), (32, 8, 128, 128, [2047, 5, 900], [1, 1, 1]), (16, 4, 256, 32, [0, 31, 32, 500, 1500], [1] * 5),
    (16, 4, 256, 128, [4000], [1]), (32, 8, 128, 64, [5000, 0, 3], [1, 0, 2]), (16, 4, 128, 64, [100], [4]), (16, 4, 128, 32, [100, 7], [8, 3]),
    (32, 8, 128, 64, [0], [70]), (32, 8, 128, 64, [61], [67]), (32, 8, 128, 32, [3, 200, 0, 1000], [100, 1, 1, 33]),
    (16, 4, 256, 64, [33], [65]), (16, 4, 256, 128, [0, 600], [40, 1]), (16, 2, 128, 64, [130], [5]), (16, 1, 128, 64, [130, 2], [1, 9]),
    (7, 7, 128, 32, [50], [33]), (12, 4, 128, 64, [77, 1], [1, 50]), (5, 1, 256, 32, [90], [30]), (15, 1, 128, 64, [20], [11]),
    (4, 2, 64, 32, [40, 3], [1, 20]), (6, 2, 80, 64, [64], [3]), (3, 3, 16, 32, [0, 100], [2, 1]), (4, 1, 240, 128, [200], [2]),
]


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("shape", ATTEND, ids=[f"{a[0]}_{a[1]}x{a[2]}_{a[3]}_{a[4][0]}_{a[5][0]}_{len(a[4])}" for a in ATTEND])
def test_attention(kind, shape):
    nq, nkv, hd, page, past, rows = shape
    rng = np.random.default_rng(nq + hd + page + sum(past))
    plan = Plan(rng, page, past, rows, pad=2)
    pool = filled(rng, kind, nkv, hd, page, plan)
    q, gate = (rng.normal(0, 1, (plan.total, nq * hd)).astype(np.float32) for _ in range(2))
    got = attention(pool, plan, nq, q, gate)
    check(got, attend_oracle(pool, plan, nq, q, gate))
    assert (got[plan.n:] == 7).all()


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("how", [dict(gate=False), dict(qs=8), dict(os=12), dict(qs=5), dict(os=3), dict(shift=1), dict(shift=2)])
@pytest.mark.parametrize("rows", [[1, 1], [40, 3]])
def test_attention_of_any_stride(kind, how, rows):
    rng = np.random.default_rng(11)
    plan = Plan(rng, 64, [100, 30], rows)
    pool = filled(rng, kind, 4, 128, 64, plan)
    q, gate = (rng.normal(0, 1, (plan.total, 16 * 128)).astype(np.float32) for _ in range(2))
    gate = gate if how.get("gate", True) else None
    got = attention(pool, plan, 16, q, gate, 16 * 128 + how.get("qs", 0), 16 * 128 + how.get("os", 0), how.get("shift", 0))
    check(got, attend_oracle(pool, plan, 16, q, gate))


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("hd", [128, 256])
def test_attention_of_many_sequences(kind, hd):
    """Lengths of every kind in one step: no rows, one position, thousands; chunks among single tokens."""
    rng = np.random.default_rng(12)
    past = [int(x) for x in np.exp(rng.uniform(0, np.log(3000), 90)) - 1]
    rows = [int(r) for r in rng.choice([1, 1, 1, 1, 0, 2, 9, 40], 90)]
    plan = Plan(rng, 32, past, rows, pad=3)
    pool = filled(rng, kind, 2, hd, 32, plan)
    q, gate = (rng.normal(0, 1, (plan.total, 8 * hd)).astype(np.float32) for _ in range(2))
    got = attention(pool, plan, 8, q, gate)
    check(got, attend_oracle(pool, plan, 8, q, gate))
    assert (got[plan.n:] == 7).all()


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("past,rows", [(131000, 1), (60001, 3), (20000, 40)])
def test_attention_of_long_contexts(kind, past, rows):
    """Some rows' results; V scales and magnitudes differ from page to page."""
    rng = np.random.default_rng(13)
    plan = Plan(rng, 128, [past, 10], [rows, 1])
    shape = (plan.pages, 1, 128, 128)
    k, v = (rng.normal(0, 1, shape).astype(np.float16) * np.exp2(rng.integers(-3, 3, shape[:2])).astype(np.float16)[..., None, None] for _ in "kv")
    pool = Pool(kind, 1, 128, 128, plan.pages, 1, k, v)
    q = rng.normal(0, 0.2, (plan.total, 512)).astype(np.float32)
    got = attention(pool, plan, 4, q, None)
    check(got, attend_oracle(pool, plan, 4, q, None, {0, rows - 1, rows}), 1e-4)


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("rows", [[1, 1, 1], [1, 30, 2]])
def test_pages_that_are_none(kind, rows):
    """Missing pages are not seen; a row without any gives 0."""
    rng = np.random.default_rng(14)
    plan = Plan(rng, 32, [200, 90, 40], rows)
    pool = filled(rng, kind, 2, 128, 32, plan)
    plan.table[0, [0, 3]] = -1, plan.pages
    plan.table[1, 1] = 1 << 30
    plan.table[2, :] = -7
    plan.upload()
    q = rng.normal(0, 1, (plan.total, 8 * 128)).astype(np.float32)
    got = attention(pool, plan, 8, q, None)
    check(got, attend_oracle(pool, plan, 8, q, None))
    assert (got[int(plan.row0[2]):] == 0).all()


@pytest.mark.parametrize("rows,max_rows", [([1, 4, 1], 2), ([9, 1, 3], 9)])
def test_bounds_of_a_step(rows, max_rows):
    """Rows past max_rows stay as they were; numbers out of order or range reach nothing; positions past the table are not seen."""
    rng = np.random.default_rng(15)
    plan = Plan(rng, 64, [100, 60, 127], rows, max_rows=max_rows)
    pool = filled(rng, F16, 2, 128, 64, plan)
    q = rng.normal(0, 1, (plan.total, 8 * 128)).astype(np.float32)
    got = attention(pool, plan, 8, q, None)
    want = attend_oracle(pool, plan, 8, q, None)
    check(got, want)
    for row in range(plan.total):
        assert row in want or (got[row] == 7).all()
    for row0, past in (([0, 5, 2, 4], [100, 60, 127]), ([-9, 1, 1 << 30, 1 << 30], [100, 60, 127]), ([1 << 30] * 4, [100] * 3),
                       ([0, 1, 2, 3], [-5, 1 << 30, 2**31 - 1])):
        p2 = Plan(rng, 64, [100, 60, 127], rows, max_rows=max_rows)
        p2.table, p2.pages, p2.row0, p2.past = plan.table, plan.pages, np.array(row0, np.int32), past
        p2.upload()
        got = attention(pool, p2, 8, q, None)
        prep(rng, Pool(I8, 2, 128, 64, plan.pages, 3), p2, 8, 0, cap=9)
    assert (got[0] == 0).all()  # no position
    full = {1: (1, plan.most * 64)}
    k, v = pool.values()
    for row, (s, n) in full.items():
        pg = plan.table[s, np.arange(n) // 64]
        see = pg >= 0
        kk, vv = k[np.where(see, pg, 0), :, np.arange(n) % 64], v[np.where(see, pg, 0), :, np.arange(n) % 64]
        ok = ~np.isnan(kk).any((1, 2))
        if ok[see].all():
            check(got, {row: po.attend(q[row].reshape(8, -1), kk, vv, see)})


@pytest.mark.parametrize("rows", [[1, 1], [20, 1]])
@pytest.mark.parametrize("hd", [128, 256])
def test_values_that_are_not_finite(rows, hd):
    """fp16 pages: infinities and NaN reach the rows that see them, and no others."""
    rng = np.random.default_rng(16)
    plan = Plan(rng, 32, [50, 70], rows)
    k, v = (rng.normal(0, 1, (plan.pages, 2, 32, hd)).astype(np.float16) for _ in "kv")
    at = lambda s, pos: (plan.table[s, pos // 32], slice(None), pos % 32)  # noqa: E731
    last = 50 + rows[0] - 1
    v[at(0, last)] = np.inf        # the last row of sequence 0 alone
    if rows[0] > 4:
        v[at(0, last - 2)] = np.nan
        k[at(0, last - 4)] = -np.inf
    pool = Pool(F16, 2, hd, 32, plan.pages, 1, k, v)
    q = np.abs(rng.normal(0, 1, (plan.total, 8 * hd))).astype(np.float32)  # scores of minus infinity there
    got = attention(pool, plan, 8, q, None)
    with np.errstate(invalid="ignore"):
        want = attend_oracle(pool, plan, 8, q, None)
    for row, w in want.items():
        assert (np.isnan(got[row]) == np.isnan(w)).all() and (np.isinf(got[row]) == np.isinf(w)).all(), row
        fine = np.isfinite(w)
        assert np.abs(got[row][fine] - w[fine]).max(initial=0) <= 3e-5
    assert not np.isfinite(got[rows[0] - 1]).all() and np.isfinite(got[rows[0]]).all()


@pytest.mark.parametrize("kind", [F16, I8])
def test_large_and_small_values(kind):
    """Scores far apart (up to 2^10 in the exponent), values from 2^-14 to 2^12: relative to the largest value seen."""
    rng = np.random.default_rng(17)
    plan = Plan(rng, 64, [900, 130], [1, 40])
    shape = (plan.pages, 2, 64, 128)
    k = (rng.normal(0, 1, shape) * np.exp2(rng.uniform(-6, 4, shape[:3]))[..., None]).astype(np.float16)
    v = (rng.normal(0, 1, shape) * np.exp2(rng.integers(-14, 12, shape[:2]))[..., None, None]).astype(np.float16)
    pool = Pool(kind, 2, 128, 64, plan.pages, 1, k, v)
    q = rng.normal(0, 3, (plan.total, 8 * 128)).astype(np.float32)
    got, want = attention(pool, plan, 8, q, None), attend_oracle(pool, plan, 8, q, None)
    vals = pool.values()[1]
    for s, j, row, pos in plan.each():
        seen = plan.seq_values(vals, s, pos + 1)
        # a score of |q||k| / sqrt(hd) <= 3 x 16 x 16 x 1.5 is off by 2^-22 of its terms: weights by 3e-4
        assert np.abs(got[row] - want[row]).max() <= 6e-4 * np.abs(seen).max(), row


@pytest.mark.parametrize("rows", [[1, 1], [37, 1]])
@pytest.mark.parametrize("zero", ["k", "v", "kv"])
def test_pages_of_zeros(rows, zero):
    """8-bit pages with the scale 0, wholly and partly seen."""
    rng = np.random.default_rng(27)
    plan = Plan(rng, 64, [20, 150], rows)
    k, v = (rng.normal(0, 1, (plan.pages, 2, 64, 128)).astype(np.float16) for _ in "kv")
    for m, x in (("k", k), ("v", v)):
        if m in zero:
            x[plan.table[0]] = 0
            x[plan.table[1, [0, 2]]] = 0
    pool = Pool(I8, 2, 128, 64, plan.pages, 1, k, v)
    q = rng.normal(0, 1, (plan.total, 8 * 128)).astype(np.float32)
    check(attention(pool, plan, 8, q, None), attend_oracle(pool, plan, 8, q, None))


def test_sequences_share_pages():
    """A prompt's pages in three tables."""
    rng = np.random.default_rng(18)
    plan = Plan(rng, 32, [100, 100, 100], [1, 1, 1])
    plan.table[1, :3], plan.table[2, :3] = plan.table[0, :3], plan.table[0, :3]
    plan.upload()
    for kind in (F16, I8):
        pool = filled(rng, kind, 2, 128, 32, plan)
        q = rng.normal(0, 1, (3, 8 * 128)).astype(np.float32)
        check(attention(pool, plan, 8, q, None), attend_oracle(pool, plan, 8, q, None))


@pytest.mark.parametrize("kind", [F16, I8])
def test_pools_past_32_bits(kind):
    """Pages whose offsets pass 2^32 bytes: written, read back and attended to."""
    rng = np.random.default_rng(19)
    nkv, hd, page = 8, 128, 128
    each = nkv * hd * page * (1 if kind == I8 else 2)
    pages = (9 << 29) // each  # 4.5 GiB
    plan = Plan(rng, page, [300], [5])
    plan.table[0, :3] = pages - 1, 2, pages // 2 + 7
    plan.pages = pages
    plan.upload()
    big = [xb.DeviceBuffer(pages * each) for _ in range(2)]
    scale = [dev(np.zeros(pages * nkv, np.float32)) for _ in range(2)]
    open_ = [dev(np.zeros(nkv * page * hd, np.float16)) for _ in range(2)]
    _held.extend(big)
    pool = Pool(kind, nkv, hd, page, 1)
    pool.c = xb.Pages(kind, nkv, hd, page, pages, 1, big[0].ptr, big[1].ptr, *(b.ptr for b in scale + open_))
    pool.ref, pool.pages = ctypes.byref(pool.c), pages
    plan.open[:] = 0
    kv, x0 = [], rng.normal(0, 1, (305, 512 * 2 + 2 * nkv * hd)).astype(np.float32)
    norms = [np.ones(hd, np.float32)] * 2
    for past, rows in (([0], [300]), ([300], [5])):
        p = Plan(rng, page, past, rows)
        p.table, p.most, p.pages, p.open = plan.table, plan.most, pages, plan.open
        p.upload()
        prep(rng, pool, p, 4, 32, x=x0[past[0]: past[0] + rows[0]], norms=norms, cap=400)
    whole = Plan(rng, page, [0], [305])
    whole.table, whole.most, whole.pages = plan.table, plan.most, pages
    whole.upload()
    bufs = [dev(np.zeros(305 * nkv * hd, np.float32)) for _ in "kv"]
    xb.ck(xb.hip().xqhip_paged_read(pool.ref, whole.ref, xb.F32, bufs[0].ptr, bufs[1].ptr, None))
    k, v = (b.download(np.float32, 305 * nkv * hd).reshape(305, nkv, hd).astype(np.float64) for b in bufs)
    vx = split_heads(x0, 4, nkv, hd, 1)[3]
    # a code is off by half a step of max / 127 (max <= 6), an fp16 value by 2^-11 of it
    assert np.abs(v - vx).max() <= (6 / 254 if kind == I8 else 6 * 2**-11)
    q = rng.normal(0, 1, (5, 32 * hd)).astype(np.float32)
    got = attention(pool, plan, 32, q, None)
    for j in range(5):
        assert np.abs(got[j] - po.attend(q[j].reshape(32, hd), k[:301 + j], v[:301 + j], np.ones(301 + j, bool))).max() <= 3e-5


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("rows", [[1] * 6, [1, 50, 1, 0, 3, 17]])
def test_attention_is_the_same_every_time(kind, rows):
    """Bit for bit: no sum's order depends on chance; after an LDS and a workspace full of NaN too."""
    rng = np.random.default_rng(20)
    plan = Plan(rng, 64, [3000, 5, 700, 64, 1200, 0], rows)
    pool = filled(rng, kind, 4, 128, 64, plan)
    q = rng.normal(0, 1, (plan.total, 16 * 128)).astype(np.float32)
    first = attention(pool, plan, 16, q, None)
    for _ in range(3):
        xb.ck(xb.hip().xqhip_lds_fill(float("nan"), None))
        assert (attention(pool, plan, 16, q, None) == first).all()


# ---- log probabilities ----------------------------------------------------------
def run_logprobs(x, tokens, inv_t=1.0, top=5, f16=False, ld=None, shift=0, outs=(1, 1, 1, 1, 1), stream=None):
    rows, vocab = x.shape
    ld, t, L = ld or vocab, np.float16 if f16 else np.float32, xb.hip()
    y = np.full(rows * ld + shift, np.nan, t)
    y[shift:].reshape(rows, ld)[:, :vocab] = x
    need = L.xqhip_token_logprobs_workspace_bytes(rows, vocab, top)
    bufs = [dev(np.full(max(1, n), 7, d)) for n, d in ((rows, np.float32), (rows, np.float32), (rows, np.int32), (rows * top, np.int32),
                                                       (rows * top, np.float32))]
    ptrs = [b.ptr if on else None for b, on in zip(bufs, outs)]
    xb.ck(L.xqhip_token_logprobs(ctypes.c_void_p(dev(y).ptr.value + shift * y.itemsize), xb.F16 if f16 else xb.F32, ld, rows, vocab, inv_t,
                                 i32(tokens).ptr if tokens is not None else None, top, *ptrs, dev(np.full(need, 0xff, np.uint8)).ptr, need, stream))
    xb.ck(L.xqhip_stream_synchronize(stream))
    lp, en = (b.download(np.float32, rows) for b in bufs[:2])
    return [lp, en, bufs[2].download(np.int32, rows), bufs[3].download(np.int32, rows * top).reshape(rows, top) if top else None,
            bufs[4].download(np.float32, rows * top).reshape(rows, top) if top else None]


def check_logprobs(got, x, tokens, inv_t, top):
    """exp's argument d = (x - m) / T carries two roundings, exp and the sum a few more: the sum, and with it log p, is off by
    1e-6 of itself (of 1 where it is larger) plus 2^-23 |d|; the entropy, sums of terms under 0.4 each of which is off by
    1e-6 |d| of itself, by 1e-5 of what it is, plus 1e-6."""
    lp, en, rank, ids, tops = got
    for r in range(len(x)):
        want = po.logprobs(x[r], tokens[r], inv_t, top)

        def near(a, b):
            return a == b or abs(a - b) <= 1e-6 * min(1, abs(b)) + 3 * 2**-23 * abs(b) + 1e-12

        assert near(lp[r], want[0]), (r, lp[r], want[0])
        assert abs(en[r] - want[1]) <= 1e-5 * abs(want[1]) + 1e-6, (r, en[r], want[1])
        assert rank[r] == want[2]
        if top:
            assert (ids[r] == want[3]).all(), (r, ids[r], want[3])
            assert all(near(a, b) for a, b in zip(tops[r], want[4]))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rows,vocab,top,inv_t", [(1, 1, 1, 1.0), (3, 2, 5, 1.0), (2, 63, 64, 0.5), (5, 64, 20, 1.0), (2, 65, 3, 2.0), (4, 1000, 64, 1.3),
                                                  (2, 4095, 20, 1.0), (2, 4097, 20, 1.0), (3, 8193, 1, 1.0), (2, 50257, 20, 0.7), (1, 248320, 5, 1.0),
                                                  (7, 248320, 64, 1.0), (70, 16385, 0, 1.0), (300, 5003, 7, 1.1)])
def test_logprobs(rows, vocab, top, inv_t, f16):
    rng = np.random.default_rng(rows + vocab)
    x = (rng.normal(0, 3, (rows, vocab)) * rng.uniform(0.2, 3, (rows, 1))).astype(np.float16 if f16 else np.float32)
    tokens = [int(t) for t in rng.integers(0, vocab, rows)]
    tokens[0] = int(np.argmax(x[0]))
    check_logprobs(run_logprobs(x, tokens, inv_t, top, f16), x, tokens, inv_t, top)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("ld,shift", [(1003, 0), (1004, 0), (1008, 0), (1008, 1), (1008, 4), (1001, 3)])
def test_logprobs_of_any_stride(ld, shift, f16):
    rng = np.random.default_rng(ld)
    x = rng.normal(0, 3, (9, 1001)).astype(np.float16 if f16 else np.float32)
    tokens = [int(t) for t in rng.integers(0, 1001, 9)]
    check_logprobs(run_logprobs(x, tokens, 1.0, 10, f16, ld, shift), x, tokens, 1.0, 10)


@pytest.mark.parametrize("vocab", [700, 1022, 1027, 8190, 8193, 30000])
def test_logprobs_of_special_rows(vocab):
    """Ties, masked tokens, rows that leave nothing or one token, infinities, NaN, tokens that are none, rows that rise or fall."""
    rng = np.random.default_rng(21)
    x = rng.normal(0, 2, (16, vocab)).astype(np.float32)
    x[0] = 1.5                                            # all the same
    x[1] = np.round(x[1])                                 # many ties
    x[2] = -np.inf                                        # nothing
    x[3, np.arange(vocab) != 77] = -np.inf                # one token
    x[4, rng.random(vocab) < 0.999] = -np.inf             # fewer than top
    x[5, [5, 600]] = np.inf
    x[6, 3:500] = np.nan
    x[7] = np.nan
    x[8] = np.arange(vocab)                               # rising
    x[9] = -np.arange(vocab)                              # falling
    x[10] *= 1e30
    x[11, 9] = 200.0                                      # sure: log p of the others near -200, its own near 0
    x[12] = np.float32(-3.4e38)                           # the type's lowest value everywhere
    x[12, 50] = 0
    x[13] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    x[14, :] = 3.0e38
    tokens = [3, 10, 4, 77, 0, 600, 4, 1, vocab - 1, vocab - 1, 20, 9, 51, 1, 5, -1]
    for t15 in (-1, vocab, 2**31 - 1):
        tokens[15] = t15
        with np.errstate(over="ignore"):
            check_logprobs(run_logprobs(x, tokens, 1.0, 20), x, tokens, 1.0, 20)


@pytest.mark.parametrize("top", [1, 20, 64])
def test_logprobs_where_one_place_holds_the_first(top):
    """All the largest logits next to each other, or at the stride of any thread count: the lists are the same."""
    rng = np.random.default_rng(22)
    x = rng.normal(0, 1, (6, 70000)).astype(np.float32)
    for r, places in enumerate((np.arange(500), 69000 + np.arange(900), np.arange(0, 70000, 64), np.arange(3, 70000, 256), np.arange(5, 70000, 1024),
                                np.arange(1, 70000, 4096))):
        x[r, places] += 50 + rng.normal(0, 1, len(places)).astype(np.float32)
    tokens = [499, 69899, 64, 3, 5, 4097]
    check_logprobs(run_logprobs(x, tokens, 1.0, top), x, tokens, 1.0, top)


@pytest.mark.parametrize("outs", [(1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 0), (0, 0, 0, 1, 0), (0, 0, 0, 0, 1), (0, 1, 0, 1, 1)])
def test_logprobs_outputs_alone(outs):
    rng = np.random.default_rng(23)
    x = rng.normal(0, 2, (3, 20000)).astype(np.float32)
    tokens = [5, 19999, 777]
    need_tokens = outs[0] or outs[2]
    all_of = run_logprobs(x, tokens, 1.0, 6)
    got = run_logprobs(x, tokens if need_tokens else None, 1.0, 6, outs=outs)
    for a, b, on in zip(got, all_of, outs):
        assert (a == b).all() if on else (a == 7).all()


# ---- together -------------------------------------------------------------------
@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("hd,nq,nkv,page", [(128, 8, 2, 64), (256, 8, 2, 32)])
def test_steps_of_several_sequences(kind, hd, nq, nkv, page):
    """Prompts of three sequences in chunks, then tokens one by one, one sequence with an image's positions: q, pages,
    attention and log probabilities of a head over the attention's output, step by step against the definition."""
    rng = np.random.default_rng(24)
    plans = [([0, 0, 0], [50, 20, 33]), ([50, 20, 33], [45, 1, 1]), ([95, 21, 34], [1, 1, 0]), ([96, 22, 34], [1, 1, 1])]
    whole = Plan(rng, page, [0, 0, 0], [100, 30, 40])
    pool = Pool(kind, nkv, hd, page, whole.pages, 3)
    model, norms = pool.raw(), [rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2)]
    head = rng.normal(0, 0.1, (nq * hd, 501)).astype(np.float32)
    for past, rows in plans:
        plan = Plan(rng, page, past, rows)
        plan.table, plan.most, plan.open, plan.pages = whole.table, whole.most, whole.open, whole.pages
        plan.upload()
        axes = np.zeros((3, plan.total), np.int32)
        for s, j, row, pos in plan.each():
            axes[:, row] = (pos, pos // 7, pos % 7) if s == 0 else pos
        x, q, g, (qn, kn), cs = prep(rng, pool, plan, nq, 32, [6, 5, 5], True, axes, norms=norms, cap=200)
        _, gx, kx, vx = split_heads(x, nq, nkv, hd, 1)
        model = appended(model, plan, kind, po.prepared(kx, kn, cs[:, None], EPS), vx)
        assert same(pool.raw(), model)
        flat, gate = q.reshape(plan.total, -1), g.reshape(plan.total, -1)
        out = attention(pool, plan, nq, flat, gate)
        check(out, attend_oracle(pool, plan, nq, flat, gate))
        logits = (out.reshape(plan.total, -1) @ head).astype(np.float32)
        tokens = [int(t) for t in logits.argmax(-1)]
        check_logprobs(run_logprobs(logits, tokens, 1.0, 5), logits, tokens, 1.0, 5)


@pytest.mark.parametrize("kind", [F16, I8])
def test_captured_steps(kind):
    """A decode step captured once and replayed at growing lengths (and with another table), eager work between; two graphs
    share one workspace, one after the other."""
    L, rng = xb.hip(), np.random.default_rng(25)
    nq, nkv, hd, page, seqs = 8, 2, 128, 32, 4
    whole = Plan(rng, page, [0] * seqs, [150] * seqs)
    pool = Pool(kind, nkv, hd, page, whole.pages, seqs)
    ref_pool = Pool(kind, nkv, hd, page, whole.pages, seqs)
    wq = 2 * nq * hd
    row = wq + 2 * nkv * hd
    norms = [rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2)]
    start = Plan(rng, page, [0] * seqs, [60, 31, 1, 95])
    steps = [start] + [Plan(rng, page, [n + i for n in (60, 31, 1, 95)], [1] * seqs) for i in range(4)]
    for p in steps:
        p.table, p.most, p.open, p.pages = whole.table, whole.most, whole.open, whole.pages
        p.upload()
    x0 = rng.normal(0, 1, (start.total, row)).astype(np.float32)
    for pl in (pool, ref_pool):
        prep(rng, pl, start, nq, 32, x=x0, norms=norms, cap=300)
    stream = ctypes.c_void_p()
    xb.ck(L.xqhip_stream_create(ctypes.byref(stream)))
    src, q, gate, out = (xb.DeviceBuffer(4 * seqs * n) for n in (row, nq * hd, nq * hd, nq * hd))
    logp = xb.DeviceBuffer(4 * seqs)
    plan = Plan(rng, page, steps[1].past, [1] * seqs)
    plan.table, plan.most, plan.open, plan.pages = whole.table, whole.most, whole.open, whole.pages
    plan.upload()
    rot = xb.rotary(dev(rope(32, 300)).ptr, 300, 32, [16])
    need = L.xqhip_paged_attention_workspace_bytes(nq, nkv, hd)
    need2 = L.xqhip_token_logprobs_workspace_bytes(seqs, nq * hd, 0)
    ws, qn, kn, tok = dev(np.full(max(need, need2), 0xff, np.uint8)), dev(norms[0]), dev(norms[1]), i32([3] * seqs)
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    graphs = []
    for _ in range(2):
        xb.ck(L.xqhip_graph_begin(stream))
        xb.ck(L.xqhip_attn_prep_paged(at(0), at(wq), at(wq + nkv * hd), 1, nq, qn.ptr, kn.ptr, EPS, ctypes.byref(rot), plan.ref, row,
                                      nq * hd, q.ptr, gate.ptr, pool.ref, stream))
        xb.ck(L.xqhip_paged_attention(q.ptr, gate.ptr, pool.ref, nq, plan.ref, nq * hd, out.ptr, nq * hd, ws.ptr, need, stream))
        xb.ck(L.xqhip_token_logprobs(out.ptr, xb.F32, nq * hd, seqs, nq * hd, 1.0, tok.ptr, 0, logp.ptr, None, None, None, None, ws.ptr,
                                     need2, stream))
        g = ctypes.c_void_p()
        xb.ck(L.xqhip_graph_end(stream, ctypes.byref(g)))
        graphs.append(g)
    for i, want_plan in enumerate(steps[1:]):
        x = rng.normal(0, 1, (seqs, row)).astype(np.float32)
        past = np.array(want_plan.past, np.int32)
        xb.ck(L.xqhip_memcpy_h2d(src.ptr, xb.ptr(x), x.nbytes, stream))
        xb.ck(L.xqhip_memcpy_h2d(plan.bufs[1].ptr, xb.ptr(past), past.nbytes, stream))
        xb.ck(L.xqhip_graph_launch(graphs[i % 2], stream))
        xb.ck(L.xqhip_stream_synchronize(stream))
        got = out.download(np.float32, seqs * nq * hd).reshape(seqs, nq, hd)
        _, q2, g2, _, _ = prep(rng, ref_pool, want_plan, nq, 32, x=x, norms=norms, cap=300)
        eager = attention(ref_pool, want_plan, nq, q2.reshape(seqs, -1), g2.reshape(seqs, -1))
        assert (got == eager).all()
        assert same(pool.raw(), ref_pool.raw())
        lp = run_logprobs(eager.reshape(seqs, -1), [3] * seqs, 1.0, 0)[0]
        assert (logp.download(np.float32, seqs) == lp).all()
    for g in graphs:
        xb.ck(L.xqhip_graph_destroy(g))
    xb.ck(L.xqhip_stream_destroy(stream))


def test_two_streams_at_once():
    L, rng = xb.hip(), np.random.default_rng(26)
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        xb.ck(L.xqhip_stream_create(ctypes.byref(s)))
        streams.append(s)
    sides = []
    for kind, rows in ((F16, [1] * 5), (I8, [60, 1, 3, 1, 1])):
        plan = Plan(rng, 64, [2000, 5, 700, 64, 1200], rows)
        pool = filled(rng, kind, 4, 128, 64, plan)
        q = rng.normal(0, 1, (plan.total, 16 * 128)).astype(np.float32)
        alone = attention(pool, plan, 16, q, None)
        need = L.xqhip_paged_attention_workspace_bytes(16, 4, 128)
        sides.append((pool, plan, dev(q), dev(np.zeros_like(q)), dev(np.full(need, 0xff, np.uint8)), need, alone))
    for _ in range(20):
        for s, (pool, plan, q, out, ws, need, _) in zip(streams, sides):
            xb.ck(L.xqhip_paged_attention(q.ptr, None, pool.ref, 16, plan.ref, 2048, out.ptr, 2048, ws.ptr, need, s))
    for s, (_, plan, _, out, _, _, alone) in zip(streams, sides):
        xb.ck(L.xqhip_stream_synchronize(s))
        assert (out.download(np.float32, plan.total * 2048).reshape(alone.shape) == alone).all()
        xb.ck(L.xqhip_stream_destroy(s))


# ---- sizes at which other kernels, or other parts of them, run --------------------
def attend_rows(pool, plan, nq, q, gate, picks):
    """attend_oracle for many rows at once (every page of the sequences there): {row: [nq][hd]} of the rows in `picks`."""
    k, v = pool.values()
    g, hd, out = nq // pool.nkv, pool.hd, {}
    for s, m in enumerate(plan.rows):
        js = np.array([j for j in range(m) if int(plan.row0[s]) + j in picks], int)
        if not len(js):
            continue
        n = min(plan.past[s] + m, plan.most * plan.page)
        kk, vv = plan.seq_values(k, s, n), plan.seq_values(v, s, n)
        rows = int(plan.row0[s]) + js
        hidden = np.arange(n)[None] > plan.past[s] + js[:, None]
        o = np.empty((len(js), nq, hd))
        for h in range(nq):
            z = q[rows].reshape(len(js), nq, hd)[:, h].astype(np.float64) @ kk[:, h // g].T / math.sqrt(hd)
            z[hidden] = -np.inf
            e = np.exp(z - z.max(-1, keepdims=True))
            o[:, h] = e @ vv[:, h // g] / e.sum(-1, keepdims=True)
        if gate is not None:
            o = o * po.sigmoid(gate[rows].reshape(len(js), nq, hd))
        out.update(zip(rows.tolist(), o))
    return out


MANY = [
    # nq, nkv, hd, page, past, rows: blocks of 64 columns with and without splits, and of 128
    (32, 8, 128, 64, [0, 100, 40], [700, 400, 1]), (16, 1, 128, 128, [40000, 3], [200, 1]), (8, 1, 256, 64, [5000, 0], [600, 1]),
    (32, 2, 256, 32, [70, 3000, 5], [40, 1, 9]), (10, 2, 128, 32, [1000, 0, 500], [333, 12, 3]), (128, 64, 128, 32, [130, 5, 61], [50, 1, 4]),
    (256, 256, 128, 32, [33, 90], [21, 1]), (256, 256, 256, 32, [40], [18]), (16, 16, 128, 64, [900] * 3, [129, 128, 127]),
    (3, 3, 128, 128, [0], [1500]), (64, 4, 128, 64, [250, 1030], [300, 5]),
]


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("shape", MANY, ids=[f"{a[0]}_{a[1]}x{a[2]}_{a[4][0]}_{a[5][0]}" for a in MANY])
def test_attention_of_many_rows(kind, shape):
    nq, nkv, hd, page, past, rows = shape
    rng = np.random.default_rng(nq + sum(rows))
    plan = Plan(rng, page, past, rows, pad=1)
    pool = filled(rng, kind, nkv, hd, page, plan)
    q, gate = (rng.normal(0, 1, (plan.total, nq * hd)).astype(np.float32) for _ in range(2))
    got = attention(pool, plan, nq, q, gate)
    check(got, attend_rows(pool, plan, nq, q, gate, set(range(plan.n))))
    assert (got[plan.n:] == 7).all()


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("most", [1, 2, 30])
def test_a_step_of_as_many_sequences_as_there_can_be(kind, most):
    rng = np.random.default_rng(28)
    rows = [int(r) for r in rng.choice([0, 1, 1, 1, most], 1024)]
    plan = Plan(rng, 32, [int(p) for p in rng.integers(0, 90, 1024)], rows, pad=1)
    pool = Pool(kind, 3, 128, 32, plan.pages, 1024, *(rng.normal(0, 1, (plan.pages, 3, 32, 128)).astype(np.float16) for _ in "kv"))
    for b in pool.open:
        xb.ck(xb.hip().xqhip_fill_u8(b.ptr, 0, 1024 * 3 * 32 * 128 * 2, None))
    was = pool.raw()
    x, q, g, (qn, kn), cs = prep(rng, pool, plan, 6, 32, cap=200)
    _, gx, kx, vx = split_heads(x, 6, 3, 128, 1)
    assert (g[:plan.n] == gx[:plan.n]).all() and (q[plan.n:] == 7).all()
    assert same(pool.raw(), appended(was, plan, kind, po.prepared(kx, kn, cs[:, None], EPS), vx))
    flat, gate = q.reshape(plan.total, -1), g.reshape(plan.total, -1)
    got = attention(pool, plan, 6, flat, gate)
    check(got, attend_oracle(pool, plan, 6, flat, gate))
    assert (got[plan.n:] == 7).all()


@pytest.mark.parametrize("kind", [F16, I8])
def test_a_prompt_of_as_many_rows_as_there_can_be(kind):
    rng = np.random.default_rng(29)
    plan = Plan(rng, 128, [1], [65535])
    plan.past[0] = 0
    plan.upload()
    pool = Pool(kind, 1, 128, 128, plan.pages)
    was = pool.raw()
    x, q, g, (qn, kn), cs = prep(rng, pool, plan, 2, 32)
    _, _, kx, vx = split_heads(x, 2, 1, 128, 1)
    assert same(pool.raw(), appended(was, plan, kind, po.prepared(kx, kn, cs[:, None], EPS), vx))
    flat = q.reshape(plan.total, -1)
    got = attention(pool, plan, 2, flat, None)
    assert np.isfinite(got).all()
    check(got, attend_rows(pool, plan, 2, flat, None, {0, 1, 31, 32, 127, 128, 4000, 32767, 50001, 65534}), 1e-4)


@pytest.mark.parametrize("nq,nkv,hd,page,past,rows", [(512, 256, 16, 32, [31, 5], [40, 1]), (300, 100, 128, 64, [0, 63], [3, 2]), (65, 1, 32, 128, [127], [1])])
@pytest.mark.parametrize("kind", [F16, I8])
def test_prep_of_many_heads(kind, nq, nkv, hd, page, past, rows):
    rng = np.random.default_rng(30)
    plan = Plan(rng, page, past, rows, pad=1)
    pool = Pool(kind, nkv, hd, page, plan.pages, len(past), *(rng.normal(0, 1, (plan.pages, nkv, page, hd)).astype(np.float16) for _ in "kv"))
    for b in pool.open:
        xb.ck(xb.hip().xqhip_fill_u8(b.ptr, 0, len(past) * nkv * page * hd * 2, None))
    was = pool.raw()
    x, q, g, (qn, kn), cs = prep(rng, pool, plan, nq, 16, cap=300)
    qx, gx, kx, vx = split_heads(x, nq, nkv, hd, 1)
    want = po.prepared(qx, qn, cs[:, None], EPS)
    assert (np.abs(q[:plan.n] - want[:plan.n]) <= 2**-23 * np.abs(want[:plan.n])).all() and (g[:plan.n] == gx[:plan.n]).all()
    assert same(pool.raw(), appended(was, plan, kind, po.prepared(kx, kn, cs[:, None], EPS), vx))


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("rows", [1, 2, 40])
def test_a_page_stands_twice_in_a_table(kind, rows):
    rng = np.random.default_rng(31)
    plan = Plan(rng, 32, [150], [rows])
    pool = filled(rng, kind, 2, 128, 32, plan)
    plan.table[0, 1] = plan.table[0, 3] = plan.table[0, 0]
    plan.upload()
    q = rng.normal(0, 1, (rows, 8 * 128)).astype(np.float32)
    check(attention(pool, plan, 8, q, None), attend_oracle(pool, plan, 8, q, None))


@pytest.mark.parametrize("kind", [F16, I8])
def test_captured_steps_of_changing_rows(kind):
    """Prep and attention captured once for steps of up to 100 rows, up to 64 of a sequence, then replayed with other divisions of the
    rows: prompts' chunks, single tokens, sequences without rows, no rows at all; eager work and synchronizations between."""
    L, rng = xb.hip(), np.random.default_rng(32)
    nq, nkv, hd, page, seqs, total = 8, 2, 128, 32, 5, 100
    steps = [[64, 20, 0, 10, 6], [1, 1, 30, 1, 1], [64, 0, 30, 1, 5], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1], [2, 33, 1, 0, 64]]
    ends = np.sum(steps, 0)
    whole = Plan(rng, page, [0] * seqs, [int(n) for n in ends])
    pool, ref_pool = (Pool(kind, nkv, hd, page, whole.pages, seqs) for _ in range(2))
    wq, norms = 2 * nq * hd, [rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2)]
    row = wq + 2 * nkv * hd
    rot = xb.rotary(dev(rope(32, 300)).ptr, 300, 32, [16])
    need = L.xqhip_paged_attention_workspace_bytes(nq, nkv, hd)
    ws, qn, kn = dev(np.full(need, 0xff, np.uint8)), dev(norms[0]), dev(norms[1])

    def plan_of(past, rows):
        p = Plan(rng, page, past, rows, pad=total - sum(rows), max_rows=64)
        p.table, p.most, p.open, p.pages = whole.table, whole.most, whole.open, whole.pages
        p.upload()
        return p

    plan = plan_of([0] * seqs, steps[0])
    src, q, gate, out = (xb.DeviceBuffer(4 * total * n) for n in (row, nq * hd, nq * hd, nq * hd))
    at = lambda f: ctypes.c_void_p(src.ptr.value + 4 * f)  # noqa: E731
    stream, g = ctypes.c_void_p(), ctypes.c_void_p()
    xb.ck(L.xqhip_stream_create(ctypes.byref(stream)))
    xb.ck(L.xqhip_graph_begin(stream))
    xb.ck(L.xqhip_attn_prep_paged(at(0), at(wq), at(wq + nkv * hd), 1, nq, qn.ptr, kn.ptr, EPS, ctypes.byref(rot), plan.ref, row, nq * hd,
                                  q.ptr, gate.ptr, pool.ref, stream))
    xb.ck(L.xqhip_paged_attention(q.ptr, gate.ptr, pool.ref, nq, plan.ref, nq * hd, out.ptr, nq * hd, ws.ptr, need, stream))
    xb.ck(L.xqhip_graph_end(stream, ctypes.byref(g)))
    past = np.zeros(seqs, np.int32)
    for rows in steps:
        now = plan_of([int(p) for p in past], rows)
        x = rng.normal(0, 1, (total, row)).astype(np.float32)
        filler = np.full(total * nq * hd, 7, np.float32)
        for buf, a in ((src, x), (plan.bufs[0], now.row0), (plan.bufs[1], past), (out, filler), (q, filler), (gate, filler)):
            xb.ck(L.xqhip_memcpy_h2d(buf.ptr, xb.ptr(np.ascontiguousarray(a)), a.nbytes, stream))
        xb.ck(L.xqhip_graph_launch(g, stream))
        xb.ck(L.xqhip_stream_synchronize(stream))
        got = out.download(np.float32, total * nq * hd).reshape(total, nq, hd)
        _, q2, g2, _, _ = prep(rng, ref_pool, now, nq, 32, x=x, norms=norms, cap=300)
        assert (q.download(np.float32, total * nq * hd).reshape(q2.shape) == q2).all()
        eager = attention(ref_pool, now, nq, q2.reshape(total, -1), g2.reshape(total, -1))
        assert (got == eager).all() and (got[now.n:] == 7).all()
        check(got, attend_oracle(ref_pool, now, nq, q2.reshape(total, -1), g2.reshape(total, -1)))
        assert same(pool.raw(), ref_pool.raw())
        past = past + np.array(rows, np.int32)
    xb.ck(L.xqhip_graph_destroy(g))
    xb.ck(L.xqhip_stream_destroy(stream))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("vocab", [1, 3, 7, 8, 9, 1023, 1024, 1025, 1029, 8191, 8192, 8193])
@pytest.mark.parametrize("masked", [0.0, 0.5, 0.99])
def test_logprobs_of_few_logits(vocab, masked, f16):
    """Rows that one block holds and the next sizes, masked tokens asked for too."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 3, (8, vocab)).astype(np.float16 if f16 else np.float32)
    x[rng.random(x.shape) < masked] = -np.inf
    x[1] = np.round(x[1])
    tokens = [int(t) for t in rng.integers(0, vocab, 8)]
    tokens[2], tokens[3] = vocab - 1, max(0, vocab - 2)
    x[3, tokens[3]] = -np.inf
    for ld in (vocab, (vocab + 7) // 8 * 8):
        for top in (0, 1, 20, 64):
            check_logprobs(run_logprobs(x, tokens, 1.0, top, f16, ld), x, tokens, 1.0, top)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rows,vocab,top", [(2, 262145, 20), (2, 300001, 64), (1, 600000, 5), (2, 1048577, 1), (1, 2500003, 64), (1, 1 << 24, 20)])
def test_logprobs_of_large_vocabularies(rows, vocab, top, f16):
    """Ranks are exact where a row's largest logits come late, early and equal."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((rows, vocab), np.float32) * 2
    x[0, -3:] = x[0].max() + 1
    x[-1, 7] = 20
    if f16:
        x = x.astype(np.float16)
    tokens = [vocab - 1, vocab // 2][:rows]
    check_logprobs(run_logprobs(x, tokens, 1.0, top, f16), x, tokens, 1.0, top)


def test_logprobs_of_as_many_rows_as_there_can_be():
    rng = np.random.default_rng(33)
    x = rng.normal(0, 3, (65535, 33)).astype(np.float32)
    tokens = [int(t) for t in rng.integers(0, 33, 65535)]
    lp, en, rank, ids, tops = run_logprobs(x, tokens, 1.0, 2)
    at = [0, 1, 32767, 40000, 65534]
    check_logprobs([a[at] for a in (lp, en, rank, ids, tops)], x[at], [tokens[i] for i in at], 1.0, 2)
    z = x.astype(np.float64) - x.max(-1, keepdims=True)
    want = z[np.arange(65535), tokens] - np.log(np.exp(z).sum(-1))
    assert np.abs(lp - want).max() <= 1e-5 and (ids[:, 0] == x.argmax(-1)).all()
    assert (rank == (x > x[np.arange(65535), tokens][:, None]).sum(-1)).all()
