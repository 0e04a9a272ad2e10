"""The kernels over paged caches run on the host (host_kernels): their own sources under AddressSanitizer, every buffer of
exactly the size that the interface asks for, workspaces and outputs full of 0xA5.  So what an index reaches is shown without a
GPU; the results are compared with the 64-bit ones as on the GPU (the same bounds, test_paged_gpu)."""
import os

import numpy as np
import pytest

import host_kernels as hk
import paged_oracle as po
import test_paged_gpu as gpu
import xqbind as xb

pytestmark = pytest.mark.skipif(not os.path.exists(hk.CLANG), reason="the compiler for the host is not there")
F16, I8 = xb.PAGES_F16, xb.PAGES_I8
ORDERS = [1, -1]  # of blocks and waves


class Plan(gpu.Plan):
    def upload(self):
        pass

    def step(self, run):
        open_ = run.buf(np.array(self.open, np.int32))
        run.call("step", len(self.past), self.total, self.max_rows, self.most, run.buf(np.array(self.row0, np.int32)),
                 run.buf(np.array(self.past, np.int32)), run.buf(self.table), open_)


class Pool:
    """gpu.Pool's arrays, in a run's buffers."""

    def __init__(self, kind, nkv, hd, page, pages, opens=1, k=None, v=None):
        self.kind, self.nkv, self.hd, self.page, self.pages, self.opens = kind, nkv, hd, page, pages, opens
        self.e = 16 if kind == I8 else 8
        self.x = [np.full((pages, nkv, page, hd), 99 if kind == I8 else np.nan, np.int8 if kind == I8 else np.float16) for _ in range(2)]
        self.scale = np.full((2, pages, nkv), np.nan, np.float32)
        self.open = np.full((2, opens, nkv, page, hd), np.nan, np.float16)
        for i, given in enumerate((k, v)):
            if given is None:
                continue
            if kind == F16:
                self.x[i][:] = given
                continue
            for p in range(pages):
                for h in range(nkv):
                    on = ~np.isnan(given[p, h].astype(np.float32)).any(-1)
                    if on.any():
                        self.x[i][p, h, on], self.scale[i, p, h] = po.codes(given[p, h][on])

    def raw(self):
        return [a.copy() for a in (*self.x, *self.scale, *self.open)]

    def pages_of(self, run):
        self.names = [run.buf(po.to_pages_k(self.x[0], self.e)), run.buf(po.to_pages_v(self.x[1], self.e))]
        extra = [run.buf(a) for a in (*self.scale, *self.open)] if self.kind == I8 else [hk.NONE] * 4
        self.names += extra
        run.call("pages", self.kind, self.nkv, self.hd, self.page, self.pages, self.opens, *self.names)

    def save(self, run):
        t = self.x[0].dtype
        run.save(self.names[0], t, (self.pages, self.nkv, self.hd // self.e, self.page, self.e))
        run.save(self.names[1], t, (self.pages, self.nkv, self.page // self.e, self.hd, self.e))
        if self.kind == I8:
            for n, a in zip(self.names[2:], (*self.scale, *self.open)):
                run.save(n, a.dtype, a.shape)

    def take(self, saved):
        """What the run left."""
        self.x = [po.from_pages_k(saved[0]), po.from_pages_v(saved[1])]
        if self.kind == I8:
            self.scale, self.open = np.stack(saved[2:4]), np.stack(saved[4:6])

    def values(self):
        if self.kind == F16:
            return [x.astype(np.float64) for x in self.x]
        return [x * s[..., None, None].astype(np.float64) for x, s in zip(self.x, self.scale)]


def rope(pairs, cap):
    ang = np.arange(cap)[:, None] * 1e4 ** (-np.arange(pairs) / max(1, pairs))
    return np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)


def prep(tmp, rng, pool, plan, nq, rotary, sections=None, inter=False, axes=None, gated=1, pad=0, x=None, norms=None, cap=None, order=1):
    """gpu.prep on the host: (projections, q, gate, norms, cos/sin of every row); the pool as it is then."""
    nkv, hd, T = pool.nkv, pool.hd, plan.total
    row = nq * hd * (2 if gated else 1) + 2 * nkv * hd + pad
    x = rng.normal(0, 1, (T, row)).astype(np.float32) if x is None else x
    qn, kn = norms or (rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2))
    cap = cap or max(p + m for p, m in zip(plan.past, plan.rows)) + 1
    run = hk.Run(tmp)
    run.call("order", order)
    pool.pages_of(run)
    plan.step(run)
    cs, angles = rope(rotary // 2, cap), np.zeros((T, rotary // 2, 2), np.float32)
    if rotary:
        sections = sections or [rotary // 2]
        run.call("rotary", run.buf(cs), cap, rotary, len(sections), int(inter), run.buf(axes) if axes is not None else hk.NONE, *sections)
        of = np.array(list(xb.rotary(1 << 20, cap, rotary, sections, inter).axis)[:rotary // 2])
        for s, j, i, p in plan.each():
            at = axes[of, i] if axes is not None else np.full(rotary // 2, p)
            ok = (at >= 0) & (at < cap)
            angles[i] = np.where(ok[:, None], cs[np.where(ok, at, 0), np.arange(rotary // 2)], np.nan)
    q, g = run.buf(np.full((T, nq * hd), 7, np.float32)), run.buf(np.full((T, nq * hd), 7, np.float32))
    run.call("prep", gated, nq, gpu.EPS, row, nq * hd, run.buf(x), run.buf(qn), run.buf(kn), q, g if gated else hk.NONE)
    run.save(q, np.float32, (T, nq, hd))
    run.save(g, np.float32, (T, nq, hd))
    pool.save(run)
    got = run.result()
    pool.take(got[2:])
    return x, got[0], got[1], (qn, kn), angles


def attention(tmp, pool, plan, nq, q, gate, order=1, out_rows=None):
    run = hk.Run(tmp)
    run.call("order", order)
    pool.pages_of(run)
    plan.step(run)
    out = run.buf(np.full((out_rows or plan.total, nq * pool.hd), 7, np.float32))
    run.call("attention", nq, nq * pool.hd, nq * pool.hd, run.buf(q), run.buf(gate) if gate is not None else hk.NONE, out)
    run.save(out, np.float32, (out_rows or plan.total, nq, pool.hd))
    return run.result()[0]


def filled(rng, kind, nkv, hd, page, plan):
    k, v = (np.full((plan.pages, nkv, page, hd), np.nan, np.float16) for _ in range(2))
    for s, (p, m) in enumerate(zip(plan.past, plan.rows)):
        for i in range((p + m + page - 1) // page):
            n = min(page, p + m - i * page)
            for x in (k, v):
                x[plan.table[s, i], :, :n] = rng.normal(0, 1, (nkv, n, hd)) * rng.uniform(0.2, 1.0)
    return Pool(kind, nkv, hd, page, plan.pages, 1, k, v)


# rows, splits and joins of every kind: the planned steps with 64 and 128 columns, several units of a row tile, query heads
# that do not divide a block's columns; single tokens over many blocks and within one
ATTEND = [a for a in gpu.ATTEND if max(a[4]) < 1000] + [
    (16, 4, 256, 64, [33], [64]), (16, 4, 256, 64, [33], [66]), (16, 4, 256, 32, [0], [65]), (16, 4, 256, 128, [200, 33], [33, 65]),
    (8, 8, 128, 32, [5] * 70, [3] * 70), (32, 2, 256, 64, [40, 500, 9], [17, 2, 30]), (256, 256, 128, 32, [20], [12]),
    (16, 16, 256, 32, [20, 3], [70, 9]), (8, 2, 128, 32, [700], [70]), (4, 1, 256, 32, [700], [70]), (2, 2, 128, 64, [130] * 3, [150] * 3)]


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("shape", ATTEND, ids=[f"{a[0]}_{a[1]}x{a[2]}_{a[3]}_{a[4][0]}_{a[5][0]}_{len(a[4])}" for a in ATTEND])
def test_attention_stays_in_its_buffers(tmp_path, kind, shape):
    nq, nkv, hd, page, past, rows = shape
    rng = np.random.default_rng(nq + hd + page + sum(past))
    plan = Plan(rng, page, past, rows, pad=2)
    pool = filled(rng, kind, nkv, hd, page, plan)
    q, gate = (rng.normal(0, 1, (plan.total, nq * hd)).astype(np.float32) for _ in range(2))
    some = set(rng.permutation(plan.n)[:40])
    for order in ORDERS[kind != I8:]:
        got = attention(tmp_path, pool, plan, nq, q, gate, order)
        gpu.check(got, gpu.attend_oracle(pool, plan, nq, q, gate, rows=some))
        assert (got[plan.n:] == 7).all() and not (got[:plan.n] == 7).all(-1).any()


@pytest.mark.parametrize("rows,hd", [([1, 1], 128), ([65], 256), ([3], 64)])
def test_a_row_past_the_buffer_is_seen(tmp_path, rows, hd):
    """An output buffer one row short: the run ends there, for each of the forms."""
    rng = np.random.default_rng(1)
    plan = Plan(rng, 64, [33] * len(rows), rows)
    pool = filled(rng, F16, 4, hd, 64, plan)
    q = rng.normal(0, 1, (plan.total, 16 * hd)).astype(np.float32)
    with pytest.raises(AssertionError, match="heap-buffer-overflow"):
        attention(tmp_path, pool, plan, 16, q, None, out_rows=plan.total - 1)


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("shape", gpu.SHAPES, ids=[f"{s[0]}_{s[1]}x{s[2]}_{s[6]}_{s[7][0]}_{s[8][0]}" for s in gpu.SHAPES])
def test_prep_stays_in_its_buffers(tmp_path, kind, shape):
    nq, nkv, hd, rotary, sections, inter, page, past, rows, gated, pad, behind = shape
    rng = np.random.default_rng(hd + page + len(past))
    plan = Plan(rng, page, past, rows, pad=behind)
    pool = Pool(kind, nkv, hd, page, plan.pages, len(past))
    if kind == I8:
        before = Plan(rng, page, [p // page * page for p in past], [p % page for p in past])
        if before.n:
            before.table, before.most, before.open = plan.table, plan.most, plan.open
            prep(tmp_path, rng, pool, before, nq, rotary, gated=gated, cap=4000)
    cap = max(past) + max(rows) + 40
    axes = rng.integers(0, cap, (len(sections), plan.total)).astype(np.int32) if sections else None
    was = pool.raw()
    x, norms = None, [rng.normal(1, 0.1, hd).astype(np.float32) for _ in range(2)]
    for order in ORDERS[kind != I8:]:
        pool.x, pool.scale, pool.open = was[:2], np.stack(was[2:4]), np.stack(was[4:])
        x, q, g, (qn, kn), cs = prep(tmp_path, rng, pool, plan, nq, rotary, sections, inter, axes, gated, pad, x=x, norms=norms, cap=cap, order=order)
        qx, gx, kx, vx = gpu.split_heads(x, nq, nkv, hd, gated)
        want, live = po.prepared(qx, qn, cs[:, None], gpu.EPS), plan.n
        assert (np.abs(q[:live] - want[:live]) <= 2**-23 * np.abs(want[:live])).all()
        assert (q[live:] == 7).all() and (g[live:] == 7).all()
        assert gpu.same(pool.raw(), gpu.appended(was, plan, kind, po.prepared(kx, kn, cs[:, None], gpu.EPS), vx))


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("out", [np.float32, np.float16])
@pytest.mark.parametrize("hd,page,past,rows", [(128, 64, [0, 63, 100], [1, 70, 0]), (48, 32, [17], [50]), (256, 128, [1], [300])])
def test_read_stays_in_its_buffers(tmp_path, kind, out, hd, page, past, rows):
    rng = np.random.default_rng(hd)
    plan = Plan(rng, page, past, rows)
    pool = filled(rng, kind, 3, hd, page, plan)
    run = hk.Run(tmp_path)
    pool.pages_of(run)
    plan.step(run)
    shape = (plan.n, 3, hd)
    k, v = (run.buf(np.full(shape, 7, out)) for _ in range(2))
    run.call("read", xb.F32 if out == np.float32 else xb.F16, k, v)
    run.save(k, out, shape)
    run.save(v, out, shape)
    for got, values in zip(run.result(), pool.values()):
        values = values.astype(np.float32) if kind == I8 else values  # (codes times their scale: one fp32 product)
        for s, j, i, p in plan.each():
            want = values[plan.table[s, p // page], :, p % page].astype(np.float32).astype(out)
            assert np.array_equal(got[i], want)


# ---- rows of an 8-bit page that are not held --------------------------------------
def steps_with_holes(tmp, rng, pool, whole, sizes, bad, nq=2, on=None):
    """Appends whole's rows to `pool` in steps of the given sizes; rows in `bad` have rotary positions outside the table.  The
    rows' keys and values [rows][nkv][hd] as an 8-bit page takes them."""
    n, cap = sum(sizes), 500
    x = (rng.normal(0, 1, (n, 2 * nq * pool.hd + 2 * pool.nkv * pool.hd)) * rng.uniform(0.1, 3, (n, 1))).astype(np.float32)
    norms, done, keys = [rng.normal(1, 0.1, pool.hd).astype(np.float32) for _ in range(2)], 0, []
    for m in sizes:
        plan = (on.Plan if on else Plan)(rng, pool.page, [whole.past[0] + done], [m])
        plan.table, plan.most, plan.open = whole.table, whole.most, whole.open
        plan.upload()
        axes = (plan.past[0] + np.arange(m, dtype=np.int32))[None].copy()
        for i, r in enumerate(range(done, done + m)):
            if r in bad:
                axes[0, i] = [-1, cap][r % 2]
        call = on.prep if on else lambda *a, **o: prep(tmp, *a, **o)
        _, q, _, (_, kn), cs = call(rng, pool, plan, nq, 32, axes=axes, x=x[done: done + m], norms=norms, cap=cap)
        _, _, kx, vx = gpu.split_heads(x[done: done + m], nq, pool.nkv, pool.hd, 1)
        assert (np.isnan(q).all((1, 2)) == [r in bad for r in range(done, done + m)]).all()
        keys.append((po.held(po.prepared(kx, kn, cs[:, None], gpu.EPS)), po.held(vx)))
        done += m
    return [np.concatenate(z) for z in zip(*keys)]


def check_holes(pool, was, whole, values, bad):
    """Codes of the rows that are held, each page's scale: the largest of its held rows, and what the page's scale said before
    where its first position was not written."""
    now = pool.raw()
    for i, x in enumerate(values):
        for at in range(whole.past[0] // pool.page, (whole.past[0] + len(x) - 1) // pool.page + 1):
            pg = whole.table[0, at]
            rows = [r for r in range(len(x)) if (whole.past[0] + r) // pool.page == at and r not in bad]
            offs = [(whole.past[0] + r) % pool.page for r in rows]
            for h in range(pool.nkv):
                if not rows:
                    assert np.array_equal(now[i][pg, h], was[i][pg, h]) and now[2 + i][pg, h] == was[2 + i][pg, h]
                    continue
                mx = np.abs(x[rows][:, h].astype(np.float64)).max()
                if 0 not in offs:
                    mx = max(mx, float(np.float16(was[2 + i][pg, h] * np.float32(127))))
                assert now[2 + i][pg, h] == np.float32(mx / 127), (i, at, h)
                assert np.array_equal(now[i][pg, h, offs], np.rint(x[rows][:, h].astype(np.float64) * 127 / mx)), (i, at, h)


HOLES = [  # positions before, rows of the steps, rows without a rotary position
    (0, [20], set(range(20))),                                 # a chunk over a page that holds codes: all as it was
    (32, [40], set(range(40))), (0, [1], {0}),                 # over two pages; one row
    (0, [10, 30], {4}), (0, [1] * 10 + [40], {4, 5, 9}),       # a hole, then a step that leaves the page
    (0, [6, 6, 6], {2, 7, 8}), (0, [10, 1, 1, 25, 1], {3, 11}), (0, [3, 70], {1, 33, 34}),
    (0, [12], {0}), (0, [1] * 12, {0}), (0, [3, 40], {0, 1, 2}), (0, [1, 1, 1, 40], {0, 1, 32})]  # the page's first position


@pytest.mark.parametrize("stale,old", [(6e4, 0.5), (np.inf, 30), (np.nan, 0.5)])
@pytest.mark.parametrize("past,sizes,bad", HOLES, ids=[f"{p}_{'_'.join(map(str, s))}_{len(b)}" for p, s, b in HOLES])
def test_rows_that_are_not_held_do_not_count(tmp_path, past, sizes, bad, stale, old):
    """Open pages hold what a sequence before left there, pages values of another size."""
    rng = np.random.default_rng(len(bad) + past)
    whole = Plan(rng, 32, [past], [sum(sizes)])
    pool = Pool(I8, 2, 128, 32, whole.pages, 1, *(rng.normal(0, old, (2, whole.pages, 2, 32, 128)).astype(np.float16)))
    pool.open[:] = stale
    was = pool.raw()
    check_holes(pool, was, whole, steps_with_holes(tmp_path, rng, pool, whole, sizes, bad), bad)


@pytest.mark.parametrize("first,stale", [(10, 6e4), (1, np.inf), (40, np.nan)])
def test_rows_before_their_page_is_there_do_not_count(tmp_path, first, stale):
    """A sequence's first rows find no page (one, a chunk, a chunk over two pages); the page that is there later takes the rest."""
    rng = np.random.default_rng(first)
    at = first // 32
    whole = Plan(rng, 32, [0], [first + 3 + 40])
    pool = Pool(I8, 2, 128, 32, whole.pages, 1, *(rng.normal(0, 0.5, (2, whole.pages, 2, 32, 128)).astype(np.float16)))
    pool.open[:] = stale
    was, table = pool.raw(), whole.table.copy()
    whole.table[0, :at + 1] = [-1, whole.pages][first % 2]
    pages = Plan(rng, 32, [0], [first])
    pages.table, pages.most, pages.open = whole.table, whole.most, whole.open
    prep(tmp_path, rng, pool, pages, 2, 32, cap=500)
    assert gpu.same(pool.raw()[:4], was[:4])
    whole.table, whole.past = table, [first]
    check_holes(pool, was, whole, steps_with_holes(tmp_path, rng, pool, whole, [3, 40], set()), set())


@pytest.mark.parametrize("hd,seqs,rows", [(256, 1024, 512), (128, 1024, 1024), (256, 60, 40)])
def test_rows_in_no_order_stay_in_the_workspace(tmp_path, hd, seqs, rows):
    """Every second sequence claims every row (row0 falls): some 65536 row tiles where a step of so many rows has 896 at most.
    What all sequences agree on comes out."""
    rng = np.random.default_rng(hd)
    plan = Plan(rng, 32, [0], [rows])
    pool = Pool(F16, 1, hd, 32, 3, 1, *rng.normal(0, 1, (2, 3, 1, 32, hd)).astype(np.float16))
    plan.table, plan.most, plan.pages, plan.open = np.full((seqs, 1), 1, np.int32), 1, 3, np.zeros(seqs, np.int32)
    run = hk.Run(tmp_path)
    pool.pages_of(run)
    run.call("step", seqs, rows, rows, 1, run.buf(np.array([[0, rows][i % 2] for i in range(seqs + 1)], np.int32)),
             run.buf(np.zeros(seqs, np.int32)), run.buf(plan.table), hk.NONE)
    q = rng.normal(0, 1, (rows, 16 * hd)).astype(np.float32)
    out = run.buf(np.full((rows, 16 * hd), 7, np.float32))
    run.call("attention", 16, 16 * hd, 16 * hd, run.buf(q), hk.NONE, out)
    run.save(out, np.float32, (rows, 16, hd))
    some = set(rng.permutation(rows)[:40])
    gpu.check(run.result()[0], gpu.attend_oracle(pool, plan, 16, q, None, rows=some))


BIG, LOW = 2**31 - 1, -2**31


@pytest.mark.parametrize("kind,hd", [(F16, 64), (I8, 128), (F16, 256)])
@pytest.mark.parametrize("max_rows", [1, 100])
@pytest.mark.parametrize("row0,past", [([0, 100] * 20, 5), ([100, 0, 50, -7, 200, 3, 3, 2], 5), ([BIG, LOW, 60, 0, 99], 5),
                                       ([LOW, BIG, 0, LOW, BIG], 31), ([0, 3, 4, 40, 100], BIG), ([0, 3, 4, 40, 100], BIG - 50),
                                       ([0, 3, 4, 40, 100], LOW), ([0, 3, 4, 40, 100], 2**20 - 20)])
def test_numbers_of_any_size(tmp_path, kind, hd, max_rows, row0, past):
    """Rows of several sequences or of none, numbers outside the step, pages and open pages that are none: nothing outside the
    buffers."""
    rng = np.random.default_rng(9)
    seqs, rows = len(row0) - 1, 100
    plan = Plan(rng, 32, [5] * seqs, [rows] * seqs)
    plan.row0, plan.total, plan.max_rows, plan.past = row0, rows, max_rows, [past] * seqs
    plan.table[0, 0], plan.table[1, 1], plan.table[2, 0] = BIG, LOW, plan.pages
    pool = Pool(kind, 2, hd, 32, plan.pages, seqs, *rng.normal(0, 1, (2, plan.pages, 2, 32, hd)).astype(np.float16))
    plan.open = np.array([BIG, LOW] + list(range(seqs - 2)), np.int64).astype(np.int32)
    x = rng.normal(0, 1, (rows, 8 * hd)).astype(np.float32)
    run = hk.Run(tmp_path)
    pool.pages_of(run)
    plan.step(run)
    ones, q = run.buf(np.ones(hd, np.float32)), run.buf(np.full((rows, 4 * hd), 7, np.float32))
    axes = rng.choice([0, 3, 39, 40, BIG, LOW, -1], (2, rows)).astype(np.int32)
    run.call("rotary", run.buf(rope(8, 40)), 40, 16, 2, 1, run.buf(axes), 4, 4)
    run.call("prep", 0, 4, gpu.EPS, 8 * hd, 4 * hd, run.buf(x), ones, ones, q, hk.NONE)
    k, v = (run.buf(np.full((rows, 2, hd), 7, np.float32)) for _ in range(2))
    run.call("read", xb.F32, k, v)
    run.call("attention", 4, 4 * hd, 4 * hd, run.buf(x[:, :4 * hd]), hk.NONE, run.buf(x[:, :4 * hd]))
    run.result()


# ---- log probabilities ----------------------------------------------------------
def logprobs(tmp, x, tokens, inv_t, top, ld):
    rows, vocab = x.shape
    run = hk.Run(tmp)
    y = np.full(rows * ld, np.nan, x.dtype)  # (nothing behind the last row's logits)
    y.reshape(rows, ld)[:, :vocab] = x
    shapes = [(np.float32, rows), (np.float32, rows), (np.int32, rows), (np.int32, rows * top), (np.float32, rows * top)]
    outs = [run.buf(np.full(n, 7, t)) if n else hk.NONE for t, n in shapes]
    run.call("logprobs", xb.F16 if x.dtype == np.float16 else xb.F32, ld, rows, vocab, inv_t, top, run.buf(y[:(rows - 1) * ld + vocab]),
             run.buf(np.array(tokens, np.int32)), *outs)
    for name, (t, n) in zip(outs, shapes):
        if n:
            run.save(name, t, (n,))
    got = run.result()
    return got[:3] + [a.reshape(rows, top) for a in got[3:]]


@pytest.mark.parametrize("t", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [1, 5, 33, 1022, 1025, 8193, 16384, 16385, 40007])
def test_logprobs_stay_in_their_buffers(tmp_path, vocab, t):
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 3, (6, vocab)).astype(t)
    x[1] = np.round(x[1])
    x[2] = 1.5
    x[3, rng.random(vocab) < 0.99] = -np.inf
    x[4, :] = np.nan
    tokens = [0, vocab - 1, vocab // 2, vocab, -1, 2**31 - 1]
    for ld, top in ((vocab, 0), (vocab, 64), ((vocab + 7) // 8 * 8, 5)):
        got = logprobs(tmp_path, x, tokens, 1.0, top, ld)
        gpu.check_logprobs(got + [np.zeros((6, 0), np.int32), np.zeros((6, 0), np.float32)][:5 - len(got)], x, tokens, 1.0, top)


def test_codes_are_the_nearest(tmp_path):
    """code_of against the quotient in 64 bits, ties to even: every fp16 value up to every maximum of two exponents and the
    subnormal ones, and to some of the other maxima."""
    run = hk.Run(tmp_path)
    run.call("codes", tmp_path / "wrong")
    run.result()
    assert (tmp_path / "wrong").read_text() == "0"


def far_rows(vocab):
    """Logits whose differences pass fp32's range, at temperatures that bring them back."""
    rng = np.random.default_rng(vocab)
    x = rng.uniform(-3.4e38, 3.4e38, (5, vocab)).astype(np.float32)
    x[1, :] = -3.4e38
    x[1, vocab // 2] = 3.4e38                # one against all
    x[2] = np.where(np.arange(vocab) % 3, -2e38, 2e38)
    x[3] = rng.normal(0, 1, vocab)           # ordinary ones beside the range's ends
    x[3, 0], x[3, vocab - 1] = np.finfo(np.float32).max, -np.finfo(np.float32).max
    x[4] = rng.normal(0, 1e-38, vocab)
    return x, [0, vocab - 1, 1, vocab - 1, 3]


@pytest.mark.parametrize("vocab", [33, 1100, 20011])
@pytest.mark.parametrize("inv_t", [1e-38, 3e-39, 2e-38, 1e-30, 0.4])
def test_logprobs_of_logits_far_apart(tmp_path, vocab, inv_t):
    x, tokens = far_rows(vocab)
    gpu.check_logprobs(logprobs(tmp_path, x, tokens, inv_t, 7, vocab + 3), x, tokens, inv_t, 7)


@pytest.mark.parametrize("kind", [F16, I8])
@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 40, 2]])
def test_heads_with_an_infinity(tmp_path, kind, rows):
    """x / sqrt(mean x^2 + eps) of a head with an infinity: 0, not a number where the infinity and its partner are.
    A page that no row began has no scale: any that is not a number counts as 0."""
    rng = np.random.default_rng(2)
    plan = Plan(rng, 32, [0, 31, 5], rows)
    pool = Pool(kind, 2, 128, 32, plan.pages, 3)
    pool.open[:] = 0
    was = pool.raw()
    x = rng.normal(0, 1, (plan.total, 2 * 4 * 128 + 4 * 128)).astype(np.float32)
    x[:, 3], x[1, 256 + 70], x[:, 1024 + 7] = np.inf, -np.inf, np.inf  # of query heads, of a key's
    with np.errstate(invalid="ignore"):
        x, q, _, (qn, kn), cs = prep(tmp_path, rng, pool, plan, 4, 32, x=x)
        qx, _, kx, vx = gpu.split_heads(x, 4, 2, 128, 1)
        want, k = po.prepared(qx, qn, cs[:, None], gpu.EPS), po.prepared(kx, kn, cs[:, None], gpu.EPS)
    assert np.array_equal(np.isnan(q), np.isnan(want))
    assert (np.abs(q - want) <= 2**-23 * np.abs(want))[~np.isnan(want)].all()
    numbers = lambda raw: raw[:2] + [np.nan_to_num(s) for s in raw[2:4]] + raw[4:]  # noqa: E731
    assert gpu.same(numbers(pool.raw()), gpu.appended(numbers(was), plan, kind, k, vx))


@pytest.mark.parametrize("steps", [[(0, 10, 6), (10, 30, 0)], [(0, 10, 6), (10, 1, 3), (11, 1, 0), (12, 20, 9), (32, 5, 2)], [(0, 20, 0), (20, 12, 5), (32, 7, 2), (39, 1, 0)],
                                   [(0, 32, 40), (32, 40, 0)], [(0, 1, 31), (1, 1, 1), (2, 60, 2), (62, 2, 3), (64, 1, 0)]])
def test_padded_steps(tmp_path, steps):
    """Steps whose last rows are padding (no rotary position), in the page where the next one goes on or past a page that is full:
    the rows' codes as of one append."""
    rng = np.random.default_rng(len(steps))
    n = max(p + m + pad for p, m, pad in steps)
    whole = Plan(rng, 32, [0], [n])
    pool = Pool(I8, 2, 128, 32, whole.pages, 1, *(rng.normal(0, 20, (2, whole.pages, 2, 32, 128)).astype(np.float16)))
    pool.open[:] = 6e4
    was, norms, keys = pool.raw(), [rng.normal(1, 0.1, 128).astype(np.float32) for _ in range(2)], []
    for past, m, pad in steps:
        plan = Plan(rng, 32, [past], [m + pad])
        plan.table, plan.most, plan.open = whole.table, whole.most, whole.open
        x = (rng.normal(0, 1, (m + pad, 8 * 128)) * rng.uniform(0.1, 3, (m + pad, 1))).astype(np.float32)
        axes = np.where(np.arange(m + pad) < m, past + np.arange(m + pad), -1)[None].astype(np.int32)
        _, _, _, (_, kn), cs = prep(tmp_path, rng, pool, plan, 2, 32, axes=axes, x=x, norms=norms, cap=500)
        _, _, kx, vx = gpu.split_heads(x, 2, 2, 128, 1)
        keys.append((po.held(po.prepared(kx, kn, cs[:, None], gpu.EPS))[:m], po.held(vx)[:m]))
    check_holes(pool, was, whole, [np.concatenate(z) for z in zip(*keys)], set())
