"""The entry points over paged caches without a GPU: the axes of a rotation's pairs, workspace sizes, and refusals (with
addresses that no call may follow)."""
import ctypes

import numpy as np
import pytest

import paged_oracle as po
import xqbind as xb

P = ctypes.c_void_p(1 << 20)  # never followed: every call here is refused
EINVAL = -1


def odd(n):
    return ctypes.c_void_p((1 << 20) + n)


def refused(rc, word=""):
    assert rc == EINVAL
    assert word in xb.hip().xqhip_last_error().decode(), xb.hip().xqhip_last_error()


def pages(type=xb.PAGES_I8, nkv=2, hd=128, page=64, pages=9, opens=4, k=P, v=P, ks=P, vs=P, ko=P, vo=P):
    return ctypes.byref(xb.Pages(type, nkv, hd, page, pages, opens, k, v, ks, vs, ko, vo))


def step(seqs=3, rows=5, max_rows=3, max_pages=4, row0=P, past=P, table=P, open=P):
    return ctypes.byref(xb.Step(seqs, rows, max_rows, max_pages, row0, past, table, open))


@pytest.mark.parametrize("rotary,sections,inter,want", [
    (16, [8], 0, [0] * 8), (16, [8], 1, [0] * 8), (16, [2, 3, 3], 0, [0, 0, 1, 1, 1, 2, 2, 2]),
    (16, [4, 2, 2], 1, [0, 1, 2, 0, 1, 2, 0, 0]), (16, [0, 8], 0, [1] * 8), (12, [2, 1, 2, 1], 0, [0, 0, 1, 2, 2, 3]),
    (64, [12, 10, 10], 1, [i % 3 if i < 30 else 0 for i in range(32)]), (0, [0], 0, [])])
def test_rotary_axes(rotary, sections, inter, want):
    r = xb.rotary(P, 10, rotary, sections, inter)
    assert list(r.axis)[:rotary // 2] == want and r.axes == len(sections) and r.rotary_dim == rotary
    if rotary and not inter:
        assert [want.count(a) for a in range(len(sections))] == sections


@pytest.mark.parametrize("a", [
    dict(rotary=15, sections=[7]), dict(rotary=258, sections=[129]), dict(rotary=-2, sections=[-1]), dict(sections=[7]),
    dict(sections=[9, -1]), dict(sections=[]), dict(sections=[2, 2, 2, 1, 1]), dict(sections=[1, 4, 3], inter=1),
    dict(cs=None), dict(cs=odd(4)), dict(positions=0)])
def test_rotary_refuses(a):
    a = dict(dict(cs=P, positions=10, rotary=16, sections=[8], inter=0), **a)
    with pytest.raises(xb.HipError, match="rotary_init"):
        xb.rotary(a["cs"], a["positions"], a["rotary"], a["sections"], a["inter"])


def rotary(dims=32, **fields):
    r = xb.rotary(P, 10, dims, [dims // 2])
    for k, v in fields.items():
        setattr(r, k, v)
    return ctypes.byref(r)


def bad_axis():
    r = xb.rotary(P, 10, 32, [16])
    r.axis[15] = 1
    return ctypes.byref(r)


BAD_PAGES = [dict(type=2), dict(type=-1), dict(nkv=0), dict(nkv=257), dict(hd=0), dict(hd=24), dict(hd=272), dict(page=16),
             dict(page=48), dict(page=256), dict(pages=0), dict(k=None), dict(v=None), dict(k=odd(8)), dict(v=odd(2)),
             dict(ks=None), dict(vs=None)]
BAD_OPENS = [dict(opens=0), dict(ko=None), dict(vo=None), dict(ko=odd(8)), dict(vo=odd(4))]
BAD_STEPS = [dict(seqs=0), dict(seqs=1025), dict(rows=0), dict(rows=65536), dict(max_rows=0), dict(max_rows=6),
             dict(max_pages=0), dict(max_pages=16385), dict(row0=None), dict(past=None), dict(table=None)]


def prep(**o):
    a = dict(q=P, k=P, v=P, gated=1, nq=8, qn=P, kn=P, eps=1e-6, rot=rotary(), step=step(), src=4096, dst=1024, qo=P, go=P,
             kv=pages())
    a.update(o)
    return xb.hip().xqhip_attn_prep_paged(*a.values(), None)


@pytest.mark.parametrize("o", [dict(q=None), dict(k=None), dict(v=None), dict(qn=None), dict(kn=None), dict(qo=None),
                               dict(go=None), dict(kv=None), dict(step=None), dict(nq=0), dict(nq=65536), dict(dst=1023),
                               dict(src=-1), dict(step=step(open=None)), dict(rot=rotary(axes=0)), dict(rot=rotary(axes=5)),
                               dict(rot=rotary(rotary_dim=31)), dict(rot=rotary(256)), dict(rot=rotary(positions=0)),
                               dict(rot=rotary(cs=None)), dict(rot=bad_axis())] +
                         [dict(kv=pages(**b)) for b in BAD_PAGES + BAD_OPENS] + [dict(step=step(**b)) for b in BAD_STEPS])
def test_prep_refuses(o):
    refused(prep(**o), "xqhip_attn_prep_paged")


@pytest.mark.parametrize("o", [dict(kv=None), dict(step=None), dict(t=2), dict(t=-1)] + [dict(kv=pages(**b)) for b in BAD_PAGES] +
                         [dict(step=step(**b)) for b in BAD_STEPS])
def test_read_refuses(o):
    a = dict(kv=pages(), step=step(), t=xb.F32, k=P, v=P)
    a.update(o)
    refused(xb.hip().xqhip_paged_read(*a.values(), None), "xqhip_paged_read")


def test_read_of_nothing():
    assert xb.hip().xqhip_paged_read(pages(), step(), xb.F16, None, None, None) == 0


@pytest.mark.parametrize("o", [dict(q=None), dict(kv=None), dict(step=None), dict(out=None), dict(nq=7), dict(nq=0), dict(nq=34),
                               dict(qs=1023), dict(os=1023), dict(ws=None), dict(ws=odd(8)), dict(n=-1)] +
                         [dict(kv=pages(**b)) for b in BAD_PAGES] + [dict(step=step(**b)) for b in BAD_STEPS])
def test_attention_refuses(o):
    need = xb.hip().xqhip_paged_attention_workspace_bytes(8, 2, 128)
    a = dict(q=P, g=P, kv=pages(), nq=8, step=step(), qs=1024, out=P, os=1024, ws=P, n=need)
    a.update(o)
    if a["n"] < 0:
        a["n"] = need - 1
    refused(xb.hip().xqhip_paged_attention(*a.values(), None), "xqhip_paged_attention")


@pytest.mark.parametrize("shape", [(7, 2, 128), (0, 1, 128), (8, 0, 128), (34, 2, 128), (8, 2, 24), (8, 2, 272), (8, 2, 0), (257, 257, 128)])
def test_attention_workspace_of_refused_shapes(shape):
    assert xb.hip().xqhip_paged_attention_workspace_bytes(*shape) == 0


@pytest.mark.parametrize("o", [dict(x=None), dict(t=2), dict(ld=99), dict(rows=0), dict(rows=65536), dict(vocab=0),
                               dict(vocab=(1 << 24) + 1), dict(it=0.0), dict(it=-1.0), dict(it=float("nan")), dict(it=float("inf")),
                               dict(tok=None), dict(top=-1), dict(top=65), dict(ws=None), dict(ws=odd(4)), dict(n=0)])
def test_logprobs_refuses(o):
    a = dict(x=P, t=xb.F32, ld=100, rows=3, vocab=100, it=1.0, tok=P, top=5, lp=P, en=P, rk=P, id=P, tl=P, ws=P, n=1 << 30)
    a.update(o)
    refused(xb.hip().xqhip_token_logprobs(*a.values(), None), "xqhip_token_logprobs")


def test_logprobs_of_nothing():
    assert xb.hip().xqhip_token_logprobs(P, xb.F32, 100, 3, 100, 1.0, None, 0, None, None, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("shape", [(0, 100, 5), (65536, 100, 5), (3, 0, 5), (3, (1 << 24) + 1, 5), (3, 100, -1), (3, 100, 65)])
def test_logprobs_workspace_of_refused_shapes(shape):
    assert xb.hip().xqhip_token_logprobs_workspace_bytes(*shape) == 0


def test_definition_of_codes_does_not_depend_on_ties():
    """The codes by one fp32 division of the exact product 127 x are those of the quotient itself, for every pair of
    fp16 significands: that is how the kernel takes them."""
    mx = np.arange(1024, 2048, 7, dtype=np.float32)
    x = np.arange(0, 2048, dtype=np.float32)
    q = (127 * x[None]) / mx[:, None]
    assert q.dtype == np.float32
    want = np.rint(127 * x.astype(np.float64)[None] / mx.astype(np.float64)[:, None])
    assert (np.rint(q) == want).all()


def test_page_layouts():
    rng = np.random.default_rng(0)
    for e in (8, 16):
        x = rng.integers(-127, 128, (3, 2, 32, 48))
        k, v = po.to_pages_k(x, e), po.to_pages_v(x, e)
        assert (po.from_pages_k(k) == x).all() and (po.from_pages_v(v) == x).all()
        assert k[1, 0].reshape(-1)[(17 // e * 32 + 5) * e + 17 % e] == x[1, 0, 5, 17]
        assert v[2, 1].reshape(-1)[(21 // e * 48 + 9) * e + 21 % e] == x[2, 1, 21, 9]
