"""The tree entry points without a GPU: trees and their masks, refusals (with
addresses that no call may follow), and that the verification's definition
samples from the target."""
import ctypes

import numpy as np
import pytest

import tree_oracle as to
import xqbind as xb

P = ctypes.c_void_p(1 << 20)  # never followed: every call here is refused
EINVAL = -1


def kv(type=xb.KV_I8, nkv=2, hd=128, cap=64, k=P, v=P, ks=P, vs=P):
    return ctypes.byref(xb.Kv(type, nkv, hd, cap, k, v, ks, vs))


def refused(rc, word=""):
    assert rc == EINVAL
    assert word in xb.hip().xqhip_last_error().decode(), xb.hip().xqhip_last_error()


@pytest.mark.parametrize("seed,n", [(0, 1), (1, 2), (2, 17), (3, 64)])
def test_tree_init(seed, n):
    par = to.random_tree(np.random.default_rng(seed), n)
    t = xb.tree(par)
    assert t.nodes == n and list(t.parent)[:n] == par and list(t.depth)[:n] == to.depths(par)
    want = to.path_masks(par)
    assert [[t.mask[i] >> j & 1 for j in range(n)] for i in range(n)] == want.astype(int).tolist()


@pytest.mark.parametrize("par", [[], [0], [-2], [-1, 1], [-1, 2], [-1, -2], [-1] * 65])
def test_tree_init_refuses(par):
    with pytest.raises(xb.HipError, match="tree_init"):
        xb.tree(par)


def broken(n=3, **fields):
    t = xb.tree([-1] + list(range(n - 1)))
    for name, (i, v) in fields.items():
        getattr(t, name)[i] = v
    return t


BAD_TREES = [broken(parent=(1, 1)), broken(parent=(0, 0)), broken(parent=(2, -3)), broken(depth=(2, 1)),
             broken(depth=(0, 3))]


def prep(**o):
    a = dict(q=P, k=P, v=P, gated=1, nq=8, rotary=32, qn=P, kn=P, eps=1e-6, rope=P, pos=P, tree=None, tokens=3,
             src=4096, dst=1024, qo=P, go=P, kv=kv())
    a.update(o)
    return xb.hip().xqhip_attn_prep_kv(*a.values(), None)


@pytest.mark.parametrize("o", [
    dict(q=None), dict(k=None), dict(v=None), dict(qn=None), dict(kn=None), dict(rope=None), dict(pos=None),
    dict(qo=None), dict(go=None), dict(kv=None), dict(nq=0), dict(tokens=0), dict(tokens=65536), dict(dst=1023),
    dict(src=-1), dict(kv=kv(type=2)), dict(kv=kv(nkv=0)), dict(kv=kv(hd=1025)), dict(kv=kv(cap=0)),
    dict(kv=kv(cap=(1 << 20) + 1)), dict(kv=kv(k=None)), dict(kv=kv(vs=None)), dict(tree=xb.tree([-1, 0])),
    *[dict(tree=t) for t in BAD_TREES]])
def test_prep_refuses(o):
    if "tree" in o:
        o = dict(o, tree=ctypes.byref(o["tree"]))
    refused(prep(**o), "xqhip_attn_prep_kv")


@pytest.mark.parametrize("cache,first,count,t", [
    (None, 0, 1, 0), (kv(type=xb.KV_F16), 0, 1, 0), (kv(), -1, 1, 0), (kv(), 0, 65, 0), (kv(), 64, 1, 0),
    (kv(), 1, 2147483647, 0), (kv(), 0, -1, 0), (kv(), 0, 1, 2), (kv(ks=None), 0, 1, 0)])
def test_read_refuses(cache, first, count, t):
    refused(xb.hip().xqhip_kv_read(cache, first, count, t, P, P, None), "xqhip_kv_read")


def test_read_of_nothing():
    assert xb.hip().xqhip_kv_read(kv(), 64, 0, xb.F16, P, P, None) == 0
    assert xb.hip().xqhip_kv_read(kv(), 0, 64, xb.F16, None, None, None) == 0


def attend(**o):
    a = dict(q=P, gate=P, kv=kv(), nq=8, tree=None, tokens=3, qs=1024, pos=P, out=P, os=1024, ws=P, size=1 << 40)
    a.update(o)
    return xb.hip().xqhip_tree_attention(*a.values(), None)


@pytest.mark.parametrize("o", [
    dict(q=None), dict(kv=None), dict(pos=None), dict(out=None), dict(tokens=0), dict(tokens=65536), dict(qs=1023),
    dict(os=1023), dict(nq=7), dict(nq=18), dict(nq=0), dict(kv=kv(k=None)), dict(kv=kv(hd=1024), nq=16, qs=1 << 16, os=1 << 16),
    dict(ws=None), dict(ws=ctypes.c_void_p(8)), dict(size=0), dict(tree=xb.tree([-1, 0])),
    *[dict(tree=t) for t in BAD_TREES]])
def test_attention_refuses(o):
    if "tree" in o:
        o = dict(o, tree=ctypes.byref(o["tree"]))
    refused(attend(**o), "xqhip_tree_attention")


def test_attention_workspace():
    need = xb.hip().xqhip_tree_attention_workspace_bytes
    assert need(7, 2, 128, 1) == need(18, 2, 128, 1) == need(8, 2, 128, 0) == need(8, 2, 2048, 1) == 0
    for nq, nkv, hd in ((32, 8, 128), (16, 4, 256), (8, 8, 64), (8, 1, 80)):
        for n in (1, 2, 63, 64, 65, 512):
            size = need(nq, nkv, hd, n)
            assert size > 0
            refused(attend(kv=kv(nkv=nkv, hd=hd), nq=nq, tokens=n, qs=1 << 14, os=1 << 14, size=size - 1), "workspace")


@pytest.mark.parametrize("group,hd", [(8, 990), (7, 1024), (4, 1024), (1, 1024)])
def test_attention_up_to_its_largest_heads(group, hd):
    """group (2 head_dim + 67) floats within 64 KiB: accepted by the size's check and refused for the workspace alone;
    one dim more, or a group of more than eight, is not (heads have up to 1024 dims)."""
    need = xb.hip().xqhip_tree_attention_workspace_bytes
    o = dict(nq=2 * group, qs=1 << 14, os=1 << 14)
    assert group * (2 * hd + 67) <= 16384 and need(2 * group, 2, hd, 3) == 16
    refused(attend(kv=kv(hd=hd), size=15, **o), "workspace")
    assert need(2 * group, 2, hd + 1, 3) == 0
    refused(attend(kv=kv(hd=hd + 1), **o), "heads")
    assert need(18, 2, 64, 3) == 0


def test_attention_sizes_for_several_lengths():
    """A prompt chunk whose blocks fill the card needs less than a few rows do: each call is checked for its own."""
    need = xb.hip().xqhip_tree_attention_workspace_bytes
    small, large = need(32, 8, 128, 1024), need(32, 8, 128, 64)
    assert small < large
    refused(attend(kv=kv(nkv=8), nq=32, tokens=64, qs=4096, os=4096, size=small), "workspace")


def linear(**o):
    a = dict(m=P, a=P, b=P, stride=4096, hist=P, pos=P, w=P, al=P, dt=P, state=P, lk=2, dk=128, lv=4, dv=128, ks=4,
             tree=xb.tree([-1, 0, 0]), out=P, os=512, ws=P, size=1 << 40)
    a.update(o)
    a["tree"] = ctypes.byref(a["tree"]) if a["tree"] is not None else None
    return xb.hip().xqhip_linear_attn_tree(*a.values(), None)


@pytest.mark.parametrize("o", [
    dict(m=None), dict(a=None), dict(b=None), dict(hist=None), dict(pos=None), dict(w=None), dict(al=None),
    dict(dt=None), dict(state=None), dict(tree=None), dict(out=None), dict(os=511), dict(stride=-1), dict(lk=0),
    dict(lk=3), dict(dk=257), dict(dv=257), dict(ks=0), dict(ks=9), dict(size=0), dict(ws=None),
    dict(ws=ctypes.c_void_p(4)), *[dict(tree=t) for t in BAD_TREES]])
def test_linear_refuses(o):
    refused(linear(**o), "xqhip_linear_attn_tree")


def verify(**o):
    a = dict(l=P, ld=100, vocab=100, tree=xb.tree([-1, 0, 0]), tok=P, draft=P, ldd=100, t=1.0, ua=P, us=P, c=P, p=P,
             o=P, ws=P, size=1 << 40)
    a.update(o)
    a["tree"] = ctypes.byref(a["tree"]) if a["tree"] is not None else None
    return xb.hip().xqhip_spec_verify(*a.values(), None)


@pytest.mark.parametrize("o", [
    dict(l=None), dict(tree=None), dict(tok=None), dict(c=None), dict(p=None), dict(o=None), dict(vocab=0),
    dict(vocab=(1 << 24) + 1, ld=1 << 25, ldd=1 << 25), dict(ld=99), dict(ldd=99), dict(t=-1.0), dict(t=float("nan")),
    dict(t=float("inf")), dict(ua=None), dict(us=None), dict(size=0), dict(ws=None), dict(ws=ctypes.c_void_p(8)),
    dict(tree=xb.tree([-1, 0, -1])), *[dict(tree=t) for t in BAD_TREES]])
def test_verify_refuses(o):
    refused(verify(**o), "xqhip_spec_verify")


def test_keep_refuses():
    L = xb.hip()
    good = (P, 16, 4, None)
    refused(L.xqhip_tree_keep(xb.rows([good]), 1, None, P, 4, None), "tree_keep")
    refused(L.xqhip_tree_keep(xb.rows([good]), 1, P, None, 4, None), "tree_keep")
    refused(L.xqhip_tree_keep(None, 1, P, P, 4, None), "tree_keep")
    refused(L.xqhip_tree_keep(xb.rows([good]), -1, P, P, 4, None), "tree_keep")
    for n in (0, 65):
        refused(L.xqhip_tree_keep(xb.rows([good]), 1, P, P, n, None), "tree_keep")
    for bad in ((None, 16, 4, None), (P, 0, 4, None), (P, 16, -1, None), (P, 1 << 31, 4, None)):
        refused(L.xqhip_tree_keep(xb.rows([good, bad]), 2, P, P, 4, None), "buffer 1")
    at = lambda f: ctypes.c_void_p(P.value + f)  # noqa: E731
    for other in ((P, 16, 4, None), (at(63), 16, 4, None), (at(16), 8, 1, None)):
        refused(L.xqhip_tree_keep(xb.rows([(P, 16, 4, None), (at(4096), 16, 4, None), other]), 3, P, P, 4, None), "0 and 2 overlap")
    assert L.xqhip_tree_keep(None, 0, P, P, 4, None) == 0


@pytest.mark.parametrize("point", [False, True])
def test_definition_samples_the_target(point):
    """The first new token's distribution is the target's, whatever was drafted: 20000 walks over three siblings and
    their children; the largest of 12 frequencies' deviations stays within 4.5 standard deviations (chance of more:
    12 x 7e-6)."""
    rng = np.random.default_rng(5)
    vocab, walks, par = 12, 20000, [-1, 0, 0, 0, 1, 2]
    logits = rng.normal(0, 1.2, (6, vocab))
    draft = np.exp(logits + rng.normal(0, 1.0, logits.shape))
    draft /= draft.sum(1, keepdims=True)
    p = np.exp(logits[0] * 0.8)
    p /= p.sum()
    seen = np.zeros(vocab)
    for _ in range(walks):
        tok = [0] + [int(rng.integers(vocab)) if point else int(rng.choice(vocab, p=draft[q])) for q in par[1:]]
        _, out = to.verify(logits, par, tok, None if point else draft, 0.8, rng.random(6), rng.random())
        seen[out[0]] += 1
    dev = np.abs(seen / walks - p) / np.sqrt(p * (1 - p) / walks)
    assert dev.max() < 4.5, dev
