"""The drafted-token operators' refusals (ds_hip_tree_*, ds_hip_kv_evict): every one is made before the device is touched, so
these run without one; none of the pointers below is read. And the definition that the verification is held to."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import tree_reference as R  # noqa: E402

PTR = 1 << 20  # an address that nothing reads


def kv(lib, rows=100, heads=4, dim=128, dtype=0, rs=None, hs=None, k=PTR, v=2 * PTR):
    hs = dim if hs is None else hs
    return lib.KvCache(k, v, heads * dim if rs is None else rs, hs, rows, heads, dim, dtype)


def refused(lib, rc, *words):
    msg = lib.load().ds_hip_last_error().decode()
    assert rc == -1
    assert all(w in msg for w in words), msg


def attention(lib, **o):
    a = dict(out=PTR, os=1024, lse=PTR, scores=None, ss=0, q=PTR, qs=1024, heads=8, cache=kv(lib), n=90,
             tree=kv(lib, rows=8), parents=PTR, nodes=8, scale=0.1, prefill=0, window=0)
    a.update(o)
    ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
    return lib.load().ds_hip_tree_attention(a["out"], a["os"], a["lse"], a["scores"], a["ss"], a["q"], a["qs"], a["heads"],
                                            ref(a["cache"]), a["n"], ref(a["tree"]), a["parents"], a["nodes"], a["scale"],
                                            a["prefill"], a["window"])


@pytest.mark.parametrize("change, words", [
    (dict(out=None), "NULL"), (dict(q=None), "NULL"), (dict(parents=None), "NULL"), (dict(cache=None), "cache is NULL"),
    (dict(tree=None), "tree is NULL"), (dict(nodes=0), "0 nodes"), (dict(nodes=129), "129 nodes"),
    (dict(nodes=9), "9 rows of 8"), (dict(n=-1), "-1 rows"), (dict(n=101), "101 rows of 100"), (dict(heads=0), "0 query"),
    (dict(heads=6), "6 query heads over 4"), (dict(qs=1020), "1024 floats"), (dict(os=1020), "1024 floats"),
    (dict(qs=1026), "16 bytes"), (dict(q=PTR + 4), "16 bytes"), (dict(out=PTR + 8), "16 bytes"),
    (dict(scores=PTR, ss=97), "score_stride 97"), (dict(prefill=-1), "prefill_len"), (dict(window=-1), "window"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
])
def test_attention_refuses(lib, change, words):
    refused(lib, attention(lib, **change), "ds_hip_tree_attention", words)


@pytest.mark.parametrize("change, words", [
    (dict(dtype=2), "unknown type"), (dict(dim=80), "head_dim 80"), (dict(dim=320), "head_dim"), (dict(heads=0), "0 heads"),
    (dict(rows=-1), "-1 rows"), (dict(k=None), "NULL arrays"), (dict(v=None), "NULL arrays"), (dict(k=PTR + 8), "16 bytes"),
    (dict(rs=514), "16 bytes"), (dict(hs=130, rs=1024), "16 bytes"), (dict(rs=508), "overlap"), (dict(hs=64, rs=512), "overlap"),
    (dict(hs=0), "overlap"), (dict(rs=-512), "overlap"), (dict(rs=128, hs=12000), "overlap"), (dict(dtype=1, rs=516), "16 bytes"),
])
def test_views_are_checked(lib, change, words):
    refused(lib, attention(lib, cache=kv(lib, **change)), "cache", words)
    L = lib.load()
    n = 90
    bad = kv(lib, **change)
    rc = L.ds_hip_kv_evict(C.byref(bad), n, 50, PTR, n, None, 0, None, 0, None, 0, 0, n, None)
    refused(lib, rc, "ds_hip_kv_evict", words)


def test_views_side_by_side_are_fine(lib):
    """Rows by head, padded rows, one head with any head stride, one row with any row stride: what is refused is another
    argument."""
    for view in (kv(lib, rs=128, hs=12800), kv(lib, rs=640), kv(lib, heads=4, rows=1, rs=3), kv(lib, dtype=1)):
        refused(lib, attention(lib, cache=view, tree=kv(lib, rows=8, dtype=view.dtype), n=min(90, view.rows), nodes=8,
                               scale=float("nan")), "scale")
    one = kv(lib, heads=1, hs=5)
    refused(lib, attention(lib, cache=one, tree=kv(lib, heads=1, rows=8), scale=float("nan")), "scale")
    refused(lib, attention(lib, tree=kv(lib, rows=8, dim=64)), "differ")
    refused(lib, attention(lib, tree=kv(lib, rows=8, heads=2)), "differ")
    refused(lib, attention(lib, tree=kv(lib, rows=8, dtype=1)), "differ")


def test_verification_refuses(lib):
    L = lib.load()
    v = lambda path=PTR, res=PTR, p=PTR, ps=500, q=None, qs=0, V=500, tok=PTR, par=PTR, n=4, u=PTR: L.ds_hip_tree_verify(  # noqa: E731
        path, res, p, ps, q, qs, V, tok, par, n, u)
    for rc, word in ((v(path=None), "NULL"), (v(res=None), "NULL"), (v(p=None), "NULL"), (v(tok=None), "NULL"),
                     (v(par=None), "NULL"), (v(u=None), "NULL")):
        refused(lib, rc, "ds_hip_tree_verify", word)
    refused(lib, v(n=-1), "-1 nodes")
    refused(lib, v(n=129), "129 nodes")
    refused(lib, v(V=0), "vocab 0")
    refused(lib, v(V=2 ** 30 + 1, ps=2 ** 31), "vocab")
    refused(lib, v(ps=499), "strides 499")
    refused(lib, v(q=PTR, qs=499), "499")
    g = lambda path=PTR, res=PTR, tgt=PTR, tok=PTR, par=PTR, n=4: L.ds_hip_tree_verify_greedy(path, res, tgt, tok, par, n)  # noqa: E731
    for rc in (g(path=None), g(res=None), g(tgt=None), g(tok=None), g(par=None)):
        refused(lib, rc, "ds_hip_tree_verify_greedy", "NULL")
    refused(lib, g(n=129), "129 nodes")


def test_commit_refuses(lib):
    L = lib.load()

    def c(**o):
        a = dict(cache=kv(lib), n=90, tree=kv(lib, rows=8), nodes=8, path=PTR, res=PTR, scores=PTR, ss=98, lse=PTR, heads=8,
                 acc=PTR, out=1 << 24, acs=98, pos=PTR, ps=98, pos0=0)
        a.update(o)
        return L.ds_hip_tree_commit(C.byref(a["cache"]), a["n"], C.byref(a["tree"]), a["nodes"], a["path"], a["res"],
                                    a["scores"], a["ss"], a["lse"], a["heads"], a["acc"], a["out"], a["acs"], a["pos"],
                                    a["ps"], a["pos0"])
    for change, word in ((dict(path=None), "NULL"), (dict(res=None), "NULL"), (dict(nodes=0), "0 nodes"),
                         (dict(nodes=200), "200 nodes"), (dict(n=93), "101 rows of 100"), (dict(n=-1), "-1 cached"),
                         (dict(tree=kv(lib, rows=7)), "8 rows of 7"), (dict(tree=kv(lib, rows=8, dim=64)), "differ"),
                         (dict(out=None), "go together"), (dict(acc=None), "go together"), (dict(scores=None), "need scores"),
                         (dict(lse=None), "need scores"), (dict(heads=6), "6 query"), (dict(ss=97), "97"),
                         (dict(acs=97), "97"), (dict(out=PTR + 4), "overlaps"), (dict(ps=97), "pos_stride"),
                         (dict(pos0=-1), "pos0"), (dict(n=2 ** 31 - 1), "cached")):
        refused(lib, c(**change), "ds_hip_tree_commit", word)


def test_eviction_refuses(lib):
    L = lib.load()

    def e(**o):
        a = dict(cache=kv(lib), n=90, keep=50, acc=PTR, acs=90, out=None, ous=0, pos=None, ps=0, pout=None, pos_s=0, sink=0,
                 recent=90, slots=None)
        a.update(o)
        return L.ds_hip_kv_evict(C.byref(a["cache"]), a["n"], a["keep"], a["acc"], a["acs"], a["out"], a["ous"], a["pos"],
                                 a["ps"], a["pout"], a["pos_s"], a["sink"], a["recent"], a["slots"])
    for change, word in ((dict(n=-1), "-1 rows"), (dict(n=2 ** 30 + 1, keep=5), "rows"), (dict(keep=-1), "-1 of 90"), (dict(keep=91), "91 of 90"),
                         (dict(n=101, keep=5), "101 rows of 100"), (dict(acc=None), "NULL"), (dict(pout=PTR, pos_s=50), "pos_out"),
                         (dict(acs=89), "strides"), (dict(pos=PTR, ps=89), "strides"), (dict(out=1 << 24, ous=49), "strides"),
                         (dict(pos=PTR, ps=90, pout=1 << 24, pos_s=49), "strides"), (dict(out=PTR, ous=50), "lie apart"),
                         (dict(out=PTR + 400, ous=90), "lie apart"), (dict(pos=PTR, ps=90, pout=PTR + 40, pos_s=90), "lie apart")):
        refused(lib, e(**change), "ds_hip_kv_evict", word)
    assert e(keep=0) == 0 and e(n=0, keep=0) == 0  # nothing stays: nothing to do, with no device either
    refused(lib, L.ds_hip_attn_kv_view(None, C.byref(kv(lib))), "NULL")


@pytest.mark.parametrize("drawn", [False, True])
def test_first_token_follows_the_target(drawn):
    """The definition keeps the target's law: whatever the drafts, the first token after the root is distributed as p. 20000
    trials over 6 tokens; 5 standard deviations of a count are at most 5 sqrt(20000 / 4) = 354."""
    rng = np.random.default_rng(5)
    V, n, trials = 6, 4, 20000
    p = rng.dirichlet(np.ones(V), n + 1).astype(np.float32)
    q = rng.dirichlet(np.ones(V), n + 1).astype(np.float32)
    parents = np.array([-1, -1, 0, -1], np.int32)  # three children of the root
    got = np.zeros(V)
    for _ in range(trials):
        tokens = rng.choice(V, n, p=q[0].astype(np.float64) / q[0].sum(dtype=np.float64)) if drawn else np.array([2, 0, 1, 2])
        path, token = R.verify(p, q if drawn else None, rng.random(n + 1, dtype=np.float32), tokens, parents, V)
        got[tokens[path[0]] if path else token] += 1
    assert np.abs(got - trials * p[0]).max() < 354
