"""GPU: drafted tokens over a KV cache (ds_hip_tree_attention, ds_hip_tree_verify, ds_hip_tree_commit, ds_hip_kv_evict)
against their plain 64-bit forms (tree_reference.py), and all of them together. Attention and the accumulated weights are held
to error bounds derived there; whole numbers and copied rows are equal."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import tree_reference as R  # noqa: E402
from tree_reference import U, Cache, normal  # noqa: E402

pytestmark = pytest.mark.gpu


def same(got, want):
    np.testing.assert_array_equal(got, want)


def within(got, want, tol, what):
    """got (f32) against want (f64): the same infinities, else within tol."""
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin].astype(np.float64), want[~fin]), what
    bad = ~(np.abs(got[fin] - want[fin]) <= np.broadcast_to(tol, want.shape)[fin])
    if bad.any():
        err = np.abs(got[fin] - want[fin])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(err / tol[fin]):.3g} of the bound")


class Attend:
    """The device buffers of one tree attention and its call."""

    def __init__(self, dev, q, cache, n, tree, parents, scale, prefill=0, window=0, pad=4, score_pad=3):
        T, H, D = q.shape
        self.dev, self.T, self.H, self.D, self.n = dev, T, H, D, n
        self.w = H * D + pad
        qq = np.full((T, self.w), np.nan, np.float32)
        qq[:, :H * D] = q.reshape(T, H * D)
        self.q = dev.DeviceBuffer.from_array(qq)
        self.ss = n + T + score_pad
        self.out = dev.DeviceBuffer.from_array(np.full((T, self.w), -7.0, np.float32))
        self.lse = dev.DeviceBuffer.from_array(np.full((H, T), -7.0, np.float32))
        self.scores = dev.DeviceBuffer.from_array(np.full((H, T, self.ss), -7.0, np.float32))
        self.parents = dev.DeviceBuffer.from_array(parents)
        self.cache, self.tree = cache, tree
        self.args = (scale, prefill, window)

    def call(self, scores=True, lse=True):
        L = self.dev.load()
        self.dev.check(L.ds_hip_tree_attention(
            self.out.ptr, self.w, self.lse.ptr if lse else None, self.scores.ptr if scores else None, self.ss, self.q.ptr,
            self.w, self.H, self.cache.ref, self.n, self.tree.ref, self.parents.ptr, self.T, *self.args), "attention")
        self.dev.check(L.ds_hip_sync(), "sync")
        return self

    def fetch(self):
        out = self.out.to_array(np.float32).reshape(self.T, self.w)
        assert (out[:, self.H * self.D:] == -7).all()  # nothing behind a row
        sc = self.scores.to_array(np.float32).reshape(self.H, self.T, self.ss)
        assert (sc[..., self.n + self.T:] == -7).all()
        return (out[:, :self.H * self.D].reshape(self.T, self.H, self.D), self.lse.to_array(np.float32).reshape(self.H, self.T),
                sc[..., :self.n + self.T])


def attend(dev, T, H, G, D, n, bf16=False, by_head=False, gap=0, pad=0, prefill=0, window=0, seed=0, chain=False, std=1.5,
           spare=3, scores=True):
    print(f"attention T={T} H={H} G={G} D={D} n={n} bf16={bf16} by_head={by_head} window=({prefill},{window}) seed={seed}",
          flush=True)
    rng = np.random.default_rng(seed)
    parents = np.arange(-1, T - 1, dtype=np.int32) if chain else R.random_tree(rng, T, pad)
    q = normal(rng, T, H, D, std=std)
    k, v = (normal(rng, n + spare, G, D, bf16=bf16) for _ in range(2))
    kt, vt = (normal(rng, T, G, D, bf16=bf16) for _ in range(2))
    dead = [i for i, c in enumerate(R.chains(parents)) if not c]
    qd, kd, vd, ktd, vtd = q.copy(), k.copy(), v.copy(), kt.copy(), vt.copy()
    for a in (kd, vd):  # the rows behind the cache are nobody's
        a[n:] = np.nan
    for a in (qd, ktd, vtd):  # a padding node's inputs hold anything
        a[dead] = np.nan
    f = lambda a: np.where(np.isnan(a), np.nan, a)  # noqa: E731
    if bf16:  # NaN as such; bf16_bits takes finite values
        fill = lambda a: np.nan_to_num(a, nan=3e38)  # noqa: E731
        kd, vd, ktd, vtd = fill(kd), fill(vd), fill(ktd), fill(vtd)
    scale = 1 / np.sqrt(D)
    scale = float(np.float32(scale))
    at = Attend(dev, f(qd), Cache(dev, kd, vd, bf16, by_head, gap), n, Cache(dev, ktd, vtd, bf16, False, gap), parents, scale,
                prefill, window)
    at.call(scores)
    out, lse, sc = at.fetch()
    wo, wl, ws, to, tl, ts = R.attention(q, k[:n], v[:n], kt, vt, n, parents, scale, prefill, window)
    within(out, wo, to, "out")
    within(lse, wl, tl, "lse")
    if scores:
        within(sc, ws, ts, "scores")
    return at


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("H, G", [(2, 2), (6, 2), (5, 1), (8, 1)])
def test_attention_heads_and_types(dev, D, bf16, H, G):
    for T, n in ((1, 0), (1, 1), (3, 40), (17, 131)):
        attend(dev, T, H, G, D, n, bf16, by_head=n % 2 == 1, gap=n % 3, seed=D + T)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_attention_cache_lengths(dev, n, bf16):
    attend(dev, 5, 2, 2, 128, n, bf16, seed=n)
    attend(dev, 2, 2, 1, 64, n, bf16, seed=n, scores=False)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128])
def test_attention_node_counts(dev, T, bf16):
    attend(dev, T, 2, 1, 128, 37, bf16, pad=T // 5, seed=T)
    attend(dev, T, 2, 2, 64, 70, bf16, chain=True, seed=T)


@pytest.mark.parametrize("n, prefill, window", [(50, 0, 1), (50, 20, 1), (50, 20, 2), (50, 20, 7), (50, 50, 3), (50, 52, 2),
                                                (50, 100, 4), (300, 10, 64), (300, 100, 150), (300, 0, 299), (300, 0, 1000),
                                                (0, 0, 2), (0, 3, 1), (700, 130, 64), (700, 0, 70)])
@pytest.mark.parametrize("bf16", [False, True])
def test_attention_window(dev, n, prefill, window, bf16):
    attend(dev, 9, 3, 1, 128, n, bf16, prefill=prefill, window=window, chain=True, seed=n + window)
    attend(dev, 20, 2, 2, 64, n, bf16, prefill=prefill, window=window, pad=3, seed=n + window)


@pytest.mark.parametrize("T, H, G, D, n, bf16", [(3, 10, 10, 128, 2000, False), (40, 4, 4, 128, 1500, False),
                                                 (12, 8, 2, 64, 5000, True), (70, 2, 1, 256, 900, True),
                                                 (1, 4, 4, 128, 7679, False), (128, 2, 2, 192, 777, False),
                                                 (100, 12, 2, 128, 200, False), (100, 12, 2, 64, 200, True),
                                                 (60, 6, 1, 256, 150, False)])
def test_attention_longer(dev, T, H, G, D, n, bf16):
    attend(dev, T, H, G, D, n, bf16, seed=T, scores=T < 40)


@pytest.mark.parametrize("std", [1e-3, 30.0])
def test_attention_flat_and_sharp(dev, std):
    """Scores that all but coincide, and scores of a few hundred."""
    attend(dev, 6, 2, 2, 128, 200, std=std, seed=7)
    attend(dev, 33, 4, 1, 128, 200, bf16=True, std=std, seed=8)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("T", [6, 40])
def test_attention_unseen_values(dev, what, bf16, T):
    """What a node does not see holds NaN, infinities or the largest values: a sibling's branch, cached rows outside the window."""
    rng = np.random.default_rng(3)
    H, G, D, n, prefill, window = 4, 2, 128, 150, 30, 40
    parents = np.array([-1, 0, 1, -1, 3, 2] + [5] * (T - 6), np.int32)  # 3 and 4 are a branch of their own
    q = normal(rng, T, H, D)
    k, v = (normal(rng, n, G, D, bf16=bf16) for _ in range(2))
    kt, vt = (normal(rng, T, G, D, bf16=bf16) for _ in range(2))
    bad = what if not bf16 or np.isfinite(what) else what
    kd, vd, ktd, vtd = k.copy(), v.copy(), kt.copy(), vt.copy()
    hide = slice(prefill, n - window)  # no node sees these
    kd[hide], vd[hide] = 0, 0
    ktd[3:5], vtd[3:5] = 0, 0
    cache, tree = Cache(dev, kd, vd, bf16), Cache(dev, ktd, vtd, bf16)
    bits = {"nan": 0x7FC1, "inf": 0x7F80, "-inf": 0xFF80, "3e+38": 0x7F61}[str(what)]
    for cch, sl in ((cache, hide), (tree, slice(3, 5))):
        for buf, raw in zip(cch.bufs, cch.raw):
            cch.view(raw)[sl] = bits if bf16 else np.float32(bad)
            buf.write(raw)
    scale = float(np.float32(D ** -0.5))
    at = Attend(dev, q, cache, n, tree, parents, scale, prefill, window).call()
    out, lse, sc = at.fetch()
    wo, wl, ws, to, tl, ts = R.attention(q, k, v, kt, vt, n, parents, scale, prefill, window)
    rest = [i for i in range(T) if i not in (3, 4)]  # 3 and 4 see themselves
    within(out[rest], wo[rest], to[rest], "out")
    within(lse[:, rest], wl[:, rest], tl[:, rest], "lse")
    within(sc[:, rest], ws[:, rest], ts[:, rest], "scores")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T", [3, 30])
def test_attention_seen_values(dev, T, bf16):
    """A V row that is not finite and seen, the cache's last one among others: its head's outputs are not finite, the other
    head's are right."""
    rng = np.random.default_rng(2)
    H, D, n = 2, 128, 77
    parents = R.random_tree(rng, T)
    q = normal(rng, T, H, D)
    k, v = (normal(rng, n, H, D, bf16=bf16) for _ in range(2))
    kt, vt = (normal(rng, T, H, D, bf16=bf16) for _ in range(2))
    scale = float(np.float32(D ** -0.5))
    wo, wl, ws, to, tl, ts = R.attention(q, k, v, kt, vt, n, parents, scale)
    for row in (0, 40, n - 1):
        cache = Cache(dev, k, v, bf16)
        cache.view(cache.raw[1])[row, 0] = 0x7F80 if bf16 else np.inf
        cache.bufs[1].write(cache.raw[1])
        out, lse, sc = Attend(dev, q, cache, n, Cache(dev, kt, vt, bf16), parents, scale).call().fetch()
        assert not np.isfinite(out[:, 0]).any()
        within(out[:, 1], wo[:, 1], to[:, 1], "out")
        within(lse, wl, tl, "lse")


def test_attention_far_offsets(dev):
    """Rows 2^30 floats apart: element offsets beyond 2^31, byte offsets beyond 2^33."""
    L = dev.load()
    rng = np.random.default_rng(4)
    n, T, H, D, rs = 3, 2, 2, 64, 1 << 30
    q, k, v, kt, vt = (normal(rng, r, H, D) for r in (T, n, n, T, T))
    big = dev.DeviceBuffer(4 * (rs * (n - 1) + 4 * H * D))
    off = 4 * H * D  # v stands right behind k in every row
    for r in range(n):
        for a, o in ((k, 0), (v, off)):
            row = np.ascontiguousarray(a[r], np.float32)
            dev.check(L.ds_hip_memcpy_h2d(big.ptr + 4 * rs * r + o, row.ctypes.data, row.nbytes), "h2d")
    tree = Cache(dev, kt, vt)

    class Far:
        st = dev.KvCache(big.ptr, big.ptr + off, rs, D, n, H, D, dev.KV_F32)
        ref = C.byref(st)
    parents = np.array([-1, 0], np.int32)
    scale = 0.125
    out, lse, sc = Attend(dev, q, Far, n, tree, parents, scale).call().fetch()
    wo, wl, ws, to, tl, ts = R.attention(q, k, v, kt, vt, n, parents, scale)
    within(out, wo, to, "out")
    within(sc, ws, ts, "scores")
    # the last row moves to the first: the far row is read and the near one written
    acc = np.array([[0.1, 2, 3]] * H, np.float32)
    ad = dev.DeviceBuffer.from_array(acc)
    dev.check(L.ds_hip_kv_evict(Far.ref, n, 2, ad.ptr, n, None, 0, None, 0, None, 0, 0, n, None), "evict")
    got = np.empty((2, H, D), np.float32)
    dev.check(L.ds_hip_memcpy_d2h(got.ctypes.data, big.ptr, got.nbytes), "d2h")
    same(got, np.stack([k[2], v[2]]).astype(np.float32))


def test_attention_repeats(dev):
    """The same call again, after larger and smaller ones, gives the same bits; outputs that are not asked for are not written."""
    a = attend(dev, 20, 4, 4, 128, 600, seed=1)
    first = a.fetch()
    attend(dev, 128, 8, 2, 256, 900, bf16=True, seed=2, scores=False)
    attend(dev, 1, 1, 1, 64, 1, seed=3)
    for _ in range(3):
        for x, y in zip(a.call().fetch(), first):
            same(x, y)
    a.lse.write(np.full(a.lse.nbytes // 4, -7.0, np.float32))
    a.scores.write(np.full(a.scores.nbytes // 4, -7.0, np.float32))
    a.call(scores=False, lse=False)
    assert (a.lse.to_array(np.float32) == -7).all() and (a.scores.to_array(np.float32) == -7).all()
    same(a.out.to_array(np.float32).reshape(20, -1)[:, :512], first[0].reshape(20, -1))


def test_attention_over_a_handles_cache(dev):
    """One token over the f32 cache of an attention handle, in the handle's own layout."""
    L = dev.load()
    rng = np.random.default_rng(6)
    hidden, H, D, n = 256, 2, 128, 77
    z = lambda *s: np.zeros(s, np.uint16)  # noqa: E731
    one = np.ones(hidden, np.float32)
    w = [z(H * D, hidden), z(H * D, hidden), z(H * D, hidden), z(hidden, H * D)]
    A = L.ds_hip_attn_create(hidden, H, D, 100, 1e-6, 1e4, *[x.ctypes.data for x in w], one.ctypes.data, one.ctypes.data, None, None)
    assert A
    try:
        view = dev.KvCache()
        dev.check(L.ds_hip_attn_kv_view(A, C.byref(view)), "view")
        assert (view.rows, view.n_heads, view.head_dim, view.dtype) == (100, H, D, dev.KV_F32)
        k, v = normal(rng, n, H, D), normal(rng, n, H, D)
        kf, vf = k.astype(np.float32), v.astype(np.float32)
        dev.check(L.ds_hip_attn_load_kv(A, kf.ctypes.data, vf.ctypes.data, n, H * D), "load")

        class Handle:
            st, ref = view, C.byref(view)
        q, kt, vt = (normal(rng, 1, H, D) for _ in range(3))
        out, lse, sc = Attend(dev, q, Handle, n, Cache(dev, kt, vt), np.array([-1], np.int32), 0.0883883461356163).call().fetch()
        wo, wl, ws, to, tl, ts = R.attention(q, k, v, kt, vt, n, [-1], 0.0883883461356163)
        within(out, wo, to, "out")
        within(lse, wl, tl, "lse")
    finally:
        L.ds_hip_attn_destroy(A)


# ---------------------------------------------------------------------------- verification
def verify(dev, p, q, u, tokens, parents, vocab, pad=0):
    L = dev.load()
    n = len(tokens)
    B = dev.DeviceBuffer.from_array
    wide = lambda a: np.concatenate([a, np.full((a.shape[0], pad), np.nan, np.float32)], 1) if pad else a  # noqa: E731
    pd, qd, ud = B(wide(p)), B(wide(q)) if q is not None else None, B(u)
    td, rd = B(np.array(list(tokens) + [0], np.int32)), B(np.array(list(parents) + [0], np.int32))
    path, res = B(np.full(n + 1, -9, np.int32)), B(np.full(2, -9, np.int32))
    dev.check(L.ds_hip_tree_verify(path.ptr, res.ptr, pd.ptr, vocab + pad, qd.ptr if qd else None, vocab + pad, vocab, td.ptr,
                                   rd.ptr, n, ud.ptr), "verify")
    dev.check(L.ds_hip_sync(), "sync")
    out = path.to_array(np.int32)
    assert out[n] == -9
    count, token = res.to_array(np.int32)
    assert (out[count:n] == -1).all()
    return list(out[:count]), int(token)


def distributions(rng, n, V, sharp=2.0):
    x = np.exp(sharp * rng.standard_normal((n + 1, V)))
    return (x / x.sum(1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 1000, 1024, 1025, 5000])
def test_verify_random_trees(dev, V, drawn):
    for seed in range(25):
        rng = np.random.default_rng(1000 * V + seed)
        n = int(rng.choice([0, 1, 2, 5, 16, 64, 100, 128])) if seed else 128
        print(f"verify V={V} drawn={drawn} seed={seed} n={n}", flush=True)
        p = distributions(rng, n, V)
        q = distributions(rng, n, V) if seed % 2 else np.where(rng.random((n + 1, V)) < 0.3, 0, p).astype(np.float32)
        parents = R.random_tree(rng, n, n // 8, width=int(rng.integers(1, 6)))
        tokens = rng.choice(min(V, 4), n) if seed % 3 == 0 else p[np.clip(parents, -1, n - 1) + 1].argmax(1) if n else []
        tokens = np.array(tokens, np.int32)
        if n > 4:
            tokens[rng.integers(0, n, 2)] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31], 2)
        u = rng.random(n + 1, dtype=np.float32) ** (1 if seed % 4 else 4)
        u = u.astype(np.float32)
        want = R.verify(p, q if drawn else None, u, tokens, parents, V)
        assert verify(dev, p, q if drawn else None, u, tokens, parents, V, pad=seed % 3) == want


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("n", [0, 1, 12])
def test_verify_full_vocabulary(dev, n, drawn):
    rng = np.random.default_rng(n)
    V = 129280
    p, q = distributions(rng, n, V, 3.0), distributions(rng, n, V, 3.0)
    parents = np.array([-1, -1, -1, 0, 0, 1, 2, 2, 3, 8, 9, 9][:n], np.int32)
    for seed in range(12):
        r = np.random.default_rng(seed)
        tokens = r.choice(V, n).astype(np.int32)
        if seed % 2:  # drafts that are taken
            for i in range(n):
                p[parents[i] + 1, tokens[i]], q[parents[i] + 1, tokens[i]] = 0.5, 0.25
        u = r.random(n + 1, dtype=np.float32)
        u[n] = [0, 1 - 2 ** -24, 0.5, 2.0 ** -24][seed % 4] if seed < 8 else u[n]
        assert verify(dev, p, q if drawn else None, u, tokens, parents, V) == R.verify(p, q if drawn else None, u, tokens,
                                                                                     parents, V), seed


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_large_vocabulary(dev, drawn):
    """More than one piece a block; the weight in the last values, in the first, in none of a block's last piece."""
    V, n = 300000, 2
    rng = np.random.default_rng(9)
    for where in (slice(0, V), slice(0, 3), slice(V - 3, V), slice(150000, 150001), slice(2040, 2060)):
        p = np.zeros((n + 1, V), np.float32)
        p[:, where] = rng.random(p[:, where].shape, dtype=np.float32) + 1e-3
        p /= p.sum(1, keepdims=True)
        q = np.full((n + 1, V), 1 / V, np.float32)
        for last in (0.0, 0.3, 1 - 2 ** -24):
            u = np.array([0.9, 0.9, last], np.float32)
            tokens, parents = np.array([5, V - 1], np.int32), np.array([-1, -1], np.int32)
            assert verify(dev, p, q if drawn else None, u, tokens, parents, V) == R.verify(p, q if drawn else None, u, tokens, parents, V)


def test_verify_borders_and_strange_values(dev):
    """Equal sides are a rejection; NaN, infinite, negative and zero probabilities; nothing left; a token twice."""
    V, n = 8, 3
    f = lambda *x: np.array(x, np.float32)  # noqa: E731
    p = np.tile(f(0.5, 0.25, 0.25, 0, 0, 0, 0, 0), (n + 1, 1))
    q = np.tile(f(1.0, 0, 0, 0, 0, 0, 0, 0), (n + 1, 1))
    chain, fan = [-1, 0, 1], [-1, -1, -1]
    nan, inf = np.nan, np.inf
    odd = p.copy()
    odd[0] = f(nan, inf, -1, 0.5, -inf, 0, 1e-45, 0.25)
    cases = [(p, q, [0.5, 0, 0, 0.5], [0, 0, 0], chain), (p, None, [0.5, 0, 0, 0.5], [0, 0, 0], chain),
             (p, q, [0.49, 0.5, 0, 0], [0, 0, 0], chain), (p, None, [0.75, 0.5, 0.9, 0], [0, 0, 1], fan),
             (p, None, [0.75, 0.5, 0.5, 0.99], [0, 1, 2], fan), (p, p, [0.999, 0.999, 0.999, 0.7], [0, 1, 2], fan),
             (p, p, [0, 0, 0, 0.3], [3, 4, 5], fan), (p * 0, q, [0, 0, 0, 0.3], [0, 1, 2], chain),
             (p * 0, None, [0, 0, 0, 0.3], [0, 1, 2], fan), (odd, None, [0, 0, 0, 0.6], [0, 1, 2], fan),
             (odd, None, [0, 0, 0, 0.0], [4, 6, 3], fan), (odd, odd, [0.9, 0.9, 0.9, 0.2], [3, 7, 6], fan),
             (np.tile(f(1, 0, 0, 0, 0, 0, 0, 0), (n + 1, 1)), None, [0.5, 0.5, 0.5, 0.5], [1, 2, 3], fan),
             (np.tile(f(1, 0, 0, 0, 0, 0, 0, 0), (n + 1, 1)), None, [0.5, 0.5, 0.5, 0.5], [0, 0, 0], chain)]
    for pp, qq, u, tokens, parents in cases:
        u = f(*u)
        want = R.verify(pp, qq, u, tokens, parents, V)
        assert verify(dev, pp, qq, u, tokens, parents, V) == want, (u, tokens, want)
    assert R.verify(p, q, f(0.5, 0, 0, 0.5), [0, 0, 0], chain, V) == ([], 2)  # rejected at the border; 0 left at token 0


def test_verify_greedy(dev):
    L = dev.load()
    B = dev.DeviceBuffer.from_array
    for seed in range(40):
        rng = np.random.default_rng(seed)
        n = int(rng.choice([0, 1, 3, 17, 64, 65, 128]))
        parents = R.random_tree(rng, n, n // 6, width=3)
        tokens = rng.choice(3, n).astype(np.int32)
        target = rng.choice([0, 1, 2, -5], n + 1, p=[0.4, 0.3, 0.2, 0.1]).astype(np.int32)
        td, tk, pr = B(target), B(np.append(tokens, 0).astype(np.int32)), B(np.append(parents, 0).astype(np.int32))
        path, res = B(np.full(n + 1, -9, np.int32)), B(np.full(2, -9, np.int32))
        dev.check(L.ds_hip_tree_verify_greedy(path.ptr, res.ptr, td.ptr, tk.ptr, pr.ptr, n), "verify")
        dev.check(L.ds_hip_sync(), "sync")
        got, (count, token) = path.to_array(np.int32), res.to_array(np.int32)
        want = R.verify_greedy(target, tokens, parents)
        assert (list(got[:count]), int(token)) == want and (got[count:n] == -1).all() and got[n] == -9


# ---------------------------------------------------------------------------- commit
def commit_case(dev, T, H, G, D, n, path, claimed, bf16, weights=True, in_place=False, seed=0, by_head=False, pos=True):
    print(f"commit T={T} H={H} G={G} D={D} n={n} path={path} claimed={claimed} bf16={bf16}", flush=True)
    L = dev.load()
    rng = np.random.default_rng(seed)
    B = dev.DeviceBuffer.from_array
    good = []
    for x in path[:max(0, min(claimed, T))]:
        if not 0 <= x < T:
            break
        good.append(x)
    cache = Cache(dev, normal(rng, n + T + 2, G, D, bf16=bf16), normal(rng, n + T + 2, G, D, bf16=bf16), bf16, by_head, 1)
    tree = Cache(dev, normal(rng, T, G, D, bf16=bf16), normal(rng, T, G, D, bf16=bf16), bf16, False, 2)
    want = cache.expect()
    for w, t in zip(want, tree.expect()):
        for k, x in enumerate(good):
            cache.view(w)[n + k] = tree.view(t)[x]
    ss, acs, ps = n + T + 1, n + T + 2, n + T + 3
    scores = rng.standard_normal((H, T, ss)).astype(np.float32) * 2
    scores[rng.random(scores.shape) < 0.1] = -np.inf
    lse = np.log(np.exp(scores[..., :n + T].astype(np.float64)).sum(-1)).astype(np.float32)
    scores[0, 0], lse[0, 0] = -np.inf, -np.inf  # a node that sees nothing
    acc = rng.random((G, acs)).astype(np.float32)
    sd, ld, ad = B(scores), B(lse), B(acc)
    out = ad if in_place else B(np.full((G, acs), -7.0, np.float32))
    pd = B(np.full((G, ps), -7, np.int32))
    pth = np.full(T, -1, np.int32)
    pth[:len(path)] = path
    path_d, res = B(pth), B(np.array([claimed, 5], np.int32))
    dev.check(L.ds_hip_tree_commit(cache.ref, n, tree.ref, T, path_d.ptr, res.ptr, sd.ptr if weights else None, ss,
                                   ld.ptr if weights else None, H, ad.ptr if weights else None, out.ptr if weights else None,
                                   acs, pd.ptr if pos else None, ps, 1000), "commit")
    dev.check(L.ds_hip_sync(), "sync")
    for g, w in zip(cache.fetch(), want):
        same(g, w)
    wp = np.full((G, ps), -7, np.int32)
    if pos:
        wp[:, n:n + len(good)] = 1000 + np.arange(len(good))
    same(pd.to_array(np.int32).reshape(G, ps), wp)
    got = out.to_array(np.float32).reshape(G, acs)
    base = acc if in_place or not weights else np.full((G, acs), -7.0, np.float32)
    if not weights:
        same(ad.to_array(np.float32).reshape(G, acs), acc)
        return
    same(got[:, n + len(good):], base[:, n + len(good):])
    cols = list(range(n)) + [n + x for x in good]
    s64 = scores.astype(np.float64)
    for g in range(G):
        add, tol = np.zeros(len(cols)), np.zeros(len(cols))
        for h in range(g * (H // G), (g + 1) * (H // G)):
            for x in good:
                if np.isfinite(lse[h, x]):
                    w = np.exp(s64[h, x, cols] - float(lse[h, x]))
                    add += w
                    # the difference is off by U of its size, the exponential by 4 U more
                    tol += w * U * (np.abs(np.where(w > 0, s64[h, x, cols] - float(lse[h, x]), 0)) + 4)
        old = np.concatenate([acc[g, :n].astype(np.float64), np.zeros(len(good))])
        tol += (len(good) * (H // G) + 1) * U * (old + add) + 1e-37
        within(got[g, :n + len(good)], old + add, tol, "acc")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_commit(dev, D, bf16):
    commit_case(dev, 5, 4, 2, D, 0, [0, 2], 2, bf16)
    commit_case(dev, 5, 4, 2, D, 300, [1, 3, 4], 3, bf16, by_head=True, in_place=True)
    commit_case(dev, 1, 3, 3, D, 255, [0], 1, bf16)
    commit_case(dev, 128, 2, 1, D, 700, list(range(128)), 128, bf16)


@pytest.mark.parametrize("path, claimed", [([], 0), ([3, 1, 2], 0), ([3, 1, 2], -4), ([3, 1, 2], 2), ([0, 9, 2], 3),
                                           ([0, -1, 2], 3), ([2, 2, 2], 3), ([7, 0], 1000)])
def test_commit_paths(dev, path, claimed):
    """Nothing accepted, fewer than the path holds, entries out of range, the same node again, a count beyond the nodes."""
    commit_case(dev, 8, 4, 2, 64, 37, path, claimed, False)
    commit_case(dev, 8, 4, 2, 64, 37, path, claimed, True, weights=False)
    commit_case(dev, 8, 4, 2, 64, 37, path, claimed, False, in_place=True, pos=False)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("path", [[0], [1, 2], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17],
                                  [3, 7, 20, 21, 39], list(range(5, 40))])
def test_commit_of_rows_within_the_cache(dev, path, bf16):
    """The drafts' rows stand in the cache itself, from n_cache on: accepted ones move down over rejected ones."""
    L = dev.load()
    rng = np.random.default_rng(len(path))
    n, T, G, D = 21, 40, 2, 128
    cache = Cache(dev, normal(rng, n + T, G, D, bf16=bf16), normal(rng, n + T, G, D, bf16=bf16), bf16)
    want = cache.expect()
    for w in want:
        v = cache.view(w)
        v[n:n + len(path)] = v[n + np.array(path)].copy()
    size = 2 if bf16 else 4
    st = cache.st
    tree = dev.KvCache(st.k + n * st.row_stride * size, st.v + n * st.row_stride * size, st.row_stride, st.head_stride, T, G, D,
                       st.dtype)
    pth = np.array(path + [-1] * (T - len(path)), np.int32)
    pd, rd = dev.DeviceBuffer.from_array(pth), dev.DeviceBuffer.from_array(np.array([len(path), 0], np.int32))
    dev.check(L.ds_hip_tree_commit(cache.ref, n, C.byref(tree), T, pd.ptr, rd.ptr, None, 0, None, 0, None, None, 0, None, 0, 0),
              "commit")
    dev.check(L.ds_hip_sync(), "sync")
    for got, w in zip(cache.fetch(), want):
        same(got, w)


# ---------------------------------------------------------------------------- eviction
def evict_case(dev, G, D, n, keep, bf16=False, by_head=False, sink=0, recent=None, acc=None, pos=True, in_place=False, seed=0,
               outputs=True):
    print(f"evict G={G} D={D} n={n} keep={keep} bf16={bf16} sink={sink} recent={recent} seed={seed}", flush=True)
    L = dev.load()
    rng = np.random.default_rng(seed)
    B = dev.DeviceBuffer.from_array
    cache = Cache(dev, normal(rng, n + 2, G, D, bf16=bf16), normal(rng, n + 2, G, D, bf16=bf16), bf16, by_head, 1)
    acs, ps = n + 3, n + 1
    a = np.full((G, acs), -3.0, np.float32)
    a[:, :n] = np.exp(rng.standard_normal((G, n))) if acc is None else acc
    p = np.stack([np.append(rng.permutation(n), -1) for _ in range(G)]).astype(np.int32)
    recent = n if recent is None else recent
    slots = R.evict_slots(a[:, :n], p[:, :n] if pos else np.tile(np.arange(n), (G, 1)), keep, sink, recent)
    want = cache.expect()
    for w in want:
        v = cache.view(w)
        old = v.copy()
        for g in range(G):
            v[:keep, g] = old[slots[g], g]
    ad, pd, sd = B(a), B(p), B(np.full((G, max(keep, 1)), -9, np.int32))
    os_ = acs if in_place else keep + 5
    po = ps if in_place else keep + 2
    ao = ad if in_place else B(np.full((G, os_), -7.0, np.float32))
    pout = pd if in_place else B(np.full((G, po), -7, np.int32))
    dev.check(L.ds_hip_kv_evict(cache.ref, n, keep, ad.ptr, acs, ao.ptr if outputs else None, os_, pd.ptr if pos else None, ps,
                                pout.ptr if outputs and pos else None, po, sink, recent, sd.ptr if outputs else None), "evict")
    dev.check(L.ds_hip_sync(), "sync")
    for got, w in zip(cache.fetch(), want):
        same(got, w)
    if not outputs:
        return
    same(sd.to_array(np.int32).reshape(G, -1)[:, :keep], slots)
    base = a if in_place else np.full((G, os_), -7.0, np.float32)
    wa = base.copy()
    wa[:, :keep] = np.take_along_axis(a, slots, 1)
    same(ao.to_array(np.uint32).reshape(G, os_), wa.view(np.uint32))
    if pos:
        wp = p.copy() if in_place else np.full((G, po), -7, np.int32)
        wp[:, :keep] = np.take_along_axis(p, slots, 1)
        same(pout.to_array(np.int32).reshape(G, po), wp)


@pytest.mark.parametrize("n, keep", [(1, 1), (2, 1), (5, 5), (64, 63), (65, 1), (100, 37), (1023, 512), (1024, 1000), (1025, 1024),
                                     (3000, 1500), (3001, 2999), (4096, 4000), (4097, 100), (7679, 4096), (8193, 8000), (16384, 5000),
                                     (20000, 9000), (32768, 16384), (32769, 16384), (70001, 30000)])
def test_evict_lengths(dev, n, keep):
    evict_case(dev, 3, 64, n, keep, seed=n)
    evict_case(dev, 2, 128, n, keep, bf16=True, by_head=True, sink=3, recent=max(0, n - n // 4), in_place=True, seed=n + 1)


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("bf16", [False, True])
def test_evict_dims(dev, D, bf16):
    evict_case(dev, 4, D, 333, 200, bf16=bf16, sink=2, recent=300)
    evict_case(dev, 1, D, 333, 200, bf16=bf16, pos=False, sink=2, recent=300)
    evict_case(dev, 4, D, 333, 200, bf16=bf16, outputs=False)


def test_evict_ties_and_strange_weights(dev):
    n = 500
    rng = np.random.default_rng(1)
    same_all = np.zeros((2, n))
    few = rng.integers(0, 3, (2, n)).astype(np.float32)
    odd = rng.choice(np.array([0.0, -0.0, 1.0, -1.0, np.nan, np.inf, -np.inf, 1e-45, -1e-45, 3e38], np.float32), (2, n))
    for acc in (same_all, few, odd, np.full((2, n), np.nan)):
        for keep in (1, 100, 250, 499):
            evict_case(dev, 2, 64, n, keep, acc=acc, seed=keep)
            evict_case(dev, 2, 64, n, keep, acc=acc, sink=20, recent=400, seed=keep)


@pytest.mark.parametrize("sink, recent", [(0, 0), (1000, 1000), (-5, 10 ** 9), (300, 301), (100, 200), (2 ** 31 - 1, 0), (0, 400)])
def test_evict_more_guarded_than_kept(dev, sink, recent):
    """Guarded rows outnumber the rows that stay: the guarded with the least weight go too."""
    for keep in (1, 50, 399):
        evict_case(dev, 2, 64, 400, keep, sink=sink, recent=recent, seed=keep)


# ---------------------------------------------------------------------------- together
@pytest.mark.parametrize("bf16", [False, True])
def test_steps_together(dev, bf16):
    """Ten steps of a decode loop with drafts over two layers' caches, held to a budget: attention, verification, commit and
    eviction fed with one another's outputs, the caches, weights and positions compared with a 64-bit simulation's each
    step. The simulation takes the eviction's choice from the library's accumulated weights (they are f32 sums: a choice
    between two rows may hang on their last bit), which it first compares with its own."""
    L = dev.load()
    rng = np.random.default_rng(11)
    B = dev.DeviceBuffer.from_array
    H, G, D, V, T, rows, budget, sink, recent = 4, 2, 64, 300, 7, 120, 60, 2, 10
    scale = 0.125
    layers = []
    n = 45
    for _ in range(2):
        k, v = normal(rng, rows, G, D, bf16=bf16), normal(rng, rows, G, D, bf16=bf16)
        acc = rng.random((G, rows)).astype(np.float32)
        pos = np.tile(np.arange(rows, dtype=np.int32), (G, 1))
        layers.append({"cache": Cache(dev, k, v, bf16), "k": k, "v": v, "acc": B(acc), "pos": B(pos), "a": acc.astype(np.float64),
                       "p": pos, "tol": np.zeros((G, rows))})
    where, evicted, accepted = n, 0, 0
    for step in range(10):
        parents = R.random_tree(rng, T, step % 2, width=2)
        p = distributions(rng, T, V, 12.0)  # a model that is mostly sure: drafts are accepted
        tokens = np.array([p[max(x, -1) + 1 if x < T else 0].argmax() for x in parents], np.int32)
        u = rng.random(T + 1, dtype=np.float32)
        bufs = [B(x) for x in (p, u, tokens, parents)]
        path, res = B(np.zeros(T, np.int32)), B(np.zeros(2, np.int32))
        work = []
        for ly in layers:
            q, kt, vt = normal(rng, T, H, D), normal(rng, T, G, D, bf16=bf16), normal(rng, T, G, D, bf16=bf16)
            work.append((Attend(dev, q, ly["cache"], n, Cache(dev, kt, vt, bf16), parents, scale), q, kt, vt))
        # the whole step without a wait between its calls
        for at, *_ in work:
            dev.check(L.ds_hip_tree_attention(at.out.ptr, at.w, at.lse.ptr, at.scores.ptr, at.ss, at.q.ptr, at.w, H, at.cache.ref,
                                              n, at.tree.ref, at.parents.ptr, T, scale, 0, 0), "attention")
        dev.check(L.ds_hip_tree_verify(path.ptr, res.ptr, bufs[0].ptr, V, None, 0, V, bufs[2].ptr, bufs[3].ptr, T, bufs[1].ptr),
                  "verify")
        for ly, (at, *_) in zip(layers, work):
            dev.check(L.ds_hip_tree_commit(ly["cache"].ref, n, at.tree.ref, T, path.ptr, res.ptr, at.scores.ptr, at.ss, at.lse.ptr,
                                           H, ly["acc"].ptr, ly["acc"].ptr, rows, ly["pos"].ptr, rows, where), "commit")
        dev.check(L.ds_hip_sync(), "sync")
        want = R.verify(p, None, u, tokens, parents, V)
        good, _ = want
        assert (list(path.to_array(np.int32)[:len(good)]), int(res.to_array(np.int32)[1])) == want
        assert res.to_array(np.int32)[0] == len(good)
        m = n + len(good)
        accepted += len(good)
        for ly, (at, q, kt, vt) in zip(layers, work):
            out, lse, sc = at.fetch()
            wo, wl, ws, to, tl, ts = R.attention(q, ly["k"][:n], ly["v"][:n], kt, vt, n, parents, scale)
            within(out, wo, to, f"out, step {step}")
            for i, x in enumerate(good):
                ly["k"][n + i], ly["v"][n + i] = kt[x], vt[x]
                ly["p"][:, n + i] = where + i
                for g in range(G):
                    ly["a"][g, n + i] = ly["tol"][g, n + i] = 0
            cols = list(range(n)) + [n + x for x in good]
            for g in range(G):
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    for x in good:
                        w = np.exp(ws[h, x, cols] - wl[h, x])
                        ly["a"][g, :m] += w
                        ly["tol"][g, :m] += w * (ts[h, x, cols] + tl[h, x] + 8 * U) + 4 * U * ly["a"][g, :m]
            got = ly["acc"].to_array(np.float32).reshape(G, rows)
            within(got[:, :m], ly["a"][:, :m], ly["tol"][:, :m] + 1e-37, f"acc, step {step}")
            same(ly["pos"].to_array(np.int32).reshape(G, rows)[:, :m], ly["p"][:, :m])
            if m > budget:
                evicted += m - budget
                dev.check(L.ds_hip_kv_evict(ly["cache"].ref, m, budget, ly["acc"].ptr, rows, ly["acc"].ptr, rows, ly["pos"].ptr, rows,
                                            ly["pos"].ptr, rows, sink, where + len(good) - recent, None), "evict")
                slots = R.evict_slots(got[:, :m], ly["p"][:, :m], budget, sink, where + len(good) - recent)
                for g in range(G):
                    ly["k"][:budget, g], ly["v"][:budget, g] = ly["k"][slots[g], g], ly["v"][slots[g], g]
                    for name in ("a", "p", "tol"):
                        ly[name][g, :budget] = ly[name][g, slots[g]]
                same(ly["pos"].to_array(np.int32).reshape(G, rows)[:, :budget], ly["p"][:, :budget])
            keep = min(m, budget)
            for raw, vals in zip(ly["cache"].fetch(), (ly["k"], ly["v"])):
                bits = R.bf16_bits(vals) if bf16 else vals.astype(np.float32).view(np.uint32)
                same(ly["cache"].view(raw)[:keep], bits[:keep])
        where += len(good)
        n = min(m, budget)
    assert accepted > 10 and evicted > 0
