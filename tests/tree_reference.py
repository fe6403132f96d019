"""Plain 64-bit forms of the drafted-token operators (ds_hip_tree_*, ds_hip_kv_evict), node by node and row by row, and
the buffers that their tests hand to the library."""
import ctypes as C

import numpy as np

U = 2.0 ** -24  # half a step of f32


def bf16_bits(a):
    """f32 -> bf16 bits, to nearest even (finite values)."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_values(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def chains(parents):
    """Each node's ancestors from the root down, itself last; [] for a padding node."""
    out = []
    for i, p in enumerate(parents):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p]:
            out.append(out[p] + [i])
        else:
            out.append([])
    return out


def random_tree(rng, n, pad=0, width=3):
    p = []
    for i in range(n):
        p.append(int(rng.integers(max(-1, i - width - 1), i)) if i else -1)
    for i in rng.choice(n, pad, replace=False) if pad else []:
        p[i] = int(rng.choice([-2, -100, i, i + 1, 2 ** 31 - 1, -2 ** 31]))
    return np.array(p, np.int32)


def attention(q, k, v, kt, vt, n, parents, scale, prefill=0, window=0):
    """q [T][H][D], k/v [rows][G][D], kt/vt [T][G][D], all f64. out, lse, scores, and per output a bound on a 32-bit kernel's
    error: a score is a sum of D products (D + 2 roundings of at most U of the sum of the products' sizes, whatever the
    order), a weight the exponential of a difference of scores (4 roundings relative to the scores' size, and 4 of its own),
    the output a sum of up to n weighted rows in chains of at most 1024 additions, over a sum of the same kind."""
    T, H, D = q.shape
    G = kt.shape[1]
    out, lse = np.zeros((T, H, D)), np.full((H, T), -np.inf)
    scores, out_tol, sc_tol = np.full((H, T, n + T), -np.inf), np.zeros((T, H, D)), np.zeros((H, T, n + T))
    lse_tol = np.zeros((H, T))
    for i, chain in enumerate(chains(parents)):
        if not chain:
            continue
        pos = n + len(chain) - 1
        sees = lambda p: window <= 0 or pos < prefill or p < prefill or p > pos - window  # noqa: E731
        rows = [j for j in range(n) if sees(j)] if window > 0 else list(range(n))
        own = [a for d, a in enumerate(chain) if sees(n + d)]
        cols = np.array(rows + [n + a for a in own])
        for h in range(H):
            g = h // (H // G)
            K, V = np.concatenate([k[rows, g], kt[own, g]]), np.concatenate([v[rows, g], vt[own, g]])
            s = scale * (K @ q[i, h])
            es = (D + 2) * U * abs(scale) * (np.abs(K) @ np.abs(q[i, h]))
            m = s.max()
            e = np.exp(s - m)
            w = e / e.sum()
            scores[h, i, cols], sc_tol[h, i, cols] = s, es + 4 * U * np.abs(s)
            lse[h, i] = m + np.log(e.sum())
            each = es.max() + 8 * U * (np.abs(s).max() + 1)
            chain_u = min(len(cols), 1024) * U
            lse_tol[h, i] = each + chain_u + 4 * U * (abs(lse[h, i]) + 1)
            out[i, h] = w @ V
            out_tol[i, h] = (2 * each + 2 * chain_u + 8 * U) * (w @ np.abs(V)) + 1e-37
    return out, lse, scores, out_tol, lse_tol, sc_tol


def probability(x):
    x = x.astype(np.float64)
    return np.where((x > 0) & np.isfinite(x), x, 0.0)


def verify(p, q, u, tokens, parents, vocab):
    """(path, token): p [n + 1][vocab], q the same or None."""
    path, at, live = [], -1, chains(parents)
    while True:
        pr = probability(p[at + 1])
        qr = None if q is None else probability(q[at + 1])
        gone, spent, c, z, hit = set(), 0.0, 0.0, 1.0, None
        for k, t in enumerate(tokens):
            if not live[k] or parents[k] != at:
                continue
            inside = 0 <= t < vocab
            if q is None:
                r = pr[t] if inside and t not in gone else 0.0
                ok = r > 0 and float(u[k]) * (1 - spent) < r
                gone.add(int(t))
                spent += r
            else:
                r = max(pr[t] - c * qr[t], 0.0) if inside else 0.0
                ok = r > 0 and float(u[k]) * qr[t] * z < r
                if not ok:
                    c += z
                    z = float(np.maximum(pr - c * qr, 0).sum())
            if ok:
                hit = k
                break
        if hit is None:
            break
        path.append(hit)
        at = hit
    w = pr.copy()
    if q is None:
        w[[t for t in gone if 0 <= t < vocab]] = 0
    else:
        w = np.maximum(pr - c * qr, 0)
    if not w.sum() > 0:
        w = pr
    if not w.sum() > 0:
        return path, -1
    cum = np.cumsum(w)
    return path, int(np.nonzero((cum > float(u[len(tokens)]) * cum[-1]) & (w > 0))[0][0])


def verify_greedy(target, tokens, parents):
    path, at, live = [], -1, chains(parents)
    while True:
        hit = [k for k, t in enumerate(tokens) if live[k] and parents[k] == at and t == target[at + 1]]
        if not hit:
            return path, int(target[at + 1])
        at = hit[0]
        path.append(at)


def evict_slots(acc, pos, keep, sink, recent_from):
    """Per head, the old row of each of the first `keep` rows."""
    heads, n = acc.shape
    slots = np.empty((heads, keep), np.int64)
    for h in range(heads):
        guarded = (pos[h] < sink) | (pos[h] >= recent_from)
        val = np.where(np.isnan(acc[h]), -np.inf, acc[h])
        gone = set(sorted(range(n), key=lambda j: (guarded[j], val[j], j))[:n - keep])
        behind = iter([j for j in range(keep, n) if j not in gone])
        slots[h] = [next(behind) if j in gone else j for j in range(keep)]
    return slots


class Cache:
    """K and V [rows][heads][dim] (f64 values of the stored type) in device memory, row by row or head by head, with a gap
    behind every row and head."""

    def __init__(self, dev, k, v, bf16=False, by_head=False, gap=0):
        rows, G, D = k.shape
        unit = 8 if bf16 else 4
        gap *= unit
        self.dev, self.bf16, self.by_head, self.shape = dev, bf16, by_head, (rows, G, D)
        if by_head:
            self.rs, self.hs = D + gap, rows * (D + gap) + gap
            total = G * self.hs
        else:
            self.hs, self.rs = D + gap, G * (D + gap) + gap
            total = rows * self.rs
        self.total = max(total, 1)
        self.bufs, self.raw = [], []
        for a in (k, v):
            raw = np.full(self.total, 0x7FC1 if bf16 else np.nan, np.uint16 if bf16 else np.float32)
            self.view(raw)[...] = bf16_bits(a) if bf16 else a
            self.raw.append(raw)
            self.bufs.append(dev.DeviceBuffer.from_array(raw))
        self.st = dev.KvCache(self.bufs[0].ptr, self.bufs[1].ptr, self.rs, self.hs, rows, G, D,
                              dev.KV_BF16 if bf16 else dev.KV_F32)

    def view(self, raw):
        rows, G, D = self.shape
        s = raw.itemsize
        return np.lib.stride_tricks.as_strided(raw, self.shape, (self.rs * s, self.hs * s, s))

    @property
    def ref(self):
        return C.byref(self.st)

    def fetch(self):
        """The raw arrays (bits) of K and V, gaps included."""
        t = np.uint16 if self.bf16 else np.uint32
        return [b.to_array(t, self.total) for b in self.bufs]

    def expect(self):
        """The uploaded bits, for a test to change and compare."""
        t = np.uint16 if self.bf16 else np.uint32
        return [r.view(t).copy() for r in self.raw]


def normal(rng, *shape, bf16=False, std=1.0):
    """f64 values that f32 (or bf16) holds exactly."""
    a = (std * rng.standard_normal(shape)).astype(np.float32)
    return (bf16_values(bf16_bits(a)) if bf16 else a).astype(np.float64)
