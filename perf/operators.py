"""The operators of a decode step with drafted tokens (speculative decoding), and their plain forms.

A step drafts a few tokens as a tree (parents[i] < i, -1 for a child of the last committed token, anything else a
padding node), runs them through the model over the KV cache, verifies them, appends the accepted ones to the cache
and, when the cache is over its budget, evicts the rows with the least accumulated attention weight.

Kinds:
  attend   ds_hip_tree_attention: the nodes' attention over the cache and over their own ancestors
  verify   ds_hip_tree_verify, ds_hip_tree_verify_greedy: the accepted path and the token after it
  commit   ds_hip_tree_commit: accepted rows into the cache, their attention weights onto the accumulated ones
  evict    ds_hip_kv_evict: the n_keep rows of each head that stay, in place

The heads are the decoder's 10 x 128 over an f32 cache of up to 7680 rows, and generic ones: shared key heads, a
bf16 cache, longer caches. The vocabulary is the decoder's 129280.
"""
import ctypes as C
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DEV = "cuda"
_HEADS = {"heads": 10, "kv_heads": 10, "dim": 128, "bf16": False, "layout": "rows"}
_SHARED = {"heads": 16, "kv_heads": 4, "dim": 128, "bf16": True, "layout": "heads"}


def listed():
    return [
        # the smallest step: a short lookup draft after a thumbnail's prompt
        {"name": "attend_5_77", "kind": "attend", "nodes": 5, "chain": True, "pad": 0, "rows": 77, "prefill": 0,
         "window": 0, "scores": False, **_HEADS},
        # a tree of drafts early in the answer to one page, its scores kept for the eviction
        {"name": "attend_16_701", "kind": "attend", "nodes": 16, "chain": False, "pad": 0, "rows": 701, "prefill": 0,
         "window": 0, "scores": True, **_HEADS},
        # a wide tree late in a long document
        {"name": "attend_64_7001", "kind": "attend", "nodes": 64, "chain": False, "pad": 0, "rows": 7001,
         "prefill": 0, "window": 0, "scores": False, **_HEADS},
        # one token over a cache with a reference part and a sliding window
        {"name": "attend_1_window", "kind": "attend", "nodes": 1, "chain": True, "pad": 0, "rows": 6500,
         "prefill": 1701, "window": 1024, "scores": False, **_HEADS},
        # shared key heads over a long bf16 cache, a padded tree
        {"name": "attend_24_120011_bf16", "kind": "attend", "nodes": 24, "chain": False, "pad": 3, "rows": 120011,
         "prefill": 0, "window": 0, "scores": False, **_SHARED},
        # lookup drafts (no draft distribution): one chain
        {"name": "verify_chain_5", "kind": "verify", "mode": "point", "nodes": 5, "chain": True, "pad": 0,
         "vocab": 129280},
        # a wide tree of lookup drafts
        {"name": "verify_tree_64", "kind": "verify", "mode": "point", "nodes": 64, "chain": False, "pad": 2,
         "vocab": 129280},
        # drafts drawn from a draft model's probabilities, several children a context
        {"name": "verify_drawn_24", "kind": "verify", "mode": "drawn", "nodes": 24, "chain": False, "pad": 0,
         "vocab": 129280},
        # the accepted part of a tree, early and late
        {"name": "commit_16_701", "kind": "commit", "nodes": 16, "accepted": 4, "rows": 701, **_HEADS},
        {"name": "commit_64_7001", "kind": "commit", "nodes": 64, "accepted": 9, "rows": 7001, **_HEADS},
        # a few rows over the budget, and a long cache cut down
        {"name": "evict_1101_1024", "kind": "evict", "rows": 1101, "keep": 1024, "sink": 4, "recent": 256, **_HEADS},
        {"name": "evict_7001_4096", "kind": "evict", "rows": 7001, "keep": 4096, "sink": 4, "recent": 512, **_HEADS},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng):
    if rng.random() < 0.4:
        return dict(_HEADS)
    kv = rng.choice([1, 2, 4, 8])
    return {"heads": kv * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv, "dim": rng.choice([64, 128, 192, 256]),
            "bf16": rng.random() < 0.5, "layout": rng.choice(["rows", "heads"])}


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "verify", "verify", "commit", "evict"])
    nodes = _log(rng, 1, 128)
    if kind == "verify":
        nodes = min(nodes, 64)
        return {"kind": kind, "mode": rng.choice(["point", "drawn", "greedy"]), "nodes": nodes,
                "chain": rng.random() < 0.4, "pad": rng.randrange(0, nodes // 4 + 1), "vocab": _log(rng, 50, 129280)}
    heads = _draw_heads(rng)
    row = 2 * heads["kv_heads"] * heads["dim"] * (2 if heads["bf16"] else 4)  # bytes of K and V
    if kind == "attend":
        rows = _log(rng, 1, max(2, min(120000, 240000000 // row)))
        rows = min(rows, 22000000000 // (4 * nodes * heads["heads"] * heads["dim"]) + 1)
        windowed = rng.random() < 0.25
        return {"kind": kind, "nodes": nodes, "chain": rng.random() < 0.3, "pad": rng.randrange(0, nodes // 4 + 1),
                "rows": rows, "prefill": rows // 3 if windowed else 0, "window": _log(rng, 1, 2000) if windowed else 0,
                "scores": rng.random() < 0.3, **heads}
    rows = _log(rng, 1, max(2, min(40000, 71000000 // row)))
    if kind == "commit":
        rows = min(rows, 4500000 // (nodes * heads["heads"]) + 1)
        return {"kind": kind, "nodes": nodes, "accepted": rng.randrange(0, min(nodes, 12) + 1), "rows": rows, **heads}
    return {"kind": kind, "rows": rows, "keep": rng.randrange(rows // 3, rows + 1), "sink": rng.randrange(0, 5),
            "recent": rng.randrange(0, rows // 4 + 1), **heads}


# ------------------------------------------------------------------ what a program has in hand

class _State:
    pass


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=_DEV)


def _parents(c, seed):
    """A chain, or a tree whose nodes have up to four children, the last `pad` nodes padding."""
    n = c["nodes"]
    if c["chain"]:
        p = list(range(-1, n - 1))
    else:
        r, p, room = random.Random(seed), [], [-1] * 4
        for i in range(n):
            p.append(room.pop(r.randrange(len(room)) if r.random() < 0.5 else 0))
            room += [i] * r.choice([1, 2, 4])
    return p[:n - c["pad"]] + [-2] * c["pad"] if c["pad"] else p


def _cache(g, c, rows):
    """K and V as [rows][kv_heads][dim], stored row by row or head by head."""
    hk, d = c["kv_heads"], c["dim"]
    shape = (rows, hk, d) if c["layout"] == "rows" else (hk, rows, d)
    kv = [_normal(g, *shape).to(torch.bfloat16 if c["bf16"] else torch.float32) for _ in range(2)]
    return [t if c["layout"] == "rows" else t.transpose(0, 1) for t in kv]


def _inputs(c, seed):
    """A case's inputs, by name."""
    g, i = _gen(seed), {}
    if c["kind"] == "verify":
        n, V = c["nodes"], c["vocab"]
        par = _parents(c, seed)
        logits = 4 * _normal(g, n + 1, V)
        top = logits.argmax(-1, keepdim=True)
        logits.scatter_add_(1, top, torch.full_like(logits[:, :1], 3.0))  # a model that is mostly sure
        i["parents"] = torch.tensor(par, dtype=torch.int32, device=_DEV)
        i["u"] = torch.rand(n + 1, generator=g, device=_DEV)
        row = torch.tensor([max(q, -1) + 1 for q in par], device=_DEV)
        nth = torch.tensor([par[:k].count(q) for k, q in enumerate(par)], device=_DEV)  # a node's place among its siblings
        guess = logits + 0.5 * _normal(g, n + 1, V)
        if c["mode"] == "drawn":
            i["q"] = torch.softmax(guess, -1)
            i["tokens"] = torch.multinomial(i["q"], n, replacement=True, generator=g)[row, nth].int()
        else:
            i["tokens"] = guess.topk(min(n, V), -1).indices[row, nth % V].int()
        if c["mode"] == "greedy":
            i["target"] = logits.argmax(-1).int()
        else:
            i["p"] = torch.softmax(logits, -1)
        return i
    H, hk, d, n = c["heads"], c["kv_heads"], c["dim"], c["rows"]
    if c["kind"] == "evict":
        i["k"], i["v"] = _cache(g, c, n)
        acc = torch.exp(2 * _normal(g, hk, n))
        i["acc"] = torch.where(torch.rand(hk, n, generator=g, device=_DEV) < 0.05, torch.zeros_like(acc), acc)
        # a head's rows stand in an order of their own once it has evicted
        i["pos"] = torch.rand(hk, n, generator=g, device=_DEV).argsort(-1).int()
        return i
    T = c["nodes"]
    i["k"], i["v"] = _cache(g, c, n + T)  # the rows behind n are free
    i["kt"], i["vt"] = _cache(g, {**c, "layout": "rows"}, T)
    if c["kind"] == "attend":
        i["q"] = 1.5 * _normal(g, T, H, d)
        i["parents"] = torch.tensor(_parents(c, seed), dtype=torch.int32, device=_DEV)
        return i
    i["scores"] = 1.5 * _normal(g, H, T, n + T)
    i["lse"] = torch.logsumexp(i["scores"], -1)
    path = sorted(random.Random(seed).sample(range(T), c["accepted"]))
    i["path"] = torch.tensor(path + [-1] * (T - len(path)), dtype=torch.int32, device=_DEV)
    i["result"] = torch.tensor([len(path), 0], dtype=torch.int32, device=_DEV)
    i["acc"] = torch.exp(_normal(g, hk, n + T))
    return i


def prepare(case, seed):
    s = _State()
    s.c, s.views = case, None
    s.i = _inputs(case, seed)
    new = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device=_DEV)  # noqa: E731
    c, o = case, {}
    if c["kind"] == "attend":
        T, H = c["nodes"], c["heads"]
        o["out"], o["lse"] = new(T, H, c["dim"]), new(H, T)
        if c["scores"]:
            o["scores"] = new(H, T, c["rows"] + T)
    elif c["kind"] == "verify":
        o["path"], o["result"] = new(c["nodes"], dtype=torch.int32), new(2, dtype=torch.int32)
    elif c["kind"] == "commit":
        o["acc"] = new(c["kv_heads"], c["rows"] + c["nodes"])
        o["pos"] = new(c["kv_heads"], c["rows"] + c["nodes"], dtype=torch.int32)
    else:
        o["acc"] = new(c["kv_heads"], c["keep"])
        o["pos"], o["slots"] = (new(c["kv_heads"], c["keep"], dtype=torch.int32) for _ in range(2))
    s.o = o
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the framework's calls

def _product():
    name = "ds_ocr_amd"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(os.getcwd(), "ds-ocr_amd", "__init__.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _views(s):
    """The host structs that describe a program's caches, kept beside them."""
    if s.views is None:
        P = _product()
        s.views = []
        for k, v in (("k", "v"), ("kt", "vt")):
            if k in s.i:
                t = s.i[k]
                s.views.append(P.KvCache(t.data_ptr(), s.i[v].data_ptr(), t.stride(0), t.stride(1), t.shape[0],
                                         t.shape[1], t.shape[2], P.KV_BF16 if s.c["bf16"] else P.KV_F32))
    return [C.byref(x) for x in s.views]


def _call(s):
    P = _product()
    L, c, i, o = P.load(), s.c, s.i, s.o
    if c["kind"] == "attend":
        cache, tree = _views(s)
        T, H, D = c["nodes"], c["heads"], c["dim"]
        scores = o["scores"].data_ptr() if c["scores"] else None
        P.check(L.ds_hip_tree_attention(o["out"].data_ptr(), H * D, o["lse"].data_ptr(), scores, c["rows"] + T,
                                        i["q"].data_ptr(), H * D, H, cache, c["rows"], tree, i["parents"].data_ptr(),
                                        T, 1 / math.sqrt(D), c["prefill"], c["window"]), "tree attention")
        return o
    if c["kind"] == "verify":
        n, V = c["nodes"], c["vocab"]
        if c["mode"] == "greedy":
            P.check(L.ds_hip_tree_verify_greedy(o["path"].data_ptr(), o["result"].data_ptr(), i["target"].data_ptr(),
                                                i["tokens"].data_ptr(), i["parents"].data_ptr(), n), "verify")
        else:
            q = i["q"].data_ptr() if c["mode"] == "drawn" else None
            P.check(L.ds_hip_tree_verify(o["path"].data_ptr(), o["result"].data_ptr(), i["p"].data_ptr(), V, q, V, V,
                                         i["tokens"].data_ptr(), i["parents"].data_ptr(), n, i["u"].data_ptr()),
                    "verify")
        return o
    if c["kind"] == "commit":
        cache, tree = _views(s)
        n, T = c["rows"], c["nodes"]
        P.check(L.ds_hip_tree_commit(cache, n, tree, T, i["path"].data_ptr(), i["result"].data_ptr(),
                                     i["scores"].data_ptr(), n + T, i["lse"].data_ptr(), c["heads"],
                                     i["acc"].data_ptr(), o["acc"].data_ptr(), n + T, o["pos"].data_ptr(), n + T, n),
                "commit")
        return _committed(s)
    cache, = _views(s)
    n, m = c["rows"], c["keep"]
    P.check(L.ds_hip_kv_evict(cache, n, m, i["acc"].data_ptr(), n, o["acc"].data_ptr(), m, i["pos"].data_ptr(), n,
                              o["pos"].data_ptr(), m, c["sink"], n - c["recent"], o["slots"].data_ptr()), "evict")
    return {**o, "k": i["k"][:m], "v": i["v"][:m]}


def _committed(s):
    """The arrays up to the accepted rows' end; what stands behind it is not the call's."""
    m, n = s.c["rows"] + s.c["accepted"], s.c["rows"]
    return {"acc": s.o["acc"][:, :m], "pos": s.o["pos"][:, n:m], "k": s.i["k"][:m], "v": s.i["v"][:m]}


# ------------------------------------------------------------------ the plain forms

def _ancestors(parents):
    """[n, n]: whether j is i or one of its ancestors; False throughout for a padding node. And the nodes' depths."""
    n = parents.numel()
    at = torch.arange(n, device=parents.device)
    inside = (parents >= 0) & (parents < at)
    up = torch.zeros(n, n, dtype=torch.float64, device=parents.device)
    up[at, parents.clamp(0, n - 1).long()] = inside.double()
    reach = torch.matrix_power(up + torch.eye(n, dtype=up.dtype, device=up.device), n) > 0
    root = parents == -1
    fine = (reach & root).any(-1)  # a chain of parents that ends at a root
    return reach & fine[:, None], reach.sum(-1) - 1, fine


def _visible(c, parents):
    """[nodes, rows + nodes]: what each node sees."""
    n, T = c["rows"], c["nodes"]
    anc, depth, fine = _ancestors(parents)
    j = torch.arange(n, device=parents.device)
    at = torch.cat([j.expand(T, n), (n + depth).expand(T, T)], 1)  # positions
    see = torch.cat([fine[:, None].expand(T, n), anc], 1)
    if c["window"]:
        here = (n + depth)[:, None]
        see = see & ((at < c["prefill"]) | (at > here - c["window"]) | (here < c["prefill"]))
    return see


def _attend(s):
    c, i = s.c, s.i
    T, H, hk, d, n = c["nodes"], c["heads"], c["kv_heads"], c["dim"], c["rows"]
    K, V = (torch.cat([i[a][:n], i[b]]).float().permute(1, 0, 2) for a, b in (("k", "kt"), ("v", "vt")))
    q = i["q"].view(T, hk, H // hk, d).permute(1, 2, 0, 3).reshape(hk, H // hk * T, d)
    x = torch.matmul(q * (1 / math.sqrt(d)), K.transpose(1, 2)).view(H, T, n + T)
    x = x.masked_fill(~_visible(c, i["parents"]), -math.inf)
    m = x.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(hk, H // hk * T, n + T), V).view(H, T, d)
    r = {"out": torch.where(z > 0, o / z, 0.0).transpose(0, 1).contiguous(), "lse": (m + torch.log(z))[..., 0]}
    if c["scores"]:
        r["scores"] = x
    return r


def _verify(s):
    c, i = s.c, s.i
    n, V, mode = c["nodes"], c["vocab"], c["mode"]
    par, tok, dev = i["parents"], i["tokens"].long(), i["parents"].device
    at = torch.arange(n, device=dev)
    anc, _, fine = _ancestors(par)
    row = par.long().clamp_min(-1) + 1
    older = (row[:, None] == row) & (at[:, None] > at) & fine  # [i, j]: j is an elder sibling of i
    known = fine & (tok >= 0) & (tok < V)
    tok = tok.clamp(0, V - 1)
    if mode == "greedy":
        ok = known & (i["target"][row] == tok)
    else:
        r = torch.where(known, i["p"][row, tok].double(), 0.0)
        u = i["u"].double()
        if mode == "point":
            r = torch.where((older & (tok[:, None] == tok)).any(-1), 0.0, r)
            ok = (r > 0) & (u[:n] * (1 - (older * r).sum(-1)) < r)
        else:
            # by the place among the siblings: the normalisers follow one from the other
            p, q = i["p"].double(), i["q"].double()
            place, a = older.sum(-1), q[row, tok]
            ok = torch.zeros_like(known)
            taken, z = torch.zeros(n + 1, 1, dtype=torch.float64, device=dev), torch.ones(n + 1, 1, dtype=torch.float64, device=dev)
            children = torch.bincount(torch.where(fine, row, n + 1), minlength=n + 2)[:n + 1, None]
            for k in range(4 if not c["chain"] else 1):  # a context has up to four children
                left = (r - taken[row, 0] * a).clamp_min(0)
                ok = torch.where(place == k, known & (left > 0) & (u[:n] * a * z[row, 0] < left), ok)
                more = children > k
                taken = torch.where(more, taken + z, taken)
                z = torch.where(more, (p - taken * q).clamp_min(0).sum(-1, keepdim=True), z)
    first = ok & ~(older & ok).any(-1)
    on = ((anc & first).sum(-1) == anc.sum(-1)) & fine
    count = on.sum()
    path = torch.where(on, at, n).sort().values
    last = torch.where(on, at, -1).amax() + 1  # the context that the path ends in
    if mode == "greedy":
        token = i["target"][last]
    else:
        w = i["p"].index_select(0, last[None])[0].double()
        if mode == "point":
            gone = torch.zeros(V + 1, dtype=torch.bool, device=dev)
            gone[torch.where(known & (row == last), tok, V)] = True
            left = torch.where(gone[:V], 0.0, w)
        else:
            left = (w - taken[last] * i["q"].index_select(0, last[None])[0].double()).clamp_min(0)
        w = torch.where(left.sum() > 0, left, w)
        cum = w.cumsum(0)
        token = ((cum > u[n] * cum[-1]) & (w > 0)).to(torch.int8).argmax()
    return {"path": torch.where(path < n, path, -1).int(), "result": torch.stack([count, token.long()]).int()}


def _commit(s):
    c, i, o = s.c, s.i, s.o
    n, T, H, hk = c["rows"], c["nodes"], c["heads"], c["kv_heads"]
    A = c["accepted"]
    path = i["path"][:A].long()
    w = torch.exp(i["scores"][:, path] - i["lse"][:, path, None]).view(hk, H // hk * A, n + T).sum(1)
    o["acc"][:, :n] = i["acc"][:, :n] + w[:, :n]
    o["acc"][:, n:n + A] = w[:, n + path]
    o["pos"][:, n:n + A] = torch.arange(n, n + A, device=path.device)
    i["k"][n:n + A], i["v"][n:n + A] = i["kt"][path], i["vt"][path]
    return _committed(s)


def _evict(s):
    c, i = s.c, s.i
    n, m, hk = c["rows"], c["keep"], c["kv_heads"]
    dev = i["acc"].device
    guarded = (i["pos"] < c["sink"]) | (i["pos"] >= n - c["recent"])
    order = i["acc"].nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).sort(dim=-1, stable=True).indices
    order = order.gather(1, guarded.gather(1, order).to(torch.int8).sort(dim=-1, stable=True).indices)
    keep = torch.ones(hk, n, dtype=torch.bool, device=dev).scatter_(1, order[:, :n - m], False)
    at = torch.arange(n, device=dev)
    movers = torch.where(keep & (at >= m), at, n).sort(-1).values
    nth = (~keep[:, :m]).cumsum(-1) - 1
    slots = torch.where(keep[:, :m], at[:m], movers.gather(1, nth.clamp_min(0)))
    h, to = torch.nonzero(~keep[:, :m], as_tuple=True)
    for t in (i["k"], i["v"]):
        t[to, h] = t[slots[h, to], h]
    return {"acc": i["acc"].gather(1, slots), "pos": i["pos"].gather(1, slots), "slots": slots.int(), "k": i["k"][:m],
            "v": i["v"][:m]}


def run(state):
    if own:
        return _call(state)
    return {"attend": _attend, "verify": _verify, "commit": _commit, "evict": _evict}[state.c["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "verify":
        rows = {"point": 1, "drawn": 2, "greedy": 0}[c["mode"]]  # the last context's distributions
        return {"bytes": 4.0 * rows * c["vocab"] + 20.0 * c["nodes"] + 12, "flops": 2.0 * rows * c["vocab"]}
    H, hk, d, n = c["heads"], c["kv_heads"], c["dim"], c["rows"]
    row = 2.0 * hk * d * (2 if c["bf16"] else 4)
    if c["kind"] == "attend":
        T = c["nodes"]
        seen = min(n, min(c["prefill"], n) + max(0, c["window"] - 1)) if c["window"] else n
        b = (seen + T) * row + 8.0 * T * H * d + 4.0 * H * T + (4.0 * H * T * (n + T) if c["scores"] else 0)
        return {"bytes": b, "flops": 4.0 * T * H * d * (seen + (T + 1) / 2)}
    if c["kind"] == "commit":
        A = c["accepted"]
        return {"bytes": 2 * A * row + 4.0 * A * H * (n + A) + 8.0 * hk * (n + A) + 16, "flops": 2.0 * A * H * (n + A)}
    moved = (n - c["keep"]) * c["keep"] / max(n, 1)
    return {"bytes": 8.0 * hk * n + 12.0 * hk * c["keep"] + 2 * moved * row, "flops": 1.0 * hk * n}


# ------------------------------------------------------------------ the same in 64 bits

def _walk64(par):
    """Every node's chain from its root down to itself, [] for padding."""
    chains = []
    for k, q in enumerate(par):
        up = [] if q == -1 else chains[q] if 0 <= q < k else None
        chains.append(up + [k] if up or q == -1 else [])
    return chains


def _attend64(c, i):
    n, T, g = c["rows"], c["nodes"], c["heads"] // c["kv_heads"]
    par = i["parents"].tolist()
    chains = _walk64(par)
    out = torch.zeros(T, c["heads"], c["dim"], dtype=torch.float64, device=_DEV)
    lse = torch.full((c["heads"], T), -math.inf, dtype=torch.float64, device=_DEV)
    scores = torch.full((c["heads"], T, n + T), -math.inf, dtype=torch.float64, device=_DEV) if c["scores"] else None
    K, V = ([i[a][:, h].double() for h in range(c["kv_heads"])] for a in ("k", "v"))
    Kt, Vt = (i[a].double() for a in ("kt", "vt"))
    for t in range(T):
        if not chains[t]:
            continue
        pos = n + len(chains[t]) - 1
        inside = lambda p: not c["window"] or pos < c["prefill"] or p < c["prefill"] or p > pos - c["window"]  # noqa: E731
        far = torch.arange(n, device=_DEV)
        if c["window"] and pos >= c["prefill"]:
            far = far[(far < c["prefill"]) | (far > pos - c["window"])]
        near = torch.tensor([a for k, a in enumerate(chains[t]) if inside(n + k)], dtype=torch.long, device=_DEV)
        every = far.numel() == n
        for h in range(c["heads"]):
            k, v = ((x[h // g][:n] if every else x[h // g][far]) for x in (K, V))
            qv = i["q"][t, h].double()
            x = torch.cat([k @ qv, Kt[near, h // g] @ qv]) / math.sqrt(c["dim"])
            if not x.numel():
                continue
            lse[h, t] = torch.logsumexp(x, 0)
            w = torch.exp(x - lse[h, t])
            out[t, h] = w[:far.numel()] @ v + w[far.numel():] @ Vt[near, h // g]
            if c["scores"]:
                scores[h, t, torch.cat([far, n + near])] = x
    return {"out": out, "lse": lse, **({"scores": scores} if c["scores"] else {})}


def _verify64(c, i):
    par, tok = i["parents"].tolist(), i["tokens"].tolist()
    n, mode = c["nodes"], c["mode"]
    host = lambda name: i[name].cpu().numpy()  # noqa: E731
    path, at = [], -1
    if mode == "greedy":
        target = host("target").tolist()
    else:
        p, u = host("p"), host("u").astype(np.float64)
        q = host("q") if mode == "drawn" else None
    while True:
        gone, spent, taken, z, found = [], 0.0, 0.0, 1.0, None
        pr = p[at + 1].astype(np.float64) if mode != "greedy" else None
        for k in range(n):
            if par[k] != at:
                continue
            t = tok[k]
            if mode == "greedy":
                hit = t == target[at + 1]
            elif mode == "point":
                r = 0.0 if t in gone else pr[t]
                hit = r > 0 and u[k] * (1 - spent) < r
                gone.append(t)
                spent += r
            else:
                qr = q[at + 1].astype(np.float64)
                r = max(pr[t] - taken * qr[t], 0.0)
                hit = r > 0 and u[k] * qr[t] * z < r
                if not hit:
                    taken += z
                    z = float(np.maximum(pr - taken * qr, 0).sum())
            if hit:
                found = k
                break
        if found is None:
            break
        path.append(found)
        at = found
    if mode == "greedy":
        token = target[at + 1]
    else:
        w = pr.copy()
        if mode == "point":
            w[gone] = 0.0
        else:
            w = np.maximum(pr - taken * q[at + 1].astype(np.float64), 0)
        w = w if w.sum() > 0 else pr
        cum = np.cumsum(w)
        token = int(np.nonzero((cum > u[n] * cum[-1]) & (w > 0))[0][0])
    return {"path": np.array(path + [-1] * (n - len(path)), np.int32), "result": np.array([len(path), token], np.int32)}


def _commit64(c, i):
    n, A, g = c["rows"], c["accepted"], c["heads"] // c["kv_heads"]
    path = i["path"][:A].tolist()
    acc = torch.zeros(c["kv_heads"], n + A, dtype=torch.float64, device=_DEV)
    acc[:, :n] = i["acc"][:, :n].double()
    cols = torch.tensor(list(range(n)) + [n + a for a in path], device=_DEV)
    for h in range(c["heads"]):
        for a in path:
            acc[h // g] += torch.exp(i["scores"][h, a, cols].double() - i["lse"][h, a].double())
    k, v = (torch.cat([i[x][:n].double()] + [i[y][a:a + 1].double() for a in path]) for x, y in (("k", "kt"), ("v", "vt")))
    pos = torch.arange(n, n + A, dtype=torch.int32).expand(c["kv_heads"], A).contiguous()
    return {"acc": acc, "pos": pos, "k": k, "v": v}


def _evict64(c, i):
    n, m = c["rows"], c["keep"]
    acc, pos = i["acc"].cpu().numpy(), i["pos"].cpu().numpy()
    slots = np.empty((c["kv_heads"], m), np.int64)
    for h in range(c["kv_heads"]):
        guarded = (pos[h] < c["sink"]) | (pos[h] >= n - c["recent"])
        rank = sorted(range(n), key=lambda j: (guarded[j], acc[h, j], j))
        out = set(rank[:n - m])
        behind = iter(j for j in range(m, n) if j not in out)
        slots[h] = [next(behind) if j in out else j for j in range(m)]
    t = torch.from_numpy(slots).to(_DEV)
    kv = [torch.stack([i[x][t[h], h].double() for h in range(c["kv_heads"])], 1) for x in ("k", "v")]
    return {"acc": i["acc"].double().gather(1, t), "pos": i["pos"].gather(1, t), "slots": slots.astype(np.int32),
            "k": kv[0], "v": kv[1]}


def exact(case, seed):
    i = _inputs(case, seed)
    return {"attend": _attend64, "verify": _verify64, "commit": _commit64, "evict": _evict64}[case["kind"]](case, i)
