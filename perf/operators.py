"""The operators over a Q8_0 KV cache that long contexts and speculative
decoding need, as calls to time: ``op`` names one.

* ``tree``    attention of a tree of drafted tokens over the cache
  (``KvQ8Cache.attend_tree``): node i sees the committed rows, its ancestors
  and itself;
* ``weigh``   causal attention that adds each row's attention weight to a
  plane per kv head (``KvQ8Cache.attend_weigh``), one token or a prompt;
* ``evict``   a cache cut down to the rows of largest accumulated weight
  (``KvQ8Cache.evict``), into another cache;
* ``blocks``  attention over the blocks of rows that a score against each
  block's mean key selects (``KvQ8Cache.attend_blocks``), one token or a
  prompt, whose new rows' means are made first (``KvQ8Cache.block_means``).

A cache is one layer's: int8 values [rows][n_kv * hd] and one f16 scale per
32 of them, K and V.  ``run`` computes an operator from elementary torch
operations, or with ``own`` calls the framework.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
_engine = None


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------

def _tree(name, n, pos, n_head, n_kv, hd, gated):
    return {"name": name, "op": "tree", "n": n, "pos": pos, "n_head": n_head, "n_kv": n_kv, "hd": hd, "gated": gated}


def _weigh(name, m, pos, n_head, n_kv, hd, gated):
    return {"name": name, "op": "weigh", "m": m, "pos": pos, "n_head": n_head, "n_kv": n_kv, "hd": hd, "gated": gated}


def _evict(name, seq, keep, n_recent, n_first, n_kv, hd):
    return {"name": name, "op": "evict", "seq": seq, "keep": keep, "n_recent": n_recent, "n_first": n_first,
            "n_kv": n_kv, "hd": hd}


def _blocks(name, m, pos, n_head, n_kv, hd, block, n_sel, n_first, n_local, gated):
    return {"name": name, "op": "blocks", "m": m, "pos": pos, "n_head": n_head, "n_kv": n_kv, "hd": hd,
            "block": block, "n_sel": n_sel, "n_first": n_first, "n_local": n_local, "gated": gated}


def listed():
    return [
        # a handful of drafts at the start of a conversation: latency counts
        _tree("tree 5 at 150", 5, 150, 8, 2, 64, False),
        # a small draft model's tree in a usual conversation
        _tree("tree 26 at 2k", 26, 2047, 16, 4, 128, True),
        # a full tree of candidates over a document
        _tree("tree 64 at 8k", 64, 8190, 16, 4, 128, True),
        # the largest: many candidates over a long document, wide model
        _tree("tree 250 at 30k", 250, 30011, 32, 8, 128, False),
        # a decode step that keeps the weights up to date, usual and long
        _weigh("weigh token at 4k", 1, 4095, 16, 4, 128, True),
        _weigh("weigh token at 60k", 1, 60000, 32, 8, 128, False),
        # a prompt whose weights decide what stays
        _weigh("weigh prompt 1500", 1500, 0, 16, 4, 128, True),
        # a running conversation held to a budget: a few rows go each time
        _evict("evict 64 of 2112", 2112, 2048, 256, 4, 4, 128),
        # a long prompt cut to a quarter
        _evict("evict 65000 to 16000", 65000, 16000, 1000, 16, 8, 128),
        # a decode step over selected blocks, moderate and very long
        _blocks("blocks token at 16k", 1, 16300, 16, 4, 128, 64, 16, 1, 2, True),
        _blocks("blocks token at 120k", 1, 120001, 32, 8, 128, 64, 32, 1, 2, False),
        # a question of 400 tokens asked about a document
        _blocks("blocks prompt 400 at 12k", 400, 12000, 16, 4, 128, 64, 16, 1, 2, True),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hd = rng.choice((64, 128, 128, 256))
    n_kv = rng.choice((1, 2, 4, 8, 16))
    return n_kv * rng.choice([g for g in (1, 2, 4, 8) if n_kv * g <= 32]), n_kv, hd


def draw(rng):
    op = rng.choice(("tree", "tree", "weigh", "weigh prompt", "evict", "blocks", "blocks prompt"))
    gated = rng.random() < 0.5
    while True:
        n_head, n_kv, hd = _heads(rng)
        if op == "tree":
            c = _tree("", _logu(rng, 1, 256), _logu(rng, 1, 60000) - 1, n_head, n_kv, hd, gated)
            fits = c["n"] * n_head * hd * (c["pos"] + c["n"]) <= 3e10 and (c["pos"] + c["n"]) * n_kv * hd <= 1e8
        elif op == "weigh":
            c = _weigh("", 1, _logu(rng, 1, 100000) - 1, n_head, n_kv, hd, gated)
            fits = c["pos"] * n_kv * hd <= 1e8
        elif op == "weigh prompt":
            c = _weigh("", _logu(rng, 2, 2500), rng.choice((0, 0, _logu(rng, 16, 6000))), n_head, n_kv, hd, gated)
            fits = c["m"] * n_head * hd * (c["pos"] + c["m"]) <= 2e10
        elif op == "evict":
            seq = _logu(rng, 40, 100000)
            keep = max(1, int(seq * rng.choice((0.1, 0.25, 0.5, 0.9, 0.98))))
            c = _evict("", seq, keep, rng.randint(0, keep // 4), rng.randint(0, keep // 8), n_kv, hd)
            fits = seq * n_kv * hd <= 1e8
        else:
            m = 1 if op == "blocks" else _logu(rng, 2, 600)
            block, n_first, n_local = rng.choice((32, 64, 128)), rng.randint(0, 2), rng.randint(1, 3)
            n_sel = n_first + n_local + rng.randint(1, 40)
            c = _blocks("", m, _logu(rng, 1, 130000 if m == 1 else 16000) - 1, n_head, n_kv, hd, block, n_sel,
                        n_first, n_local, gated)
            fits = c["pos"] * n_kv * hd <= 1.3e8 and m * n_kv * n_sel * block * hd <= 3e8
        if fits:
            del c["name"]
            return c


def _pairs(pos, m):
    """Rows seen by tokens at pos .. pos + m - 1, summed."""
    return m * pos + m * (m + 1) // 2


def work(case):
    c = case
    row = c["n_kv"] * c["hd"] * 34 / 32     # one plane's bytes of a cache row
    if c["op"] == "evict":
        return {"bytes": 8 * c["n_kv"] * c["seq"] + c["keep"] * (4 * row + 8 * c["n_kv"]), "flops": 0}
    m = c.get("m") or c["n"]
    rows, width = c["pos"] + m, c["n_head"] * c["hd"]
    io = 4 * m * width * (3 if c["gated"] else 2)
    if c["op"] == "tree":
        depth = 2 * math.log2(m + 1)        # about what a node sees of its tree
        return {"bytes": 2 * rows * row + io + 4 * m, "flops": 4 * m * width * (c["pos"] + depth)}
    if c["op"] == "weigh":
        # the weights of a prompt are sums over its tokens: the plane is read and written once
        return {"bytes": 2 * rows * row + io + 4 * c["n_kv"] * (c["pos"] + rows + m), "flops": 4 * width * _pairs(c["pos"], m)}
    seen = min(c["n_sel"] * c["block"], rows)
    means = rows // c["block"]
    return {"bytes": min(2 * rows, 2 * m * seen) * row + means * row + io + 4 * m * c["n_kv"] * c["n_sel"]
            + (m * row if m > 1 else 0),
            "flops": 4 * width * m * seen + 2 * m * c["n_kv"] * c["hd"] * means}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _quantise(x):
    """Rows of f32 as Q8_0 blocks: int8 codes and one f16 scale per 32."""
    b = x.unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1) / 127.0).half()
    df = d.float()
    inv = torch.where(df > 0, 1.0 / df, torch.zeros_like(df))
    q = (b * inv[..., None]).round().clamp(-127, 127)
    return q.to(torch.int8).flatten(-2).contiguous(), d.contiguous()


def _cache(rows, max_seq, c, g):
    """Keys that share a part over stretches of 48 rows (a topic), a few rows
    that every query attends to, and values; rows past `rows` hold zeros."""
    per = c["n_kv"] * c["hd"]
    topic = _randn((rows // 48 + 1, per), g, 0.7)
    k = _randn((rows, per), g, 0.8) + topic.repeat_interleave(48, 0)[:rows]
    k *= 1 + (torch.rand((rows, 1), generator=g, device=DEV) < 0.02)
    planes = {}
    for n, x in (("k", k), ("v", _randn((rows, per), g))):
        planes[n + "_qs"] = torch.zeros((max_seq, per), dtype=torch.int8, device=DEV)
        planes[n + "_d"] = torch.zeros((max_seq, per // 32), dtype=torch.float16, device=DEV)
        planes[n + "_qs"][:rows], planes[n + "_d"][:rows] = _quantise(x)
    return planes


def _parents(n, seed):
    """Nodes in drafting order: each hangs on an earlier one or on the last
    committed token, mostly on the more recent ones."""
    r = np.random.RandomState(seed % (1 << 31))
    back = np.minimum(r.geometric(0.25, n), np.arange(n) + 1)
    return (np.arange(n) - back).astype(np.int32)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "evict":
        s.update(_cache(c["seq"], c["seq"], c, g))
        s["weight"] = torch.exp(_randn((c["n_kv"], c["seq"]), g, 1.5))
        gaps = torch.randint(1, 4, (c["n_kv"], c["seq"]), generator=g, device=DEV, dtype=torch.int32)
        order = gaps.cumsum(1).int() - 1
        s["n_tokens"] = 3 * c["seq"]
        s["position"] = order + (s["n_tokens"] - 1 - order[:, -1:])
        s["position"][:, 0] = 0
        s["position"] = s["position"].int().contiguous()
        per = c["n_kv"] * c["hd"]
        s["to"] = {n: torch.zeros((c["keep"], per if n.endswith("qs") else per // 32), device=DEV,
                                  dtype=torch.int8 if n.endswith("qs") else torch.float16)
                   for n in ("k_qs", "k_d", "v_qs", "v_d")}
        s["to"]["weight"] = torch.zeros((c["n_kv"], c["keep"]), device=DEV)
        s["to"]["position"] = torch.zeros((c["n_kv"], c["keep"]), device=DEV, dtype=torch.int32)
        return s
    m = c.get("m") or c["n"]
    rows = c["pos"] + m
    s.update(_cache(rows, rows, c, g))
    s["q"] = _randn((m, c["n_head"] * c["hd"]), g, 1.2)
    s["gate"] = _randn((m, c["n_head"] * c["hd"]), g) if c["gated"] else None
    s["out"] = torch.zeros((m, c["n_head"] * c["hd"]), device=DEV)
    if c["op"] == "tree":
        s["parents"] = torch.from_numpy(_parents(c["n"], seed)).to(DEV)
    elif c["op"] == "weigh":
        s["weight"] = torch.exp(_randn((c["n_kv"], rows), g))
        s["position"] = torch.arange(rows, device=DEV, dtype=torch.int32).repeat(c["n_kv"], 1).contiguous()
    else:
        s["mean_qs"], s["mean_d"] = _block_means(s["k_qs"], s["k_d"], c, 0, c["pos"] // c["block"] * c["block"])
        grow = rows // c["block"] + 1 - s["mean_qs"].shape[0]
        s["mean_qs"] = torch.nn.functional.pad(s["mean_qs"], (0, 0, 0, grow))
        s["mean_d"] = torch.nn.functional.pad(s["mean_d"], (0, 0, 0, grow))
        s["sel"] = torch.zeros((m, c["n_kv"], c["n_sel"]), device=DEV, dtype=torch.int32)
    return s


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def _values(qs, d, n_kv):
    """Codes and scales as f32 values [n_kv][rows][hd]."""
    x = (qs.float().unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)
    return x.unflatten(-1, (n_kv, -1)).transpose(0, 1).contiguous()


def _by_kv(x, n_kv, hd):
    """[m][n_head * hd] as [n_kv][m * group][hd]."""
    m = x.shape[0]
    return x.view(m, n_kv, -1, hd).transpose(0, 1).reshape(n_kv, -1, hd).contiguous()


def _back(x, m):
    """[n_kv][m * group][hd] as [m][n_head * hd]."""
    return x.unflatten(1, (m, -1)).transpose(0, 1).reshape(m, -1)


def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _gated(out, gate):
    return out if gate is None else out * (1.0 / (1.0 + torch.exp(-gate)))


def _plain_tree(s):
    c, n = s["case"], s["case"]["n"]
    group = c["n_head"] // c["n_kv"]
    up = torch.eye(n, device=DEV)           # one step towards the root, then two, four, ...
    at = s["parents"].long()
    step = torch.zeros((n, n), device=DEV)
    step[torch.arange(n, device=DEV)[at >= 0], at[at >= 0]] = 1
    for _ in range(max(1, n.bit_length())):
        up = ((up + step @ up) > 0).float()
        step = ((step @ step) > 0).float()
    seen = torch.cat([torch.ones((n, c["pos"]), device=DEV), up], 1) > 0
    K, V = (_values(s[x + "_qs"], s[x + "_d"], c["n_kv"]) for x in "kv")
    w = _by_kv(s["q"], c["n_kv"], c["hd"]) @ K.transpose(1, 2) / math.sqrt(c["hd"])
    w.masked_fill_(~seen.repeat_interleave(group, 0), -math.inf)
    return _gated(_back(_softmax(w) @ V, n), s["gate"])


def _plain_weigh(s):
    c, m, pos = s["case"], s["case"]["m"], s["case"]["pos"]
    group, rows = c["n_head"] // c["n_kv"], pos + m
    K, V = (_values(s[x + "_qs"], s[x + "_d"], c["n_kv"]) for x in "kv")
    w = _by_kv(s["q"], c["n_kv"], c["hd"]) @ K.transpose(1, 2) / math.sqrt(c["hd"])
    late = torch.arange(rows, device=DEV) > torch.arange(pos, rows, device=DEV)[:, None]
    w.masked_fill_(late.repeat_interleave(group, 0), -math.inf)
    p = _softmax(w)
    total = p.sum(1)
    s["weight"][:, :pos] += total[:, :pos]
    s["weight"][:, pos:] = total[:, pos:]
    s["position"][:, pos:] = torch.arange(pos, rows, device=DEV, dtype=torch.int32)
    return {"out": _gated(_back(p @ V, m), s["gate"]), "weight": s["weight"], "position": s["position"]}


def _plain_evict(s):
    c, keep = s["case"], s["case"]["keep"]
    safe = (s["position"] < c["n_first"]) | (s["position"] >= s["n_tokens"] - c["n_recent"])
    rank = torch.where(safe, torch.full_like(s["weight"], math.inf), s["weight"])
    best = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :keep]
    kept = torch.zeros_like(safe).scatter_(1, best, True)
    source = torch.arange(keep, device=DEV).repeat(c["n_kv"], 1)
    source[~kept[:, :keep]] = kept[:, keep:].nonzero()[:, 1] + keep
    got = {}
    for n in ("k_qs", "k_d", "v_qs", "v_d"):
        x = s[n].unflatten(1, (c["n_kv"], -1))
        got[n] = x[source.T, torch.arange(c["n_kv"], device=DEV)].flatten(1)
    for n in ("weight", "position"):
        got[n] = s[n].gather(1, source)
    return got


def _block_means(qs, d, c, row0, row1):
    """Mean keys of the whole blocks of rows row0 .. row1, as Q8_0 blocks."""
    b = c["block"]
    n = (row1 - row0) // b
    x = qs[row0:row0 + n * b].double().unflatten(-1, (-1, 32)) * d[row0:row0 + n * b].double()[..., None]
    return _quantise((x.flatten(-2).unflatten(0, (n, b)).sum(1) / b).float())


def _plain_blocks(s):
    c, m, pos, b = s["case"], s["case"]["m"], s["case"]["pos"], s["case"]["block"]
    n_kv, hd, n_sel = c["n_kv"], c["hd"], c["n_sel"]
    if m > 1:                                # the new rows' whole blocks
        lo, hi = pos // b, (pos + m) // b
        s["mean_qs"][lo:hi], s["mean_d"][lo:hi] = _block_means(s["k_qs"], s["k_d"], c, lo * b, hi * b)
    own_block = torch.arange(pos, pos + m, device=DEV) // b          # [m]
    n_blocks = (pos + m - 1) // b + 1
    q = s["q"].double().view(m, n_kv, -1, hd).sum(2).float()
    qq, qd = _quantise(q)
    Q = (qq.double().unflatten(-1, (-1, 32)) * qd.double()[..., None]).flatten(-2)     # [m][n_kv][hd]
    M = s["mean_qs"][:n_blocks].double().unflatten(-1, (-1, 32)) * s["mean_d"][:n_blocks].double()[..., None]
    M = M.flatten(-2).unflatten(-1, (n_kv, hd))                      # [blocks][n_kv][hd]
    score = (Q.transpose(0, 1).contiguous() @ M.permute(1, 2, 0).contiguous()).float()  # [n_kv][m][blocks]
    blk, at = torch.arange(n_blocks, device=DEV), own_block[:, None]
    score = torch.where((blk < c["n_first"]) | (blk > at - c["n_local"]), torch.full_like(score, math.inf), score)
    score = torch.where(blk > at, torch.full_like(score, -math.inf), score)
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    best = torch.where(order.indices[..., :n_sel] > at, n_blocks + n_sel, order.indices[..., :n_sel])
    best = torch.nn.functional.pad(best, (0, max(0, n_sel - n_blocks)), value=n_blocks + n_sel)
    sel = best.sort(-1).values.transpose(0, 1)                       # [m][n_kv][n_sel], ascending
    rows = (sel[..., None] * b + torch.arange(b, device=DEV)).flatten(-2)               # [m][n_kv][n_sel * b]
    seen = rows <= torch.arange(pos, pos + m, device=DEV)[:, None, None]
    at = rows.clamp(max=pos + m - 1)
    kv = torch.arange(n_kv, device=DEV)[None, :, None]
    K, V = ((s[x + "_qs"].view(-1, n_kv, hd // 32, 32)[at, kv].float()
             * s[x + "_d"].view(-1, n_kv, hd // 32)[at, kv].float()[..., None]).flatten(-2) for x in "kv")
    w = s["q"].view(m, n_kv, -1, hd) @ K.transpose(2, 3) / math.sqrt(hd)
    w.masked_fill_(~seen[:, :, None], -math.inf)
    out = _gated((_softmax(w) @ V).reshape(m, -1), s["gate"])
    got = {"out": out, "sel": torch.where(sel >= n_blocks, torch.full_like(sel, -1), sel).int()}
    if m > 1:
        got.update(mean_qs=s["mean_qs"], mean_d=s["mean_d"])
    return got


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------

def _bind(s):
    """The handles over the state's tensors that a program keeps."""
    from vxg_amd import engine as E
    global _engine
    if _engine is None:
        _engine = E.HipEngine(0)
    c = s["case"]
    p = {n: v.data_ptr() for n, v in s.items() if isinstance(v, torch.Tensor)}
    h = {"cache": E.KvQ8Cache.over(_engine, p["k_qs"], p["k_d"], p["v_qs"], p["v_d"], s["k_qs"].shape[0], c["n_kv"],
                                   c["hd"])}
    if "weight" in s:
        h["weights"] = E.KvWeights.over(_engine, p["weight"], p["position"], s["weight"].shape[1], c["n_kv"])
    if "mean_qs" in s:
        h["means"] = E.KvBlockMeans.over(_engine, p["mean_qs"], p["mean_d"], s["mean_qs"].shape[0], c["block"])
    if "to" in s:
        t = {n: v.data_ptr() for n, v in s["to"].items()}
        h["to"] = E.KvQ8Cache.over(_engine, t["k_qs"], t["k_d"], t["v_qs"], t["v_d"], c["keep"], c["n_kv"], c["hd"])
        h["to_weights"] = E.KvWeights.over(_engine, t["weight"], t["position"], c["keep"], c["n_kv"])
    h["p"] = p
    s["handles"] = h
    return h


def _run_own(s):
    c, h = s["case"], s.get("handles") or _bind(s)
    cache, p, stream = h["cache"], h["p"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "tree":
        cache.attend_tree(p["q"], c["n_head"], p["parents"], c["n"], c["pos"], p["out"], p.get("gate", 0), stream)
        return s["out"]
    if c["op"] == "weigh":
        cache.attend_weigh(h["weights"], p["q"], c["n_head"], c["m"], c["pos"], c["pos"], p["out"], p.get("gate", 0),
                           stream)
        return {"out": s["out"], "weight": s["weight"], "position": s["position"]}
    if c["op"] == "evict":
        cache.evict(h["weights"], c["seq"], c["keep"], s["n_tokens"], c["n_recent"], c["n_first"], h["to"],
                    h["to_weights"], stream)
        return s["to"]
    if c["m"] > 1:
        cache.block_means(h["means"], c["pos"], c["m"], stream)
    cache.attend_blocks(h["means"], p["q"], c["n_head"], c["m"], c["pos"], c["n_sel"], c["n_first"], c["n_local"],
                        p["out"], p.get("gate", 0), p["sel"], stream)
    got = {"out": s["out"], "sel": s["sel"]}
    if c["m"] > 1:
        got.update(mean_qs=s["mean_qs"], mean_d=s["mean_d"])
    return got


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "weigh": _plain_weigh, "evict": _plain_evict, "blocks": _plain_blocks}[
        state["case"]["op"]](state)


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------

def _head64(s, x, kv, hd):
    """One kv head's keys or values in 64 bits: [rows][hd]."""
    qs = s[x + "_qs"][:, kv * hd:(kv + 1) * hd].double()
    return qs * s[x + "_d"][:, kv * hd // 32:(kv + 1) * hd // 32].double().repeat_interleave(32, 1)


def _exact_dense(s, seen):
    """(out, sums of the weights per kv head) for queries [m][...] of which
    query i sees the rows seen[i]."""
    c = s["case"]
    hd, group, m = c["hd"], c["n_head"] // c["n_kv"], s["q"].shape[0]
    out = torch.zeros((m, c["n_head"], hd), device=DEV, dtype=torch.float64)
    total = torch.zeros((c["n_kv"], seen.shape[1]), device=DEV, dtype=torch.float64)
    q = s["q"].double().view(m, c["n_head"], hd)
    for kv in range(c["n_kv"]):
        K, V = _head64(s, "k", kv, hd), _head64(s, "v", kv, hd)
        for h in range(kv * group, (kv + 1) * group):
            for r in range(0, m, 256):
                a = torch.mm(q[r:r + 256, h], K.T) / hd ** 0.5
                a[~seen[r:r + 256]] = -math.inf
                a = torch.softmax(a, -1)
                total[kv] += a.sum(0)
                out[r:r + 256, h] = torch.mm(a, V)
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double()).view(m, c["n_head"], hd)
    return out.view(m, -1), total


def _exact_blocks(s):
    c, m, b, hd = s["case"], s["case"]["m"], s["case"]["block"], s["case"]["hd"]
    group = c["n_head"] // c["n_kv"]
    code, scale = s["mean_qs"].cpu().numpy().copy(), s["mean_d"].cpu().numpy().copy()

    def blocks_of(x):
        x = x.reshape(-1, 32)
        d = (np.abs(x).max(1) / np.float32(127)).astype(np.float16)
        df = d.astype(np.float32)
        inv = np.where(df > 0, np.float32(1) / np.where(df > 0, df, np.float32(1)), np.float32(0)).astype(np.float32)
        return np.clip(np.rint(x * inv[:, None]), -127, 127), d

    if m > 1:
        for k in range(c["pos"] // b, (c["pos"] + m) // b):
            rows = slice(k * b, (k + 1) * b)
            x = s["k_qs"][rows].cpu().numpy().astype(np.float64)
            x = x * np.repeat(s["k_d"][rows].cpu().numpy().astype(np.float64), 32, 1)
            q, d = blocks_of((x.sum(0) / b).astype(np.float32))
            code[k], scale[k] = q.reshape(-1), d
    out = torch.zeros((m, c["n_head"], hd), device=DEV, dtype=torch.float64)
    q_all, heads = s["q"].cpu().numpy(), [(_head64(s, "k", kv, hd), _head64(s, "v", kv, hd)) for kv in range(c["n_kv"])]
    mean = code.astype(np.float64) * np.repeat(scale.astype(np.float64), 32, 1)
    for i in range(m):
        last = c["pos"] + i
        n = last // b + 1
        forced = [k for k in range(n) if k < c["n_first"] or k > n - 1 - c["n_local"]]
        for kv in range(c["n_kv"]):
            qs = q_all[i].reshape(c["n_head"], hd)[kv * group:(kv + 1) * group]
            qq, qd = blocks_of(qs.astype(np.float64).sum(0).astype(np.float32))
            qv = (qq * qd.astype(np.float64)[:, None]).reshape(-1)
            score = (mean[:n, kv * hd:(kv + 1) * hd] @ qv).astype(np.float32)
            rest = sorted(set(range(n)) - set(forced), key=lambda k: (-score[k], k))
            take = forced + rest[:max(0, c["n_sel"] - len(forced))]
            at = np.concatenate([np.arange(k * b, min((k + 1) * b, last + 1)) for k in sorted(take)])
            at = torch.from_numpy(at).to(DEV)
            K, V = heads[kv]
            a = torch.softmax(torch.from_numpy(qs).to(DEV).double() @ K[at].T.contiguous() / hd ** 0.5, -1)
            out[i, kv * group:(kv + 1) * group] = a @ V[at]
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double()).view(m, c["n_head"], hd)
    got = {"out": out.view(m, -1), "sel": None}
    if m > 1:
        got.update(mean_qs=None, mean_d=None)
    return got


def exact(case, seed):
    """What ``run`` returns, from the definitions; codes, indices and moved
    rows have no value of their own here."""
    c = case
    if c["op"] == "evict":
        return None
    s = prepare(c, seed)
    if c["op"] == "blocks":
        return _exact_blocks(s)
    m = c.get("m") or c["n"]
    seen = torch.zeros((m, c["pos"] + m), dtype=torch.bool)
    seen[:, :c["pos"]] = True
    if c["op"] == "tree":
        up = s["parents"].tolist()
        for i in range(m):
            k = i
            while k >= 0:
                seen[i, c["pos"] + k] = True
                k = up[k]
        return _exact_dense(s, seen.to(DEV))[0]
    for i in range(m):
        seen[i, c["pos"]:c["pos"] + i + 1] = True
    out, total = _exact_dense(s, seen.to(DEV))
    before = s["weight"].double()
    before[:, c["pos"]:] = 0
    return {"out": out, "weight": before + total, "position": None}
