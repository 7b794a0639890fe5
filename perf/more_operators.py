"""The operators of serving many conversations from one paged Q8_0 KV cache, as
calls to time: ``op`` names one.

* ``write``   the attention preparation of a batch's new tokens into pages
  (``KvPagesQ8.prep``): each head's query and key normalised, rotated by
  positions of one axis or of several (time, height, width), K and V quantised
  into their sequences' pages, and those rows read back as values
  (``KvPagesQ8.read``);
* ``read``    whole sequences read back from their pages as values
  (``KvPagesQ8.read``);
* ``attend``  attention of each sequence's new token, or its new token and the
  ones drafted after it, over the pages (``KvPagesQ8.attend``);
* ``verify``  drafted tokens accepted or not by the model's probabilities and
  given random numbers, and the token that follows (``HipEngine.verify_drafts``).

Pages are int8 values [pages][n_kv][page][hd] and one f16 scale per 32 of them.
A sequence's row r lies in page table[sequence][r // page]; a batch's tokens are
the last rows of their sequences.  ``run`` computes an operator from elementary
torch operations, or with ``own`` calls the framework.
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

def _write(name, n_seq, most, past, n_head, n_kv, hd, page, gated, axes, dtype, mix):
    """`most` tokens at most to a sequence (all of them if there is one sequence)
    after up to `past` rows; axes: "one", "sections" or "interleaved"."""
    return {"name": name, "op": "write", "n_seq": n_seq, "most": most, "past": past, "n_head": n_head, "n_kv": n_kv,
            "hd": hd, "page": page, "gated": gated, "axes": axes, "dtype": dtype, "mix": mix}


def _read(name, n_seq, lo, hi, n_kv, hd, page, dtype, mix):
    return {"name": name, "op": "read", "n_seq": n_seq, "lo": lo, "hi": hi, "n_kv": n_kv, "hd": hd, "page": page,
            "dtype": dtype, "mix": mix}


def _attend(name, n_seq, most, lo, hi, n_head, n_kv, hd, page, gated, dtype, mix):
    """Sequences of lo to hi rows, 1 to `most` new tokens each."""
    return {"name": name, "op": "attend", "n_seq": n_seq, "most": most, "lo": lo, "hi": hi, "n_head": n_head,
            "n_kv": n_kv, "hd": hd, "page": page, "gated": gated, "dtype": dtype, "mix": mix}


def _verify(name, n_seq, most, vocab, drafts, dtype, mix):
    """0 to `most` drafted tokens to a sequence (all of them if there is one);
    drafts: whether the draft model's logits are there."""
    return {"name": name, "op": "verify", "n_seq": n_seq, "most": most, "vocab": vocab, "drafts": drafts,
            "dtype": dtype, "mix": mix}


def listed():
    return [
        # one conversation's decode step: latency counts
        _write("write 1 token", 1, 1, 700, 16, 4, 128, 16, True, "one", "f32", 1),
        # a decode step of many conversations, a wide model
        _write("write 64 tokens", 64, 1, 8000, 32, 8, 128, 32, False, "one", "f32", 2),
        # a prompt with images: positions of three axes
        _write("write 1900 image prompt", 1, 1900, 0, 16, 4, 128, 64, True, "interleaved", "bf16", 3),
        # conversations of ordinary length, handed on as bf16 rows
        _read("read 40 of 50 to 1500", 40, 50, 1500, 4, 128, 16, "bf16", 4),
        # a long document's cache for an operator outside of the pages
        _read("read 60000", 1, 60000, 60000, 8, 128, 64, "f32", 5),
        # one short conversation, a small model: latency counts
        _attend("attend 1 at 500", 1, 1, 500, 500, 8, 2, 64, 16, False, "f32", 6),
        # a serving batch of unlike lengths
        _attend("attend 32 of 150 to 8000", 32, 1, 150, 8000, 16, 4, 128, 16, True, "f32", 7),
        # a few long documents, a wide model: the largest
        _attend("attend 8 of 20000 to 30000", 8, 1, 20000, 30000, 32, 8, 128, 64, False, "bf16", 8),
        # a serving batch that drafts up to five tokens ahead
        _attend("attend 24 x 6 of 300 to 4000", 24, 6, 300, 4000, 16, 4, 128, 32, True, "f32", 9),
        # one conversation, four drafted tokens
        _verify("verify 1 x 4", 1, 4, 151936, True, "f32", 10),
        # a serving batch with a draft model
        _verify("verify 48 x 5", 48, 5, 151936, True, "f32", 11),
        # drafts from text seen before, without probabilities of their own
        _verify("verify 16 x 8 given", 16, 8, 248320, False, "bf16", 12),
    ]


def _logu(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "write prompt", "read", "attend", "attend", "attend drafts", "verify", "verify"))
    hd, page, mix = rng.choice((64, 128, 128, 256)), rng.choice((16, 32, 64, 128)), rng.randint(100, 1 << 30)
    gated, dtype = rng.random() < 0.5, rng.choice(("f32", "bf16"))
    while True:
        n_kv = rng.choice((1, 2, 4, 8))
        n_head = n_kv * rng.choice((1, 2, 4, 5, 7, 8))
        axes = rng.choice(("one", "sections", "interleaved"))
        if op == "write":
            c = _write("", _logu(rng, 1, 256), rng.choice((1, 1, 4)), _logu(rng, 1, 20000), n_head, n_kv, hd, page,
                       gated, axes, dtype, mix)
            fits = c["n_seq"] * c["most"] * n_head * hd <= 4e6
        elif op == "write prompt":
            c = _write("", rng.choice((1, 1, 3)), _logu(rng, 20, 3000), rng.choice((0, 1000)), n_head, n_kv, hd, page,
                       gated, axes, dtype, mix)
            fits = c["n_seq"] * c["most"] * n_head * hd <= 4e6
        elif op == "read":
            lo = _logu(rng, 1, 20000)
            c = _read("", _logu(rng, 1, 100), lo, _logu(rng, lo, 60000), n_kv, hd, page, dtype, mix)
            fits = c["n_seq"] * c["hi"] * n_kv * hd <= 6.1e7
        elif op == "verify":
            c = _verify("", _logu(rng, 1, 64), rng.randint(1, 9), rng.choice((32000, 50257, 151936, _logu(rng, 500, 250000))),
                        rng.random() < 0.6, dtype, mix)
            fits = c["n_seq"] * (c["most"] + 1) * c["vocab"] <= 4.4e7
        else:
            lo = _logu(rng, 1, 20000)
            most = 1 if op == "attend" else _logu(rng, 2, 40)
            c = _attend("", _logu(rng, 1, 200), most, lo, _logu(rng, lo, 60000), n_head, n_kv, hd, page, gated,
                        dtype, mix)
            fits = (c["n_seq"] * c["hi"] * n_kv * hd <= 2.4e8 and c["lo"] >= most
                    and c["n_seq"] * c["hi"] * n_head * most <= 1.5e8)
        if fits:
            del c["name"]
            return c


def _mix(c):
    return np.random.RandomState(c["mix"])


def _shape(c):
    """(rows, new tokens) of each sequence, by the case alone."""
    r, n = _mix(c), c["n_seq"]
    if c["op"] == "verify":
        return np.zeros(n, np.int64), 1 + (r.randint(0, c["most"] + 1, n) if n > 1 else np.full(n, c["most"]))
    if c["op"] == "write":
        new = r.randint(1, c["most"] + 1, n) if n > 1 else np.full(n, c["most"])
        return new + r.randint(0, c["past"] + 1, n), new
    rows = np.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"]), n)).round().astype(np.int64)
    if c["op"] == "read":
        return rows, rows
    return rows, np.minimum(r.randint(1, c["most"] + 1, n), rows)


def _size(c):
    return 2 if c["dtype"] == "bf16" else 4


def work(case):
    c = case
    rows, new = _shape(c)
    if c["op"] == "verify":
        read = new.sum() + ((new - 1).sum() if c["drafts"] else 0)
        return {"bytes": float(read * c["vocab"] * _size(c) + 8 * new.sum() + 24 * c["n_seq"]), "flops": float(3 * read * c["vocab"])}
    per = c["n_kv"] * c["hd"]
    row = 2 * per * 34 / 32                 # K and V of a row as codes and scales
    if c["op"] == "read":
        return {"bytes": float(rows.sum() * (row + 2 * per * _size(c))), "flops": float(2 * rows.sum() * per)}
    wide = c["n_head"] * c["hd"]
    if c["op"] == "write":
        q = wide * (2 if c["gated"] else 1)
        return {"bytes": float(new.sum() * ((q + 2 * per) * _size(c) + 4 * q + row + 8 * per)),
                "flops": float(new.sum() * 10 * (wide + 2 * per))}
    seen = (new * rows - new * (new - 1) // 2).sum()
    return {"bytes": float(rows.sum() * row + new.sum() * wide * (4 + _size(c) + (4 if c["gated"] else 0))),
            "flops": float(4 * wide * seen)}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _typed(x, c):
    return x.bfloat16() if c["dtype"] == "bf16" else x


def _quantise(x):
    """f32 [..., n] as Q8_0 blocks: int8 codes and one f16 scale per 32."""
    b = x.unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1) / 127.0).half()
    df = d.float()
    inv = torch.where(df > 0, 1.0 / df, torch.zeros_like(df))
    q = (b * inv[..., None]).round().clamp(-127, 127)
    return q.to(torch.int8).flatten(-2).contiguous(), d.contiguous()


def _pages(c, rows, g, filled):
    """Pages in an order of their own, a few of nobody's among them; every
    sequence's table a little longer than it needs."""
    need = -(-rows // c["page"])
    total, wide = int(need.sum()), int(need.max()) + 2
    n_pages = total + 1 + total // 16
    order = torch.randperm(n_pages, generator=g, device=DEV)[:total].int()
    table = torch.zeros((c["n_seq"], wide), dtype=torch.int32, device=DEV)
    cols = torch.arange(wide, device=DEV)
    table[cols < torch.from_numpy(need).to(DEV)[:, None]] = order
    s = {"table": table, "seq_len": torch.from_numpy(rows).int().to(DEV)}
    shape = (n_pages, c["n_kv"], c["page"], c["hd"])
    for x in "kv":
        if filled:
            # keys share a part over a page (a topic), a few rows draw every query
            a = _randn(shape, g, 0.8 if x == "k" else 1.0)
            if x == "k":
                a += _randn((n_pages, c["n_kv"], 1, c["hd"]), g, 0.6)
                a *= 1 + (torch.rand((n_pages, 1, c["page"], 1), generator=g, device=DEV) < 0.02)
            s[x + "_qs"], s[x + "_d"] = _quantise(a)
            del a
        else:
            s[x + "_qs"] = torch.zeros(shape, dtype=torch.int8, device=DEV)
            s[x + "_d"] = torch.zeros(shape[:3] + (c["hd"] // 32,), dtype=torch.float16, device=DEV)
    return s


def _axis_of_pair(c):
    """Which axis's position turns each pair of a head's dims."""
    half = c["hd"] // 2
    if c["axes"] == "one":
        return [0] * half
    if c["axes"] == "interleaved":
        return [i % 3 for i in range(half)]
    first = half // 4
    second = first + (half - first) // 2
    return [0 if i < first else 1 if i < second else 2 for i in range(half)]


def _positions(c, rows, new):
    """[axes][tokens]: one axis counts rows.  With three, the first tenth of a
    sequence's new tokens is text, then comes an image of 28 columns, then text that
    goes on behind it."""
    at = np.concatenate([np.arange(r - n, r) for r, n in zip(rows, new)])
    if c["axes"] == "one":
        return at[None].astype(np.int32)
    j = np.concatenate([np.arange(n) for n in new])
    n = np.repeat(new, new)
    begin = at - j
    head, end = n // 10, n - n // 5
    i = j - head
    image = (j >= head) & (j < end)
    high = (end - head + 27) // 28
    after = begin + head + np.maximum(high, 28) + (j - end)
    text = np.where(j < head, at, after)
    return np.stack([np.where(image, begin + head, text), np.where(image, begin + head + i // 28, text),
                     np.where(image, begin + head + i % 28, text)]).astype(np.int32)


def prepare(case, seed):
    c, g = case, _gen(seed)
    rows, new = _shape(c)
    n = int(new.sum())
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    s = {"case": c, "n_tok": n, "tok_start": torch.from_numpy(start).to(DEV)}
    if c["op"] == "verify":
        return _prepare_verify(c, g, s, n)
    s.update(_pages(c, rows, g, c["op"] != "write"))
    per, wide = c["n_kv"] * c["hd"], c["n_head"] * c["hd"] if "n_head" in c else 0
    if c["op"] == "attend":
        s["q"] = _randn((n, wide), g, 1.2)
        s["gate"] = _randn((n, wide), g) if c["gated"] else None
        s["out"] = torch.zeros((n, wide), device=DEV, dtype=torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)
        return s
    back = torch.bfloat16 if c["op"] == "read" and c["dtype"] == "bf16" else torch.float32
    s["k_out"], s["v_out"] = (torch.zeros((n, per), device=DEV, dtype=back) for _ in "kv")
    if c["op"] == "write":
        q_rows = wide * (2 if c["gated"] else 1)
        s["qkv"] = _typed(_randn((n, q_rows + 2 * per), g), c)
        s["q_norm"], s["k_norm"] = (1 + _randn((c["hd"],), g, 0.2) for _ in "qk")
        s["rope_pos"] = torch.from_numpy(_positions(c, rows, new)).to(DEV)
        s["axis"] = torch.tensor(_axis_of_pair(c), device=DEV)
        s["q_out"] = torch.zeros((n, wide), device=DEV)
        s["gate_out"] = torch.zeros((n, wide), device=DEV) if c["gated"] else None
    return s


def _prepare_verify(c, g, s, n):
    """Rows where one token stands out more or less; a draft model near the
    target, its tokens drawn from it, or tokens that were copied."""
    v = c["vocab"]
    s["temperature"] = torch.tensor([0.0, 0.7, 1.0, 1.0], device=DEV)[
        torch.randint(0, 4, (c["n_seq"],), generator=g, device=DEV)] if c["n_seq"] > 1 else torch.ones(1, device=DEV)
    logits = _randn((n, v), g, 2.0)
    top = torch.randint(0, v, (n,), generator=g, device=DEV)
    logits[torch.arange(n, device=DEV), top] += 8 + 8 * torch.rand(n, generator=g, device=DEV)
    s["logits"] = _typed(logits, c)
    tokens = top.roll(1)
    s["draft_logits"] = None
    if c["drafts"]:
        s["draft_logits"] = _typed(logits + _randn((n, v), g, 0.5), c)
        t = s["temperature"].clamp(min=0.05)[_seq_of(s, c)]
        u = torch.rand((n, v), generator=g, device=DEV).clamp_(min=1e-30)
        tokens = (s["draft_logits"].float() / t[:, None] - torch.log(-torch.log(u))).argmax(-1).roll(1)
    s["tokens"] = tokens.int()
    s["u_accept"] = torch.rand(n, generator=g, device=DEV)
    s["u_next"] = torch.rand(c["n_seq"], generator=g, device=DEV)
    counts = s["tok_start"][1:] - s["tok_start"][:-1]
    s["seq_len"] = (counts + torch.randint(0, 4000, (c["n_seq"],), generator=g, device=DEV)).int()
    for x in ("n_accept", "next", "new_len"):
        s[x] = torch.zeros(c["n_seq"], dtype=torch.int32, device=DEV)
    return s


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def _seq_of(s, c):
    """The sequence of each token."""
    counts = (s["tok_start"][1:] - s["tok_start"][:-1]).long()
    return torch.repeat_interleave(torch.arange(c["n_seq"], device=DEV), counts, output_size=s["n_tok"])


def _slots(s, c):
    """(page, row in it) of each token."""
    seq = _seq_of(s, c)
    back = s["tok_start"][1:].long()[seq] - torch.arange(s["n_tok"], device=DEV)
    row = s["seq_len"].long()[seq] - back
    return s["table"][seq, row // c["page"]].long(), row % c["page"]


def _values(s, x, page, at):
    """f32 values of rows [..., n_kv, hd]."""
    code, d = s[x + "_qs"][page, :, at], s[x + "_d"][page, :, at]
    return (code.float().unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)


def _head_norm(x, weight):
    """64 bits: x [..., hd] times weight over its root mean square."""
    return x * (1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)) * weight.double()


def _turn(x, s, c):
    """64 bits: pairs (i, i + hd / 2) turned by the position of their axis."""
    half = c["hd"] // 2
    freq = 10000.0 ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / c["hd"])
    angle = s["rope_pos"].double()[s["axis"]].T * freq              # [tokens][half]
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_write(s):
    c, n = s["case"], s["n_tok"]
    per, hd = c["n_kv"] * c["hd"], c["hd"]
    x = s["qkv"].double()
    q_rows = x.shape[1] - 2 * per
    q = x[:, :q_rows].unflatten(1, (c["n_head"], -1))
    k, v = x[:, q_rows:q_rows + per].unflatten(1, (c["n_kv"], hd)), x[:, q_rows + per:].unflatten(1, (c["n_kv"], hd))
    q_out = _turn(_head_norm(q[..., :hd], s["q_norm"]), s, c).float().reshape(n, -1)
    k = _turn(_head_norm(k, s["k_norm"]), s, c).float()
    page, at = _slots(s, c)
    for name, rows in (("k", k), ("v", v.float())):
        s[name + "_qs"][page, :, at], s[name + "_d"][page, :, at] = _quantise(rows)
    got = {"q": q_out, "k": _values(s, "k", page, at).reshape(n, -1), "v": _values(s, "v", page, at).reshape(n, -1)}
    if c["gated"]:
        got["gate"] = q[..., hd:].float().reshape(n, -1)
    return got


def _plain_read(s):
    page, at = _slots(s, s["case"])
    return {x: _values(s, x, page, at).flatten(1).to(s["k_out"].dtype) for x in "kv"}


def _plain_attend(s):
    c, n = s["case"], s["n_tok"]
    hd, n_kv, group, page = c["hd"], c["n_kv"], c["n_head"] // c["n_kv"], c["page"]
    rows, new = _shape(c)
    longest, most = int(rows.max()), int(new.max())
    row = torch.arange(longest, device=DEV)
    at = s["table"].long()[:, row // page]                          # [sequences][rows]
    K, V = (_values(s, x, at, (row % page).expand_as(at)).transpose(1, 2).contiguous() for x in "kv")
    seq = _seq_of(s, c)
    j = torch.arange(n, device=DEV) - s["tok_start"].long()[seq]
    q = torch.zeros((c["n_seq"], most, n_kv, group, hd), device=DEV)
    q[seq, j] = s["q"].view(n, n_kv, group, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(c["n_seq"], n_kv, most * group, hd)
    w = q @ K.transpose(2, 3).contiguous() / math.sqrt(hd)          # [sequences][n_kv][most * group][rows]
    counts = s["tok_start"][1:] - s["tok_start"][:-1]
    upto = (s["seq_len"] - counts)[:, None] + torch.arange(most, device=DEV)            # a token's own row
    late = row > torch.minimum(upto, s["seq_len"][:, None] - 1)[..., None]              # [sequences][most][rows]
    w.masked_fill_(late.repeat_interleave(group, 1)[:, None], -math.inf)
    e = torch.exp(w - w.amax(-1, keepdim=True))
    out = (e / e.sum(-1, keepdim=True)) @ V
    out = out.view(c["n_seq"], n_kv, most, group, hd).permute(0, 2, 1, 3, 4)[seq, j].reshape(n, -1)
    if s["gate"] is not None:
        out = out * (1.0 / (1.0 + torch.exp(-s["gate"])))
    return out.to(s["out"].dtype)


def _probabilities(logits, t):
    """64 bits: softmax of rows at their temperatures; at zero, all of it on the
    lowest of the largest."""
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t))[:, None]))
    p = w / w.sum(-1, keepdim=True)
    ids = torch.arange(x.shape[1], device=DEV)
    first = torch.where(x == top, ids, x.shape[1]).amin(-1, keepdim=True)
    return torch.where(t[:, None] > 0, p, (ids == first).double())


def _plain_verify(s):
    c, n, v = s["case"], s["n_tok"], s["case"]["vocab"]
    seq, start = _seq_of(s, c), s["tok_start"].long()
    j = torch.arange(n, device=DEV) - start[seq]
    t = s["temperature"].double()
    p = _probabilities(s["logits"], t[seq])
    x = s["tokens"].long().roll(-1)                                 # the token drafted after each row
    at = torch.arange(n, device=DEV)
    if s["draft_logits"] is not None:
        q = _probabilities(s["draft_logits"], t[seq])
        q_x = torch.where(t[seq] > 0, q[at, x], torch.ones(n, device=DEV, dtype=torch.float64))
    else:
        q, q_x = None, torch.ones(n, device=DEV, dtype=torch.float64)
    good = s["u_accept"].double().roll(-1) * q_x < p[at, x]
    drafts = (start[1:] - start[:-1]) - 1
    good &= j < drafts[seq]
    run_ = torch.zeros((c["n_seq"], int(c["most"]) + 1), device=DEV)
    run_[seq, j] = good.float()
    n_accept = run_.cumprod(1).sum(1).long()
    row = start[:-1] + n_accept
    refused = n_accept < drafts
    r = p[row]
    if q is not None:
        left = torch.where((t > 0)[:, None], (r - q[row]).clamp(min=0), r)
    else:
        left = r.scatter(1, x[row][:, None], 0.0)
    left = torch.where((t > 0)[:, None] & refused[:, None], left, r)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, r)
    c_sum = left.cumsum(-1)
    ids = torch.arange(v, device=DEV)
    over = torch.where(c_sum > s["u_next"].double()[:, None] * c_sum[:, -1:], ids, v).amin(-1)
    last = torch.where(left > 0, ids, 0).amax(-1)
    return {"n_accept": n_accept.int(), "next": torch.minimum(over, last).int(),
            "new_len": (s["seq_len"] - (drafts - n_accept)).int()}


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
    h = {"p": p, "dtype": E.DTYPE_BF16 if c["dtype"] == "bf16" else E.DTYPE_F32, "f32": E.DTYPE_F32}
    if c["op"] != "verify":
        h["pages"] = E.KvPagesQ8.over(_engine, p["k_qs"], p["k_d"], p["v_qs"], p["v_d"], s["k_qs"].shape[0], c["page"],
                                      c["n_kv"], c["hd"])
        h["batch"] = E.PagedBatch(p["table"], p["seq_len"], p["tok_start"], c["n_seq"], s["table"].shape[1], s["n_tok"])
    if c["op"] == "write":
        h["params"] = E.GqaParams(p["q_norm"], p["k_norm"], 0, 0, 0, c["n_head"], int(c["gated"]), c["hd"], 1, 10000.0, 1e-6)
        h["axes"] = E.RopeAxes.of(_axis_of_pair(c))
    s["handles"] = h
    return h


def _run_own(s):
    c, h = s["case"], s.get("handles") or _bind(s)
    p, stream = h["p"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "verify":
        _engine.verify_drafts(p["logits"], p.get("draft_logits", 0), h["dtype"], c["vocab"], p["tokens"], p["tok_start"],
                              c["n_seq"], s["n_tok"], p["u_accept"], p["u_next"], p["n_accept"], p["next"],
                              p["temperature"], p["seq_len"], p["new_len"], stream=stream)
        return {x: s[x] for x in ("n_accept", "next", "new_len")}
    if c["op"] == "attend":
        h["pages"].attend(h["batch"], p["q"], c["n_head"], p["out"], p.get("gate", 0), h["dtype"], stream)
        return s["out"]
    if c["op"] == "read":
        h["pages"].read(h["batch"], p["k_out"], p["v_out"], h["dtype"], stream=stream)
        return {"k": s["k_out"], "v": s["v_out"]}
    wide, per, size = s["qkv"].shape[1], c["n_kv"] * c["hd"], s["qkv"].element_size()
    k_cur = p["qkv"] + (wide - 2 * per) * size
    h["pages"].prep(h["batch"], h["params"], p["qkv"], k_cur, k_cur + per * size, p["q_out"], p.get("gate_out", 0),
                    h["axes"], p["rope_pos"], wide, wide, h["dtype"], stream)
    h["pages"].read(h["batch"], p["k_out"], p["v_out"], h["f32"], stream=stream)
    got = {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    if c["gated"]:
        got["gate"] = s["gate_out"]
    return got


def run(state):
    if own:
        return _run_own(state)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}[
        state["case"]["op"]](state)


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------

def _where(c, s, i, rows):
    """(pages, rows in them) of the given rows of sequence i, as numpy indices."""
    page = s["table"][i].cpu().numpy()[rows // c["page"]]
    return torch.from_numpy(page.astype(np.int64)).to(DEV), torch.from_numpy(rows % c["page"]).to(DEV)


def _rows64(s, x, page, at):
    """[n_kv][rows][hd] in 64 bits."""
    code, d = s[x + "_qs"][page, :, at].double(), s[x + "_d"][page, :, at].double()
    return (code * d.repeat_interleave(32, -1)).transpose(0, 1)


def _exact_write(c, s, new):
    x = s["qkv"].double().cpu().numpy()
    n, hd, per = x.shape[0], c["hd"], c["n_kv"] * c["hd"]
    half = hd // 2
    pos, axis = s["rope_pos"].cpu().numpy(), _axis_of_pair(c)
    angle = np.stack([pos[axis[i]].astype(np.float64) * 10000.0 ** (-2.0 * i / hd) for i in range(half)], -1)

    def head(a, weight):
        a = a / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-6) * weight.double().cpu().numpy()
        z = (a[..., :half] + 1j * a[..., half:]) * np.exp(1j * angle)[:, None]
        return np.concatenate([z.real, z.imag], -1)

    def held(a):
        """The value that a block of 32 keeps of each: in 8 bits."""
        b = a.astype(np.float32).reshape(-1, 32)
        d = (np.abs(b).max(1) / np.float32(127)).astype(np.float16)
        f = d.astype(np.float32)
        inv = np.where(f > 0, np.float32(1) / np.where(f > 0, f, np.float32(1)), np.float32(0)).astype(np.float32)
        return (np.clip(np.rint(b * inv[:, None]), -127, 127) * d.astype(np.float64)[:, None]).reshape(n, -1)

    q_rows = x.shape[1] - 2 * per
    q = x[:, :q_rows].reshape(n, c["n_head"], -1)
    got = {"q": head(q[..., :hd], s["q_norm"]).reshape(n, -1),
           "k": held(head(x[:, q_rows:q_rows + per].reshape(n, c["n_kv"], hd), s["k_norm"])), "v": held(x[:, q_rows + per:])}
    if c["gated"]:
        got["gate"] = q[..., hd:].reshape(n, -1)
    return got


def exact(case, seed):
    """What ``run`` returns, from the definitions; accepted counts and tokens
    have no value of their own here."""
    c = case
    if c["op"] == "verify":
        return None
    s = prepare(c, seed)
    rows, new = _shape(c)
    if c["op"] == "write":
        return _exact_write(c, s, new)
    if c["op"] == "read":
        got = {"k": [], "v": []}
        for i, r in enumerate(rows):
            page, at = _where(c, s, i, np.arange(r))
            for x in "kv":
                got[x].append(_rows64(s, x, page, at).transpose(0, 1).reshape(r, -1))
        return {x: torch.cat(a) for x, a in got.items()}
    group, hd = c["n_head"] // c["n_kv"], c["hd"]
    out, first = [], 0
    for i, (r, m) in enumerate(zip(rows, new)):
        page, at = _where(c, s, i, np.arange(r))
        K, V = _rows64(s, "k", page, at), _rows64(s, "v", page, at)
        q = s["q"][first:first + m].double().view(m, c["n_kv"], group, hd)
        for t in range(m):
            upto = int(r - m + t + 1)
            a = (K[:, :upto] @ q[t].transpose(1, 2).contiguous()) / hd ** 0.5           # [n_kv][rows][group]
            a = torch.softmax(a, 1)
            out.append((a.transpose(1, 2).contiguous() @ V[:, :upto].contiguous()).reshape(-1))
        first += m
    out = torch.stack(out)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())
