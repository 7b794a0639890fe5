"""Shared by the tests of the paged Q8_0 KV cache: pages as host planes, a
batch's rows, and the formulas in 64 bits.

Bar of an attention output: that of kv_ops_util (the same operand widths and
sums), and half a step of bf16, 2^-8 of the value, where that is the output's
type.  Prepared queries are one rounding from 64 bits: 2^-24 of the value and
2^-45 of the head's largest (the steps before it).  Codes, scales and what is read
back are exact."""
import numpy as np

from kv_ops_util import attention, raises  # noqa: F401  (re-exported)
from vxg_amd import engine

PLANES = ("k_qs", "k_d", "v_qs", "v_d")


class HostPages:
    def __init__(self, n_pages, page, n_kv, hd, seed, zero=False):
        r = np.random.default_rng(seed)
        self.n_pages, self.page, self.n_kv, self.hd = n_pages, page, n_kv, hd
        shape = (n_pages, n_kv, page)
        for x in "kv":
            qs = r.integers(-127, 128, shape + (hd,)).astype(np.int8)
            lo, hi = (0.002, 0.02) if x == "k" else (1e-4, 0.05)
            d = np.exp(r.uniform(np.log(lo), np.log(hi), shape + (hd // 32,))).astype(np.float16)
            setattr(self, x + "_qs", qs * 0 if zero else qs)
            setattr(self, x + "_d", d * np.float16(0) if zero else d)

    def upload(self, eng):
        g = eng.kv_pages(self.n_pages, self.page, self.n_kv, self.hd)
        for n in PLANES:
            getattr(g, n).upload(getattr(self, n))
        return g

    def download(self, g):
        return {n: getattr(g, n).download(np.int8 if n.endswith("qs") else np.uint16, getattr(self, n).shape) for n in PLANES}

    def bits(self):
        return {n: getattr(self, n) if n.endswith("qs") else getattr(self, n).view(np.uint16).copy() for n in PLANES}

    def good(self, pages):
        return (pages >= 0) & (pages < self.n_pages)

    def rows(self, x, table, n):
        """([n][n_kv][hd] in 64 bits, which of them have a page) of a sequence's rows 0 .. n - 1."""
        r = np.arange(n)
        pages = table[r // self.page]
        at = np.where(self.good(pages), pages, 0), slice(None), r % self.page
        v = getattr(self, x + "_qs")[at].astype(np.float64) * np.repeat(getattr(self, x + "_d")[at].astype(np.float64), 32, -1)
        return v, self.good(pages)


class Batch:
    """Tables with pages in a random order, lengths and token ranges."""

    def __init__(self, lens, new, page, seed, spare_pages=2, spare_cols=1, tail=0, bare=False):
        r = np.random.default_rng(seed)
        self.lens, self.new = np.asarray(lens, np.int32), np.asarray(new, np.int32)
        self.n_seq, self.page, self.bare = len(lens), page, bare
        need = -(-np.maximum(self.lens, 0) // page)
        self.n_pages = int(need.sum()) + spare_pages
        order = r.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((self.n_seq, int(need.max(initial=0)) + spare_cols), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.n_tok = int(self.start[-1]) + tail
        self.owner = np.full(self.n_tok, -1)
        self.row = np.full(self.n_tok, -1)
        for i in range(self.n_seq):
            for j in range(self.new[i]):
                self.owner[self.start[i] + j] = i
                self.row[self.start[i] + j] = self.lens[i] - self.new[i] + j

    def put(self, d):
        """The device's batch (``d``: Dev)."""
        self.dev = [d.put(self.table), d.put(self.lens)] + ([] if self.bare else [d.put(self.start)])
        return engine.PagedBatch(self.dev[0].ptr, self.dev[1].ptr, 0 if self.bare else self.dev[2].ptr, self.n_seq,
                                 self.table.shape[1], self.n_tok)


class _Rows:
    """A sequence's rows with the names kv_ops_util.attention reads."""

    def __init__(self, K, V, n_kv, hd):
        self.rows, self.n_kv, self.hd, self._x = K.shape[0], n_kv, hd, {"k": K, "v": V}

    def values(self, x):
        return self._x[x]


def paged_attention(host, batch, q, n_head, gate=None):
    """(out, bar) [n_tok][n_head * hd] in 64 bits; a token that sees nothing is 0,
    a buffer row of nobody NaN in both."""
    out = np.full(q.shape, np.nan)
    bar = np.full(q.shape, np.nan)
    for i in range(batch.n_seq):
        n = max(int(batch.lens[i]), 0)
        K, okay = host.rows("k", batch.table[i], n)
        V, _ = host.rows("v", batch.table[i], n)
        for t in range(batch.start[i], batch.start[i + 1]):
            sees = okay & (np.arange(n) <= batch.row[t])
            out[t], bar[t] = 0.0, 0.0
            if sees.any():
                o, _, b, _ = attention(_Rows(K, V, host.n_kv, host.hd), q[t:t + 1], sees[None],
                                       None if gate is None else gate[t:t + 1])
                out[t], bar[t] = o[0], b
    return out, bar


def quantise(x):
    """KvQ8Block::quantize of f32 [..., 32 n]: (codes, f16 scales)."""
    b = np.asarray(x, np.float32).reshape(x.shape[:-1] + (-1, 32))
    a = np.abs(b)
    amax = np.where(np.isnan(a), np.float32(0), a).max(-1)
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        d = (amax / np.float32(127)).astype(np.float16)
        f = d.astype(np.float32)
        inv = np.where(f > 0, np.float32(1) / f, np.float32(0)).astype(np.float32)
        q = np.rint(b * inv[..., None])
        q = np.where(np.isnan(q), 0, np.clip(q, -127, 127)).astype(np.int8)
    return q.reshape(x.shape), d


def prepared(x, weight, bias, pos, axis, rope_dim, base, neox, eps):
    """64 bits: x [n_tok][heads][hd] with bias [heads][hd], normalised, turned by
    pos [axes][n_tok]."""
    x = np.asarray(x, np.float64)
    if bias is not None:
        x = x + np.asarray(bias, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(weight, np.float64)
    dim = min(rope_dim, x.shape[-1])
    half = dim // 2
    out = x.copy()
    for i in range(half):
        angle = pos[axis[i]].astype(np.float64) * np.float64(np.float32(base)) ** (-2.0 * i / dim)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        i0, i1 = (i, i + half) if neox else (2 * i, 2 * i + 1)
        out[..., i0] = x[..., i0] * c - x[..., i1] * s
        out[..., i1] = x[..., i0] * s + x[..., i1] * c
    return out


def to_bf16(x):
    """(bits, the values they hold in f32), rounded to nearest even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    bits = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32)
