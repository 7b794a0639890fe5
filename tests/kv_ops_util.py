"""Shared by the tests of the operators over the Q8_0 KV cache: random caches
as host planes, their device copies, and the operators' formulas in 64 bits.

Bar of an attention output.  A head's output is a convex combination of V
rows, so the error is measured in units of max|V|.  With S the largest
sum |q_d K_td| / sqrt(hd), a score's error is at most
S ((hd + 8) 2^-24 + 2^-21): f32 sums of hd products of a 22-bit query, the
scale products and the factor.  A weight's relative error is that plus 2^-20
(exp2, two 22-bit operands), it enters numerator and denominator, and the sums
over L rows run in pieces of at most L / 16 + 64 f32 additions each:
  |out - ref| <= max|V| (2 S ((hd + 8) 2^-24 + 2^-21) + 2 (L / 16 + 64) 2^-24 + 2^-19).
A row's accumulated weight, a sum of weights, has that bar relative to itself
plus 2^-22 of the largest weight (exp2 results near zero).
"""
import numpy as np

from vxg_amd import engine


def f16(bits):
    return np.asarray(bits, np.uint16).view(np.float16)


class HostCache:
    """Planes of one layer's cache on the host: int8 codes and f16 scales."""

    def __init__(self, rows, n_kv, hd, seed, spread=1.0):
        r = np.random.default_rng(seed)
        per = n_kv * hd
        self.rows, self.n_kv, self.hd, self.per = rows, n_kv, hd, per
        self.k_qs = r.integers(-127, 128, (rows, per)).astype(np.int8)
        self.v_qs = r.integers(-127, 128, (rows, per)).astype(np.int8)
        self.k_d = (r.uniform(0.002, 0.02, (rows, per // 32)) * spread).astype(np.float16)
        self.v_d = np.exp(r.uniform(np.log(1e-4), np.log(0.05), (rows, per // 32))).astype(np.float16)

    def values(self, x):
        """[rows][n_kv][hd] in 64 bits."""
        qs, d = getattr(self, x + "_qs"), getattr(self, x + "_d")
        return (qs.astype(np.float64) * np.repeat(d.astype(np.float64), 32, 1)).reshape(-1, self.n_kv, self.hd)

    def upload(self, eng, max_seq=None):
        c = eng.kv_q8_cache(max_seq or self.rows, self.n_kv, self.hd)
        for n in ("k_qs", "k_d", "v_qs", "v_d"):
            getattr(c, n).upload(getattr(self, n))
        return c

    @staticmethod
    def download(cache, rows):
        per = cache.n_kv * cache.head_dim
        return {n: getattr(cache, n).download(np.int8 if n.endswith("qs") else np.uint16,
                                              (rows, per if n.endswith("qs") else per // 32))
                for n in ("k_qs", "k_d", "v_qs", "v_d")}

    def bits(self, rows):
        return {n: (getattr(self, n)[rows] if n.endswith("qs") else getattr(self, n)[rows].view(np.uint16))
                for n in ("k_qs", "k_d", "v_qs", "v_d")}


def attention(host, q, sees, gate=None):
    """q [m][n_head * hd], sees [m][rows] (or [m][n_kv][rows]) truth values:
    (out [m][n_head * hd], weights summed over tokens and the group's heads
    [n_kv][rows], the outputs' bar), in 64 bits.  Rows nobody sees may hold
    anything."""
    m, hd, n_kv = q.shape[0], host.hd, host.n_kv
    n_head = q.shape[1] // hd
    group = n_head // n_kv
    K, V = host.values("k"), host.values("v")
    out = np.zeros((m, n_head, hd))
    total = np.zeros((n_kv, host.rows))
    S = vmax = 0.0
    longest = 1
    qh = q.astype(np.float64).reshape(m, n_head, hd)
    for i in range(m):
        for kv in range(n_kv):
            t = np.flatnonzero(sees[i] if sees.ndim == 2 else sees[i, kv])
            k, v = K[t, kv], V[t, kv]
            x = qh[i, kv * group:(kv + 1) * group]
            s = x @ k.T / np.sqrt(hd)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[i, kv * group:(kv + 1) * group] = p @ v
            total[kv, t] += p.sum(0)
            S = max(S, (np.abs(x) @ np.abs(k).T).max() / np.sqrt(hd))
            vmax = max(vmax, np.abs(v).max())
            longest = max(longest, t.size)
    if gate is not None:
        out *= (1 / (1 + np.exp(-gate.astype(np.float64)))).reshape(out.shape)
    rel = 2 * S * ((hd + 8) * 2.0 ** -24 + 2.0 ** -21) + 2 * (longest / 16 + 64) * 2.0 ** -24 + 2.0 ** -19
    return out.reshape(m, -1), total, vmax * rel, rel


def ancestors(parents):
    """[n][n]: node i sees j (itself and its ancestors)."""
    n = len(parents)
    a = np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            a[i] |= a[p]
    return a


def depths(parents):
    d = []
    for i, p in enumerate(parents):
        d.append(d[p] + 1 if 0 <= p < i else 0)
    return d


def random_tree(n, seed, kind="mixed"):
    r = np.random.default_rng(seed)
    if kind == "chain":
        return np.arange(n, dtype=np.int32) - 1
    if kind == "roots":
        return np.full(n, -1, np.int32)
    return (np.arange(n) - np.minimum(r.geometric(0.25, n), np.arange(n) + 1)).astype(np.int32)


class Dev:
    """Device copies of host arrays, freed together."""

    def __init__(self, eng):
        self.eng, self.bufs = eng, []

    def put(self, a):
        b = self.eng.to_device(np.ascontiguousarray(a))
        self.bufs.append(b)
        return b

    def room(self, nbytes):
        b = self.eng.alloc(nbytes)
        self.bufs.append(b)
        return b

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.eng.synchronize()
        for b in self.bufs:
            b.free()


def raises(code, call, *a, **kw):
    import pytest
    with pytest.raises(engine.BackendError) as e:
        call(*a, **kw)
    assert e.value.code == code, e.value
