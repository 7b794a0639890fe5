"""GPU: verification of drafted tokens against its definition in 64 bits.  The
random numbers are kept away from the borders where the order of a 64-bit sum
decides (2^-40 of the whole; the sums themselves are good to 2^-45), so counts and
tokens have to be equal."""
import numpy as np
import pytest

from kv_ops_util import Dev
from kv_pages_util import to_bf16
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def probabilities(x, t):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    if not t > 0:
        p = np.zeros(x.size)
        p[np.argmax(x)] = 1.0       # the lowest of the largest; id 0 where all are -inf
        return p
    if m == -np.inf:
        return np.zeros(x.size)
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, 0.0 if m == np.inf else np.exp((x - m) / np.float64(t)))
    return w / w.sum()


NONE = 0xFFFFFFFF


class Case:
    def __init__(self, counts, vocab, drafts, dtype="f32", temperature=1.0, seed=0, spread=1.0, pad=0, near=0.4, tail=0):
        r = np.random.default_rng(seed)
        self.counts, self.vocab, self.dtype, self.stride = np.asarray(counts), vocab, dtype, vocab + pad
        self.start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        n = self.n_tok = max(1, int(self.start[-1]) + tail)
        self.n_seq = len(counts)
        t = np.broadcast_to(np.float32(temperature), (self.n_seq,)).astype(np.float32)
        self.t = None if temperature is None else t
        base = r.standard_normal((n, self.stride)) * 2 * spread
        base[np.arange(n), r.integers(0, vocab, n)] += 6 * spread
        self.p = self.typed(base)
        self.q = self.typed(base + near * spread * r.standard_normal(base.shape)) if drafts else None
        self.tokens = np.zeros(n, np.uint32)
        for i in range(self.n_seq):
            for j in range(self.start[i] + 1, self.start[i + 1]):
                d = (self.q if drafts else self.p)[j - 1, :vocab]
                tt = 1.0 if self.t is None else max(float(t[i]), 0.2)
                pr = probabilities(d, tt)
                self.tokens[j] = r.choice(vocab, p=pr) if pr.sum() > 0 else 0
        self.u, self.un = r.random(n).astype(np.float32), r.random(self.n_seq).astype(np.float32)
        self.lens = r.integers(20, 90, self.n_seq).astype(np.int32)

    def typed(self, x):
        x = np.asarray(x, np.float32)
        return to_bf16(x)[1] if self.dtype == "bf16" else x

    def want(self):
        """(accepted, next, new lengths), moving the random numbers off the borders."""
        acc, nxt, V = np.zeros(self.n_seq, np.uint32), np.zeros(self.n_seq, np.uint32), self.vocab
        for i in range(self.n_seq):
            a, e = self.start[i], self.start[i + 1]
            if e <= a:
                nxt[i] = NONE
                continue
            t = 1.0 if self.t is None else self.t[i]
            row, without, q = a, None, None
            while row < e - 1:
                x = int(self.tokens[row + 1])
                p = probabilities(self.p[row, :V], t)
                px = p[x] if x < V else 0.0
                if not t > 0:
                    good = px == 1.0
                else:
                    q = None if self.q is None else probabilities(self.q[row, :V], t)
                    qx = 1.0 if q is None else q[x] if x < V else 0.0
                    if qx > 0 and abs(float(self.u[row + 1]) * qx - px) <= 2.0 ** -40 * px:
                        self.u[row + 1] *= np.float32(0.5)
                    good = np.float64(self.u[row + 1]) * qx < px
                if not good:
                    without = x
                    break
                row += 1
            acc[i] = row - a
            p = probabilities(self.p[row, :V], t)
            if not t > 0:
                nxt[i] = np.argmax(p)
                continue
            r = p
            if without is not None:
                if q is not None:
                    r = np.maximum(p - q, 0)
                else:
                    r = p.copy()
                    if without < V:
                        r[without] = 0
                if not r.sum() > 0:
                    r = p
            if not r.sum() > 0:
                continue
            c = np.cumsum(r.astype(np.longdouble))
            for _ in range(60):
                target = np.longdouble(self.un[i]) * c[-1]
                if np.abs(c - target)[r > 0].min() > 2.0 ** -40 * c[-1] or self.un[i] == 0:
                    break
                self.un[i] = np.float32(self.un[i] * np.float32(0.99))
            over = np.flatnonzero(c > target)
            nxt[i] = over[0] if over.size else np.flatnonzero(r > 0)[-1]
        return acc, nxt, self.lens - (np.maximum(self.counts, 1) - 1 - acc.astype(np.int64)).astype(np.int32)

    def run(self, eng, bare=False, in_place=False):
        with Dev(eng) as d:
            put = lambda x: None if x is None else d.put(to_bf16(x)[0] if self.dtype == "bf16" else x)  # noqa: E731
            p, q = put(self.p), put(self.q)
            tok, st, t = d.put(self.tokens), d.put(self.start), None if self.t is None else d.put(self.t)
            u, un, ln = d.put(self.u), d.put(self.un), d.put(self.lens)
            new = ln if in_place else d.room(4 * self.n_seq)
            acc, nxt = d.room(4 * self.n_seq), d.room(4 * self.n_seq)
            eng.verify_drafts(p.ptr, q.ptr if q else 0, engine.DTYPE_BF16 if self.dtype == "bf16" else engine.DTYPE_F32,
                              self.vocab, tok.ptr, 0 if bare else st.ptr, self.n_seq, self.n_tok, u.ptr, un.ptr, acc.ptr,
                              nxt.ptr, t.ptr if t else 0, ln.ptr, new.ptr, self.stride, eng.stream)
            eng.synchronize()
            return (acc.download(np.uint32, (self.n_seq,)), nxt.download(np.uint32, (self.n_seq,)),
                    new.download(np.int32, (self.n_seq,)))

    def check(self, eng, **kw):
        want = self.want()
        got = self.run(eng, **kw)
        for w, g, name in zip(want, got, ("accepted", "next", "length")):
            assert np.array_equal(w, g), (name, np.flatnonzero(w != g)[:8], w[w != g][:8], g[w != g][:8])
        return want


@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 2047, 2048, 2049, 8191, 8193, 50257])
@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_against_the_definition(eng, vocab, drafts, dtype):
    Case([1, 5, 3, 0, 9, 2], vocab, drafts, dtype, seed=vocab, pad=vocab % 3, tail=2).check(eng)


@pytest.mark.parametrize("temperature", [None, 0.0, -1.0, float("nan"), 1e-3, 0.3, 5.0, 1e30, float("inf")])
@pytest.mark.parametrize("drafts", [True, False])
def test_temperatures(eng, temperature, drafts):
    Case([4, 1, 6, 2], 3001, drafts, temperature=temperature, seed=4).check(eng)


def test_many_sequences_at_temperatures_of_their_own(eng):
    r = np.random.default_rng(3)
    c = Case(r.integers(0, 7, 300), 600, True, seed=3, near=0.7)
    c.t = r.choice(np.array([0, 0.5, 1, 2], np.float32), 300)
    acc, _, _ = c.check(eng, in_place=True)
    assert acc.max() >= 4 and (acc == 0).any()


def test_a_sampled_token_each(eng):
    """No drafts: plain sampling, without ranges."""
    Case([1] * 130, 5000, False, seed=8).check(eng, bare=True)


@pytest.mark.parametrize("drafts", [True, False])
def test_a_long_draft(eng, drafts):
    c = Case([40, 33], 4000, drafts, seed=2, near=0.02, spread=3.0)
    c.u[:] *= np.float32(0.3)
    c.check(eng)


def test_ids_outside_the_vocabulary_are_refused(eng):
    for drafts in (True, False):
        c = Case([3, 3], 100, drafts, seed=1)
        c.tokens[1], c.tokens[5] = 100, NONE
        acc, _, _ = c.check(eng)
        assert acc[0] == 0


def test_masked_and_broken_logits(eng):
    """-inf and NaN have no probability, infinite logits have all of it; rows
    with nothing answer 0."""
    V = 2500
    c = Case([2, 2, 2, 2, 1, 1, 2], V, True, seed=6)
    c.p[c.start[0], 5:] = -np.inf
    c.p[c.start[1], ::2] = np.nan
    c.p[c.start[2], [7, 2100]] = np.inf
    c.p[c.start[3], :] = -np.inf
    c.p[c.start[4], :] = np.nan
    c.p[c.start[5], 2:] = -3e38
    c.q[c.start[6], :] = -np.inf
    _, nxt, _ = c.check(eng)
    assert nxt[3] == 0 and nxt[4] == 0
    c.t = np.zeros(7, np.float32)
    c.check(eng)


def test_a_draft_model_equal_to_the_model_is_always_accepted(eng):
    c = Case([8, 3], 7000, True, seed=6)
    c.q = c.p.copy()
    c.u[:] = np.float32(1 - 2.0 ** -24)
    acc, _, _ = c.check(eng)
    assert list(acc) == [7, 2]


def test_random_numbers_at_their_ends(eng):
    for u in (0.0, 1 - 2.0 ** -24):
        for drafts in (True, False):
            c = Case([1, 4, 3], 1000, drafts, seed=5)
            c.u[:], c.un[:] = np.float32(u), np.float32(u)
            c.check(eng)


def test_what_is_emitted_is_distributed_as_the_model(eng):
    """First emitted tokens of 1,000 sequences with one draft each from the same
    two rows: counts within five standard deviations of 1000 p."""
    V, n = 12, 1000
    r = np.random.default_rng(0)
    p, q = r.standard_normal(V).astype(np.float32) * 1.5, r.standard_normal(V).astype(np.float32) * 1.5
    c = Case([2] * n, V, True, seed=1)
    c.p[:], c.q[:] = p, q
    c.tokens[1::2] = r.choice(V, n, p=probabilities(q, 1.0))
    acc, nxt, _ = c.check(eng)
    first = np.where(acc == 1, c.tokens[1::2], nxt)
    want = n * probabilities(p, 1.0)
    assert np.all(np.abs(np.bincount(first, minlength=V) - want) <= 5 * np.sqrt(want * (1 - want / n)) + 1)


def test_replayed(eng):
    """A captured verification with other logits and numbers at each replay."""
    c = Case([3, 5, 1], 3000, True, seed=11)
    with Dev(eng) as d:
        p, q, tok, st, t = d.put(c.p), d.put(c.q), d.put(c.tokens), d.put(c.start), d.put(c.t)
        u, un, ln = d.put(c.u), d.put(c.un), d.put(c.lens)
        acc, nxt, new = (d.room(12) for _ in range(3))

        def call(s):
            eng.verify_drafts(p.ptr, q.ptr, engine.DTYPE_F32, c.vocab, tok.ptr, st.ptr, 3, c.n_tok, u.ptr, un.ptr, acc.ptr,
                              nxt.ptr, t.ptr, ln.ptr, new.ptr, stream=s)
        call(eng.stream)
        eng.synchronize()
        graph = eng.capture(call)
        for seed in range(5):
            n = Case([[3, 5, 1], [1, 1, 7], [4, 0, 5], [9, 0, 0], [2, 2, 2]][seed], 3000, True, seed=20 + seed, tail=[0, 0, 0, 0, 3][seed])
            want = n.want()
            for buf, a in ((p, n.p), (q, n.q), (tok, n.tokens), (st, n.start), (u, n.u), (un, n.un), (ln, n.lens)):
                buf.upload(a)
            graph.launch()
            eng.synchronize()
            for buf, w in zip((acc, nxt, new), want):
                assert np.array_equal(buf.download(w.dtype, (3,)), w), seed
        graph.free()
