"""GPU parity of attention that keeps its weights
(``vxt_hip_attn_weigh_q8_dev``) and of eviction by them
(``vxt_hip_kv_q8_evict_dev``), against the formulas in 64 bits (kv_ops_util,
which derives the bars) and, for the rows kept, exactly."""
import numpy as np
import pytest

from kv_ops_util import Dev, HostCache, attention, raises
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def causal(pos, m, rows):
    return np.arange(rows)[None] <= pos + np.arange(m)[:, None]


def run_weigh(eng, host, q, pos, tok_pos, weight, position, gate=None):
    """(out, weight plane, position plane) after one call on planes like the given ones."""
    m, width = q.shape
    cache = host.upload(eng)
    w = eng.kv_weights(weight.shape[1], host.n_kv)
    w.weight.upload(weight)
    w.position.upload(position)
    with Dev(eng) as d:
        out = d.room(q.nbytes)
        g = d.put(gate).ptr if gate is not None else 0
        cache.attend_weigh(w, d.put(q).ptr, width // host.hd, m, pos, tok_pos, out.ptr, g, eng.stream)
        eng.synchronize()
        got = (out.download(np.float32, q.shape), w.weight.download(np.float32, weight.shape),
               w.position.download(np.uint32, position.shape))
    cache.free()
    w.free()
    return got


WEIGH = [
    # m, pos, n_head, n_kv, hd, gated
    (1, 0, 4, 4, 32, False),
    (1, 31, 8, 1, 64, True),
    (1, 32, 6, 2, 128, False),
    (1, 1000, 16, 4, 128, True),
    (1, 333, 4, 2, 256, True),
    (1, 9000, 8, 2, 64, False),
    (1, 5000, 4, 2, 32, True),
    (1, 5000, 2, 1, 256, False),
    (2, 0, 2, 1, 64, False),
    (3, 127, 8, 1, 128, True),
    (17, 40, 10, 2, 32, False),
    (65, 0, 4, 4, 128, False),
    (130, 61, 7, 1, 64, True),
    (40, 700, 4, 2, 256, False),
    (300, 0, 16, 4, 128, True),
    (500, 900, 4, 1, 64, False),
    (700, 1500, 6, 2, 128, True),      # a group of three, many segments and pieces
    (1300, 0, 5, 1, 32, False),
]


@pytest.mark.parametrize("case", WEIGH)
def test_weigh_parity(eng, case):
    m, pos, n_head, n_kv, hd, gated = case
    r = np.random.default_rng(m + pos)
    rows, plane = pos + m, pos + m + 9
    host = HostCache(rows, n_kv, hd, seed=m * 3 + pos)
    q = r.standard_normal((m, n_head * hd)).astype(np.float32)
    gate = r.standard_normal(q.shape).astype(np.float32) if gated else None
    weight = r.exponential(1.0, (n_kv, plane)).astype(np.float32)
    weight[:, pos:] = np.nan                               # the call's rows are set, the rest left
    position = r.integers(0, 1 << 31, (n_kv, plane)).astype(np.uint32)
    out, w, p = run_weigh(eng, host, q, pos, 5000, weight, position, gate)
    ref, total, tol, rel = attention(host, q, causal(pos, m, rows), gate)
    assert np.abs(out - ref).max() <= tol
    want = total.copy()
    want[:, :pos] += weight[:, :pos]
    bar = rel * total + 2.0 ** -22 * total.max() + 2.0 ** -23 * np.abs(want)
    assert (np.abs(w[:, :rows] - want) <= bar).all()
    assert np.isnan(w[:, rows:]).all()                     # rows behind: as they were
    assert np.array_equal(p[:, :pos], position[:, :pos]) and np.array_equal(p[:, rows:], position[:, rows:])
    assert np.array_equal(p[:, pos:rows], np.tile(5000 + np.arange(m, dtype=np.uint32), (n_kv, 1)))
    again = run_weigh(eng, host, q, pos, 5000, weight, position, gate)
    assert np.array_equal(again[0], out) and np.array_equal(again[1][:, :rows], w[:, :rows])


def test_weights_of_a_prompt_and_of_its_tokens_agree(eng):
    """One batch, or the same tokens one call each."""
    m, n_head, n_kv, hd = 50, 8, 2, 64
    host = HostCache(m, n_kv, hd, seed=2)
    q = np.random.default_rng(2).standard_normal((m, n_head * hd)).astype(np.float32)
    zero = np.zeros((n_kv, m), np.float32), np.zeros((n_kv, m), np.uint32)
    out, w, p = run_weigh(eng, host, q, 0, 0, *zero)
    w1, p1 = zero
    outs = []
    for i in range(m):
        o, w1, p1 = run_weigh(eng, host, q[i:i + 1], i, i, w1, p1)
        outs.append(o[0])
    ref, total, tol, rel = attention(host, q, causal(0, m, m))
    assert np.abs(out - np.stack(outs)).max() <= 2 * tol
    assert (np.abs(w - w1) <= 2 * (rel * total + 2.0 ** -22 * total.max() + m * 2.0 ** -24 * total)).all()
    assert np.array_equal(p, p1)
    assert abs(w.sum() - m * n_head) <= 1e-3 * m * n_head   # every token's heads give 1 each


def evict_plan(weight, position, seq, keep, n_tokens, n_recent, n_first):
    """Source row of every kept row, one kv head, by the rule itself."""
    w = weight[:seq].astype(np.float64)
    rank = np.where(np.isnan(w), -np.inf, w)
    safe = (position[:seq] < n_first) | (position[:seq].astype(np.int64) >= n_tokens - n_recent)
    order = sorted(range(seq), key=lambda i: (not safe[i], np.isnan(w[i]) and not safe[i], -rank[i] if not safe[i] else 0, i))
    kept = np.zeros(seq, bool)
    kept[order[:keep]] = True
    src = np.arange(min(keep, seq))
    src[~kept[:keep]] = np.flatnonzero(kept[keep:]) + keep
    return src


def check_evict(eng, host, weight, position, seq, keep, n_tokens, n_recent, n_first, other):
    n_kv, hd = host.n_kv, host.hd
    cache = host.upload(eng)
    w = eng.kv_weights(weight.shape[1], n_kv)
    w.weight.upload(weight)
    w.position.upload(position)
    kept = min(keep, seq)
    to = eng.kv_q8_cache(kept + 2, n_kv, hd) if other else None
    tw = eng.kv_weights(kept + 3, n_kv) if other else None
    if other:
        for b in (to.k_qs, to.v_qs, to.k_d, to.v_d, tw.weight, tw.position):
            b.upload(np.full(b.nbytes, 7, np.uint8))
    cache.evict(w, seq, keep, n_tokens, n_recent, n_first, to, tw, eng.stream)
    eng.synchronize()
    c, tp = (to, tw) if other else (cache, w)
    got = HostCache.download(c, c.max_seq)
    gw = tp.weight.download(np.uint32, (n_kv, tp.max_seq))
    gp = tp.position.download(np.uint32, (n_kv, tp.max_seq))
    bits = host.bits(slice(None))
    for k in range(n_kv):
        src = evict_plan(weight[k], position[k], seq, keep, n_tokens, n_recent, n_first)
        for x, wide in (("k_qs", hd), ("v_qs", hd), ("k_d", hd // 32), ("v_d", hd // 32)):
            cols = slice(k * wide, (k + 1) * wide)
            assert np.array_equal(got[x][:kept, cols], bits[x][src, cols]), (x, k)
            rest = got[x][kept:, cols]
            assert (rest.view(np.uint8) == 7).all() if other else np.array_equal(rest, bits[x][kept:, cols])
        assert np.array_equal(gw[k, :kept], weight[k].view(np.uint32)[src])
        assert np.array_equal(gp[k, :kept], position[k][src])
        if other:
            assert (gw[k, kept:] == 0x07070707).all() and (gp[k, kept:] == 0x07070707).all()
        else:
            assert np.array_equal(gw[k, kept:], weight[k].view(np.uint32)[kept:])
            assert np.array_equal(gp[k, kept:], position[k][kept:])
    for b in (cache, w, to, tw):
        if b is not None:
            b.free()


EVICT = [
    # seq, keep, n_recent, n_first, n_kv, hd
    (1, 1, 0, 0, 1, 32),
    (2, 1, 1, 0, 2, 64),
    (65, 64, 8, 2, 4, 128),
    (100, 7, 3, 1, 3, 64),
    (1000, 999, 0, 0, 2, 256),
    (1025, 1, 0, 0, 1, 128),
    (2112, 2048, 256, 4, 4, 128),
    (5000, 1250, 200, 16, 2, 64),
    (8191, 8000, 100, 0, 1, 32),
    (16384, 100, 0, 0, 1, 32),     # the most rows that one workgroup selects among
    (16385, 16384, 30, 4, 2, 64),
    (20000, 1, 0, 0, 3, 32),
    (20001, 6000, 5990, 10, 1, 128),   # nothing but the protected stays
    (70001, 16000, 1000, 16, 1, 32),
    (540001, 530000, 1000, 16, 1, 32),   # stretches of more than one batch
    (10, 64, 8, 2, 2, 64),        # fewer rows than are kept
    (64, 64, 8, 2, 2, 64),
]


@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("case", EVICT)
def test_evict_parity(eng, case, other):
    seq, keep, n_recent, n_first, n_kv, hd = case
    r = np.random.default_rng(seq + keep)
    plane = seq + 5
    host = HostCache(plane, n_kv, hd, seed=seq)
    weight = np.exp(r.standard_normal((n_kv, plane)) * 2).astype(np.float32)
    position = np.stack([np.sort(r.choice(4 * plane, plane, replace=False)) for _ in range(n_kv)]).astype(np.uint32)
    check_evict(eng, host, weight, position, seq, keep, 4 * plane, n_recent, n_first, other)


@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("size", [(700, 300), (17001, 7000)])
@pytest.mark.parametrize("kind", ["equal", "zeros", "two values", "nan", "inf", "negative", "close", "all protected"])
def test_evict_orders(eng, kind, size, other):
    """Ties go to the lower row, NaN last, -0 with 0, neighbours in f32 apart."""
    (seq, keep), n_kv, hd = size, 2, 32
    r = np.random.default_rng(3)
    host = HostCache(seq, n_kv, hd, seed=3)
    w = {"equal": np.full((n_kv, seq), 3.25), "zeros": r.choice([0.0, -0.0], (n_kv, seq)),
         "two values": r.choice([1.0, 2.0], (n_kv, seq)), "nan": r.standard_normal((n_kv, seq)),
         "inf": r.standard_normal((n_kv, seq)), "negative": -r.exponential(1, (n_kv, seq)),
         "close": np.float32(1) + r.integers(0, 40, (n_kv, seq)) * np.float32(2.0 ** -23),
         "all protected": r.standard_normal((n_kv, seq))}[kind].astype(np.float32)
    if kind == "nan":
        w[r.random(w.shape) < 0.6] = np.nan
    if kind == "inf":
        w[r.random(w.shape) < 0.3] = np.inf
        w[r.random(w.shape) < 0.3] = -np.inf
    position = np.tile(np.arange(seq, dtype=np.uint32), (n_kv, 1))
    if kind == "all protected":        # positions a caller never set: as many rows stay as asked for
        position[:] = 0
    check_evict(eng, host, w, position, seq, keep, seq, 20, 5, other)


def test_decode_with_a_budget(eng):
    """Tokens one after the other, each weighed, the cache cut back when it is
    full: outputs, weights and kept rows follow a 64-bit model of the same."""
    n_head, n_kv, hd, full, keep, steps = 4, 2, 64, 40, 24, 60
    r = np.random.default_rng(7)
    src = HostCache(steps, n_kv, hd, seed=7)
    cache, w = eng.kv_q8_cache(full, n_kv, hd), eng.kv_weights(full, n_kv)
    model = HostCache(full, n_kv, hd, seed=7)
    mw, mp = np.zeros((n_kv, full)), np.zeros((n_kv, full), np.uint32)
    rows = 0
    with Dev(eng) as d:
        out = d.room(4 * n_head * hd)
        K, V = d.put(src.values("k").reshape(steps, -1).astype(np.float32)), d.put(src.values("v").reshape(steps, -1).astype(np.float32))
        for t in range(steps):
            if rows == full:
                cache.evict(w, rows, keep, t, 6, 2, stream=eng.stream)
                eng.synchronize()
                gp = w.position.download(np.uint32, (n_kv, full))
                gw = w.weight.download(np.float32, (n_kv, full))
                # by the device's own weights: near ties may fall either way
                last_w, last_p = before
                for k in range(n_kv):
                    s = evict_plan(last_w[k], last_p[k], rows, keep, t, 6, 2)
                    assert np.array_equal(gp[k, :keep], last_p[k][s])
                    mw[k, :keep], mp[k, :keep] = mw[k][s], mp[k][s]
                rows = keep
            q = r.standard_normal((1, n_head * hd)).astype(np.float32)
            cache.append(K.ptr + 4 * t * n_kv * hd, V.ptr + 4 * t * n_kv * hd, rows, eng.stream)
            cache.attend_weigh(w, d.put(q).ptr, n_head, 1, rows, t, out.ptr, 0, eng.stream)
            eng.synchronize()
            for x in ("k_qs", "k_d", "v_qs", "v_d"):
                h = HostCache.download(cache, full)[x]
                setattr(model, x, h if x.endswith("qs") else h.view(np.float16))
            mp[:, rows] = t
            mw[:, rows] = 0
            ref, total, tol, rel = attention(model, q, (np.arange(full) <= rows)[None])
            mw[:, :rows + 1] += total[:, :rows + 1]
            before = w.weight.download(np.float32, (n_kv, full)), w.position.download(np.uint32, (n_kv, full))
            assert np.abs(out.download(np.float32, q.shape) - ref).max() <= tol
            assert np.array_equal(before[1][:, :rows + 1], mp[:, :rows + 1])
            assert np.allclose(before[0][:, :rows + 1], mw[:, :rows + 1], rtol=steps * rel, atol=steps * 2.0 ** -22)
            rows += 1
    cache.free()
    w.free()


def test_weigh_nonfinite_rows_behind_are_not_read(eng):
    for m in (1, 9):
        pos, n_kv, hd = 40, 2, 64
        host = HostCache(pos + m + 60, n_kv, hd, seed=1)
        host.k_d[pos + m:] = np.nan
        host.v_d[pos + m:] = np.inf
        q = np.random.default_rng(1).standard_normal((m, 4 * hd)).astype(np.float32)
        zero = np.zeros((n_kv, host.rows), np.float32), np.zeros((n_kv, host.rows), np.uint32)
        out, w, _ = run_weigh(eng, host, q, pos, 0, *zero)
        ref, total, tol, rel = attention(host, q, causal(pos, m, host.rows))
        assert np.abs(out - ref).max() <= tol
        assert (np.abs(w - total) <= rel * total + 2.0 ** -22 * total.max()).all()


def test_a_later_row_that_is_not_finite_spares_earlier_tokens(eng):
    """Causal batch: token m's V row is Inf in one block: tokens before it are
    as without it, it and later ones NaN in that block's dims."""
    m, pos, n_kv, hd = 12, 70, 1, 64
    q = np.random.default_rng(1).standard_normal((m, 2 * hd)).astype(np.float32)
    host, bad = HostCache(pos + m, n_kv, hd, seed=1), HostCache(pos + m, n_kv, hd, seed=1)
    bad.v_d[pos + 5, 1] = np.inf
    bad.v_qs[pos + 5, 32:64] = 0
    zero = np.zeros((n_kv, pos + m), np.float32), np.zeros((n_kv, pos + m), np.uint32)
    a, wa, _ = run_weigh(eng, host, q, pos, 0, *zero)
    b, wb, _ = run_weigh(eng, bad, q, pos, 0, *zero)
    a, b = a.reshape(m, 2, hd), b.reshape(m, 2, hd)
    assert np.array_equal(a[:5], b[:5]) and np.array_equal(a[5:, :, :32], b[5:, :, :32])
    assert np.isnan(b[5:, :, 32:]).all() and np.array_equal(wa, wb)


def test_spare_rows_of_a_tile_see_what_their_token_sees(eng):
    """Twenty tokens of a group of three leave rows of a tile spare.  Only the
    last token sees the last row, whose scale is infinite, with a score of
    -inf: its weight is 0, whatever another token's queries would make of it."""
    m, n_head, n_kv, hd = 20, 3, 1, 64
    host = HostCache(m, n_kv, hd, seed=6)
    host.k_qs[-1] = 1
    q = np.abs(np.random.default_rng(6).standard_normal((m, n_head * hd))).astype(np.float32)
    q[-1] *= -1
    ref, total, tol, rel = attention(host, q, np.where(np.arange(m)[None] == m - 1, False, causal(0, m, m)))
    host.k_d[-1] = np.inf
    out, w, _ = run_weigh(eng, host, q, 0, 0, np.zeros((n_kv, m), np.float32), np.zeros((n_kv, m), np.uint32))
    assert np.abs(out - ref).max() <= tol
    assert w[0, -1] == 0 and (np.abs(w - total) <= rel * total + 2.0 ** -22 * total.max()).all()


@pytest.mark.parametrize("m", [1, 21, 150])
def test_tensors_at_any_float(eng, m):
    """Queries, gate and output four bytes past a 16-byte boundary, and a stream
    that is not the context's."""
    pos, n_head, n_kv, hd = 300, 8, 2, 128
    host = HostCache(pos + m, n_kv, hd, seed=m)
    r = np.random.default_rng(m)
    q, gate = (r.standard_normal((m, n_head * hd)).astype(np.float32) for _ in range(2))
    cache, w = host.upload(eng), eng.kv_weights(pos + m, n_kv)
    parents = np.arange(m, dtype=np.int32) - 1
    one = np.zeros(1, np.float32)
    other = engine.HipEngine()
    s = other.stream
    with Dev(eng) as d:
        w.weight.upload(np.zeros((n_kv, pos + m), np.float32))
        w.position.upload(np.zeros((n_kv, pos + m), np.uint32))
        Q, G = (d.put(np.concatenate([one, x.ravel()])) for x in (q, gate))
        P = d.put(parents)
        outs = [d.room(q.nbytes + 8) for _ in range(3)]
        means = eng.kv_block_means((pos + m) // 32, 32, n_kv, hd)
        for b in outs:
            b.upload(np.full(b.nbytes, 7, np.uint8))
        eng.synchronize()
        cache.attend_weigh(w, Q.ptr + 4, n_head, m, pos, 0, outs[0].ptr + 4, G.ptr + 4, s)
        cache.attend_tree(Q.ptr + 4, n_head, P.ptr, m, pos, outs[1].ptr + 4, G.ptr + 4, s)
        cache.block_means(means, 0, pos + m, s)
        cache.attend_blocks(means, Q.ptr + 4, n_head, m, pos, 64, 1, 1, outs[2].ptr + 4, G.ptr + 4, 0, s)
        other.synchronize()
        ref, _, tol, _ = attention(host, q, causal(pos, m, pos + m), gate)
        for b in outs:
            got = b.download(np.float32, (q.size + 2,))
            assert np.abs(got[1:-1].reshape(q.shape) - ref).max() <= tol
            assert (got[[0, -1]].view(np.uint32) == 0x07070707).all()   # nothing beside it
    other.close()
    for b in (cache, w, means):
        b.free()


def test_refusals(eng):
    A, S, U = engine.VXT_E_ARG, engine.VXT_E_SHAPE, engine.VXT_E_UNSUPPORTED
    cache, w = eng.kv_q8_cache(100, 2, 64), eng.kv_weights(100, 2)
    short, heads = eng.kv_weights(50, 2), eng.kv_weights(100, 1)
    to, tw, other = eng.kv_q8_cache(30, 2, 64), eng.kv_weights(30, 2), eng.kv_q8_cache(30, 2, 32)
    with Dev(eng) as d:
        b = d.room(1 << 20).ptr
        g = cache.attend_weigh
        raises(A, g, w, 0, 4, 1, 0, 0, b)
        raises(A, g, w, b, 4, 1, 0, 0, 0)
        raises(S, g, w, b, 5, 1, 0, 0, b)
        raises(U, g, w, b, 18, 1, 0, 0, b)
        raises(S, g, w, b, 4, 0, 0, 0, b)
        raises(S, g, w, b, 4, 2, 99, 0, b)
        raises(S, g, w, b, 4, 1, 100, 0, b)
        raises(S, g, w, b, 4, 2, 0, 0xffffffff, b)
        raises(S, g, short, b, 4, 1, 50, 0, b)
        raises(S, g, heads, b, 4, 1, 0, 0, b)
        raises(A, g, engine.KvWeights.over(eng, 0, b, 100, 2), b, 4, 1, 0, 0, b)
        raises(A, g, engine.KvWeights.over(eng, b + 2, b, 100, 2), b, 4, 1, 0, 0, b)
        raises(A, g, engine.KvWeights.over(eng, b, b + 1, 100, 2), b, 4, 1, 0, 0, b)
    e = cache.evict
    raises(S, e, w, 0, 10, 100)
    raises(S, e, w, 101, 10, 100)
    raises(S, e, w, 100, 0, 100)
    raises(S, e, w, 100, 10, 100, 9, 2)
    raises(S, e, w, 100, 10, 100, 0xffffffff, 2)
    raises(S, e, short, 60, 10, 100)
    raises(A, e, w, 100, 10, 100, 0, 0, to, None)
    raises(A, e, w, 100, 10, 100, 0, 0, None, tw)
    raises(S, e, w, 100, 31, 100, 0, 0, to, tw)
    raises(S, e, w, 100, 10, 100, 0, 0, other, tw)
    raises(A, e, w, 100, 10, 100, 0, 0, cache, tw)
    raises(A, e, w, 100, 10, 100, 0, 0, to, w)
    for x in (cache, w, short, heads, to, tw, other):
        x.free()


def test_captured_and_replayed(eng):
    """Weigh and evict into another cache in one graph, replayed with new
    queries and weights, eager calls of other sizes in between."""
    n_kv, hd, n_head, pos, keep = 2, 64, 8, 400, 100
    host = HostCache(pos + 1, n_kv, hd, seed=5)
    cache, to = host.upload(eng), eng.kv_q8_cache(keep, n_kv, hd)
    w, tw = eng.kv_weights(pos + 1, n_kv), eng.kv_weights(keep, n_kv)
    r = np.random.default_rng(5)
    with Dev(eng) as d:
        q, out = d.room(4 * n_head * hd), d.room(4 * n_head * hd)

        def call(s):
            cache.attend_weigh(w, q.ptr, n_head, 1, pos, pos, out.ptr, 0, s)
            cache.evict(w, pos + 1, keep, pos + 1, 10, 2, to, tw, s)

        def load(k):
            x = np.random.default_rng(k)
            q.upload(x.standard_normal(n_head * hd).astype(np.float32))
            w.weight.upload(x.exponential(1, (n_kv, pos + 1)).astype(np.float32))
            w.position.upload(np.tile(np.arange(pos + 1, dtype=np.uint32), (n_kv, 1)))

        def state():
            eng.synchronize()
            return [out.download(np.float32, (n_head * hd,)), w.weight.download(np.float32, (n_kv, pos + 1)),
                    tw.weight.download(np.float32, (n_kv, keep)), tw.position.download(np.uint32, (n_kv, keep)),
                    *HostCache.download(to, keep).values()]

        load(0)
        call(eng.stream)
        eng.synchronize()
        graph = eng.capture(call)
        for k in range(4):
            load(k)
            graph.launch(1)
            a = state()
            load(k)
            call(eng.stream)
            b = state()
            assert all(np.array_equal(x, y) for x, y in zip(a, b)), k
            load(k + 10)
            cache.attend_weigh(w, q.ptr, n_head, 1, 30 + 50 * k, 0, out.ptr, 0, eng.stream)
            eng.synchronize()
        graph.free()
    for x in (cache, to, w, tw):
        x.free()
    assert r is not None


def test_a_large_selection_replayed(eng):
    """A selection over several workgroups, whose counts each replay starts anew."""
    n_kv, hd, seq, keep = 2, 32, 17001, 600
    host = HostCache(seq, n_kv, hd, seed=8)
    cache, to = host.upload(eng), eng.kv_q8_cache(keep, n_kv, hd)
    w, tw = eng.kv_weights(seq, n_kv), eng.kv_weights(keep, n_kv)
    pos = np.tile(np.arange(seq, dtype=np.uint32), (n_kv, 1))
    w.position.upload(pos)
    w.weight.upload(np.ones((n_kv, seq), np.float32))

    def call(s):
        cache.evict(w, seq, keep, seq, 50, 4, to, tw, s)

    call(eng.stream)
    eng.synchronize()
    graph = eng.capture(call)
    for k in range(4):
        weight = np.random.default_rng(k).choice(np.float32([0.5, 1, 2, 3]), (n_kv, seq))
        w.weight.upload(weight)
        graph.launch(1)
        eng.synchronize()
        got = tw.position.download(np.uint32, (n_kv, keep))
        for kv in range(n_kv):
            assert np.array_equal(got[kv], evict_plan(weight[kv], pos[kv], seq, keep, seq, 50, 4)), k
        cache.evict(w, 700 + k, 20, seq, 5, 2, to, tw, eng.stream)   # an eager call between, in the same workspace
        eng.synchronize()
    graph.free()
    for x in (cache, to, w, tw):
        x.free()


def test_rows_behind_four_gigabytes(eng):
    """Planes of more than 2^32 bytes: the last 64 rows hold values, the rows
    ahead of them scales of zero (scores and values of 0, codes whatever was
    there), which the reference counts without listing them."""
    n_kv, hd, n_head, rows, tail = 16, 256, 32, 8224 * 128, 64
    per, first = n_kv * hd, rows - tail
    assert first * per > 1 << 32
    host = HostCache(tail, n_kv, hd, seed=9)
    K, V = host.values("k"), host.values("v")
    r = np.random.default_rng(9)
    cache, w = eng.kv_q8_cache(rows, n_kv, hd), eng.kv_weights(rows, n_kv)
    means = eng.kv_block_means(rows // 128, 128, n_kv, hd)
    memcpy = engine.load_library().vxt_hip_memcpy

    def copy(dst, src, nbytes, kind):
        err = engine._errbuf()
        engine._check(memcpy(eng.ctx, dst, src, nbytes, kind, err, len(err)), err)

    zero = np.zeros(rows * per // 32, np.uint16)
    for plane, b, per_row in ((cache.k_d, host.k_d, per // 16), (cache.v_d, host.v_d, per // 16),
                              (cache.k_qs, host.k_qs, per), (cache.v_qs, host.v_qs, per)):
        if per_row != per:
            plane.upload(zero)
        copy(plane.ptr + first * per_row, np.ascontiguousarray(b).ctypes.data, b.nbytes, 0)
    means.d.upload(zero[:rows // 128 * per // 32])
    w.weight.upload(np.ones((n_kv, rows), np.float32))
    w.position.upload(np.tile(np.arange(rows, dtype=np.uint32), (n_kv, 1)))

    def want(q, sees, zeros):
        """(out, weights of the tail's rows, bar) with `zeros` rows of scores and values of 0."""
        m = q.shape[0]
        out, total, S = np.zeros((m, n_head, hd)), np.zeros((n_kv, tail)), 0.0
        for i in range(m):
            t = np.flatnonzero(sees[i])
            for h in range(n_head):
                k, x = h // (n_head // n_kv), q[i].astype(np.float64).reshape(n_head, hd)[h]
                s = K[t, k] @ x / np.sqrt(hd)
                top = max(s.max(), 0.0)
                e = np.exp(s - top)
                p = e / (e.sum() + zeros * np.exp(-top))
                out[i, h] = p @ V[t, k]
                total[k, t] += p
                S = max(S, (np.abs(K[t, k]) @ np.abs(x)).max() / np.sqrt(hd))
        rel = 2 * S * ((hd + 8) * 2.0 ** -24 + 2.0 ** -21) + 2 * (rows / 16 + 64) * 2.0 ** -24 + 2.0 ** -19
        return out.reshape(m, -1), total, np.abs(V).max() * rel, rel

    def query(m):
        return (8 * r.standard_normal((m, n_head * hd))).astype(np.float32)

    with Dev(eng) as d:
        q = query(3)
        out, sees = d.room(q.nbytes), np.zeros((3, tail), bool)
        sees[:, :tail - 3] = True
        sees[:, tail - 3:] = [[1, 0, 0], [1, 1, 0], [1, 0, 1]]
        cache.attend_tree(d.put(q).ptr, n_head, d.put(np.array([-1, 0, 0], np.int32)).ptr, 3, rows - 3, out.ptr, 0, eng.stream)
        eng.synchronize()
        ref, _, tol, _ = want(q, sees, first)
        assert np.abs(out.download(np.float32, q.shape) - ref).max() <= tol < np.abs(ref).max() / 10
        for m in (1, 2):
            q = query(m)
            cache.attend_weigh(w, d.put(q).ptr, n_head, m, rows - m, rows - m, out.ptr, 0, eng.stream)
            eng.synchronize()
            ref, total, tol, rel = want(q, causal(tail - m, m, tail), first)
            assert np.abs(out.download(np.float32, q.shape) - ref).max() <= tol
            got = w.weight.download(np.float32, (n_kv, rows))[:, -tail:]   # the call's own rows
            assert (np.abs(got[:, -m:] - total[:, -m:]) <= rel * total[:, -m:] + 2.0 ** -22 * total.max()).all()
        q = query(1)
        cache.attend_blocks(means, d.put(q).ptr, n_head, 1, rows - 1, 4, 1, 2, out.ptr, 0, 0, eng.stream)
        eng.synchronize()
        ref, _, tol, _ = want(q, np.ones((1, tail), bool), 4 * 128 - tail)
        assert np.abs(out.download(np.float32, q.shape) - ref).max() <= tol
        # rows 5, 6, 7 go, the last three take their places
        weight = np.ones((n_kv, rows), np.float32)
        weight[:, 5:8] = 0
        w.weight.upload(weight)
        cache.evict(w, rows, rows - 3, rows, 0, 0, stream=eng.stream)
        eng.synchronize()
        got = HostCache.download(cache, 8)
        for x, b in host.bits(slice(tail - 3, None)).items():
            assert np.array_equal(got[x][5:8], b), x
        assert np.array_equal(w.position.download(np.uint32, (n_kv, rows))[:, 5:8], np.tile(np.arange(rows - 3, rows), (n_kv, 1)))
        # of the last four rows the second and fourth move up
        cache.keep_path(d.put(np.array([2, 1, 3, 0, 0], np.uint32)).ptr, 4, rows - 4, eng.stream)
        eng.synchronize()
        last = np.empty((4, per), np.int8)
        copy(last.ctypes.data, cache.v_qs.ptr + (rows - 4) * per, last.nbytes, 1)
        assert np.array_equal(last, host.v_qs[[-3, -1, -2, -1]])
    for b in (cache, w, means):
        b.free()
