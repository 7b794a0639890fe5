"""GPU parity of the attention of a drafted tree over the Q8_0 KV cache
(``vxt_hip_attn_tree_q8_dev``, ``vxt_hip_attn_tree_step_q8_dev``) and of keeping
an accepted path (``vxt_hip_kv_q8_keep_path_dev``), against the formulas in
64 bits (kv_ops_util, which derives the bar)."""
import numpy as np
import pytest

from kv_ops_util import Dev, HostCache, ancestors, attention, depths, raises, random_tree
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def sees_of(parents, pos, rows):
    n = len(parents)
    s = np.zeros((n, rows), bool)
    s[:, :pos] = True
    s[:, pos:pos + n] = ancestors(parents)
    return s


def run_tree(eng, host, q, parents, pos, gate=None, cache=None, stream=None):
    n, width = q.shape
    own = cache is None
    cache = cache or host.upload(eng)
    with Dev(eng) as d:
        out = d.room(q.nbytes)
        g = d.put(gate).ptr if gate is not None else 0
        cache.attend_tree(d.put(q).ptr, width // host.hd, d.put(np.asarray(parents, np.int32)).ptr, n, pos, out.ptr,
                          g, eng.stream if stream is None else stream)
        eng.synchronize()
        got = out.download(np.float32, q.shape)
    if own:
        cache.free()
    return got


CASES = [
    # n, pos, n_head, n_kv, hd, kind, gated
    (1, 0, 4, 4, 32, "mixed", False),
    (1, 100, 4, 4, 32, "mixed", False),        # the smallest buffers, more than one tile
    (1, 500, 16, 4, 128, "mixed", True),
    (3, 31, 2, 1, 64, "roots", False),
    (5, 150, 8, 2, 64, "mixed", False),
    (8, 64, 8, 1, 128, "chain", True),
    (13, 0, 6, 2, 64, "mixed", True),          # a group of three, nothing committed
    (26, 1000, 16, 4, 128, "mixed", True),
    (31, 97, 16, 2, 32, "mixed", False),
    (33, 1, 4, 2, 256, "mixed", True),
    (64, 700, 10, 2, 128, "mixed", False),     # a group of five
    (100, 333, 4, 4, 128, "chain", False),
    (129, 40, 14, 2, 64, "mixed", False),      # a group of seven
    (256, 500, 8, 2, 128, "mixed", True),
    (256, 0, 1, 1, 128, "chain", False),
    (7, 33, 2, 2, 256, "mixed", False),
    (9, 210, 3, 1, 32, "mixed", True),
    (4, 2000, 4, 2, 32, "mixed", True),        # many partial sums to a row
    (4, 2000, 2, 2, 256, "mixed", False),
    (255, 5000, 8, 8, 64, "roots", False),
]


@pytest.mark.parametrize("case", CASES)
def test_tree_parity(eng, case):
    n, pos, n_head, n_kv, hd, kind, gated = case
    r = np.random.default_rng(n + pos)
    host = HostCache(pos + n, n_kv, hd, seed=n * 7 + pos)
    q = r.standard_normal((n, n_head * hd)).astype(np.float32)
    gate = r.standard_normal(q.shape).astype(np.float32) if gated else None
    parents = random_tree(n, n, kind)
    got = run_tree(eng, host, q, parents, pos, gate)
    ref, _, tol, _ = attention(host, q, sees_of(parents, pos, pos + n), gate)
    assert np.abs(got - ref).max() <= tol


def test_tree_of_one_is_the_decode_step(eng):
    """One node: the rows a plain decode attention reads, within both bars."""
    host = HostCache(700, 4, 128, seed=5)
    r = np.random.default_rng(5)
    q = r.standard_normal((1, 16 * 128)).astype(np.float32)
    cache = host.upload(eng)
    got = run_tree(eng, host, q, [-1], 699, cache=cache)
    with Dev(eng) as d:
        out = d.room(q.nbytes)
        cache.attend(d.put(q).ptr, 16, 700, out.ptr, 0, eng.stream)
        eng.synchronize()
        plain = out.download(np.float32, q.shape)
    cache.free()
    _, _, tol, _ = attention(host, q, np.ones((1, 700), bool))
    assert np.abs(got - plain).max() <= tol + 1e-4 * np.abs(host.values("v")).max()


def test_bad_parents_hang_on_the_committed_rows(eng):
    """Parents out of range (itself, a later node, below -1) count as -1."""
    n, pos = 40, 77
    host = HostCache(pos + n, 2, 64, seed=1)
    q = np.random.default_rng(1).standard_normal((n, 8 * 64)).astype(np.float32)
    bad = random_tree(n, 3)
    bad[[0, 5, 9, 20, 39]] = [0, 5, 30, -7, 1 << 30]
    clean = bad.copy()
    clean[[0, 5, 9, 20, 39]] = -1
    a = run_tree(eng, host, q, bad, pos)
    b = run_tree(eng, host, q, clean, pos)
    assert np.array_equal(a, b)
    ref, _, tol, _ = attention(host, q, sees_of(clean, pos, pos + n))
    assert np.abs(a - ref).max() <= tol


@pytest.mark.parametrize("n_head,n_kv,hd", [(4, 2, 64), (8, 1, 128), (2, 2, 256)])
def test_values_that_are_not_finite_stay_with_those_who_see_them(eng, n_head, n_kv, hd):
    """Inf and NaN scales in rows of one branch (K or V) change no node of
    another branch; a node that sees such a V row is NaN in that block's dims
    and as before elsewhere; one that sees such a K row is NaN."""
    pos = 45
    parents = np.array([-1, 0, 0, 1, 2, -1, 5, 4, 3], np.int32)
    n = len(parents)
    host = HostCache(pos + n, n_kv, hd, seed=3)
    q = np.random.default_rng(2).standard_normal((n, n_head * hd)).astype(np.float32)
    clean = run_tree(eng, host, q, parents, pos)
    sees = ancestors(parents)
    group = n_head // n_kv
    for value in (np.inf, np.nan):
        bad = HostCache(pos + n, n_kv, hd, seed=3)
        bad.v_d[pos + 2, 0] = value          # kv head 0, first block
        bad.v_qs[pos + 2, :32] = 0
        got = run_tree(eng, bad, q, parents, pos).reshape(n, n_head, hd)
        ref = clean.reshape(n, n_head, hd)
        hit = np.zeros((n, n_head, hd), bool)
        hit[sees[:, 2], :group, :32] = True
        assert np.isnan(got[hit]).all()
        assert np.array_equal(got[~hit], ref[~hit])
        bad = HostCache(pos + n, n_kv, hd, seed=3)
        bad.k_d[pos + 5, 0] = value
        bad.k_qs[pos + 5, :32] = 0
        got = run_tree(eng, bad, q, parents, pos).reshape(n, n_head, hd)
        hit = np.zeros((n, n_head, hd), bool)
        hit[sees[:, 5], :group] = True
        assert np.isnan(got[hit]).all()
        assert np.array_equal(got[~hit], ref[~hit])


def test_rows_behind_the_tree_are_not_read(eng):
    """Rows past pos + n hold NaN scales: nothing of them arrives."""
    n, pos = 9, 50
    host = HostCache(pos + n + 40, 2, 128, seed=8)
    host.k_d[pos + n:] = np.nan
    host.v_d[pos + n:] = np.inf
    q = np.random.default_rng(8).standard_normal((n, 8 * 128)).astype(np.float32)
    parents = random_tree(n, 8)
    got = run_tree(eng, host, q, parents, pos)
    ref, _, tol, _ = attention(host, q, sees_of(parents, pos, host.rows))
    assert np.abs(got - ref).max() <= tol


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 30.0])
def test_query_magnitudes(eng, scale):
    n, pos = 6, 200
    host = HostCache(pos + n, 2, 128, seed=9, spread=0.5)
    q = (np.random.default_rng(9).standard_normal((n, 4 * 128)) * scale).astype(np.float32)
    parents = random_tree(n, 9)
    got = run_tree(eng, host, q, parents, pos)
    ref, _, tol, _ = attention(host, q, sees_of(parents, pos, pos + n))
    assert np.abs(got - ref).max() <= tol


@pytest.mark.parametrize("v_scale", [1e-7, 3e-5, 1.0, 300.0])
def test_value_magnitudes(eng, v_scale):
    """V scales from f16 subnormals to its upper range."""
    n, pos = 20, 100
    host = HostCache(pos + n, 2, 64, seed=10)
    host.v_d = (np.random.default_rng(10).uniform(0.5, 2, host.v_d.shape) * v_scale).astype(np.float16)
    q = np.random.default_rng(10).standard_normal((n, 4 * 64)).astype(np.float32)
    parents = random_tree(n, 10)
    got = run_tree(eng, host, q, parents, pos)
    ref, _, tol, _ = attention(host, q, sees_of(parents, pos, pos + n))
    assert np.abs(got - ref).max() <= tol


def test_tree_step_prepares_each_node_at_its_depth(eng):
    """The whole step: gates, biases, norms, rotation at rope_pos + depth, the
    cache rows written, then the attention over what was written."""
    import oracle
    n_head, n_kv, hd, pos, rope_pos, n = 8, 2, 64, 60, 1000, 21
    r = np.random.default_rng(4)
    host = HostCache(pos + n, n_kv, hd, seed=4)
    parents = random_tree(n, 4)
    qn, kn = (r.standard_normal(hd) * 0.5 + 1).astype(np.float32), (r.standard_normal(hd) * 0.5 + 1).astype(np.float32)
    rows = 2 * n_head * hd
    q_raw = r.standard_normal((n, rows + 5)).astype(np.float32)     # strided rows
    k = r.standard_normal((n, n_kv * hd + 3)).astype(np.float32)
    v = r.standard_normal((n, n_kv * hd + 3)).astype(np.float32)
    cache = host.upload(eng)
    alone = host.upload(eng)
    with Dev(eng) as d:
        p = engine.GqaParams(d.put(qn).ptr, d.put(kn).ptr, 0, 0, 0, n_head, 1, hd // 2, 1, 1e6, 1e-6)
        out = d.room(4 * n * n_head * hd)
        dq, dk, dv = d.put(q_raw), d.put(k), d.put(v)
        cache.step_tree(p, dq.ptr, dk.ptr, dv.ptr, d.put(parents).ptr, n, pos, rope_pos, out.ptr,
                        q_stride=q_raw.shape[1], kv_stride=k.shape[1], stream=eng.stream)
        # each node prepared on its own, as a decode step at that position
        qo, go = d.room(4 * n * n_head * hd), d.room(4 * n * n_head * hd)
        for i, depth in enumerate(depths(parents)):
            alone.prep(p, dq.ptr + 4 * i * q_raw.shape[1], dk.ptr + 4 * i * k.shape[1], dv.ptr + 4 * i * v.shape[1],
                       pos + i, rope_pos + depth, qo.ptr + 4 * i * n_head * hd, go.ptr + 4 * i * n_head * hd,
                       stream=eng.stream)
        eng.synchronize()
        got = out.download(np.float32, (n, n_head * hd))
        q1, g1 = qo.download(np.float32, got.shape), go.download(np.float32, got.shape)
    a, b = HostCache.download(cache, pos + n), HostCache.download(alone, pos + n)
    for x in a:
        assert np.array_equal(a[x], b[x]), x
        setattr(host, x, a[x] if x.endswith("qs") else a[x].view(np.float16))
    ref, _, tol, _ = attention(host, q1, sees_of(parents, pos, pos + n), g1)
    assert np.abs(got - ref).max() <= tol
    assert oracle is not None
    cache.free()
    alone.free()


@pytest.mark.parametrize("path", [[], [0], [0, 1, 2], [2], [0, 3, 7, 11], [1, 4, 5, 9, 10, 11], list(range(12)), [11]])
def test_keep_path(eng, path):
    n, pos, n_kv, hd = 12, 35, 2, 64
    host = HostCache(pos + n + 4, n_kv, hd, seed=6)
    cache = host.upload(eng)
    want = host.bits(slice(None))
    want = {k: v.copy() for k, v in want.items()}
    before = host.bits(slice(None))
    for j, i in enumerate(path):
        for x in want:
            want[x][pos + j] = before[x][pos + i]
    with Dev(eng) as d:
        p = np.zeros(1 + n, np.uint32)
        p[0] = len(path)
        p[1:1 + len(path)] = path
        cache.keep_path(d.put(p).ptr, n, pos, eng.stream)
        eng.synchronize()
    got = HostCache.download(cache, host.rows)
    for x in want:
        assert np.array_equal(got[x], want[x]), x
    cache.free()


@pytest.mark.parametrize("path,ends", [([0, 3, 3, 5], 2), ([0, 5, 2], 2), ([1, 12], 1), ([4, 0xffffffff], 1), ([0, 1, 0], 2)])
def test_keep_path_ends_where_it_stops_ascending(eng, path, ends):
    n, pos = 12, 3
    host = HostCache(pos + n, 1, 32, seed=6)
    cache = host.upload(eng)
    want = {k: v.copy() for k, v in host.bits(slice(None)).items()}
    before = host.bits(slice(None))
    for j, i in enumerate(path[:ends]):
        for x in want:
            want[x][pos + j] = before[x][pos + i]
    with Dev(eng) as d:
        p = np.zeros(1 + n, np.uint32)
        p[0] = 0xffffffff if path[-1] == 0xffffffff else len(path)
        p[1:1 + len(path)] = path
        cache.keep_path(d.put(p).ptr, n, pos, eng.stream)
        eng.synchronize()
    got = HostCache.download(cache, host.rows)
    for x in want:
        assert np.array_equal(got[x], want[x]), x
    cache.free()


def test_tree_refusals(eng):
    cache = eng.kv_q8_cache(300, 2, 64)
    with Dev(eng) as d:
        b = d.room(1 << 20).ptr
        A, S, U = engine.VXT_E_ARG, engine.VXT_E_SHAPE, engine.VXT_E_UNSUPPORTED
        t = cache.attend_tree
        raises(A, t, 0, 4, b, 1, 0, b)
        raises(A, t, b, 4, 0, 1, 0, b)
        raises(A, t, b, 4, b, 1, 0, 0)
        raises(S, t, b, 3, b, 1, 0, b)
        raises(S, t, b, 0, b, 1, 0, b)
        raises(U, t, b, 18, b, 1, 0, b)
        raises(S, t, b, 4, b, 0, 0, b)
        raises(U, t, b, 4, b, 257, 0, b)
        raises(S, t, b, 4, b, 1, 300, b)
        raises(S, t, b, 4, b, 2, 299, b)
        raises(A, cache.keep_path, 0, 4, 0)
        raises(U, cache.keep_path, b, 257, 0)
        raises(S, cache.keep_path, b, 4, 297)
        p = engine.GqaParams(0, 0, 0, 0, 0, 4, 0, 64, 1, 1e6, 1e-6)
        st = cache.step_tree
        raises(A, st, p, b, b, b, 0, 3, 0, 0, b, 4 * 64, 2 * 64)
        raises(S, st, p, b, b, b, b, 3, 0, 0, b, 4 * 64 - 1, 2 * 64)
        raises(U, st, p, b, b, b, b, 257, 0, 0, b, 4 * 64, 2 * 64)
        raises(A, st, p, b, b, b, b, 3, 0, 0, 0, 4 * 64, 2 * 64)
    cache.free()


def test_tree_captured_and_replayed(eng):
    """A captured call replayed with other trees and queries in the same
    buffers, eager calls of another size between the replays."""
    n, pos, n_head, n_kv, hd = 24, 300, 8, 2, 128
    host = HostCache(pos + n, n_kv, hd, seed=12)
    cache = host.upload(eng)
    r = np.random.default_rng(12)
    with Dev(eng) as d:
        q = d.room(4 * n * n_head * hd)
        par, out = d.room(4 * n), d.room(4 * n * n_head * hd)
        call = lambda s: cache.attend_tree(q.ptr, n_head, par.ptr, n, pos, out.ptr, 0, s)  # noqa: E731
        par.upload(random_tree(n, 0))
        q.upload(np.zeros((n, n_head * hd), np.float32))
        call(eng.stream)
        eng.synchronize()
        g = eng.capture(call)
        for k in range(4):
            x = r.standard_normal((n, n_head * hd)).astype(np.float32)
            parents = random_tree(n, k, ("mixed", "chain", "roots", "mixed")[k])
            q.upload(x)
            par.upload(parents)
            g.launch(2)
            got = out.download(np.float32, x.shape)
            eager = run_tree(eng, host, x, parents, pos, cache=cache)
            assert np.array_equal(got, eager), k
            run_tree(eng, host, x[:3], parents[:3], 17 * k, cache=cache)
        g.free()
    cache.free()
