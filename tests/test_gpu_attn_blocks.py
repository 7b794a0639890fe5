"""GPU parity of block means (``vxt_hip_kv_q8_block_means_dev``) and of the
attention over selected blocks (``vxt_hip_attn_blocks_q8_dev``): means and
selections exactly by the rule, outputs against 64 bits (kv_ops_util, which
derives the bar)."""
import numpy as np
import pytest

from kv_ops_util import Dev, HostCache, attention, raises
from vxg_amd import engine

pytestmark = pytest.mark.gpu
NONE = 0xffffffff


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def q8_blocks(x):
    """KvQ8Block::quantize of f32 rows of 32 (llm_prefill.rs:27-42)."""
    x = np.asarray(x, np.float32).reshape(-1, 32)
    with np.errstate(over="ignore", invalid="ignore"):
        amax = np.fmax.reduce(np.abs(x), axis=1, initial=0.0)
        d = (amax.astype(np.float32) / np.float32(127)).astype(np.float16)
        df = d.astype(np.float32)
        inv = np.where(df > 0, np.float32(1) / np.where(df > 0, df, 1), 0).astype(np.float32)
        q = np.rint(x * inv[:, None])
        q = np.where(np.isnan(q), 0, np.clip(q, -127, 127)).astype(np.int8)
    return q, d


def means_of(host, block):
    """(codes [blocks][per], f16 scales) of every whole block."""
    n = host.rows // block
    x = host.values("k")[:n * block].reshape(n, block, host.per)
    q, d = q8_blocks((x.sum(1) / block).astype(np.float32))
    return q.reshape(n, host.per), d.reshape(n, host.per // 32)


def selection(host, mean, q, pos, block, n_sel, n_first, n_local):
    """[m][n_kv] lists of blocks by the rule."""
    code, scale = mean
    m, hd, n_kv = q.shape[0], host.hd, host.n_kv
    group = q.shape[1] // hd // n_kv
    all_ = []
    for i in range(m):
        own = (pos + i) // block
        per_head = []
        for kv in range(n_kv):
            x = q[i].reshape(-1, hd)[kv * group:(kv + 1) * group].astype(np.float64).sum(0).astype(np.float32)
            qq, qd = q8_blocks(x)
            forced = {b for b in range(own + 1) if b < n_first or own - b < n_local}
            rest = []
            for b in range(own + 1):
                if b in forced:
                    continue
                c = code[b, kv * hd:(kv + 1) * hd].reshape(-1, 32).astype(np.int64)
                s = scale[b, kv * hd // 32:(kv + 1) * hd // 32].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    v = np.float32((qd.astype(np.float64) * s * (c * qq).sum(1)).sum())
                rest.append((np.isnan(v), -v if not np.isnan(v) else 0, b))
            take = sorted(forced | {b for *_, b in sorted(rest)[:max(0, n_sel - len(forced))]})
            per_head.append(take if own + 1 > n_sel else list(range(own + 1)))
        all_.append(per_head)
    return all_


def run_blocks(eng, host, mean, q, pos, block, n_sel, n_first, n_local, gate=None):
    m, width = q.shape
    cache = host.upload(eng)
    means = eng.kv_block_means(max(1, mean[0].shape[0]), block, host.n_kv, host.hd)
    if mean[0].size:
        means.qs.upload(mean[0])
        means.d.upload(mean[1])
    with Dev(eng) as d:
        out, sel = d.room(q.nbytes), d.room(4 * m * host.n_kv * n_sel)
        g = d.put(gate).ptr if gate is not None else 0
        dq = d.put(q)
        cache.attend_blocks(means, dq.ptr, width // host.hd, m, pos, n_sel, n_first, n_local, out.ptr, g, sel.ptr,
                            eng.stream)
        eng.synchronize()
        got = out.download(np.float32, q.shape), sel.download(np.uint32, (m, host.n_kv, n_sel))
        # the selection is optional
        cache.attend_blocks(means, dq.ptr, width // host.hd, m, pos, n_sel, n_first, n_local, out.ptr, g, 0, eng.stream)
        eng.synchronize()
        assert np.array_equal(out.download(np.float32, q.shape), got[0], equal_nan=True)
    cache.free()
    means.free()
    return got


def check(eng, host, q, pos, block, n_sel, n_first, n_local, gate=None, mean=None):
    m = q.shape[0]
    mean = mean or means_of(host, block)
    out, sel = run_blocks(eng, host, mean, q, pos, block, n_sel, n_first, n_local, gate)
    want = selection(host, mean, q, pos, block, n_sel, n_first, n_local)
    sees = np.zeros((m, host.n_kv, host.rows), bool)
    for i in range(m):
        for kv in range(host.n_kv):
            take = want[i][kv]
            assert sel[i, kv, :len(take)].tolist() == take, (i, kv)
            assert (sel[i, kv, len(take):] == NONE).all()
            for b in take:
                sees[i, kv, b * block:(b + 1) * block] = True
            sees[i, kv, pos + i + 1:] = False
    ref, _, tol, _ = attention(host, q, sees, gate)
    assert np.abs(out - ref).max() <= tol
    return sel


CASES = [
    # m, pos, n_head, n_kv, hd, block, n_sel, n_first, n_local, gated
    (1, 0, 4, 4, 32, 32, 1, 0, 1, False),
    (1, 63, 4, 2, 64, 64, 4, 1, 1, True),
    (1, 64, 4, 2, 64, 64, 1, 0, 1, False),
    (1, 1000, 16, 4, 128, 64, 8, 1, 2, True),
    (1, 5000, 8, 1, 64, 32, 40, 0, 1, False),
    (1, 4095, 6, 2, 128, 128, 5, 2, 3, False),
    (1, 2000, 4, 2, 256, 64, 9, 1, 1, True),
    (1, 40000, 8, 2, 32, 32, 100, 1, 2, False),
    (3, 126, 4, 2, 64, 64, 2, 0, 1, False),       # the tokens cross a block's end
    (17, 500, 10, 2, 32, 32, 6, 1, 1, True),
    (70, 0, 4, 1, 128, 32, 2, 0, 1, False),
    (40, 900, 16, 4, 128, 64, 8, 1, 2, True),
    (9, 700, 2, 2, 256, 128, 3, 0, 2, False),
    (18, 34000, 4, 2, 32, 32, 20, 1, 2, False),   # many tokens, more than 1,024 blocks
    (2, 20000, 4, 1, 256, 64, 30, 2, 1, True),
]


@pytest.mark.parametrize("case", CASES)
def test_blocks_parity(eng, case):
    m, pos, n_head, n_kv, hd, block, n_sel, n_first, n_local, gated = case
    r = np.random.default_rng(pos + m)
    host = HostCache(pos + m, n_kv, hd, seed=pos * 3 + m)
    q = r.standard_normal((m, n_head * hd)).astype(np.float32)
    gate = r.standard_normal(q.shape).astype(np.float32) if gated else None
    check(eng, host, q, pos, block, n_sel, n_first, n_local, gate)


def test_all_blocks_is_plain_attention(eng):
    """With as many blocks taken as there are, every row up to the token."""
    m, pos = 5, 411
    host = HostCache(pos + m, 2, 64, seed=1)
    q = np.random.default_rng(1).standard_normal((m, 4 * 64)).astype(np.float32)
    none = np.zeros((0, 128), np.int8), np.zeros((0, 4), np.float16)
    out, sel = run_blocks(eng, host, none, q, pos, 32, 50, 0, 1)
    ref, _, tol, _ = attention(host, q, np.arange(pos + m)[None] <= pos + np.arange(m)[:, None])
    assert np.abs(out - ref).max() <= tol
    assert (sel[:, :, (pos + m - 1) // 32 + 1:] == NONE).all()


@pytest.mark.parametrize("kind", ["equal", "zero query", "nan", "inf", "subnormal"])
def test_selection_orders(eng, kind):
    """Equal scores take the lowest blocks, NaN scores come last."""
    pos, n_kv, hd, block = 1500, 2, 64, 32
    host = HostCache(pos + 1, n_kv, hd, seed=4)
    q = np.random.default_rng(4).standard_normal((1, 4 * hd)).astype(np.float32)
    code, scale = means_of(host, block)
    if kind == "equal":
        code[:], scale[:] = code[0], scale[0]
    if kind == "zero query":
        q[:] = 0
    if kind == "nan":
        scale[::2, 0] = np.nan
        scale[1::4, 3] = np.nan
    if kind == "inf":
        scale[5:30, :] = np.inf
        code[5:10, :32] = 0
    if kind == "subnormal":
        scale[:] = (np.random.default_rng(1).integers(1, 900, scale.shape).astype(np.uint16)).view(np.float16)
    check(eng, host, q, pos, block, 7, 1, 1, mean=(code, scale))


def test_unselected_rows_do_not_arrive(eng):
    """NaN and Inf scales in every block that was not taken."""
    pos, n_kv, hd, block, n_sel = 900, 1, 128, 64, 4
    host = HostCache(pos + 1, n_kv, hd, seed=2)
    q = np.random.default_rng(2).standard_normal((1, 8 * hd)).astype(np.float32)
    mean = means_of(host, block)
    want = selection(host, mean, q, pos, block, n_sel, 1, 1)[0][0]
    bad = np.ones(host.rows, bool)
    for b in want:
        bad[b * block:(b + 1) * block] = False
    host.k_d[bad] = np.nan
    host.v_d[bad] = np.inf
    check(eng, host, q, pos, block, n_sel, 1, 1, mean=mean)


@pytest.mark.parametrize("n_kv,hd,block", [(1, 32, 32), (3, 64, 64), (2, 128, 128), (2, 256, 32)])
def test_block_means(eng, n_kv, hd, block):
    """Every mean bit by bit; blocks that are not full, and those the rows do
    not touch, are left as they were."""
    rows = 5 * block + 17
    host = HostCache(rows, n_kv, hd, seed=block + hd)
    host.k_d[3, 0] = np.float16(6e-8)                       # a subnormal scale
    want_q, want_d = means_of(host, block)
    cache = host.upload(eng)
    n = rows // block + 1
    means = eng.kv_block_means(n, block, n_kv, hd)
    for row0, n_rows, lo, hi in [(0, rows, 0, 5), (block + 5, 1, 0, 0), (2 * block - 1, 1, 1, 2),
                                 (block + 3, 2 * block, 1, 3), (4 * block, block - 1, 0, 0), (0, 0, 0, 0)]:
        for b in (means.qs, means.d):
            b.upload(np.full(b.nbytes, 9, np.uint8))
        cache.block_means(means, row0, n_rows, eng.stream)
        eng.synchronize()
        q = means.qs.download(np.int8, (n, n_kv * hd))
        d = means.d.download(np.uint16, (n, n_kv * hd // 32))
        assert np.array_equal(q[lo:hi], want_q[lo:hi]) and np.array_equal(d[lo:hi], want_d[lo:hi].view(np.uint16))
        rest = np.ones(n, bool)
        rest[lo:hi] = False
        assert (q[rest] == 9).all() and (d[rest] == 0x0909).all()
    cache.free()
    means.free()


def test_decode_over_blocks(eng):
    """Tokens appended one after the other, the means kept up with them."""
    n_head, n_kv, hd, block, n_sel, steps = 4, 2, 64, 32, 4, 200
    r = np.random.default_rng(6)
    src = HostCache(steps, n_kv, hd, seed=6)
    cache, means = eng.kv_q8_cache(steps, n_kv, hd), eng.kv_block_means(steps // block, block, n_kv, hd)
    with Dev(eng) as d:
        K = d.put(src.values("k").reshape(steps, -1).astype(np.float32))
        V = d.put(src.values("v").reshape(steps, -1).astype(np.float32))
        out, sel = d.room(4 * n_head * hd), d.room(4 * n_kv * n_sel)
        for t in range(steps):
            cache.append(K.ptr + 4 * t * n_kv * hd, V.ptr + 4 * t * n_kv * hd, t, eng.stream)
            cache.block_means(means, t, 1, eng.stream)
            q = r.standard_normal((1, n_head * hd)).astype(np.float32)
            cache.attend_blocks(means, d.put(q).ptr, n_head, 1, t, n_sel, 1, 1, out.ptr, 0, sel.ptr, eng.stream)
            if t % 13 and t % block > 1:
                continue
            eng.synchronize()
            now = HostCache(t + 1, n_kv, hd, seed=0)
            for x, a in HostCache.download(cache, t + 1).items():
                setattr(now, x, a if x.endswith("qs") else a.view(np.float16))
            want = selection(now, means_of(now, block), q, t, block, n_sel, 1, 1)[0]
            got = sel.download(np.uint32, (n_kv, n_sel))
            sees = np.zeros((1, n_kv, t + 1), bool)
            for kv in range(n_kv):
                assert got[kv][got[kv] != NONE].tolist() == want[kv]
                for b in want[kv]:
                    sees[0, kv, b * block:(b + 1) * block] = True
            ref, _, tol, _ = attention(now, q, sees)
            assert np.abs(out.download(np.float32, q.shape) - ref).max() <= tol
    cache.free()
    means.free()


def test_refusals(eng):
    A, S, U = engine.VXT_E_ARG, engine.VXT_E_SHAPE, engine.VXT_E_UNSUPPORTED
    cache, means = eng.kv_q8_cache(1000, 2, 64), eng.kv_block_means(10, 32, 2, 64)
    odd = eng.kv_block_means(10, 48, 2, 64)
    with Dev(eng) as d:
        b = d.room(1 << 20).ptr
        f = cache.attend_blocks
        raises(A, f, means, 0, 4, 1, 0, 4, 1, 1, b)
        raises(A, f, means, b, 4, 1, 0, 4, 1, 1, 0)
        raises(S, f, means, b, 5, 1, 0, 4, 1, 1, b)
        raises(U, f, means, b, 18, 1, 0, 4, 1, 1, b)
        raises(S, f, means, b, 4, 0, 0, 4, 1, 1, b)
        raises(S, f, means, b, 4, 1, 1000, 4, 1, 1, b)
        raises(S, f, means, b, 4, 2, 999, 4, 1, 1, b)
        raises(S, f, means, b, 4, 1, 100, 4, 1, 0, b)
        raises(S, f, means, b, 4, 1, 100, 4, 3, 2, b)
        raises(S, f, means, b, 4, 1, 100, 0, 0, 1, b)
        raises(S, f, means, b, 4, 1, 900, 4, 1, 1, b)       # fewer means than blocks
        raises(U, f, odd, b, 4, 1, 100, 4, 1, 1, b)
        raises(A, f, engine.KvBlockMeans.over(eng, 0, b, 10, 32), b, 4, 1, 100, 4, 1, 1, b)
        raises(A, f, engine.KvBlockMeans.over(eng, b + 8, b, 10, 32), b, 4, 1, 100, 4, 1, 1, b)
        long = engine.KvQ8Cache.over(eng, b, b, b, b, 1 << 22, 2, 64)
        raises(U, long.attend_blocks, engine.KvBlockMeans.over(eng, b, b, 1 << 20, 32), b, 4, 1, 14336 * 32, 4, 1, 1, b)
    m = cache.block_means
    raises(S, m, means, 0, 1001)
    raises(S, m, means, 1001, 0)
    raises(S, m, means, 0, 352)
    raises(U, m, odd, 0, 10)
    for x in (cache, means, odd):
        x.free()


def test_captured_and_replayed(eng):
    pos, n_kv, hd, n_head, block, n_sel = 800, 2, 64, 8, 32, 5
    host = HostCache(pos + 1, n_kv, hd, seed=5)
    cache, means = host.upload(eng), eng.kv_block_means(26, block, n_kv, hd)
    cache.block_means(means, 0, pos, eng.stream)
    with Dev(eng) as d:
        q, out, sel = d.room(4 * n_head * hd), d.room(4 * n_head * hd), d.room(4 * n_kv * n_sel)
        call = lambda s: cache.attend_blocks(means, q.ptr, n_head, 1, pos, n_sel, 1, 1, out.ptr, 0, sel.ptr, s)  # noqa: E731
        q.upload(np.zeros(n_head * hd, np.float32))
        call(eng.stream)
        eng.synchronize()
        g = eng.capture(call)
        for k in range(4):
            q.upload(np.random.default_rng(k).standard_normal(n_head * hd).astype(np.float32))
            g.launch(1)
            a = out.download(np.float32, (n_head * hd,)), sel.download(np.uint32, (n_kv, n_sel))
            call(eng.stream)
            eng.synchronize()
            assert np.array_equal(a[0], out.download(np.float32, (n_head * hd,)))
            assert np.array_equal(a[1], sel.download(np.uint32, (n_kv, n_sel)))
            cache.attend_blocks(means, q.ptr, n_head, 1, 50 + 100 * k, n_sel, 1, 1, out.ptr, 0, 0, eng.stream)
            eng.synchronize()
        g.free()
    cache.free()
    means.free()
