"""GPU parity of the operators over the Q8_0 KV cache at their limits: the most
blocks to select from, a prompt of thousands of tokens, the widest tree; bars
of kv_ops_util and kv_ops_bits."""
import numpy as np
import pytest

from kv_ops_bits import row_bar, row_errors
from kv_ops_util import Dev, HostCache, ancestors, random_tree
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def dense(host, q, sees):
    """(out, weights summed per kv head) in 64 bits, a head at a time."""
    m, hd = q.shape[0], host.hd
    n_head = q.shape[1] // hd
    group = n_head // host.n_kv
    K, V = host.values("k"), host.values("v")
    out, total = np.zeros((m, n_head, hd)), np.zeros((host.n_kv, host.rows))
    for h in range(n_head):
        s = q.astype(np.float64).reshape(m, n_head, hd)[:, h] @ K[:, h // group].T / np.sqrt(hd)
        s[~sees] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ V[:, h // group]
        total[h // group] += p.sum(0)
    return out.reshape(m, -1), total


def q8(x):
    """f32 rows of 32 as codes and f32 scales."""
    x = x.reshape(-1, 32)
    d = (np.abs(x).max(1) / np.float32(127)).astype(np.float16).astype(np.float32)
    inv = np.where(d > 0, np.float32(1) / np.where(d > 0, d, 1), 0).astype(np.float32)
    return np.clip(np.rint(x * inv[:, None]), -127, 127).astype(np.int64), d.astype(np.float64)


@pytest.mark.parametrize("hd,block,n_sel,n_first,n_local,short", [
    (32, 32, 40, 1, 2, 0), (64, 32, 3000, 2, 1, 9), (32, 128, 14335, 1, 1, 0), (32, 32, 14336, 0, 1, 5)])
def test_the_most_blocks(eng, hd, block, n_sel, n_first, n_local, short):
    """14,336 blocks, of which a few, many, all but one and all are taken."""
    n_head, rows = 2, 14336 * block - short
    host = HostCache(rows, 1, hd, seed=n_sel)
    r = np.random.default_rng(hd)
    q = r.standard_normal((1, n_head * hd)).astype(np.float32)
    cache, means = host.upload(eng), eng.kv_block_means(14336, block, 1, hd)
    print(hd, block, n_sel, flush=True)
    with Dev(eng) as d:
        out, sel = d.room(q.nbytes), d.room(4 * n_sel)
        cache.block_means(means, 0, rows, eng.stream)
        cache.attend_blocks(means, d.put(q).ptr, n_head, 1, rows - 1, n_sel, n_first, n_local, out.ptr, 0, sel.ptr, eng.stream)
        eng.synchronize()
        got, taken = out.download(np.float32, q.shape), sel.download(np.uint32, (n_sel,))
        code = means.qs.download(np.int8, (14336, hd)).astype(np.int64).reshape(14336, -1, 32)
        scale = means.d.download(np.uint16, (14336, hd // 32)).view(np.float16).astype(np.float64)
    qq, qd = q8(q.astype(np.float64).reshape(n_head, hd).sum(0).astype(np.float32))
    own = 14335
    b = np.arange(14336)
    score = ((qd * scale) * (code * qq).sum(2)).sum(1).astype(np.float32).astype(np.float64)
    score[(b < n_first) | (b > own - n_local)] = np.inf
    want = np.sort(np.lexsort((b, -score))[:n_sel])
    assert np.array_equal(taken, want)
    sees = np.isin(np.arange(rows) // block, want)[None]
    ref, _ = dense(host, q, sees)
    assert row_errors(got, ref, hd).max() <= row_bar(host, q, rows)
    cache.free()
    means.free()


@pytest.mark.parametrize("m,pos,n_head,n_kv,hd", [(4500, 300, 8, 1, 32), (3000, 0, 3, 1, 64), (2200, 0, 2, 2, 128), (1300, 2000, 2, 1, 256)])
def test_a_long_weighed_prompt(eng, m, pos, n_head, n_kv, hd):
    host = HostCache(pos + m, n_kv, hd, seed=m)
    q = np.random.default_rng(m).standard_normal((m, n_head * hd)).astype(np.float32)
    cache, w = host.upload(eng), eng.kv_weights(host.rows, n_kv)
    before = np.random.default_rng(1).exponential(1, (n_kv, host.rows)).astype(np.float32)
    w.weight.upload(before)
    with Dev(eng) as d:
        out = d.room(q.nbytes)
        cache.attend_weigh(w, d.put(q).ptr, n_head, m, pos, 7, out.ptr, 0, eng.stream)
        eng.synchronize()
        got, gw = out.download(np.float32, q.shape), w.weight.download(np.float32, before.shape)
        gp = w.position.download(np.uint32, before.shape)
    ref, total = dense(host, q, np.arange(host.rows)[None] <= pos + np.arange(m)[:, None])
    bar = row_bar(host, q, host.rows)
    assert row_errors(got, ref, hd).max() <= bar
    total[:, :pos] += before[:, :pos]
    assert (np.abs(gw / total - 1) <= bar + 2.0 ** -22 * total.max() / total).all()
    assert np.array_equal(gp[:, pos:], np.tile(7 + np.arange(m, dtype=np.uint32), (n_kv, 1)))
    cache.free()
    w.free()


@pytest.mark.parametrize("n_head,n_kv,hd,pos", [(8, 1, 256, 3000), (16, 2, 128, 31), (64, 8, 32, 5000)])
def test_the_widest_tree(eng, n_head, n_kv, hd, pos):
    n = 256
    host = HostCache(pos + n, n_kv, hd, seed=n + pos)
    q = np.random.default_rng(hd).standard_normal((n, n_head * hd)).astype(np.float32)
    parents = random_tree(n, hd)
    sees = np.ones((n, pos + n), bool)
    sees[:, pos:] = ancestors(parents)
    cache = host.upload(eng)
    with Dev(eng) as d:
        out = d.room(q.nbytes)
        cache.attend_tree(d.put(q).ptr, n_head, d.put(parents).ptr, n, pos, out.ptr, 0, eng.stream)
        eng.synchronize()
        got = out.download(np.float32, q.shape)
    ref, _ = dense(host, q, sees)
    assert row_errors(got, ref, hd).max() <= row_bar(host, q, host.rows)
    cache.free()
