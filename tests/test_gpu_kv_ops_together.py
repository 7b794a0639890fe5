"""GPU: drafted trees and a row budget on one cache, as the header has them go
together: a weighed prompt, a tree's attention, its accepted path kept, the
kept tokens weighed at their rows, rows evicted, block means made anew and a
token over selected blocks -- each against 64 bits on what the cache holds."""
import numpy as np
import pytest

from kv_ops_util import Dev, HostCache, ancestors, attention
from test_gpu_kv_evict import evict_plan
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def held(cache, rows):
    h = HostCache(rows, cache.n_kv, cache.head_dim, seed=0)
    for x, a in HostCache.download(cache, rows).items():
        setattr(h, x, a if x.endswith("qs") else a.view(np.float16))
    return h


@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 64), (4, 1, 128), (6, 2, 32)])
def test_trees_under_a_budget(eng, n_head, n_kv, hd):
    full, keep, m, block = 160, 96, 70, 32
    r = np.random.default_rng(hd)
    cache, w = eng.kv_q8_cache(full, n_kv, hd), eng.kv_weights(full, n_kv)
    means = eng.kv_block_means(full // block, block, n_kv, hd)
    per = n_kv * hd

    def queries(n):
        return r.standard_normal((n, n_head * hd)).astype(np.float32)

    with Dev(eng) as d:
        def append(n, row):
            K, V = (d.put(r.standard_normal((n, per)).astype(np.float32)) for _ in range(2))
            for i in range(n):
                cache.append(K.ptr + 4 * i * per, V.ptr + 4 * i * per, row + i, eng.stream)

        def planes():
            eng.synchronize()
            return w.weight.download(np.float32, (n_kv, full)), w.position.download(np.uint32, (n_kv, full))

        append(m, 0)
        q, out = queries(m), d.room(4 * 64 * n_head * hd * 2)
        cache.attend_weigh(w, d.put(q).ptr, n_head, m, 0, 0, out.ptr, 0, eng.stream)
        rows, tokens = m, m
        for step in range(6):
            parents = np.array([-1, 0, 0, 1, 1, 3, 4, -1, 7, 5, 9, 2], np.int32)
            path = [[0, 1, 3, 5, 9, 10], [0, 2, 11], [7, 8], [0], [0, 1, 4, 6], [0, 1, 3, 5]][step]
            n = len(parents)
            if rows + n > full:
                before = planes()
                cache.evict(w, rows, keep, tokens, 10, 2, stream=eng.stream)
                after = planes()
                for k in range(n_kv):
                    src = evict_plan(before[0][k], before[1][k], rows, keep, tokens, 10, 2)
                    assert np.array_equal(after[0][k, :keep], before[0][k][src])
                    assert np.array_equal(after[1][k, :keep], before[1][k][src])
                rows = keep
                cache.block_means(means, 0, rows, eng.stream)
            append(n, rows)
            q = queries(n)
            cache.attend_tree(d.put(q).ptr, n_head, d.put(parents).ptr, n, rows, out.ptr, 0, eng.stream)
            eng.synchronize()
            now = held(cache, rows + n)
            sees = np.ones((n, rows + n), bool)
            sees[:, rows:] = ancestors(parents)
            ref, _, tol, _ = attention(now, q, sees)
            tree_out = out.download(np.float32, q.shape)
            assert np.abs(tree_out - ref).max() <= tol
            cache.keep_path(d.put(np.array([len(path)] + path, np.uint32)).ptr, n, rows, eng.stream)
            before = planes()
            c = len(path)
            cache.attend_weigh(w, d.put(q[path]).ptr, n_head, c, rows, tokens, out.ptr, 0, eng.stream)
            after = planes()
            now = held(cache, rows + c)
            ref, total, tol, rel = attention(now, q[path], np.arange(rows + c)[None] <= rows + np.arange(c)[:, None])
            got = out.download(np.float32, (c, n_head * hd))
            assert np.abs(got - ref).max() <= tol
            assert np.abs(got - tree_out[path]).max() <= 2 * tol      # the same rows seen, in the tree and behind it
            want = total.copy()
            want[:, :rows] += before[0][:, :rows]
            assert (np.abs(after[0][:, :rows + c] - want) <= rel * total + 2.0 ** -22 * total.max() + 2.0 ** -23 * want).all()
            assert np.array_equal(after[1][:, rows:rows + c], np.tile(tokens + np.arange(c, dtype=np.uint32), (n_kv, 1)))
            assert np.array_equal(after[1][:, :rows], before[1][:, :rows])
            cache.block_means(means, rows if step else 0, c if step else rows + c, eng.stream)
            rows, tokens = rows + c, tokens + c
            sel = d.room(4 * n_kv * 3)
            cache.attend_blocks(means, d.put(q[path[-1:]]).ptr, n_head, 1, rows - 1, 3, 1, 1, out.ptr, 0, sel.ptr, eng.stream)
            eng.synchronize()
            taken = sel.download(np.uint32, (1, n_kv, 3))
            assert (taken[:, :, 0] == 0).all() and (taken[:, :, 2] == (rows - 1) // block).all()
            sees = (taken[:, :, :, None] == np.arange(rows) // block).any(2)
            ref, _, tol, _ = attention(now, q[path[-1:]], sees)
            assert np.abs(out.download(np.float32, (1, n_head * hd)) - ref).max() <= tol
    for b in (cache, w, means):
        b.free()
