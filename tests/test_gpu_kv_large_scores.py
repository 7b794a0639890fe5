"""GPU: attention over the Q8_0 KV cache with scores of any size.  Two rows have
the same, largest score and the others lie far below it: each of the two has
half of the weight, and an output is the mean of their values, whatever the
scores' magnitude.

Bars.  The two weights are the same number, exactly, so an output's error is
that of two products and a division: three roundings of 22 bits, 2^-20 of the
larger value.  A row's weight is a sum of m * group halves, each right to three
roundings of f32 and an exp2 (2^-21), added in f32.
"""
import numpy as np
import pytest

from kv_ops_util import Dev, HostCache, ancestors, random_tree
from vxg_amd import engine

pytestmark = pytest.mark.gpu
A, B = 3, 40


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def twins(rows, n_kv, hd, n_tok, n_head, k, seed):
    """Scores 2^k code / (64 sqrt(hd)): 100 in rows A and B, at most 60 elsewhere."""
    host = HostCache(rows, n_kv, hd, seed)
    r = np.random.default_rng(seed)
    host.k_qs[:, ::hd] = r.integers(-100, 61, (rows, n_kv))
    host.k_qs[[A, B], ::hd] = 100
    host.k_d[:] = 2.0 ** -6
    q = np.zeros((n_tok, n_head, hd), np.float32)
    q[:, :, 0] = 2.0 ** k
    return host, q.reshape(n_tok, -1)


@pytest.mark.parametrize("form,m,rows,n_head,n_kv,hd", [
    ("weigh", 1, 300, 4, 2, 64), ("weigh", 1, 5000, 8, 1, 128), ("weigh", 1, 700, 2, 1, 256), ("weigh", 1, 90, 3, 1, 32),
    ("weigh", 7, 300, 4, 2, 64), ("weigh", 300, 400, 8, 2, 128), ("weigh", 40, 900, 2, 2, 256), ("weigh", 33, 90, 3, 1, 32),
    ("tree", 1, 300, 4, 2, 64), ("tree", 30, 2000, 8, 2, 128), ("tree", 9, 500, 4, 2, 256), ("tree", 200, 600, 4, 4, 32),
    ("blocks", 1, 300, 4, 2, 64), ("blocks", 20, 3000, 16, 4, 128), ("blocks", 5, 900, 2, 1, 256)])
@pytest.mark.parametrize("k", [11, 14, 20, 25, 26, 27, 28, 32, 60])
def test_two_rows_share(eng, form, m, rows, n_head, n_kv, hd, k):
    host, q = twins(rows, n_kv, hd, m, n_head, k, seed=rows + m)
    pos, group = rows - m, n_head // n_kv
    cache = host.upload(eng)
    held, total = [cache], None
    with Dev(eng) as d:
        out, Q = d.room(q.nbytes), d.put(q).ptr
        if form == "tree":
            cache.attend_tree(Q, n_head, d.put(random_tree(m, m)).ptr, m, pos, out.ptr, 0, eng.stream)
        elif form == "weigh":
            w = eng.kv_weights(rows, n_kv)
            held.append(w)
            w.weight.upload(np.zeros((n_kv, rows), np.float32))
            cache.attend_weigh(w, Q, n_head, m, pos, 0, out.ptr, 0, eng.stream)
            eng.synchronize()
            total = w.weight.download(np.float32, (n_kv, rows))
        else:
            nb = (rows - 1) // 32 + 1
            means = eng.kv_block_means(nb, 32, n_kv, hd)
            held.append(means)
            cache.attend_blocks(means, Q, n_head, m, pos, nb, 1, 1, out.ptr, 0, 0, eng.stream)
        eng.synchronize()
        got = out.download(np.float32, q.shape).reshape(m, n_kv, group, hd)
    V = host.values("v")
    want = ((V[A] + V[B]) / 2)[None, :, None]
    big = np.maximum(np.abs(V[A]), np.abs(V[B]))[None, :, None]
    assert (np.abs(got - want) <= 2.0 ** -20 * big + 2.0 ** -36 * np.abs(V).max()).all()
    if total is not None:
        full = m * group / 2
        assert (np.abs(total[:, [A, B]] / full - 1) <= 2.0 ** -21 + (m * group + 8) * 2.0 ** -24).all()
        rest = np.delete(total, [A, B], axis=1)
        assert (np.abs(rest) <= full * np.exp(-40 * 2.0 ** k / (64 * np.sqrt(hd))) * 1.01 + 2.0 ** -100).all()
    for b in held:
        b.free()
