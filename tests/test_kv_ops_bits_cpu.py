"""What the bars of kv_ops_bits see, in a model of the operands on the CPU: two
f16 terms of each pass, one term of any does not."""
import numpy as np
import pytest

from kv_ops_bits import row_bar, row_errors, sink, sink_bar
from kv_ops_util import HostCache, attention


def f16_terms(x, n, up=1.0):
    """x as n f16 terms after a factor, in 64 bits."""
    left, total = x * up, np.zeros_like(x)
    for _ in range(n):
        t = left.astype(np.float16).astype(np.float64)
        total, left = total + t, left - t
    return total / up


def model(host, q, sees, terms=(2, 2, 2), up=2.0 ** 13):
    """Attention with queries, weights and values in that many f16 terms, the
    weights relative to the row's largest and `up` times as large."""
    m, hd = q.shape[0], host.hd
    n_head = q.shape[1] // hd
    K, V = host.values("k"), host.values("v")
    out = np.zeros((m, n_head, hd))
    for i in range(m):
        t = np.flatnonzero(sees[i])
        for h in range(n_head):
            kv = h // (n_head // host.n_kv)
            x = q[i].astype(np.float64).reshape(n_head, hd)[h]
            s = K[t, kv] @ f16_terms(x, terms[0], 2.0 ** (14 - np.floor(np.log2(np.abs(x).max())))) / np.sqrt(hd)
            p = np.exp(s - s.max())
            top = np.abs(V[t, kv]).max()
            out[i, h] = f16_terms(p, terms[1], up) @ f16_terms(V[t, kv], terms[2], 2.0 ** (13 - np.floor(np.log2(top)))) / p.sum()
    return out.reshape(m, -1)


@pytest.mark.parametrize("m,rows,n_head,n_kv,hd", [(1, 700, 4, 2, 64), (3, 1500, 4, 1, 128), (5, 160, 2, 2, 32),
                                                   (1, 5000, 2, 1, 256), (2, 9000, 4, 2, 64)])
def test_random_rows_tell_one_term_from_two(m, rows, n_head, n_kv, hd):
    host = HostCache(rows, n_kv, hd, seed=rows)
    q = np.random.default_rng(m).standard_normal((m, n_head * hd)).astype(np.float32)
    sees = np.arange(rows)[None] <= rows - m + np.arange(m)[:, None]
    ref, _, _, _ = attention(host, q, sees)
    bar = row_bar(host, q, rows)
    assert bar < 3e-5
    assert row_errors(model(host, q, sees), ref, hd).max() <= bar
    for terms in ((1, 2, 2), (2, 1, 2), (2, 2, 1)):
        assert row_errors(model(host, q, sees, terms), ref, hd).max() > 2 * bar, terms


@pytest.mark.parametrize("gap", [8, 10, 12])
def test_a_row_above_the_others_tells_the_weights_range(gap):
    host, q, g = sink(1024, 1, 64, gap, 1, 2, seed=gap)
    sees = np.ones((1, 1024), bool)
    ref, _, _, _ = attention(host, q, sees)
    err = [np.abs(model(host, q, sees, up=up) / ref - 1).max() for up in (2.0 ** 13, 1.0)]
    assert err[0] <= sink_bar(g, 1024)
    assert gap < 10 or err[1] > sink_bar(g, 1024)
