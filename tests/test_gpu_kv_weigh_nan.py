"""GPU: a token whose queries hold NaN, in a weighed prompt
(``vxt_hip_attn_weigh_q8_dev``), gives NaN to the rows that it sees and to
nothing else: no other token's output, no row behind it, no other kv head."""
import numpy as np
import pytest

from kv_ops_util import Dev, HostCache, attention
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def weigh(eng, host, q, pos):
    m, width = q.shape
    cache, w = host.upload(eng), eng.kv_weights(host.rows, host.n_kv)
    w.weight.upload(np.zeros((host.n_kv, host.rows), np.float32))
    with Dev(eng) as d:
        out = d.room(q.nbytes)
        cache.attend_weigh(w, d.put(q).ptr, width // host.hd, m, pos, 0, out.ptr, 0, eng.stream)
        eng.synchronize()
        got = out.download(np.float32, q.shape), w.weight.download(np.float32, (host.n_kv, host.rows))
    cache.free()
    w.free()
    return got


@pytest.mark.parametrize("m,pos,n_head,n_kv,hd,token", [
    (2, 0, 2, 2, 32, 0), (9, 40, 4, 2, 64, 3), (40, 0, 4, 1, 64, 0), (40, 0, 4, 1, 64, 17), (40, 5, 4, 1, 64, 39),
    (130, 61, 7, 1, 64, 80), (20, 0, 3, 1, 64, 19), (300, 0, 16, 4, 128, 33), (300, 700, 16, 4, 128, 200),
    (40, 700, 4, 2, 256, 8), (700, 1500, 6, 2, 128, 350)])
def test_a_token_of_nan_reaches_the_rows_it_sees_alone(eng, m, pos, n_head, n_kv, hd, token):
    host = HostCache(pos + m, n_kv, hd, seed=m + token)
    q = np.random.default_rng(m).standard_normal((m, n_head * hd)).astype(np.float32)
    clean, _ = weigh(eng, host, q, pos)
    bad = q.copy()
    bad[token, 5] = np.nan                 # query head 0, kv head 0
    out, w = weigh(eng, host, bad, pos)
    hit = np.zeros((m, n_head, hd), bool)
    hit[token, 0] = True
    assert np.isnan(out.reshape(hit.shape)[hit]).all()
    assert np.array_equal(out.reshape(hit.shape)[~hit], clean.reshape(hit.shape)[~hit])
    sees = np.arange(host.rows)[None] <= pos + np.arange(m)[:, None]
    _, total, _, rel = attention(host, q, sees)
    rest = np.arange(m) != token
    _, total[0], _, _ = (x if i != 1 else x[0] for i, x in enumerate(attention(host, q[rest], sees[rest])))
    behind = np.arange(host.rows) > pos + token
    assert np.isnan(w[0, ~behind]).all()
    assert (np.abs(w[0] - total[0]) <= rel * total[0] + 2.0 ** -22 * total.max())[behind].all()
    assert (np.abs(w[1:] - total[1:]) <= rel * total[1:] + 2.0 ** -22 * total.max()).all()
