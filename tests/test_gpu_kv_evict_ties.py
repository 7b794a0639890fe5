"""GPU parity of eviction (``vxt_hip_kv_q8_evict_dev``) where the threshold
falls among equal weights of many rows: which of them stay goes by the row,
whatever the row count is to a power of two."""
import numpy as np
import pytest

from kv_ops_util import HostCache
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def sources(weight, position, keep, n_tokens, n_recent, n_first):
    """Source row of every kept row of a head, by the rule: protected rows,
    then by weight, NaN last, the lower row among equals."""
    seq = weight.size
    safe = (position < n_first) | (position.astype(np.int64) >= n_tokens - n_recent)
    rank = np.where(safe, np.inf, np.where(np.isnan(weight), -np.inf, weight))
    order = np.lexsort((np.arange(seq), -rank, np.isnan(weight) & ~safe, ~safe))
    kept = np.zeros(seq, bool)
    kept[order[:keep]] = True
    src = np.arange(keep)
    src[~kept[:keep]] = np.flatnonzero(kept[keep:]) + keep
    return src


def weights_of(kind, seq, keep, r):
    w = np.full(seq, 1.5, np.float32)
    if kind == "a pair":             # two early neighbours at the threshold, of which one stays
        w = r.permutation(np.arange(2, seq + 2)).astype(np.float32) * np.float32(2.0 ** -21)
        order = np.argsort(-w)
        at = 480
        w[[at, order[keep - 1]]] = w[[order[keep - 1], at]]
        j = int(np.flatnonzero(w == np.sort(w)[seq - keep - 1])[0])
        w[[at + 1, j]] = w[[j, at + 1]]
        w[at + 1] = w[at]
    if kind == "a few":
        w[:] = r.permutation(seq).astype(np.float32)
        w[r.choice(4000, 900, replace=False)] = np.float32(seq)
    if kind == "zeros":
        w[:] = 0
        w[r.choice(seq, min(keep // 3, seq), replace=False)] = 2
    return w


@pytest.mark.parametrize("seq,keep", [(300001, 1), (300001, 27), (300001, 530), (300001, 150000), (1000001, 1), (1000001, 2),
                                      (1000001, 50), (1000001, 999999), (262145, 3), (524287, 1000)])
@pytest.mark.parametrize("kind", ["equal", "a pair", "a few", "zeros"])
def test_threshold_among_equals(eng, kind, seq, keep):
    n_kv, hd = 1, 32
    r = np.random.default_rng(seq + keep)
    host = HostCache(seq, n_kv, hd, seed=1)
    w = weights_of(kind, seq, keep, r)[None]
    position = np.arange(seq, dtype=np.uint32)[None]
    n_first, n_recent = (0, 0) if keep < 20 else (2, 5)
    src = sources(w[0], position[0], keep, seq, n_recent, n_first)
    cache, weights = host.upload(eng), eng.kv_weights(seq, n_kv)
    to, tw = eng.kv_q8_cache(keep, n_kv, hd), eng.kv_weights(keep, n_kv)
    weights.weight.upload(w)
    weights.position.upload(position)
    bits = host.bits(slice(None))
    print(kind, seq, keep, flush=True)
    cache.evict(weights, seq, keep, seq, n_recent, n_first, to, tw, eng.stream)
    cache.evict(weights, seq, keep, seq, n_recent, n_first, stream=eng.stream)
    eng.synchronize()
    for c, planes in ((to, tw), (cache, weights)):
        assert np.array_equal(planes.position.download(np.uint32, (planes.max_seq,))[:keep], position[0][src])
        assert np.array_equal(planes.weight.download(np.float32, (planes.max_seq,))[:keep], w[0][src])
        got = HostCache.download(c, c.max_seq)
        for x, b in bits.items():
            assert np.array_equal(got[x][:keep], b[src]), x
            assert np.array_equal(got[x][keep:], b[keep:] if c is cache else b[:0]), x
    for b in (cache, weights, to, tw):
        b.free()
