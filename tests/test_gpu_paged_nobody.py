"""GPU: rows of a batch's buffers that belong to no sequence.  They are there
(preparation may load them), and whatever they hold, results have the same bits
and their own rows of the results stay as they were."""
import numpy as np
import pytest

from kv_ops_util import Dev
from kv_pages_util import Batch, HostPages
from test_gpu_paged_rows import axis_map
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


@pytest.mark.parametrize("n_tok,dtype", [(1, "f32"), (40, "bf16"), (1100, "f32")])
def test_rows_of_nobody_change_nothing(eng, n_tok, dtype):
    """Before the first sequence's tokens and behind the last one's: whatever
    values and positions the rows hold, the others' results have the same bits."""
    r = np.random.default_rng(n_tok)
    n_head, n_kv, hd, page, lead, tail = 4, 2, 64, 16, 3, 5
    b = Batch([n_tok + 20], [n_tok], page, seed=2, tail=lead + tail)
    b.start = np.array([lead, lead + n_tok], np.int32)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=3, zero=True)
    n, per, wide = b.n_tok, n_kv * hd, n_head * hd
    clean = r.standard_normal((n, wide + 2 * per)).astype(np.float32)
    nobody = np.r_[0:lead, lead + n_tok:n]
    pos = r.integers(0, 9000, (3, n)).astype(np.int32)
    kind = engine.DTYPE_BF16 if dtype == "bf16" else engine.DTYPE_F32
    struct, _ = axis_map("interleaved", hd // 2)
    norm = np.ones(hd, np.float32)
    results = []
    for value, where in ((0.0, 0), (np.nan, -2 ** 31), (np.inf, 2 ** 31 - 1)):
        x, at = clean.copy(), pos.copy()
        x[nobody], at[:, nobody] = value, where
        if dtype == "bf16":
            x = np.ascontiguousarray(x).view(np.uint32) >> 16
            x = x.astype(np.uint16)
        esz = x.itemsize
        with Dev(eng) as d:
            dx, g, db = d.put(x), host.upload(eng), b.put(d)
            p = engine.GqaParams(d.put(norm).ptr, d.put(norm).ptr, 0, 0, 0, n_head, 0, hd, 1, 1e4, 1e-6)
            q, k, v = (d.put(np.full((n, w), 7.0, np.float32)) for w in (wide, per, per))
            g.prep(db, p, dx.ptr, dx.ptr + wide * esz, dx.ptr + (wide + per) * esz, q.ptr, 0, struct, d.put(at).ptr,
                   wide + 2 * per, wide + 2 * per, kind, eng.stream)
            g.read(db, k.ptr, v.ptr, stream=eng.stream)
            eng.synchronize()
            results.append([q.download(np.float32, (n, wide)), k.download(np.float32, (n, per)),
                            v.download(np.float32, (n, per))] + list(host.download(g).values()))
            g.free()
    for got in results:
        for a, first in zip(got, results[0]):
            assert np.array_equal(a, first)
        for a in got[:3]:
            assert np.all(a[nobody] == 7.0) and np.isfinite(a).all()
