"""GPU parity of a drafted tree's whole attention step
(``vxt_hip_attn_tree_step_q8_dev``) with the oracle's restatement of
step_full_gqa_q8 (llm_prefill.rs:259-367): each node prepared by it at the
tree's cache row and at its depth's position, attention by it over the rows the
node sees.  Bars as for a plain step (test_gpu_attn_step): V's cache rows bit
for bit, K's within a quantisation step, outputs within 1e-4 max|V|."""
import numpy as np
import pytest

import oracle
from kv_ops_util import ancestors, depths, random_tree
from test_gpu_attn_step import Case, check_k_cache, empty_blocks
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


@pytest.mark.parametrize("n_head,n_kv,hd,gated,norms,neox,rope_dim,biases,n,pos,rope_pos,kind", [
    (8, 2, 64, True, True, True, 64, False, 21, 60, 1000, "mixed"),
    (16, 4, 128, True, True, True, 32, True, 40, 100, 30000, "mixed"),
    (8, 8, 128, False, True, False, 128, False, 9, 0, 0, "chain"),
    (4, 1, 256, True, False, False, 64, True, 12, 33, 123456, "mixed"),
    (6, 2, 64, False, False, True, 64, True, 1, 9, 9, "mixed"),
    (2, 2, 32, True, True, False, 7, False, 30, 1, 40, "roots"),
    (4, 2, 64, False, False, False, 0, False, 64, 5, 70, "mixed")])
def test_tree_step_parity(eng, n_head, n_kv, hd, gated, norms, neox, rope_dim, biases, n, pos, rope_pos, kind):
    case = Case(eng, n_head, n_kv, hd, gated, norms, neox, rope_dim, biases, seed=hd + n)
    cache = eng.kv_q8_cache(pos + n, n_kv, hd)
    parents = random_tree(n, n, kind)
    kb, vb = empty_blocks(pos + n, case.kvd), empty_blocks(pos + n, case.kvd)
    per = case.kvd // 32
    bufs = []
    try:
        for t in range(pos):                 # the committed rows
            _, k, v = case.tokens(1)
            bk, bv = eng.to_device(k), eng.to_device(v)
            cache.append(bk.ptr, bv.ptr, t, eng.stream)
            eng.synchronize()
            bk.free()
            bv.free()
        if pos:
            kb[:pos * per], vb[:pos * per] = (cache.blocks(x, pos).reshape(-1, 34) for x in "kv")
        q, k, v = case.tokens(n)
        bufs = [eng.to_device(np.ascontiguousarray(x)) for x in (q, k, v, parents)]
        out = eng.alloc(4 * n * n_head * hd)
        bufs.append(out)
        cache.step_tree(case.params, bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, bufs[3].ptr, n, pos, rope_pos, out.ptr,
                        q_stride=case.p.q_rows, kv_stride=case.kvd, stream=eng.stream)
        eng.synchronize()
        got = out.download(np.float32, (n, n_head * hd))
        qi, ki, vi = case.host_inputs(q, k, v)
        heads = [case.p.prep(qi[i], ki[i], vi[i], kb, vb, pos + i, rope_pos + depth)[:2]
                 for i, depth in enumerate(depths(parents))]
        k_dev, v_dev = (cache.blocks(x, pos + n).reshape(-1, 34) for x in "kv")
        assert np.array_equal(v_dev, vb)
        check_k_cache(k_dev, kb, case.exact_k)
        sees = ancestors(parents)
        for i, (qh, qg) in enumerate(heads):
            rows = np.concatenate([np.arange(pos), pos + np.flatnonzero(sees[i])])
            bk, bv = (np.ascontiguousarray(x.reshape(pos + n, per, 34)[rows]) for x in (k_dev, v_dev))
            ref = oracle.attn_q8(qh, bk, bv, rows.size, n_head, n_kv, hd, gate=qg)
            assert np.abs(got[i] - ref).max() <= 1e-4 * np.abs(oracle.q8_dequant(bv.reshape(-1))).max(), i
    finally:
        for b in bufs:
            b.free()
        cache.free()
        case.free()
