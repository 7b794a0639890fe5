"""GPU: how many bits the operands of attention over the Q8_0 KV cache keep --
drafted trees, weighed tokens and prompts, selected blocks -- by the bars of
kv_ops_bits, which derives them."""
import numpy as np
import pytest

from kv_ops_bits import row_bar, row_errors, sink, sink_bar
from kv_ops_util import Dev, HostCache, ancestors, attention, random_tree
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def run(eng, host, q, form, block=32, n_sel=0):
    """(out, sees) of the last rows' tokens by one of the calls."""
    m, width = q.shape
    n_head, pos = width // host.hd, host.rows - m
    sees = np.arange(host.rows)[None] <= pos + np.arange(m)[:, None]
    cache = host.upload(eng)
    held = [cache]
    with Dev(eng) as d:
        out, Q = d.room(q.nbytes), d.put(q).ptr
        if form == "tree":
            parents = random_tree(m, m)
            sees[:, pos:] = ancestors(parents)
            cache.attend_tree(Q, n_head, d.put(parents).ptr, m, pos, out.ptr, 0, eng.stream)
        elif form == "weigh":
            w = eng.kv_weights(host.rows, host.n_kv)
            held.append(w)
            w.weight.upload(np.zeros((host.n_kv, host.rows), np.float32))
            cache.attend_weigh(w, Q, n_head, m, pos, 0, out.ptr, 0, eng.stream)
        else:
            nb = (host.rows - 1) // block + 1
            n_sel = n_sel or nb
            means, sel = eng.kv_block_means(nb, block, host.n_kv, host.hd), d.room(4 * m * host.n_kv * n_sel)
            held.append(means)
            cache.block_means(means, 0, host.rows, eng.stream)
            cache.attend_blocks(means, Q, n_head, m, pos, n_sel, 1, 1, out.ptr, 0, sel.ptr, eng.stream)
            eng.synchronize()
            taken = sel.download(np.uint32, (m, host.n_kv, n_sel))
            of = np.arange(host.rows) // block
            sees = sees[:, None] & (taken[:, :, :, None] == of).any(2)
        eng.synchronize()
        got = out.download(np.float32, q.shape)
    for b in held:
        b.free()
    return got, sees


RANDOM = [
    # form, tokens, rows, n_head, n_kv, hd, block, n_sel
    ("tree", 1, 500, 4, 4, 32, 0, 0), ("tree", 5, 155, 8, 2, 64, 0, 0), ("tree", 26, 2073, 16, 4, 128, 0, 0),
    ("tree", 64, 764, 10, 2, 128, 0, 0), ("tree", 7, 2040, 2, 2, 256, 0, 0), ("tree", 200, 1200, 4, 2, 64, 0, 0),
    ("weigh", 1, 1000, 16, 4, 128, 0, 0), ("weigh", 1, 9000, 8, 2, 64, 0, 0), ("weigh", 1, 5000, 2, 1, 256, 0, 0),
    ("weigh", 1, 5000, 4, 2, 32, 0, 0), ("weigh", 17, 60, 10, 2, 32, 0, 0), ("weigh", 130, 191, 7, 1, 64, 0, 0),
    ("weigh", 300, 300, 16, 4, 128, 0, 0), ("weigh", 40, 740, 4, 2, 256, 0, 0),
    ("blocks", 1, 1000, 16, 4, 128, 64, 8), ("blocks", 1, 5000, 8, 1, 64, 32, 40), ("blocks", 40, 940, 16, 4, 128, 64, 8),
    ("blocks", 9, 700, 2, 2, 256, 128, 3), ("blocks", 17, 517, 10, 2, 32, 32, 6), ("blocks", 2, 9000, 4, 2, 64, 64, 0),
]


@pytest.mark.parametrize("case", RANDOM, ids=lambda c: "-".join(map(str, c)))
def test_errors_to_the_outputs_norm(eng, case):
    form, m, rows, n_head, n_kv, hd, block, n_sel = case
    host = HostCache(rows, n_kv, hd, seed=rows + m)
    q = np.random.default_rng(m).standard_normal((m, n_head * hd)).astype(np.float32)
    got, sees = run(eng, host, q, form, block, n_sel)
    ref, _, _, _ = attention(host, q, sees)
    assert row_errors(got, ref, hd).max() <= row_bar(host, q, rows)


@pytest.mark.parametrize("form,m,rows,n_head,n_kv,hd,block", [
    ("weigh", 1, 1024, 4, 2, 64, 0), ("weigh", 1, 4000, 8, 1, 128, 0), ("weigh", 1, 700, 2, 1, 256, 0),
    ("weigh", 1, 3000, 3, 1, 32, 0), ("weigh", 6, 1030, 4, 2, 64, 0), ("weigh", 70, 1100, 8, 2, 128, 0),
    ("tree", 1, 1000, 4, 1, 64, 0), ("tree", 9, 3000, 8, 2, 128, 0), ("tree", 60, 1100, 4, 2, 256, 0),
    ("tree", 250, 4000, 64, 16, 64, 0), ("weigh", 500, 2000, 64, 16, 64, 0),
    ("blocks", 1, 1024, 4, 1, 128, 64), ("blocks", 1, 3999, 8, 2, 64, 32), ("blocks", 200, 3000, 16, 4, 128, 64),
    ("blocks", 150, 2000, 8, 8, 64, 128)])
@pytest.mark.parametrize("gap", [8, 10, 12])
def test_a_row_far_above_the_others(eng, form, m, rows, n_head, n_kv, hd, block, gap):
    """What the others add to the output is as exact as f32 weights make it,
    though one row, of value zero, has almost all of the weight."""
    host, q, g = sink(rows, n_kv, hd, gap, m, n_head, seed=rows)
    got, sees = run(eng, host, q, form, block)
    ref, _, _, _ = attention(host, q, sees)
    assert np.abs(got / ref - 1).max() <= sink_bar(g, rows)


LARGE = [("weigh", 1, 1024, 4, 2, 64, 0), ("weigh", 1, 700, 2, 1, 256, 0), ("blocks", 1, 1024, 4, 1, 128, 64),
         ("blocks", 200, 1500, 4, 1, 64, 64), ("weigh", 70, 1100, 8, 2, 128, 0), ("tree", 9, 3000, 8, 2, 128, 0)]


@pytest.mark.parametrize("case,large", [(c, x) for c in LARGE for x in (0.9, 300.0, 60000.0) if x < 1e4 or c in LARGE[:4]])
def test_a_scale_far_above_the_others(eng, case, large):
    """All rows weigh alike; one has a large scale and codes of zero.  By
    kv_ops.hpp a product of weight and scale is right to 2^-36 of the weight
    times the largest scale, a weight to 2^-38 of one times the power of two
    that the largest scale takes from it; in the rows kernel a scale to 2^-31 of
    the largest, a thousandth of 0.0101 at 60000, which is left out."""
    form, m, rows, n_head, n_kv, hd, block = case
    host, q, _ = sink(rows, n_kv, hd, 0, m, n_head, seed=rows)
    host.v_qs[0] = 64
    host.v_d[:] = 0.0101
    host.v_qs[7], host.v_d[7] = 0, large
    got, sees = run(eng, host, q, form, block)
    ref, _, _, _ = attention(host, q, sees)
    bar = 2.0 ** -21 + 2 * (rows / 16 + 64) * 2.0 ** -24 + 2.0 ** -36 * large / 0.0101 + 2.0 ** -37 * max(1, large)
    if case not in LARGE[:4]:
        bar += 2.0 ** -31 * large / 0.0101
    assert np.abs(got / ref - 1).max() <= bar
