"""GPU: rows of a paged cache written (head norms, rotation by one axis or
several, quantised) and read back.  Queries to one rounding from 64 bits, codes,
scales and values read back to the bit; what belongs to nobody stays as it was."""
import ctypes as C

import numpy as np
import pytest

from kv_ops_util import Dev
from kv_pages_util import PLANES, Batch, HostPages, prepared, quantise, to_bf16
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def axis_map(kind, half):
    if kind == "one":
        return None, [0] * half
    a = [i % 3 for i in range(half)] if kind == "interleaved" else [0] * (half // 4) + [1] * (half // 2) + [2] * (half - half // 4 - half // 2)
    return engine.RopeAxes(3, (C.c_uint8 * 128)(*a)), a


CASES = [
    # n_head, n_kv, hd, page, lens, new, gated, neox, axes, rope_dim, norms, biases, dtype
    (8, 2, 64, 16, [5, 33, 16], [1, 1, 1], True, 1, "one", 64, True, False, "f32"),
    (4, 4, 128, 32, [40, 1, 0, 70], [33, 1, 0, 2], False, 0, "sections", 128, True, True, "f32"),
    (5, 1, 256, 64, [300], [300], True, 1, "interleaved", 256, True, False, "bf16"),
    (7, 7, 32, 128, [130, 129], [130, 3], False, 1, "one", 20, False, True, "bf16"),
    (16, 2, 128, 128, [1000, 17, 129, 128, 127, 2], [1, 1, 1, 1, 1, 1], True, 0, "interleaved", 64, True, False, "bf16"),
    (3, 3, 64, 16, [50, 60], [7, 60], False, 1, "sections", 7, True, True, "f32"),      # an odd rope_dim: three pairs
    (2, 1, 32, 16, [9], [9], False, 1, "one", 0, False, False, "f32"),                  # nothing but rounding
    (40, 8, 64, 32, [64] * 70, [1] * 70, False, 1, "one", 64, True, False, "f32"),      # more heads than waves, 70 sequences
]


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,new,gated,neox,axes,rope_dim,norms,biases,dtype,bare",
                         [c + (False,) for c in CASES] + [c + (True,) for c in CASES if set(c[5]) == {1}])
def test_written_rows(eng, n_head, n_kv, hd, page, lens, new, gated, neox, axes, rope_dim, norms, biases, dtype, bare):
    r = np.random.default_rng(hd + len(lens))
    b = Batch(lens, new, page, seed=len(lens), tail=0 if bare else 2, bare=bare)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=3)
    n, per, q_rows = b.n_tok, n_kv * hd, n_head * hd * (2 if gated else 1)
    width = q_rows + 2 * per + 3            # rows further apart than they are wide, odd
    x = (r.standard_normal((n, width)) * np.exp(r.uniform(-3, 3, (n, 1)))).astype(np.float32)
    x[0, :32] = 0
    if dtype == "bf16":
        raw, x = to_bf16(x)
    else:
        raw = x
    qn, kn = ((r.standard_normal(hd) * 0.3 + 1).astype(np.float32) for _ in range(2))
    qb, kb, vb = (r.standard_normal(k).astype(np.float32) for k in (q_rows, per, per))
    struct, at = axis_map(axes, min(rope_dim, hd) // 2)
    pos = None if axes == "one" else r.integers(0, 70000, (3, n)).astype(np.int32)
    esz = raw.itemsize
    with Dev(eng) as d:
        dx = d.put(raw)
        p = engine.GqaParams(d.put(qn).ptr if norms else 0, d.put(kn).ptr if norms else 0, d.put(qb).ptr if biases else 0,
                             d.put(kb).ptr if biases else 0, d.put(vb).ptr if biases else 0, n_head, int(gated), rope_dim,
                             neox, 1e6 if hd == 128 else 1e4, 1e-6)
        g = host.upload(eng)
        fill = np.full((n, n_head * hd), 7.0, np.float32)
        dq, dg, db = d.put(fill), d.put(fill), b.put(d)
        dt = engine.DTYPE_BF16 if dtype == "bf16" else engine.DTYPE_F32
        g.prep(db, p, dx.ptr, dx.ptr + q_rows * esz, dx.ptr + (q_rows + per) * esz, dq.ptr, dg.ptr if gated else 0, struct,
               0 if pos is None else d.put(pos).ptr, width, width, dt, eng.stream)
        ko, vo = (d.put(np.full((n, per + 5), 9.0, np.float32)) for _ in range(2))
        g.read(db, ko.ptr, vo.ptr, engine.DTYPE_F32, per + 5, eng.stream)
        eng.synchronize()
        got_q, got_g = dq.download(np.float32, fill.shape), dg.download(np.float32, fill.shape)
        got_k, got_v = (a.download(np.float32, (n, per + 5)) for a in (ko, vo))
        got = host.download(g)
        g.free()

    mine = b.owner >= 0
    where = np.where(mine, b.row, 0)[None].repeat(3, 0) if pos is None else pos
    q = x[:, :q_rows].reshape(n, n_head, -1)
    if biases:
        q = q.astype(np.float64) + qb.reshape(n_head, -1)
    want = prepared(q[..., :hd], qn if norms else None, None, where, at, rope_dim, p.rope_freq_base, neox, 1e-6)
    bar = 2.0 ** -24 * np.abs(want) + 2.0 ** -45 * np.abs(want).max(-1, keepdims=True)
    have = got_q.reshape(n, n_head, hd)
    assert np.all(np.abs(have - want)[mine] <= bar[mine])
    assert np.all(got_q[~mine] == 7.0)
    if gated:
        assert np.array_equal(got_g.reshape(n, n_head, hd)[mine], q[..., hd:].astype(np.float32)[mine])
    assert np.all(got_g[~mine if gated else slice(None)] == 7.0)

    k, v = x[:, q_rows:q_rows + per].reshape(n, n_kv, hd), x[:, q_rows + per:q_rows + 2 * per].reshape(n, n_kv, hd)
    if biases:
        v = (v.astype(np.float64) + vb.reshape(n_kv, hd)).astype(np.float32)
    k = prepared(k, kn if norms else None, kb.reshape(n_kv, hd) if biases else None, where, at, rope_dim, p.rope_freq_base,
                 neox, 1e-6).astype(np.float32)
    want = {m: a.copy() for m, a in host.bits().items()}
    for t in np.flatnonzero(mine):
        page_no, in_page = b.table[b.owner[t], b.row[t] // page], b.row[t] % page
        for name, rows, back in (("k", k, got_k), ("v", v, got_v)):
            qs, dd = quantise(rows[t])
            want[name + "_qs"][page_no, :, in_page], want[name + "_d"][page_no, :, in_page] = qs, dd.view(np.uint16)
            values = qs.astype(np.float32) * np.repeat(dd.astype(np.float32), 32, -1)
            assert np.array_equal(back[t, :per], values.reshape(-1)), (t, name)
    for m in PLANES:
        assert np.array_equal(got[m], want[m]), m
    for back in (got_k, got_v):
        assert np.all(back[~mine] == 9.0) and np.all(back[:, per:] == 9.0)


def test_tokens_without_a_row_or_a_page(eng):
    """More tokens than rows, pages that are none, lengths past the table: nothing
    written, zeros read, the others as ever."""
    n_kv, hd, page = 2, 64, 16
    b = Batch([40, 20, 3], [40, 20, 3], page, seed=5, spare_cols=0)
    b.table[0, 1], b.table[0, 2], b.table[1, 0] = b.n_pages, -7, 2 ** 31 - 1
    b.lens[2] = 2                                      # three tokens, two rows
    host = HostPages(b.n_pages, page, n_kv, hd, seed=1)
    x = np.random.default_rng(0).standard_normal((b.n_tok, n_kv * hd)).astype(np.float32)
    row = np.concatenate([np.arange(40), np.arange(20), [-1, 0, 1]])
    seq = np.repeat([0, 1, 2], [40, 20, 3])
    with Dev(eng) as d:
        g, db, dx = host.upload(eng), b.put(d), d.put(x)
        p = engine.GqaParams(0, 0, 0, 0, 0, 0, 0, 0, 1, 1e4, 0.0)
        g.prep(db, p, 0, dx.ptr, dx.ptr, 0, kv_stride=n_kv * hd, stream=eng.stream)
        ko, vo = (d.put(np.full(x.shape, 9.0, np.float32)) for _ in range(2))
        g.read(db, ko.ptr, vo.ptr, stream=eng.stream)
        eng.synchronize()
        got, k, v = host.download(g), ko.download(np.float32, x.shape), vo.download(np.float32, x.shape)
        g.free()
    want = {m: a.copy() for m, a in host.bits().items()}
    for t in range(b.n_tok):
        page_no = b.table[seq[t], row[t] // page] if row[t] >= 0 else -1
        if not 0 <= page_no < b.n_pages:
            assert np.all(k[t] == 0) and np.all(v[t] == 0)
            continue
        qs, dd = quantise(x[t].reshape(n_kv, hd))
        for m in "kv":
            want[m + "_qs"][page_no, :, row[t] % page], want[m + "_d"][page_no, :, row[t] % page] = qs, dd.view(np.uint16)
        assert np.array_equal(k[t], (qs.astype(np.float32) * np.repeat(dd.astype(np.float32), 32, -1)).reshape(-1))
    for m in PLANES:
        assert np.array_equal(got[m], want[m]), m


@pytest.mark.parametrize("hd,page,n_kv", [(32, 16, 3), (64, 32, 1), (128, 128, 4), (256, 64, 2)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_whole_sequences_read_back(eng, hd, page, n_kv, dtype):
    lens = [1, 0, page, 3 * page + 1, 700]
    b = Batch(lens, lens, page, seed=hd, tail=1)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=hd)
    per = n_kv * hd
    kind = np.uint16 if dtype == "bf16" else np.float32
    with Dev(eng) as d:
        g, db = host.upload(eng), b.put(d)
        fill = np.full((b.n_tok, per), 77, kind)
        ko, vo = d.put(fill), d.put(fill)
        g.read(db, ko.ptr, vo.ptr, engine.DTYPE_BF16 if dtype == "bf16" else engine.DTYPE_F32, stream=eng.stream)
        eng.synchronize()
        got = {"k": ko.download(kind, fill.shape), "v": vo.download(kind, fill.shape)}
        g.free()
    for x in "kv":
        for i, n in enumerate(lens):
            want = host.rows(x, b.table[i], n)[0].reshape(n, per).astype(np.float32)     # exact in f32
            have = got[x][b.start[i]:b.start[i + 1]]
            assert np.array_equal(have, to_bf16(want)[0] if dtype == "bf16" else want)
        assert np.all(got[x][b.start[-1]:] == 77)


def test_values_that_are_not_finite(eng):
    """An infinite value makes its block's scale infinite, NaN counts as nothing
    in a maximum and is code 0: KvQ8Block's rules; neighbours stay."""
    n_kv, hd, page = 1, 64, 16
    b = Batch([4], [4], page, seed=0)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=1)
    x = np.random.default_rng(1).standard_normal((4, hd)).astype(np.float32)
    x[1, 3], x[2, 40], x[3, :] = np.inf, np.nan, 3e38
    with Dev(eng) as d:
        g, db, dx = host.upload(eng), b.put(d), d.put(x)
        g.prep(db, engine.GqaParams(0, 0, 0, 0, 0, 0, 0, 0, 1, 1e4, 0.0), 0, dx.ptr, dx.ptr, 0, kv_stride=hd, stream=eng.stream)
        eng.synchronize()
        got = host.download(g)
        g.free()
    for t in range(4):
        qs, dd = quantise(x[t].reshape(1, hd))
        for m in "kv":
            assert np.array_equal(got[m + "_qs"][b.table[0, 0], :, t], qs), (t, m)
            assert np.array_equal(got[m + "_d"][b.table[0, 0], :, t], dd.view(np.uint16)), (t, m)


def test_far_positions(eng):
    """Angles of positions up to 2^30, where f32 holds no fraction of a turn."""
    n_kv, hd, page = 1, 128, 16
    pos = np.array([[0, 1, 100003, 16777217, 2 ** 30 + 1, -5]], np.int32)
    n = pos.shape[1]
    b = Batch([n], [n], page, seed=0)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=1)
    x = np.random.default_rng(2).standard_normal((n, 3 * hd)).astype(np.float32)
    with Dev(eng) as d:
        g, db, dx, dq = host.upload(eng), b.put(d), d.put(x), d.room(4 * n * hd)
        g.prep(db, engine.GqaParams(0, 0, 0, 0, 0, 1, 0, hd, 1, 1e6, 0.0), dx.ptr, dx.ptr + 4 * hd, dx.ptr + 8 * hd, dq.ptr,
               rope_pos=d.put(pos).ptr, q_stride=3 * hd, kv_stride=3 * hd, stream=eng.stream)
        eng.synchronize()
        got = dq.download(np.float32, (n, 1, hd))
        g.free()
    want = prepared(x[:, None, :hd], None, None, pos, [0] * 64, hd, 1e6, 1, 0.0)
    # pow and the product are good to an ulp each: 2^-52 of an angle, twice
    bar = 2.0 ** -24 * np.abs(want) + (2.0 ** -50 * np.abs(pos[0])[:, None, None] + 2.0 ** -45) * np.abs(want).max()
    assert np.all(np.abs(got - want) <= bar)
