"""GPU: the paged operators in the forms that their sizes choose: attention of
one token a sequence in blocks of four query rows, with what masks and stores it
has; preparation of several tokens to a workgroup; results that the last-level
cache does not hold read back.  Oracles and bars as in kv_pages_util."""
import numpy as np
import pytest

from kv_ops_util import Dev
from kv_pages_util import PLANES, Batch, HostPages, paged_attention, prepared, quantise, to_bf16
from test_gpu_paged_attn import check, queries, run
from test_gpu_paged_rows import axis_map
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


# ---- attention: up to four heads to a kv head and no more tokens than sequences ----

GROUPS = [(4, 1), (2, 2), (4, 2), (6, 2), (3, 1)]


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n_head,n_kv", GROUPS)
@pytest.mark.parametrize("new", [None, [1, 0, 2, 0, 2], [3, 1, 0, 0, 1]], ids=str)
def test_four_rows_to_a_block(eng, hd, n_head, n_kv, new):
    """Split and whole sequences, a page that is none, NaN and infinite scales
    behind every sequence's last row, a gate, both types; `new` None: one token
    each and no ranges."""
    bare = new is None
    b = Batch([260, 100, 77, 131, 1023], new or [1] * 5, 32, seed=hd + n_head, bare=bare)
    b.table[3, 1] = b.n_pages + 5
    assert b.n_tok <= b.n_seq and n_head // n_kv <= 4
    host = HostPages(b.n_pages, 32, n_kv, hd, seed=n_head)
    for i in (0, 1, 2, 4):
        host.v_d[b.table[i, b.lens[i] // 32], :, b.lens[i] % 32:] = np.nan
        host.k_d[b.table[i, b.lens[i] // 32], :, b.lens[i] % 32:] = np.inf
    q, gate = queries(b, n_head, hd, 3), queries(b, n_head, hd, 4)
    with np.errstate(invalid="ignore"):
        want, bar = paged_attention(host, b, q, n_head, gate)
        plain, plain_bar = paged_attention(host, b, q, n_head)
    for dtype in ("f32", "bf16"):
        check(run(eng, host, b, n_head, q, gate, dtype), want, bar, dtype)
    out = run(eng, host, b, n_head, q)
    check(out, plain, plain_bar)
    assert np.array_equal(out, run(eng, host, b, n_head, q))


@pytest.mark.parametrize("hd,page", [(32, 16), (128, 16), (128, 64), (128, 128), (256, 16)])
def test_four_rows_lengths_and_pages(eng, hd, page):
    """Every end of a tile and a page, sequences of none, tokens that see nothing."""
    lens = [1, 15, 16, 17, 31, 32, 33, 0, 47, 127, 128, 129, 4097, 2 * page, page + 1]
    b = Batch(lens, [1] * len(lens), page, seed=page, bare=True)
    b.table[-1, :] = -3                               # no page at all
    host = HostPages(b.n_pages, page, 2, hd, seed=1)
    q = queries(b, 8, hd, 2)
    want, bar = paged_attention(host, b, q, 8)
    assert np.all(want[7] == 0) and np.all(want[-1] == 0)
    check(run(eng, host, b, 8, q), want, bar)


@pytest.mark.parametrize("hd", [32, 128, 256])
def test_four_rows_scales_and_scores_far_apart(eng, hd):
    """V's scales grow along the rows by powers of two, 2^-14 beside 2^14;
    queries of three sizes."""
    b = Batch([700, 64, 90], [1, 1, 1], 32, seed=3, bare=True)
    host = HostPages(b.n_pages, 32, 2, hd, seed=2)
    for j in range(-(-700 // 32)):
        host.v_d[b.table[0, j]] = np.float16(2.0 ** (j - 14))
    host.v_d[b.table[1, 0]], host.v_d[b.table[1, 1]] = np.float16(2.0 ** -14), np.float16(2.0 ** 14)
    q = queries(b, 8, hd, 3)
    for scale in (2.0 ** -20, 1.0, 2.0 ** 9):
        x = q * np.float32(scale)
        check(run(eng, host, b, 8, x), *paged_attention(host, b, x, 8))


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_four_rows_of_values_that_are_not_finite(eng, hd):
    """A query of NaN stays with its row; a row of NaN in the pages with the
    sequence that sees it."""
    b = Batch([300, 90, 40], [1, 1, 1], 16, seed=3, bare=True)
    host = HostPages(b.n_pages, 16, 2, hd, seed=2)
    q = queries(b, 8, hd, 3)
    want, bar = paged_attention(host, b, q, 8)
    want, bar = want.reshape(3, 8, hd), bar.reshape(3, 8, hd)
    bad = q.reshape(3, 8, hd).copy()
    bad[0, 5, 7] = np.nan
    host.v_d[b.table[1, 2], 1, 3] = np.nan            # kv head 1 of sequence 1
    host.k_d[b.table[2, 0], 0, 9] = np.nan            # kv head 0 of sequence 2
    out = run(eng, host, b, 8, bad.reshape(3, -1)).reshape(want.shape)
    broken = np.zeros((3, 8), bool)
    broken[0, 5] = broken[1, 4:] = broken[2, :4] = True
    assert np.isnan(out[broken]).all()
    assert np.all(np.abs(out - want)[~broken] <= bar[~broken])


def test_four_rows_captured(eng):
    """One graph over one token a sequence at 128 dims, replayed while lengths
    and tables change, against the formula at every replay."""
    n_kv, hd, page, n_head = 2, 128, 32, 8
    b = Batch([900] * 4, [1] * 4, page, seed=9, bare=True)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=2)
    q = queries(b, n_head, hd, 3)
    r = np.random.default_rng(1)
    with Dev(eng) as d:
        g, db, dq, do = host.upload(eng), b.put(d), d.put(q), d.put(np.zeros_like(q))
        g.attend(db, dq.ptr, n_head, do.ptr, stream=eng.stream)
        eng.synchronize()
        graph = eng.capture(lambda s: g.attend(db, dq.ptr, n_head, do.ptr, stream=s))
        for lens in ([1, 2, 3, 4], [900, 3, 17, 130], [900] * 4, [0, 33, 1, 899], [128, 129, 256, 257]):
            b.lens[:], b.row[:] = lens, np.array(lens) - 1
            b.table[:] = np.roll(b.table, 1, axis=0)
            q = r.permutation(q)
            for buf, a in zip(b.dev + [dq, do], (b.table, b.lens, q, np.full_like(q, 5.0))):
                buf.upload(a)
            graph.launch()
            eng.synchronize()
            check(do.download(np.float32, q.shape), *paged_attention(host, b, q, n_head))
        graph.free()
        g.free()


# ---- preparation: more than 1,023 tokens, two to eight to a workgroup ----

@pytest.mark.parametrize("new,n_head,n_kv,hd,gated,neox,axes,rope_dim,dtype", [
    ([700, 0, 3, 328], 4, 1, 64, True, 1, "interleaved", 64, "bf16"),     # 1,033 with the tail: two, the last alone
    ([1] * 130 + [900, 2, 560], 2, 2, 32, False, 1, "one", 32, "f32"),    # 1,594: three
    ([2600], 3, 3, 128, True, 0, "sections", 96, "f32"),                  # 2,602: five
    ([4000, 1, 98], 5, 1, 64, False, 1, "sections", 40, "bf16"),          # 4,101: eight, the last five
    ([513, 520], 9, 1, 256, False, 1, "one", 256, "f32"),                 # 1,035
], ids=lambda v: str(v)[:24])
def test_several_tokens_to_a_workgroup(eng, new, n_head, n_kv, hd, gated, neox, axes, rope_dim, dtype):
    r = np.random.default_rng(hd + len(new))
    page, tail = 64, 2
    past = r.integers(0, 90, len(new))
    b = Batch(np.asarray(new) + past, new, page, seed=len(new), tail=tail)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=3)
    n, per, q_rows = b.n_tok, n_kv * hd, n_head * hd * (2 if gated else 1)
    assert n >= 1024
    width = q_rows + 2 * per
    x = (r.standard_normal((n, width)) * np.exp(r.uniform(-2, 2, (n, 1)))).astype(np.float32)
    x[n - tail:] = np.nan                             # rows of nobody may hold anything
    raw = x
    if dtype == "bf16":
        raw, x = to_bf16(np.nan_to_num(x))
        raw[n - tail:] = 0x7FC0
    qn, kn = ((r.standard_normal(hd) * 0.3 + 1).astype(np.float32) for _ in range(2))
    struct, at = axis_map(axes, min(rope_dim, hd) // 2)
    pos = None
    if axes != "one":
        pos = r.integers(0, 70000, (3, n)).astype(np.int32)
        pos[:, n - tail:] = -2 ** 31
    esz = raw.itemsize
    with Dev(eng) as d:
        dx, g, db = d.put(raw), host.upload(eng), b.put(d)
        p = engine.GqaParams(d.put(qn).ptr, d.put(kn).ptr, 0, 0, 0, n_head, int(gated), rope_dim, neox, 1e4, 1e-6)
        fill = np.full((n, n_head * hd), 7.0, np.float32)
        dq, dg = d.put(fill), d.put(fill)
        g.prep(db, p, dx.ptr, dx.ptr + q_rows * esz, dx.ptr + (q_rows + per) * esz, dq.ptr, dg.ptr if gated else 0, struct,
               0 if pos is None else d.put(pos).ptr, width, width,
               engine.DTYPE_BF16 if dtype == "bf16" else engine.DTYPE_F32, eng.stream)
        eng.synchronize()
        got_q, got_g, got = dq.download(np.float32, fill.shape), dg.download(np.float32, fill.shape), host.download(g)
        g.free()
    mine = b.owner >= 0
    assert mine.sum() == n - tail
    where = np.where(mine, b.row, 0)[None].repeat(3, 0) if pos is None else pos
    x, where = np.where(mine[:, None], x, 0), np.where(mine, where, 0)
    q = x[:, :q_rows].reshape(n, n_head, -1)
    want = prepared(q[..., :hd], qn, None, where, at, rope_dim, 1e4, neox, 1e-6)
    bar = 2.0 ** -24 * np.abs(want) + 2.0 ** -45 * np.abs(want).max(-1, keepdims=True)
    assert np.all(np.abs(got_q.reshape(want.shape) - want)[mine] <= bar[mine])
    if gated:
        assert np.array_equal(got_g.reshape(n, n_head, hd)[mine], q[..., hd:][mine])
    assert np.all(got_q[~mine] == 7.0) and np.all(got_g[~mine if gated else slice(None)] == 7.0)
    k = prepared(x[:, q_rows:q_rows + per].reshape(n, n_kv, hd), kn, None, where, at, rope_dim, 1e4, neox, 1e-6)
    held = host.bits()
    to = b.table[b.owner[mine], b.row[mine] // page], slice(None), b.row[mine] % page
    for name, rows in (("k", k.astype(np.float32)), ("v", x[:, q_rows + per:].reshape(n, n_kv, hd))):
        qs, dd = quantise(rows[mine])
        held[name + "_qs"][to], held[name + "_d"][to] = qs, dd.view(np.uint16)
    for m in PLANES:
        assert np.array_equal(got[m], held[m]), m


# ---- read-back of results of 2^28 bytes ----

@pytest.mark.parametrize("n_kv,hd,dtype", [(8, 128, "f32"), (16, 128, "bf16")])
def test_results_past_the_last_level_cache(eng, n_kv, hd, dtype):
    """Sequences of 20,001 and 13,000 rows on a few pages that they share."""
    page, lens = 128, [20001, 13000]
    b = Batch([page * 6], [1], page, seed=1, spare_pages=0)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=2)
    r = np.random.default_rng(3)
    table = r.integers(0, b.n_pages, (2, 160)).astype(np.int32)
    table[0, 40], table[1, 101] = -1, b.n_pages       # no pages: zeros
    start = np.array([0, 20001, 33001], np.int32)
    n, per = 33004, n_kv * hd
    kind = np.uint16 if dtype == "bf16" else np.float32
    assert 2 * n * per * np.dtype(kind).itemsize >= 1 << 28
    with Dev(eng) as d:
        g = host.upload(eng)
        dt, dl, ds = d.put(table), d.put(np.array(lens, np.int32)), d.put(start)
        db = engine.PagedBatch(dt.ptr, dl.ptr, ds.ptr, 2, table.shape[1], n)
        fill = np.full((n, per), 77, kind)
        ko, vo = d.put(fill), d.put(fill)
        g.read(db, ko.ptr, vo.ptr, engine.DTYPE_BF16 if dtype == "bf16" else engine.DTYPE_F32, stream=eng.stream)
        eng.synchronize()
        for x, buf in (("k", ko), ("v", vo)):
            got = buf.download(kind, fill.shape)
            assert np.all(got[start[-1]:] == 77)
            for i, rows in enumerate(lens):
                for a in range(0, rows, 4000):        # in pieces: the oracle is in 64 bits
                    at = np.arange(a, min(a + 4000, rows))
                    no = table[i, at // page]
                    ok = host.good(no)
                    where = np.where(ok, no, 0), slice(None), at % page
                    want = (getattr(host, x + "_qs")[where].astype(np.float32)
                            * np.repeat(getattr(host, x + "_d")[where].astype(np.float32), 32, -1)).reshape(-1, per)
                    want = np.where(ok[:, None], want, np.float32(0))
                    have = got[start[i] + a:start[i] + a + len(at)]
                    assert np.array_equal(have, to_bf16(want)[0] if dtype == "bf16" else want), (x, i, a)
        g.free()
