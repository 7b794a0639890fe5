"""GPU: the operators of the paged KV cache and the verification of drafts used
together, as a server's loop uses them, and at the ends of their ranges.  Bars as
where each is tested by itself."""
import numpy as np
import pytest

from kv_ops_util import Dev
from kv_pages_util import PLANES, Batch, HostPages, paged_attention, prepared, quantise
from test_gpu_paged_rows import axis_map
from test_gpu_verify_drafts import Case
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def write_rows(host, table, rows, k, v):
    """Rows of K and V, quantised, into the host's planes."""
    for r, kr, vr in zip(rows, k, v):
        at = table[r // host.page], slice(None), r % host.page
        for x, val in (("k", kr), ("v", vr)):
            qs, dd = quantise(val)
            getattr(host, x + "_qs")[at], getattr(host, x + "_d")[at] = qs, dd


def set_rows(b, lens, new):
    """The batch's lengths and tokens, within the buffers that it has."""
    b.lens[:], b.new[:] = lens, new
    b.start[:] = np.concatenate([[0], np.cumsum(new)])
    b.owner[:], b.row[:] = -1, -1
    for i in range(b.n_seq):
        at = np.arange(b.start[i], b.start[i + 1])
        b.owner[at], b.row[at] = i, b.lens[i] - b.new[i] + at - b.start[i]


@pytest.mark.parametrize("captured", [False, True])
def test_a_loop_of_drafts(eng, captured):
    """Four sequences, six steps of a committed token and 0 to 4 drafts each:
    prepared into the pages, attended, verified; the lengths that the verification
    leaves on the device are the next step's, and refused rows are written over.
    `captured`: preparation, attention and verification are one graph."""
    n_head, n_kv, hd, page, vocab, most = 6, 2, 64, 16, 700, 5
    n_seq, half, base = 4, hd // 2, 1e4
    r = np.random.default_rng(31 + captured)
    b = Batch([120] * n_seq, [most] * n_seq, page, seed=4)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=5)
    struct, at = axis_map("interleaved", half)
    qn, kn = ((r.standard_normal(hd) * 0.3 + 1).astype(np.float32) for _ in range(2))
    lens, n = np.array([40, 1, 17, 64]), b.n_tok
    per, wide = n_kv * hd, n_head * hd
    start = Case([most] * n_seq, vocab, True, seed=0)
    with Dev(eng) as d:
        g, db = host.upload(eng), b.put(d)
        p = engine.GqaParams(d.put(qn).ptr, d.put(kn).ptr, 0, 0, 0, n_head, 0, hd, 1, base, 1e-6)
        x, pos = d.room(4 * n * (wide + 2 * per)), d.room(4 * 3 * n)
        q, out = d.put(np.zeros((n, wide), np.float32)), d.put(np.zeros((n, wide), np.float32))
        lp, lq, tok, u, un, t = (d.put(a) for a in (start.p, start.q, start.tokens, start.u, start.un, start.t))
        acc, nxt = d.room(4 * n_seq), d.room(4 * n_seq)
        dlen, dstart = b.dev[1], b.dev[2]
        width = wide + 2 * per

        def step(s):
            g.prep(db, p, x.ptr, x.ptr + 4 * wide, x.ptr + 4 * (wide + per), q.ptr, 0, struct, pos.ptr, width, width,
                   engine.DTYPE_F32, s)
            g.attend(db, q.ptr, n_head, out.ptr, stream=s)
            eng.verify_drafts(lp.ptr, lq.ptr, engine.DTYPE_F32, vocab, tok.ptr, dstart.ptr, n_seq, n, u.ptr, un.ptr,
                              acc.ptr, nxt.ptr, t.ptr, dlen.ptr, dlen.ptr, stream=s)
        graph = None
        for i in range(6):
            new = r.integers(1, most + 1, n_seq)
            set_rows(b, lens + new, new)
            c = Case(new, vocab, True, seed=50 + i, tail=n - int(new.sum()))
            c.lens = b.lens.copy()
            want_acc, want_next, want_len = c.want()
            xs = r.standard_normal((n, width)).astype(np.float32)
            ps = r.integers(0, 5000, (3, n)).astype(np.int32)
            for buf, a in ((x, xs), (pos, ps), (lp, c.p), (lq, c.q), (tok, c.tokens), (u, c.u), (un, c.un), (t, c.t),
                           (dlen, b.lens), (dstart, b.start), (out, np.full((n, wide), 5.0, np.float32))):
                buf.upload(np.ascontiguousarray(a))
            if captured and i == 1:
                graph = eng.capture(step)      # run once above, replayed from here
            if graph is None:
                step(eng.stream)
            else:
                graph.launch()
            eng.synchronize()

            mine = b.owner >= 0
            want_q = prepared(xs[:, :wide].reshape(n, n_head, hd), qn, None, ps, at, hd, base, 1, 1e-6)
            got_q = q.download(np.float32, (n, n_head, hd))
            bar = 2.0 ** -24 * np.abs(want_q) + 2.0 ** -45 * np.abs(want_q).max(-1, keepdims=True)
            assert np.all(np.abs(got_q - want_q)[mine] <= bar[mine]), i
            k = prepared(xs[:, wide:wide + per].reshape(n, n_kv, hd), kn, None, ps, at, hd, base, 1, 1e-6).astype(np.float32)
            v = xs[:, wide + per:].reshape(n, n_kv, hd)
            for s in range(n_seq):
                rows = slice(b.start[s], b.start[s + 1])
                write_rows(host, b.table[s], b.row[rows], k[rows], v[rows])
            got, want = host.download(g), host.bits()
            for m in PLANES:
                assert np.array_equal(got[m], want[m]), (i, m)
            a, bar = paged_attention(host, b, got_q.reshape(n, wide), n_head)
            have = out.download(np.float32, (n, wide))
            assert np.all(np.abs(have - a)[mine] <= bar[mine]) and np.all(have[~mine] == 5.0), i
            lens = dlen.download(np.int32, (n_seq,))
            assert np.array_equal(acc.download(np.uint32, (n_seq,)), want_acc), i
            assert np.array_equal(nxt.download(np.uint32, (n_seq,)), want_next), i
            assert np.array_equal(lens, want_len), i

        # what is left, read back
        set_rows_len = np.minimum(lens, b.n_tok // n_seq)
        set_rows(b, lens, set_rows_len)
        dlen.upload(b.lens)
        dstart.upload(b.start)
        ko, vo = d.room(4 * n * per), d.room(4 * n * per)
        g.read(db, ko.ptr, vo.ptr, stream=eng.stream)
        eng.synchronize()
        for name, buf in (("k", ko), ("v", vo)):
            have = buf.download(np.float32, (n, per))
            for s in range(n_seq):
                rows, _ = host.rows(name, b.table[s], int(lens[s]))
                assert np.array_equal(have[b.start[s]:b.start[s + 1]], rows[-set_rows_len[s]:].reshape(-1, per).astype(np.float32))
        if graph is not None:
            graph.free()
        g.free()


def test_pages_behind_four_gigabytes(eng):
    """The last of 40,000 pages of 131,072 values each (a plane of 5.2 GB)."""
    n_pages, page, n_kv, hd, n_head = 40000, 128, 8, 128, 16
    b = Batch([200], [200], page, seed=0, spare_pages=1)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=1)
    r = np.random.default_rng(2)
    k, v = (r.standard_normal((200, n_kv * hd)).astype(np.float32) for _ in range(2))
    q = r.standard_normal((200, n_head * hd)).astype(np.float32)
    write_rows(host, b.table[0], np.arange(200), k.reshape(200, n_kv, hd), v.reshape(200, n_kv, hd))
    want, bar = paged_attention(host, b, q, n_head)
    g = eng.kv_pages(n_pages, page, n_kv, hd)
    with Dev(eng) as d:
        b.table = np.where(b.table >= 0, b.table + n_pages - b.n_pages, -1).astype(np.int32)
        db = b.put(d)
        p = engine.GqaParams(0, 0, 0, 0, 0, 0, 0, 0, 1, 1e4, 0.0)
        g.prep(db, p, 0, d.put(k).ptr, d.put(v).ptr, 0, kv_stride=n_kv * hd, stream=eng.stream)
        ko, vo, out = (d.room(4 * 200 * w * hd) for w in (n_kv, n_kv, n_head))
        g.read(db, ko.ptr, vo.ptr, stream=eng.stream)
        g.attend(db, d.put(q).ptr, n_head, out.ptr, stream=eng.stream)
        eng.synchronize()
        for name, val, buf in (("k", k, ko), ("v", v, vo)):
            qs, dd = quantise(val)
            rows = qs.astype(np.float32) * np.repeat(dd.astype(np.float32), 32, -1)
            assert np.array_equal(buf.download(np.float32, val.shape), rows), name
        assert np.all(np.abs(out.download(np.float32, q.shape) - want) <= bar)
    g.free()


def test_ranges_that_fall(eng):
    """Preparation and reading take the tokens that they find, the attention
    writes nothing, and the verification still ends."""
    n_kv, hd, page, n_head = 1, 64, 16, 4
    b = Batch([40, 40, 40], [3, 3, 3], page, seed=3)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=1)
    c = Case([3, 3, 3], 500, True, seed=3)
    b.start[:] = c.start[:] = [0, 7, 2, 9]
    n = b.n_tok
    with Dev(eng) as d:
        g, db = host.upload(eng), b.put(d)
        q, out = d.put(np.ones((n, n_head * hd), np.float32)), d.put(np.full((n, n_head * hd), 5.0, np.float32))
        g.attend(db, q.ptr, n_head, out.ptr, stream=eng.stream)
        ko, vo = d.room(4 * n * hd), d.room(4 * n * hd)
        g.read(db, ko.ptr, vo.ptr, stream=eng.stream)
        eng.synchronize()
        assert np.all(out.download(np.float32, (n, n_head * hd)) == 5.0)
        rows, _ = host.rows("k", b.table[0], 40)
        assert np.array_equal(ko.download(np.float32, (n, hd))[:2], rows[33:35].reshape(2, hd).astype(np.float32))
        g.free()
    c.run(eng)


def test_a_prompt_beside_single_tokens(eng):
    """A prompt of 500 tokens after 300 rows (its blocks split over the rows), one
    from nothing, and single tokens in one batch."""
    n_head, n_kv, hd, page = 8, 2, 128, 64
    b = Batch([800, 130, 1000, 1], [500, 130, 1, 1], page, seed=8, tail=3)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=9)
    q = np.random.default_rng(1).standard_normal((b.n_tok, n_head * hd)).astype(np.float32)
    want, bar = paged_attention(host, b, q, n_head)
    mine = b.owner >= 0
    with Dev(eng) as d:
        g, db, out = host.upload(eng), b.put(d), d.put(np.full(q.shape, 5.0, np.float32))
        dq = d.put(q)
        first = None
        for _ in range(3):                 # the same bits each time
            g.attend(db, dq.ptr, n_head, out.ptr, stream=eng.stream)
            eng.synchronize()
            have = out.download(np.float32, q.shape)
            first = have if first is None else first
            assert np.array_equal(have, first)
        g.free()
    assert np.all(np.abs(have - want)[mine] <= bar[mine]) and np.all(have[~mine] == 5.0)
