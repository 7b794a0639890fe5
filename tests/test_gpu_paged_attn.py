"""GPU: attention over the pages of a Q8_0 KV cache against the formula in 64
bits: lengths from none to long, groups of 1 to 8, pages that end inside a tile,
several new tokens a sequence, rows that are nobody's, values that are not finite
where they are not seen, other streams and replayed graphs."""
import numpy as np
import pytest

from kv_ops_util import Dev
from kv_pages_util import Batch, HostPages, paged_attention, to_bf16
from vxg_amd import engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = engine.HipEngine()
    yield e
    e.close()


def run(eng, host, b, n_head, q, gate=None, dtype="f32", stream=None, fill=5.0):
    kind = np.uint16 if dtype == "bf16" else np.float32
    start = to_bf16(np.full(q.shape, fill, np.float32))[0] if dtype == "bf16" else np.full(q.shape, fill, np.float32)
    with Dev(eng) as d:
        g, db, dq, do = host.upload(eng), b.put(d), d.put(q), d.put(start)
        dg = d.put(gate).ptr if gate is not None else 0
        g.attend(db, dq.ptr, n_head, do.ptr, dg, engine.DTYPE_BF16 if dtype == "bf16" else engine.DTYPE_F32,
                 eng.stream if stream is None else stream)
        eng.synchronize()
        out = do.download(kind, q.shape)
        g.free()
    return (out.astype(np.uint32) << 16).view(np.float32) if dtype == "bf16" else out


def check(out, want, bar, dtype="f32", fill=5.0):
    mine = ~np.isnan(want).all(1)
    if dtype == "bf16":
        bar = bar + 2.0 ** -8 * (np.abs(want) + bar)
    assert np.all(np.abs(out - want)[mine] <= bar[mine]), np.nanmax((np.abs(out - want) / np.maximum(bar, 1e-30))[mine])
    assert np.all(out[~mine] == fill)


def queries(b, n_head, hd, seed, scale=1.0):
    return (np.random.default_rng(seed).standard_normal((b.n_tok, n_head * hd)) * scale).astype(np.float32)


CASES = [
    # n_head, n_kv, hd, page, lens, new, gated, dtype
    (8, 2, 64, 16, [1], [1], False, "f32"),
    (4, 4, 32, 16, [15, 16, 17, 31, 32, 33, 0, 47], [1] * 8, True, "f32"),
    (8, 1, 128, 32, [127, 128, 129, 500], [1, 1, 1, 1], False, "bf16"),
    (6, 2, 256, 64, [63, 65, 257], [1, 2, 3], True, "f32"),
    (10, 2, 128, 128, [900, 1, 130], [1, 1, 5], False, "f32"),
    (7, 1, 64, 16, [400, 55], [9, 1], True, "bf16"),
    (16, 2, 128, 16, [300, 40, 9], [5, 0, 9], False, "f32"),
    (5, 5, 128, 32, [220], [40], False, "f32"),
    (4, 2, 256, 16, [70, 150], [20, 1], True, "bf16"),
    (8, 2, 64, 64, [2049, 17, 640], [1, 1, 1], True, "f32"),
]


@pytest.mark.parametrize("n_head,n_kv,hd,page,lens,new,gated,dtype", CASES)
def test_against_64_bits(eng, n_head, n_kv, hd, page, lens, new, gated, dtype):
    b = Batch(lens, new, page, seed=hd + page, tail=3)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=page)
    q = queries(b, n_head, hd, seed=hd)
    gate = queries(b, n_head, hd, seed=1) if gated else None
    want, bar = paged_attention(host, b, q, n_head, gate)
    out = run(eng, host, b, n_head, q, gate, dtype)
    check(out, want, bar, dtype)
    assert np.array_equal(out, run(eng, host, b, n_head, q, gate, dtype))      # the same bits each time


@pytest.mark.parametrize("n_seq", [2, 63, 64, 65, 200])
def test_many_sequences(eng, n_seq):
    r = np.random.default_rng(n_seq)
    lens = (2.0 ** r.uniform(0, 9, n_seq)).astype(int)
    lens[r.integers(0, n_seq)] = 1500
    b = Batch(lens, [1] * n_seq, 32, seed=n_seq, bare=True)
    host = HostPages(b.n_pages, 32, 2, 64, seed=n_seq)
    q = queries(b, 8, 64, n_seq)
    check(run(eng, host, b, 8, q), *paged_attention(host, b, q, 8))


def test_a_thousand_sequences_of_ragged_tokens(eng):
    r = np.random.default_rng(7)
    new = r.integers(0, 4, 1024)
    lens = new + r.integers(0, 60, 1024)
    b = Batch(lens, new, 16, seed=7)
    host = HostPages(b.n_pages, 16, 1, 32, seed=7)
    q = queries(b, 4, 32, 7)
    check(run(eng, host, b, 4, q), *paged_attention(host, b, q, 4))


@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 8, 64), (8, 1, 128), (2, 1, 256)])
def test_one_long_sequence(eng, n_head, n_kv, hd):
    """Split over its length and joined."""
    b = Batch([30011], [1], 64, seed=1, spare_cols=4)
    host = HostPages(b.n_pages, 64, n_kv, hd, seed=2)
    q = queries(b, n_head, hd, 3)
    check(run(eng, host, b, n_head, q), *paged_attention(host, b, q, n_head))


def test_drafts_over_a_long_and_a_short_sequence(eng):
    b = Batch([9000, 12], [6, 4], 16, seed=1)
    host = HostPages(b.n_pages, 16, 2, 128, seed=2)
    q = queries(b, 16, 128, 3)
    check(run(eng, host, b, 16, q), *paged_attention(host, b, q, 16))


def test_shared_pages(eng):
    """Two sequences with the same first pages."""
    b = Batch([100, 90], [1, 1], 32, seed=1)
    b.table[1, :2] = b.table[0, :2]
    host = HostPages(b.n_pages, 32, 2, 64, seed=2)
    q = queries(b, 4, 64, 3)
    check(run(eng, host, b, 4, q), *paged_attention(host, b, q, 4))


@pytest.mark.parametrize("page", [16, 32, 128])
def test_pages_out_of_range_are_seen_by_none(eng, page):
    b = Batch([10 * page, 3 * page, 2 * page], [3, 1, 1], page, seed=4, spare_cols=0)
    b.table[0, 1], b.table[0, 6], b.table[1, 2] = -1, b.n_pages, -2 ** 31
    b.table[2, :] = b.n_pages + 5                     # a token that sees nothing
    host = HostPages(b.n_pages, page, 2, 64, seed=2)
    q = queries(b, 8, 64, 3)
    want, bar = paged_attention(host, b, q, 8)
    assert np.all(want[-1] == 0)
    check(run(eng, host, b, 8, q), want, bar)


def test_lengths_and_ranges_out_of_range(eng):
    """A length past the table counts to its end, one below zero as none, ranges
    behind the buffer end with it."""
    b = Batch([64, 40, 16], [1, 2, 1], 16, seed=3, spare_cols=0)
    host = HostPages(b.n_pages, 16, 1, 64, seed=2)
    q = queries(b, 4, 64, 3)
    want, bar = paged_attention(host, b, q, 4)
    b.lens[0] = 2 ** 31 - 1
    check(run(eng, host, b, 4, q), want, bar)
    b.lens[0], b.lens[1] = 64, -9
    want[1:3], bar[1:3] = 0, 0
    check(run(eng, host, b, 4, q), want, bar)
    b.start[:] = [0, 1, 3, 99]
    check(run(eng, host, b, 4, q), want, bar)


def test_rows_behind_the_last_and_drafts_that_are_not_finite(eng):
    """What a page holds behind a sequence's rows, and a drafted row's NaN or
    infinity, reach no token that does not see them."""
    b = Batch([37, 50, 16], [4, 1, 2], 16, seed=3)
    host = HostPages(b.n_pages, 16, 2, 64, seed=2)
    q = queries(b, 8, 64, 3)
    want, bar = paged_attention(host, b, q, 8)
    bad = {n: getattr(host, n) for n in ("k_d", "v_d")}
    for i, n in enumerate(b.lens):
        for row in range(n, -(-n // 16) * 16):
            for x, v in (("k_d", np.nan), ("v_d", np.inf)):
                bad[x][b.table[i, row // 16], :, row % 16] = v
    check(run(eng, host, b, 8, q), want, bar)
    for x, v in (("k_d", np.inf), ("v_d", np.nan)):   # the last drafted row of sequence 0, token 3
        bad[x][b.table[0, 36 // 16], :, 36 % 16] = v
    out = run(eng, host, b, 8, q)
    assert np.isnan(out[3]).all()
    out[3] = want[3]
    check(out, want, bar)


def test_queries_that_are_not_finite_stay_with_their_rows(eng):
    b = Batch([300, 50], [3, 1], 32, seed=3)
    host = HostPages(b.n_pages, 32, 2, 64, seed=2)
    q = queries(b, 8, 64, 3)
    want, bar = paged_attention(host, b, q, 8)
    q = q.reshape(-1, 8, 64)
    q[1, 5, 7] = np.nan
    out = run(eng, host, b, 8, q.reshape(want.shape)).reshape(q.shape)
    assert np.isnan(out[1, 5]).all()
    out[1, 5] = want.reshape(q.shape)[1, 5]
    check(out.reshape(want.shape), want, bar)


@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** 5, 2.0 ** 12])
def test_scores_of_any_size(eng, scale):
    b = Batch([333, 80], [2, 1], 16, seed=3)
    host = HostPages(b.n_pages, 16, 2, 128, seed=2)
    q = queries(b, 4, 128, 3, scale)
    check(run(eng, host, b, 4, q), *paged_attention(host, b, q, 4))


def test_scales_that_lie_far_apart(eng):
    """Values whose scales grow along the rows by powers of two, and a page of
    scales 2^-14 beside one of 2^14."""
    b = Batch([700, 64], [1, 3], 32, seed=3)
    host = HostPages(b.n_pages, 32, 2, 64, seed=2)
    for j in range(-(-700 // 32)):
        host.v_d[b.table[0, j]] = np.float16(2.0 ** (j - 14))
    host.v_d[b.table[1, 0]], host.v_d[b.table[1, 1]] = np.float16(2.0 ** -14), np.float16(2.0 ** 14)
    q = queries(b, 8, 64, 3)
    check(run(eng, host, b, 8, q), *paged_attention(host, b, q, 8))


def test_unaligned_tensors_and_another_stream(eng):
    """Everything but the value planes one element behind where an allocation
    starts, on another context's stream."""
    b = Batch([200, 33], [2, 1], 16, seed=3)
    host = HostPages(b.n_pages, 16, 2, 64, seed=2)
    q, gate = queries(b, 8, 64, 3), queries(b, 8, 64, 4)
    want, bar = paged_attention(host, b, q, 8, gate)
    other = engine.HipEngine()
    with Dev(eng) as d:
        def off(a):
            return d.put(np.concatenate([np.zeros(1, a.dtype), a.reshape(-1)])).ptr + a.itemsize
        g = engine.KvPagesQ8.over(eng, d.put(host.k_qs).ptr, off(host.k_d), d.put(host.v_qs).ptr, off(host.v_d), b.n_pages, 16,
                                  2, 64)
        db = engine.PagedBatch(off(b.table), off(b.lens), off(b.start), 2, b.table.shape[1], b.n_tok)
        for dtype, kind in ((engine.DTYPE_F32, np.float32), (engine.DTYPE_BF16, np.uint16)):
            do = d.put(np.zeros(q.size + 1, kind))
            eng.synchronize()
            g.attend(db, off(q), 8, do.ptr + do.nbytes // (q.size + 1), off(gate), dtype, other.stream)
            other.synchronize()
            out = do.download(kind, (q.size + 1,))
            assert out[0] == 0
            out = out[1:].reshape(q.shape)
            if dtype == engine.DTYPE_BF16:
                check((out.astype(np.uint32) << 16).view(np.float32), want, bar, "bf16")
            else:
                check(out, want, bar)
    other.close()


def test_a_captured_call_follows_its_lengths(eng):
    """One graph, replayed while lengths, tables and token ranges change in
    device memory, against eager calls."""
    n_kv, hd, page, n_head = 2, 64, 16, 8
    b = Batch([500, 500, 500, 500], [3, 3, 3, 3], page, seed=9)
    host = HostPages(b.n_pages, page, n_kv, hd, seed=2)
    q = queries(b, n_head, hd, 3)
    r = np.random.default_rng(1)
    with Dev(eng) as d:
        g, db, dq, do = host.upload(eng), b.put(d), d.put(q), d.put(np.zeros_like(q))
        g.attend(db, dq.ptr, n_head, do.ptr, stream=eng.stream)
        eng.synchronize()
        graph = eng.capture(lambda s: g.attend(db, dq.ptr, n_head, do.ptr, stream=s))
        for step in range(6):
            b.lens[:] = [[1, 2, 3, 4], [500, 3, 17, 130], [500, 500, 500, 500], [0, 33, 1, 499], [128, 129, 256, 257], [64, 5, 9, 500]][step]
            b.new[:] = np.minimum(r.integers(0, 4, 4), b.lens)
            b.start[:] = np.concatenate([[0], np.cumsum(b.new)])
            for buf, a in zip(b.dev, (b.table, b.lens, b.start)):
                buf.upload(a)
            do.upload(np.full_like(q, 5.0))
            graph.launch()
            eng.synchronize()
            out = do.download(np.float32, q.shape)
            for t in range(b.n_tok):
                i = int(np.searchsorted(b.start, t, side="right")) - 1
                b.owner[t] = i if t < b.start[-1] else -1
                b.row[t] = b.lens[i] - b.new[i] + t - b.start[i] if b.owner[t] >= 0 else -1
            check(out, *paged_attention(host, b, q, n_head))
        graph.free()
        g.free()


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n_head,n_kv,new", [
    (4, 1, [1, 1, 1, 1, 1]),            # one token, up to four heads: four rows to a block
    (2, 2, [2, 3, 0, 1, 9]),            # eight
    (6, 2, [2, 1, 3, 0, 1]),            # eight, at 128 dims 16
    (10, 2, [2, 3, 1, 4, 1]),           # 16 (256 dims: eight), blocks of three tokens
    (16, 2, [9, 1, 30, 2, 0]),          # 16, two column tiles where the sums fit
    (7, 1, [40, 3, 0, 25, 7]),
    (3, 3, [100, 60, 70, 99, 90]),
], ids=str)
def test_every_form(eng, hd, n_head, n_kv, new):
    """The kernels' forms by rows to a block, with a page that is none, NaN in the
    rows behind every sequence's last, a gate and both types."""
    b = Batch([260, 100, 77, 131, 1024], new, 32, seed=hd + n_head, tail=2)
    b.table[3, 1] = b.n_pages + 5
    host = HostPages(b.n_pages, 32, n_kv, hd, seed=n_head)
    for i in (0, 1, 2):
        host.v_d[b.table[i, b.lens[i] // 32], :, b.lens[i] % 32:] = np.nan
        host.k_d[b.table[i, b.lens[i] // 32], :, b.lens[i] % 32:] = np.inf
    q, gate = queries(b, n_head, hd, 3), queries(b, n_head, hd, 4)
    want, bar = paged_attention(host, b, q, n_head, gate)
    for dtype in ("f32", "bf16"):
        check(run(eng, host, b, n_head, q, gate, dtype), want, bar, dtype)
    r = run(eng, host, b, n_head, q)
    assert np.array_equal(r, run(eng, host, b, n_head, q))


def test_rows_of_nan_in_a_block_of_sixteen(eng):
    """A query of NaN, and one of infinities, stay with their rows."""
    b = Batch([300, 90], [5, 4], 16, seed=3)
    host = HostPages(b.n_pages, 16, 1, 128, seed=2)
    q = queries(b, 8, 128, 3)
    want, bar = paged_attention(host, b, q, 8)
    bad = q.reshape(b.n_tok, 8, 128).copy()
    bad[1, 3, 5], bad[6, 0, :] = np.nan, np.inf
    out = run(eng, host, b, 8, bad.reshape(q.shape)).reshape(bad.shape)
    fine = np.ones((b.n_tok, 8), bool)
    fine[1, 3] = fine[6, 0] = False
    err = np.abs(out - want.reshape(bad.shape)).max(-1)
    assert np.all(err[fine] <= bar.reshape(bad.shape).max(-1)[fine])
    assert np.all(np.isnan(out[1, 3]))
