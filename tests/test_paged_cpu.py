"""CPU-side checks of the paged cache and the verification of drafts: what is
refused before any device is asked for, the ctypes mirrors, and the arithmetic
of ``csrc/paged_rows.hpp`` compiled for the host -- rows of bad tables, lengths
and token ranges, and that a batch's units and slots stay within what the host
allows for."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from vxg_amd import build, engine

LIB = engine.load_library()
PTR = 0x10000   # an address that nothing reads: the calls end at a check


def pages(**kw):
    a = dict(k_qs=PTR, k_d=PTR, v_qs=PTR, v_d=PTR, n_pages=4, page=16, n_kv=2, head_dim=64)
    a.update(kw)
    return engine.KvPagesQ8View(**a)


def batch(**kw):
    a = dict(table=PTR, seq_len=PTR, tok_start=PTR, n_seq=2, table_stride=3, n_tok=4)
    a.update(kw)
    return engine.PagedBatch(**a)


def params(**kw):
    a = dict(n_head=4, gated_q=0, rope_dim=64, rope_neox=1, rope_freq_base=1e4, eps=1e-6)
    a.update(kw)
    return engine.GqaParams(**a)


def ref(x):
    return None if x is None else C.byref(x)


def prep(ctx=None, g=pages(), b=batch(), p=params(), axes=None, pos=None, q=PTR, qs=256, k=PTR, v=PTR, kvs=128, dt=0,
         qo=PTR, go=None):
    buf = C.create_string_buffer(256)
    rc = LIB.vxt_hip_attn_prep_paged_q8_dev(ctx, ref(g), ref(b), ref(p), ref(axes), pos, q, qs, k, v, kvs, dt, qo, go,
                                            None, buf, len(buf))
    return rc, buf.value


def read(ctx=None, g=pages(), b=batch(), k=PTR, v=PTR, dt=0, stride=128):
    buf = C.create_string_buffer(256)
    return LIB.vxt_hip_kv_paged_q8_read_dev(ctx, ref(g), ref(b), k, v, dt, stride, None, buf, len(buf)), buf.value


def attend(ctx=None, g=pages(), b=batch(), q=PTR, n_head=4, gate=None, out=PTR, dt=0):
    buf = C.create_string_buffer(256)
    return LIB.vxt_hip_attn_paged_q8_dev(ctx, ref(g), ref(b), q, n_head, gate, out, dt, None, buf, len(buf)), buf.value


def verify(ctx=None, logits=PTR, draft=PTR, dt=0, vocab=100, stride=100, tokens=PTR, start=PTR, n_seq=2, n_tok=5,
           temperature=PTR, u=PTR, un=PTR, seq_len=PTR, new_len=PTR, acc=PTR, nxt=PTR):
    buf = C.create_string_buffer(256)
    rc = LIB.vxt_hip_verify_drafts_dev(ctx, logits, draft, dt, vocab, stride, tokens, start, n_seq, n_tok, temperature, u,
                                       un, seq_len, new_len, acc, nxt, None, buf, len(buf))
    return rc, buf.value


ARG, SHAPE, UNSUPPORTED = engine.VXT_E_ARG, engine.VXT_E_SHAPE, engine.VXT_E_UNSUPPORTED

BAD_PAGES = [(dict(k_qs=None), ARG), (dict(v_d=None), ARG), (dict(page=0), UNSUPPORTED), (dict(page=48), UNSUPPORTED),
             (dict(page=256), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=512), UNSUPPORTED),
             (dict(n_pages=0), SHAPE), (dict(n_pages=1 << 31), SHAPE), (dict(n_kv=0), SHAPE),
             (dict(n_kv=65536), UNSUPPORTED), (dict(k_qs=PTR + 8), ARG), (dict(v_d=PTR + 1), ARG)]
BAD_BATCH = [(dict(table=None), ARG), (dict(seq_len=None), ARG), (dict(n_seq=0), SHAPE), (dict(n_seq=1025), SHAPE),
             (dict(n_tok=0), SHAPE), (dict(n_tok=(1 << 24) + 1), SHAPE), (dict(tok_start=None), SHAPE),
             (dict(table_stride=0), SHAPE), (dict(table_stride=1 << 27), SHAPE), (dict(table=PTR + 2), ARG),
             (dict(seq_len=PTR + 1), ARG), (dict(tok_start=PTR + 2), ARG)]


@pytest.mark.parametrize("call", [prep, read, attend], ids=lambda f: f.__name__)
def test_bad_pages_and_batches_are_refused(call):
    assert call(g=None)[0] == ARG and call(b=None)[0] == ARG
    for kw, code in BAD_PAGES:
        rc, msg = call(g=pages(**kw))
        assert rc == code and msg and b"context" not in msg, (kw, rc, msg)
    for kw, code in BAD_BATCH:
        rc, msg = call(b=batch(**kw))
        assert rc == code and msg and b"context" not in msg, (kw, rc, msg)


def axes(n, *at):
    return engine.RopeAxes(n, (C.c_uint8 * 128)(*at))


@pytest.mark.parametrize("call,kw,code", [
    (prep, dict(p=None), ARG), (prep, dict(k=None), ARG), (prep, dict(v=None), ARG), (prep, dict(dt=2), ARG),
    (prep, dict(p=params(gated_q=2)), ARG), (prep, dict(p=params(rope_neox=3)), ARG),
    (prep, dict(p=params(eps=-1.0)), ARG), (prep, dict(p=params(eps=float("nan"))), ARG),
    (prep, dict(p=params(eps=float("inf"))), ARG),
    (prep, dict(p=params(rope_freq_base=0.0)), ARG), (prep, dict(p=params(rope_freq_base=float("inf"))), ARG),
    (prep, dict(kvs=127), SHAPE), (prep, dict(qs=255), SHAPE), (prep, dict(qs=256, p=params(gated_q=1), go=PTR), SHAPE),
    (prep, dict(qo=None), ARG), (prep, dict(p=params(gated_q=1), qs=512), ARG), (prep, dict(p=params(n_head=0)), SHAPE),
    (prep, dict(axes=axes(0)), SHAPE), (prep, dict(axes=axes(9)), SHAPE), (prep, dict(axes=axes(2, 0, 1, 2)), SHAPE),
    (prep, dict(pos=PTR + 2), ARG), (prep, dict(q=PTR + 2), ARG), (prep, dict(dt=1, k=PTR + 1), ARG),
    (read, dict(k=None), ARG), (read, dict(v=None), ARG), (read, dict(dt=7), ARG), (read, dict(stride=127), SHAPE),
    (read, dict(k=PTR + 2), ARG), (read, dict(dt=1, v=PTR + 1), ARG),
    (attend, dict(q=None), ARG), (attend, dict(out=None), ARG), (attend, dict(n_head=0), SHAPE),
    (attend, dict(n_head=5), SHAPE), (attend, dict(n_head=18), UNSUPPORTED), (attend, dict(dt=3), ARG),
    (attend, dict(q=PTR + 2), ARG), (attend, dict(gate=PTR + 1), ARG), (attend, dict(out=PTR + 2), ARG),
    (verify, dict(logits=None), ARG), (verify, dict(tokens=None), ARG), (verify, dict(u=None), ARG),
    (verify, dict(un=None), ARG), (verify, dict(acc=None), ARG), (verify, dict(nxt=None), ARG), (verify, dict(dt=2), ARG),
    (verify, dict(vocab=0), SHAPE), (verify, dict(vocab=(1 << 24) + 1, stride=1 << 25), SHAPE),
    (verify, dict(stride=99), SHAPE), (verify, dict(n_seq=0), SHAPE), (verify, dict(n_seq=1025), SHAPE),
    (verify, dict(n_tok=0), SHAPE), (verify, dict(start=None), SHAPE), (verify, dict(seq_len=None), ARG),
    (verify, dict(logits=PTR + 2), ARG), (verify, dict(tokens=PTR + 2), ARG), (verify, dict(acc=PTR + 1), ARG),
    (verify, dict(vocab=1 << 24, stride=1 << 24, n_tok=1 << 24), UNSUPPORTED),
    (verify, dict(n_tok=1 << 23), UNSUPPORTED),                     # 2^24 rows with the drafts'
    (attend, dict(b=batch(n_tok=(1 << 23) + 1)), UNSUPPORTED),      # times four heads
])
def test_bad_arguments_are_refused(call, kw, code):
    rc, msg = call(**kw)
    assert rc == code and msg and b"context" not in msg, (rc, msg)


@pytest.mark.parametrize("call", [prep, read, attend, verify], ids=lambda f: f.__name__)
@pytest.mark.parametrize("ctx", [None, 0x1000])
def test_good_arguments_end_at_the_context(call, ctx):
    rc, msg = call(ctx=ctx)
    assert rc == ARG and b"context" in msg


def test_struct_layouts():
    assert C.sizeof(engine.KvPagesQ8View) == 48 and engine.KvPagesQ8View.n_pages.offset == 32
    assert C.sizeof(engine.PagedBatch) == 40 and engine.PagedBatch.n_tok.offset == 32
    assert C.sizeof(engine.RopeAxes) == 132
    a = engine.RopeAxes.of([0, 2, 1])
    assert a.n_axes == 3 and list(a.axis[:3]) == [0, 2, 1]
    for bad in ([], [0] * 129, [8], [-1]):
        with pytest.raises(engine.BackendError):
            engine.RopeAxes.of(bad)


HARNESS = r"""
#include <cstdint>
#include <cstddef>
#include "paged_rows.hpp"
using namespace vxt;

static PagedDev dev(const int32_t* table, const int32_t* len, const int32_t* start, const uint32_t* v) {
  return PagedDev{table, len, start, v[0], v[1], v[2], v[3], v[4]};
}
// row and element index (or -1) of each token that the ranges of sequence i hold
extern "C" void rows(const int32_t* table, const int32_t* len, const int32_t* start, const uint32_t* v, uint32_t i,
                     uint32_t* range, int64_t* at, uint32_t n_kv, uint32_t kvh, uint32_t per) {
  const PagedDev b = dev(table, len, start, v);
  const SeqRange r = seq_range(b, i);
  range[0] = r.tok; range[1] = r.n; range[2] = r.len;
  for (uint32_t t = r.tok; t < r.tok + r.n; ++t) {
    const int32_t row = row_of_token(r, t);
    uint32_t page = 0;
    at[t] = row >= 0 && page_of(b, i, row, page) ? (int64_t)page_at(b.shift, n_kv, page, kvh, (uint32_t)row & ((1u << b.shift) - 1u), per) : -1;
  }
}
// {units, the host's bound, slots, the host's bound, pieces to a unit, blocks, least pieces}
extern "C" void cut(const int32_t* len, const int32_t* start, const uint32_t* v, uint32_t tb, uint32_t n_kv, uint32_t places,
                    uint64_t* res) {
  const PagedDev b = dev(nullptr, len, start, v);
  uint64_t work = 0, blocks = 0;
  for (uint32_t i = 0; i < b.n_seq; ++i) {
    const SeqRange r = seq_range(b, i);
    work += (uint64_t)blocks_of(r.n, tb) * pieces_of(r.len);
    blocks += blocks_of(r.n, tb);
  }
  const uint64_t least = least_pieces(work, n_kv, places);
  uint64_t units = 0, slots = 0, c = least;
  for (int round = 0;; ++round) {
    units = slots = 0;
    for (uint32_t i = 0; i < b.n_seq; ++i) {
      const SeqRange r = seq_range(b, i);
      const uint64_t u = (uint64_t)blocks_of(r.n, tb) * units_of(r.len, (uint32_t)c);
      units += u;
      if (units_of(r.len, (uint32_t)c) > 1) slots += u;
    }
    if (round == 8 || !more_pieces(units, blocks, n_kv, places)) break;
    c += 1 + c / 16;
  }
  res[0] = units; res[1] = most_units(b, tb, n_kv, places); res[2] = slots; res[3] = most_slots(b, tb, n_kv, places);
  res[4] = c; res[5] = blocks; res[6] = least; res[7] = work;
}
// the tiles of a sequence, as its units take them
extern "C" int tiles(uint32_t len, uint32_t c) {
  const uint32_t units = units_of(len, c), each = unit_tiles(len, units), all = (len + 31u) / 32u;
  if (each > 4u * c || (uint64_t)each * units < all) return 1;
  return 0;
}
"""


@pytest.fixture(scope="module")
def rows_lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src, so = d / "h.cpp", d / "h.so"
    src.write_text("#define __host__\n#define __device__\n" + HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I" + build.CSRC, str(src), "-o", str(so)], check=True)
    return C.CDLL(str(so))


def _p(a):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


def _head(n_seq, stride, n_tok, shift, n_pages):
    return np.array([n_seq, stride, n_tok, shift, n_pages], np.uint32)


@pytest.mark.parametrize("seed", range(40))
def test_rows_of_any_table_stay_inside(rows_lib, seed):
    r = np.random.default_rng(seed)
    n_seq, stride, shift, n_pages, n_kv, per = int(r.integers(1, 9)), int(r.integers(1, 6)), int(r.integers(4, 8)), int(r.integers(1, 7)), 3, 8
    n_tok = int(r.integers(1, 50))
    wild = np.array([-2**31, -5, -1, 0, 1, n_pages - 1, n_pages, 2**31 - 1])
    table = np.where(r.random((n_seq, stride)) < 0.5, r.integers(0, n_pages, (n_seq, stride)), r.choice(wild, (n_seq, stride))).astype(np.int32)
    lens = np.where(r.random(n_seq) < 0.6, r.integers(0, stride * 2**shift + 1, n_seq), r.choice([-2**31, -1, 2**31 - 1], n_seq)).astype(np.int32)
    start = np.where(r.random(n_seq + 1) < 0.7, np.sort(r.integers(0, n_tok + 1, n_seq + 1)), r.choice([-2**31, -3, n_tok + 9, 2**31 - 1], n_seq + 1)).astype(np.int32)
    head = _head(n_seq, stride, n_tok, shift, n_pages)
    for bare in (False, True):
        if bare:
            head[2] = n_tok = n_seq
        for i in range(n_seq):
            rng, at = np.zeros(3, np.uint32), np.full(n_tok, -9, np.int64)
            rows_lib.rows(_p(table), _p(lens), None if bare else _p(start), _p(head), i, _p(rng), _p(at), n_kv, 2, per)
            tok, n, length = (int(x) for x in rng)
            assert tok + n <= n_tok and length <= stride << shift
            if 0 <= lens[i] <= stride << shift:
                assert length == lens[i]
            for t in range(tok, tok + n):
                row = length - n + t - tok
                page = table[i, row >> shift] if row >= 0 else -1
                want = (((int(page) * n_kv + 2) << shift) + (row & (2**shift - 1))) * per if 0 <= page < n_pages else -1
                assert at[t] == want


@pytest.mark.parametrize("seed", range(60))
def test_units_and_slots_stay_within_the_hosts_bounds(rows_lib, seed):
    r = np.random.default_rng(1000 + seed)
    n_seq, shift = int(2 ** r.uniform(0, 10)), int(r.integers(4, 8))
    stride = int(2 ** r.uniform(0, 17 if seed % 3 else 6))
    most = stride << shift
    lens = (most * r.random(n_seq) ** r.choice([0.2, 1, 6])).astype(np.int32)
    new = np.minimum((2 ** r.uniform(0, 9 if seed % 2 else 3, n_seq)).astype(np.int32) - (r.random(n_seq) < 0.1), 400).astype(np.int32)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    head = _head(n_seq, stride, max(1, int(start[-1])), shift, 10)
    for tb in (1, 2, 8, 32):
        for n_kv in (1, 3, 8, 700):
            for places in (1, 256, 768, 1280):
                res = np.zeros(8, np.uint64)
                rows_lib.cut(_p(lens), _p(start), _p(head), tb, n_kv, places, _p(res))
                units, units_most, slots, slots_most, c, blocks, least, work = (int(x) for x in res)
                assert units <= units_most and slots <= slots_most, res
                assert least == min(1 << 24, max(1, -(-work * n_kv // places))) and c >= least
                # no more than there are places for, but for one unit to a block
                assert units * n_kv <= places + n_kv * blocks
    for _ in range(50):
        assert rows_lib.tiles(int(2 ** r.uniform(0, 31)) - 1, int(2 ** r.uniform(0, 20))) == 0
