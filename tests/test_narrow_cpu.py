"""The search by counts that eviction selects with (``csrc/narrow.hpp``),
compiled for the host: what it answers against a sort, and that it ends.  The
counts here are made as the kernels make them: a number counts when it lies in
the range, in its bin."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from vxg_amd import build

HARNESS = r"""
#include <algorithm>
#include <cstdint>
#include <vector>
#include "narrow.hpp"

// x ascending.  {low end, width, wanted of it, held by it, rounds}; 1 where a
// bin is out of range or the search goes on for more than eight rounds.
extern "C" int search(const uint32_t* x, uint64_t n, uint32_t lo, uint32_t width, uint32_t need, uint32_t* res) {
  struct Endless {};
  uint32_t rounds = 0, n_eq = (uint32_t)n;
  try {
    const vxt::Range r = vxt::narrow({lo, width}, need, n_eq, [&](vxt::Range in, uint32_t shift, uint32_t& want, uint32_t& held) {
      if (++rounds > 8 || (in.width >> shift) >= vxt::kBins) throw Endless();
      std::vector<uint32_t> c(vxt::kBins, 0);
      // x - lo <= width, in 32 bits: x from lo to the end of the range, which may lie behind 2^32
      for (int part = 0; part < 2; ++part) {
        const uint64_t end = (uint64_t)in.lo + in.width;
        const uint64_t from = part ? 0 : in.lo, to = part ? (end >> 32 ? end - (1ull << 32) + 1 : 0) : std::min<uint64_t>(end, 0xffffffffu) + 1;
        const uint32_t* p = std::lower_bound(x, x + n, from, [](uint32_t a, uint64_t b) { return a < b; });
        const uint32_t* q = std::lower_bound(x, x + n, to, [](uint32_t a, uint64_t b) { return a < b; });
        while (p < q) {   // a bin after the other
          const uint32_t b = (*p - in.lo) >> shift;
          const uint64_t next = (uint64_t)*p + ((1ull << shift) - ((*p - in.lo) & ((1u << shift) - 1u)));
          const uint32_t* e = std::lower_bound(p, q, next, [](uint32_t a, uint64_t b2) { return a < b2; });
          c[b] += (uint32_t)(e - p);
          p = e;
        }
      }
      uint32_t above = 0;
      for (int b = (int)vxt::kBins - 1; b >= 0; --b) {
        if (above < want && want <= above + c[b]) {
          want -= above;
          held = c[b];
          return (uint32_t)b;
        }
        above += c[b];
      }
      throw Endless();
    });
    const uint32_t v[5] = {r.lo, r.width, need, n_eq, rounds};
    std::copy(v, v + 5, res);
    return 0;
  } catch (Endless) {
    return 1;
  }
}
"""


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    d = tmp_path_factory.mktemp("narrow")
    src, lib = d / "narrow_host.cpp", d / "narrow_host.so"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-D__host__=", "-D__device__=", "-I" + build.CSRC,
                    str(src), "-o", str(lib)], check=True)
    f = C.CDLL(os.fspath(lib)).search
    u32p = np.ctypeslib.ndpointer(np.uint32, flags="C")
    f.argtypes, f.restype = [u32p, C.c_uint64, C.c_uint32, C.c_uint32, C.c_uint32, u32p], C.c_int

    def run(x, lo, width, need):
        """The kept ones' count by the answer: those above the last range and,
        of one value, as many as are wanted."""
        res = np.zeros(5, np.uint32)
        assert f(x, x.size, lo, width, need, res) == 0, (x.size, need, "does not end")
        low, w, want, held, rounds = (int(v) for v in res)
        assert rounds <= 4
        assert w == 0 or want == held
        at_least = x.size - int(np.searchsorted(x, low, "left"))
        return low, at_least if want == held else at_least - held + want

    return run


def rows_as_keys(rows, seq):
    """Lower rows first: ~row, ascending, and the range of them all."""
    return np.sort(~np.asarray(rows, np.uint32)), (~(seq - 1)) & 0xffffffff, seq - 1


SEQS = [16385, 65000, 262143, 262144, 262145, 300000, 300001, 524287, 524289, 540001, 600000, 1000000, 1048575, 1048577,
        4194303, 8388607]


@pytest.mark.parametrize("seq", SEQS)
def test_one_weight_everywhere(search, seq):
    """Of seq rows that weigh alike the first `keep` stay."""
    x, lo, width = rows_as_keys(np.arange(seq), seq)
    r = np.random.default_rng(seq)
    keeps = {1, 2, 27, 50, 100, 530, 1000, 2500, seq // 2, seq - 2, seq - 1, *r.integers(1, seq, 150).tolist(),
             *range(1, 2500, 13)}
    for keep in sorted(keeps):
        if keep < seq:
            low, kept = search(x, lo, width, keep)
            assert kept == keep and (~low & 0xffffffff) == keep - 1, keep


@pytest.mark.parametrize("seq", SEQS)
def test_two_rows_of_one_weight(search, seq):
    """Adjacent, of which the earlier one stays; wherever they lie."""
    for first in [*range(2500), *range(seq - 600, seq - 1), *range(2500, seq - 1, seq // 700 + 1)]:
        x, lo, width = rows_as_keys([first, first + 1], seq)
        low, kept = search(x, lo, width, 1)
        assert kept == 1 and (~low & 0xffffffff) == first, first


@pytest.mark.parametrize("seq", SEQS)
def test_some_rows_of_one_weight(search, seq):
    r = np.random.default_rng(seq + 1)
    for n in (3, 20, 700):
        for top in (4 * n, seq // 100 + 4 * n, seq):
            x, lo, width = rows_as_keys(r.choice(min(top, seq), n, replace=False), seq)
            for need in {1, 2, n // 2, n - 1, *r.integers(1, n, 20).tolist()}:
                low, kept = search(x, lo, width, need)
                assert kept == need


@pytest.mark.parametrize("lo,width", [(0, 0xffffffff), (0, 0xff800000), (0x7fffff, 0xff000001), (0xff000000, 0xffffff),
                                      (0xff800000, 0x7fffff), (0x3f800000, 511), (0x3f800000, 512), (0xfffffe00, 511),
                                      (0xfffffdff, 512), (7, 0)])
def test_keys(search, lo, width):
    """Any range of the keys themselves, up to the whole and to its upper end, many alike among them."""
    r = np.random.default_rng(width % 1000003)
    for n in (1, 2, 50, 5000):
        x = lo + r.integers(0, width + 1, n, dtype=np.uint64)
        if n > 2:
            x[r.random(n) < 0.5] = x[:3].max()
            x[:2] = lo, lo + width
        x = np.sort(x).astype(np.uint32)
        for need in {1, n, *r.integers(1, n + 1, 60).tolist()}:
            low, kept = search(x, lo, width, need)
            assert kept == need and low <= x[n - need]
