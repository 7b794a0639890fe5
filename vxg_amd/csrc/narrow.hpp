// narrow.hpp -- the need-th largest of a set of 32-bit numbers by counts over
// equal bins of a shrinking range: the arithmetic of it alone, apart from how
// the numbers are counted, so that it runs on the host as on the device (a host
// compiler takes it with __host__ and __device__ defined as nothing).
//
// A range is its low end and its width, the number x in it when x - lo <=
// width in 32 bits.  With the high end in place of the width, the end of the
// topmost bin, which is partial unless the width + 1 is a multiple of the
// bin's, would pass 2^32.
#pragma once

#include <stdint.h>

namespace vxt {

constexpr uint32_t kBins = 512;

struct Range {
  uint32_t lo, width;
};

// Numbers x of the range are in bin (x - lo) >> shift, below kBins.
__host__ __device__ inline uint32_t bin_shift(uint32_t width) {
  return width >= kBins ? 23u - (uint32_t)__builtin_clz(width) : 0u;
}

// Bin `bin`, at most width >> shift: what the range has of it.
__host__ __device__ inline Range bin_of(Range r, uint32_t bin, uint32_t shift) {
  const uint32_t off = bin << shift, left = r.width - off, most = (1u << shift) - 1u;
  return {r.lo + off, left < most ? left : most};
}

// Narrows r, of which n_eq numbers are counted and the `need` largest wanted
// (1 <= need <= n_eq), until all its numbers are wanted or it is one value.
// count(range, shift, need, n_eq) returns the bin of the need-th largest and
// sets what is wanted of that bin and what it holds.  A width of 512 or more
// falls below a 256th of itself, a smaller one to 0: at most four rounds.
template <class Count>
__host__ __device__ __attribute__((always_inline)) inline Range narrow(Range r, uint32_t& need, uint32_t& n_eq, Count count) {
  while (r.width != 0 && need != n_eq) {
    const uint32_t shift = bin_shift(r.width);
    const uint32_t bin = count(r, shift, need, n_eq);
    r = bin_of(r, bin, shift);
  }
  return r;
}

}  // namespace vxt
