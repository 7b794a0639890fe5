// paged_rows.hpp -- where a batch's rows lie in the pages of a KV cache, and how
// the attention over them is cut into workgroups: the arithmetic alone, so that it
// runs on the host as on the device (a host compiler takes it with __host__ and
// __device__ defined as nothing).
//
// Tables, lengths and token ranges come from device memory that no check on the
// host sees.  Whatever they hold, a length is cut to what the table holds, a
// token range to the batch's tokens, and a row whose page number is out of range
// is nobody's.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace vxt {

struct PagedDev {
  const int32_t* table;      // [n_seq][stride]
  const int32_t* seq_len;    // [n_seq]
  const int32_t* tok_start;  // null (a token each) or [n_seq + 1]
  uint32_t n_seq, stride, n_tok;
  uint32_t shift, n_pages;   // 2^shift rows to a page
};

struct SeqRange {
  uint32_t tok, n, len;   // first token, tokens, rows
};

__host__ __device__ inline uint32_t clamp_u32(int32_t v, uint32_t most) {
  return v < 0 ? 0u : (uint32_t)v < most ? (uint32_t)v : most;
}

// Tokens [tok, end) of sequence i: rows [0, 1) of none where there are none.
__host__ __device__ inline SeqRange token_range(const int32_t* tok_start, uint32_t n_tok, uint32_t i) {
  if (!tok_start) return {i, i < n_tok ? 1u : 0u, 0u};
  const uint32_t tok = clamp_u32(tok_start[i], n_tok), end = clamp_u32(tok_start[i + 1], n_tok);
  return {tok, end > tok ? end - tok : 0u, 0u};
}

__host__ __device__ inline SeqRange seq_range(const PagedDev& b, uint32_t i) {
  SeqRange r = token_range(b.tok_start, b.n_tok, i);
  r.len = clamp_u32(b.seq_len[i], b.stride << b.shift);
  return r;
}

// The row of token t of a sequence; below 0: it has none.
__host__ __device__ inline int32_t row_of_token(const SeqRange& r, uint32_t t) {
  return (int32_t)r.len - (int32_t)r.n + (int32_t)(t - r.tok);
}

// The page of row `row` (>= 0, below the sequence's length) of sequence i;
// false if it is out of range.
__host__ __device__ inline bool page_of(const PagedDev& b, uint32_t i, int32_t row, uint32_t& page) {
  page = (uint32_t)b.table[(size_t)i * b.stride + ((uint32_t)row >> b.shift)];
  return page < b.n_pages;
}

// Element index of (page, head, row of the page) in a plane of `per` values to a
// head's row.
__host__ __device__ inline size_t page_at(uint32_t shift, uint32_t n_kv, uint32_t page, uint32_t kvh, uint32_t r, uint32_t per) {
  return ((((size_t)page * n_kv + kvh) << shift) + r) * per;
}

// ---- the attention's cut --------------------------------------------------------
// A sequence's tokens go in blocks of `tb`, its rows in pieces of 128 (a tile
// of 32 to each of a workgroup's waves); a unit is a block over about `c` pieces,
// and a workgroup to each of its kv heads.  c is chosen for `places`, the
// workgroups that run at once: where the blocks leave room to, it grows until all
// units have a place -- with a few more units than places a second round would
// run nearly empty -- and is what brings their number down to that plus one to a
// block otherwise.  Blocks of more than one unit leave partial sums in slots,
// numbered apart.
constexpr uint32_t kPieceRows = 128;

__host__ __device__ inline uint32_t pieces_of(uint32_t rows) { return (rows + kPieceRows - 1u) / kPieceRows; }
__host__ __device__ inline uint32_t blocks_of(uint32_t n, uint32_t tb) { return (n + tb - 1u) / tb; }

// The least c, from the sum of blocks * pieces over the sequences: ceil(work *
// n_kv / places).
__host__ __device__ inline uint32_t least_pieces(uint64_t work, uint32_t n_kv, uint32_t places) {
  const uint64_t w = work * n_kv;
  uint64_t c = (uint64_t)((double)w / places);   // off by one at most
  if (c && (c - 1u) * places >= w) --c;
  if (c * places < w) ++c;
  return c < 1 ? 1u : c > 0x01000000u ? 0x01000000u : (uint32_t)c;
}

// Whether c is to grow: the units have no place each, and could have.
__host__ __device__ inline bool more_pieces(uint64_t units, uint64_t blocks, uint32_t n_kv, uint32_t places) {
  return units * n_kv > places && 2u * blocks * n_kv <= places;
}

// Units to a block of a sequence of `len` rows.
__host__ __device__ inline uint32_t units_of(uint32_t len, uint32_t c) {
  const uint32_t u = (pieces_of(len) + c - 1u) / c;
  return u ? u : 1u;
}

// Tiles of 32 rows to a unit: a sequence's units are as even as its tiles allow.
__host__ __device__ inline uint32_t unit_tiles(uint32_t len, uint32_t units) {
  const uint32_t t = (len + 31u) / 32u;
  return t ? (t + units - 1u) / units : 1u;
}

// At most so many blocks, units and slots (host: from the batch's sizes alone).
__host__ __device__ inline uint64_t most_blocks(const PagedDev& b, uint32_t tb) {
  const uint64_t m = (uint64_t)b.n_tok / tb + b.n_seq;
  return m < b.n_tok ? m : b.n_tok;
}
__host__ __device__ inline uint64_t most_units(const PagedDev& b, uint32_t tb, uint32_t n_kv, uint32_t places) {
  const uint64_t blocks = most_blocks(b, tb), all = blocks * units_of(b.stride << b.shift, 1);
  const uint64_t m = places / n_kv + blocks;
  return m < all ? m : all;
}
__host__ __device__ inline uint64_t most_slots(const PagedDev& b, uint32_t tb, uint32_t n_kv, uint32_t places) {
  const uint32_t units = units_of(b.stride << b.shift, 1);
  const uint64_t all = most_blocks(b, tb) * units, m = 2ull * places / n_kv;
  return units < 2 ? 0 : m < all ? m : all;
}

}  // namespace vxt
