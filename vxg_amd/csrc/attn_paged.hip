// attn_paged.hip -- attention of a batch's new tokens over the pages of a Q8_0
// KV cache.  Token j of a sequence's n new ones, in row len - n + j, attends to
// rows [0, len - n + j]:
//   out = sum_t softmax(q . K_t / sqrt(hd)) V_t, times 1 / (1 + exp(-gate)).
// A token that sees no row (none, or on pages that are out of range) gets 0.
//
// Cut (paged_rows.hpp): a unit is a block of tokens over a stretch of rows, a
// workgroup to each of its kv heads, all of about the same work whatever the mix
// of lengths.  Lengths are known on the device alone, so every wave finds its unit
// by itself, by one scan over the sequences (64 at a time, a lane to each), and
// the grid is what the batch's sizes allow for at most.
//
// Measured (whole calls; query / kv heads of 128 dims).  32 / 8 heads, 8 sequences of
// 20,000 to 30,000 rows, 437 MB: 95 us, 4.6 TB/s, memory beside the vector unit (some
// 460 operations a wave and tile; 75 us with all rows in the L2s).  16 / 4, 32 sequences
// of 150 to 8,000: 26 us, of which the scan and the first tile's chain of loads take
// 6, the tiles 8 to 12, the join 5; 24 of 300 to 4,000 with 1 to 6 tokens: 25 us, the
// same chain.  Units for as many workgroups as run at once, 768
// of one column tile and four rows: 95 and 28 us; for 512, 114 and 33; for 1,024, 100
// and 29; for 1,536, 98 and 34.
#include "kv_pages.hpp"

#include <algorithm>
#include <type_traits>

namespace vxt {

namespace {

// ---- the cut, by every lane of a wave ------------------------------------------

// Sum over the wave, in every lane.
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
  auto near = [&](auto ctrl) {
    const uint32_t lo = dpp_u32<decltype(ctrl)::value>((uint32_t)v), hi = dpp_u32<decltype(ctrl)::value>((uint32_t)(v >> 32));
    v += (uint64_t)hi << 32 | lo;
  };
  near(std::integral_constant<int, 0xB1>{});    // quad_perm [1,0,3,2]
  near(std::integral_constant<int, 0x4E>{});    // quad_perm [2,3,0,1]
  near(std::integral_constant<int, 0x141>{});   // row_half_mirror
  near(std::integral_constant<int, 0x140>{});   // row_mirror
  const auto l16 = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  const auto h16 = __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  v = ((uint64_t)h16[0] << 32 | l16[0]) + ((uint64_t)h16[1] << 32 | l16[1]);
  const auto l32 = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  const auto h32 = __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  return ((uint64_t)h32[0] << 32 | l32[0]) + ((uint64_t)h32[1] << 32 | l32[1]);
}

// A lane's sequences are [lane * per, lane * per + per), the first of them kept;
// before: units (slots) of the lanes below.
struct CutScan {
  SeqRange first;
  uint32_t per, c, units, slots, units_before, slots_before, all_units;
  bool bad, any;   // ranges that fall; the lane has a sequence
};

__device__ __forceinline__ CutScan scan_cut(const PagedDev& b, uint32_t tb, uint32_t n_kv, uint32_t places) {
  CutScan s;
  const uint32_t lane = threadIdx.x & 63u;
  s.per = (b.n_seq + 63u) / 64u;
  const uint32_t i0 = lane * s.per, n = i0 < b.n_seq ? min(s.per, b.n_seq - i0) : 0u;
  s.first = seq_range(b, min(i0, b.n_seq - 1u));
  auto range = [&](uint32_t k) { return k == 0 ? s.first : seq_range(b, i0 + k); };
  uint64_t work = 0;
  uint32_t blocks = 0;
  bool falls = false;
  s.any = n != 0;
  for (uint32_t k = 0; k < n; ++k) {
    const SeqRange r = range(k);
    work += (uint64_t)blocks_of(r.n, tb) * pieces_of(r.len);
    blocks += blocks_of(r.n, tb);
    falls |= b.tok_start && clamp_u32(b.tok_start[i0 + k + 1u], b.n_tok) < r.tok;
  }
  s.bad = __builtin_amdgcn_ballot_w64(falls) != 0;
  s.c = (uint32_t)__builtin_amdgcn_readfirstlane((int)least_pieces(wave_sum_u64(work), n_kv, places));
  blocks = lane63(lane_scan_u32(blocks));
  uint32_t u, t;
  for (int round = 0;; ++round) {
    s.units = s.slots = 0;
    for (uint32_t k = 0; k < n; ++k) {
      const SeqRange r = range(k);
      const uint32_t nc = units_of(r.len, s.c), x = blocks_of(r.n, tb) * nc;
      s.units += x;
      s.slots += nc > 1 ? x : 0u;
    }
    u = lane_scan_u32(s.units);
    s.all_units = lane63(u);
    if (round == 8 || !more_pieces(s.all_units, blocks, n_kv, places)) break;
    s.c += 1u + s.c / 16u;
  }
  t = lane_scan_u32(s.slots);
  s.units_before = u - s.units;
  s.slots_before = t - s.slots;
  return s;
}

struct Unit {
  SeqRange r;
  uint32_t seq, nc, nb, at, slot;   // units to a block, blocks, units before the sequence, slots before it
};

// Told to the compiler as scalars.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ Unit uniform(const Unit& u) {
  return Unit{SeqRange{uniform(u.r.tok), uniform(u.r.n), uniform(u.r.len)}, uniform(u.seq), uniform(u.nc), uniform(u.nb), uniform(u.at), uniform(u.slot)};
}

// The sequence that unit (BY_UNIT) or token `which` is of.
template <bool BY_UNIT>
__device__ __forceinline__ bool find_cut(const PagedDev& b, const CutScan& s, uint32_t tb, uint32_t which, Unit& o) {
  const uint64_t m = __builtin_amdgcn_ballot_w64(BY_UNIT ? s.units_before + s.units > which : s.first.tok <= which && s.any);
  if (m == 0) return false;
  // the first lane that reaches past the unit; the last whose tokens begin at or before it
  const int l = BY_UNIT ? __builtin_ctzll(m) : 63 - __builtin_clzll(m);
  o.at = (uint32_t)__builtin_amdgcn_readlane((int)s.units_before, l);
  o.slot = (uint32_t)__builtin_amdgcn_readlane((int)s.slots_before, l);
  for (uint32_t k = 0; k < s.per; ++k) {
    o.seq = (uint32_t)l * s.per + k;
    if (o.seq >= b.n_seq) return false;
    if (k == 0)
      o.r = SeqRange{(uint32_t)__builtin_amdgcn_readlane((int)s.first.tok, l), (uint32_t)__builtin_amdgcn_readlane((int)s.first.n, l),
                     (uint32_t)__builtin_amdgcn_readlane((int)s.first.len, l)};
    else
      o.r = seq_range(b, o.seq);
    o.nc = units_of(o.r.len, s.c);
    o.nb = blocks_of(o.r.n, tb);
    const uint32_t u = o.nb * o.nc;
    if (BY_UNIT ? which < o.at + u : which - o.r.tok < o.r.n) return true;
    o.at += u;
    o.slot += o.nc > 1 ? u : 0u;
  }
  return false;
}

// Rows that some token of block `blk` sees: [0, upto).
__device__ __forceinline__ int block_upto(const SeqRange& r, uint32_t tb, uint32_t blk) {
  return (int)r.len - (int)r.n + (int)min((blk + 1u) * tb, r.n);
}

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

struct AttnArgs {
  PagedAttn a;
  uint32_t group, tb, max_slots, places;
  float* ml;   // [slot][kv head][rows][2]: reference (base 2; -inf: nothing seen), sum
  float* o;    // [slot][kv head][rows][hd]
};

// Four results from `at` on, by their gates.
__device__ __forceinline__ void store_out(const PagedAttn& a, size_t at, float4v x, float4u gate) {
  if (a.gate) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= 1.0f / (1.0f + expf(-gate[j]));
  }
  if (a.out_bf16) {
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4), aligned(2)));
    u16x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = f32_to_bf16(x[j]);
    *reinterpret_cast<u16x4*>(static_cast<uint16_t*>(a.out) + at) = y;
  } else
    *reinterpret_cast<float4u*>(static_cast<float*>(a.out) + at) = x;
}

// Waves to a SIMD that the registers are to leave room for.  256 dims: two (one, 8
// sequences of 20,000 to 30,000 rows, 4 kv heads, 104 for 95 us); 128 dims and 16 rows:
// two, three spill (12 sequences of 2,000 to 20,000 rows, 4 kv heads: 1 to 4 tokens of
// 5 heads 38 us, with three 45; 1 to 40 tokens 181 and 164).
constexpr int waves_of(int hd, int nt, int rt) { return hd == 256 ? 2 : hd == 128 ? (rt == 16 ? 2 : 3) : nt == 1 ? 4 : 3; }

// A workgroup to a unit and kv head: 4 waves, each on its own tiles of 32 rows.
// A block's query rows (token, head of the group) are columns of
// v_mfma_f32_16x16x32_f16, in one of three forms by their number (RT to a column
// tile), each row in two f16 terms:
//   16: a column each, both terms products into the same sums;
//    8: column n is row n % 8, term n / 8: half the products;
//    4: columns 0 .. 3 and 7 .. 4 are the two terms, and columns 8 on the same again,
//       which hold the weights of a second 32-dim block, so that a set of weights
//       serves two blocks.
// Then,
//   S (positions x columns) = K Q^T per 32-dim block, K's codes exact, then
//     S += d_k * block, and the two terms' columns added, if there are two: every
//     lane holds 8 positions' scores of its column's row;
//   O^T (dims x columns) += V^T W with V's codes exact and W = weight * d_v, per
//     32-dim block, as the first or the second f16 term of the lane's column.
// A lane's 8 positions are those of its operand in the second product, so no
// weight leaves its lane.  K, V and the scales go through a wave's own LDS as rows
// (V is read transposed there), loaded a tile ahead.
// V's scales carry the power of two that brings the largest that the wave has met
// up to [1/2, 1) (2^-13 at most for a larger one), so that with weights of at most
// 2^15 the products stay below 2^15; where a tile brings a larger one, the sums
// move by the difference, a power of two.  Numbers otherwise as in kv_ops.hpp.
template <int HD, int NT, int RT>
__global__ __launch_bounds__(256, waves_of(HD, NT, RT)) void paged_attn_kernel(PagesDev c, PagedDev b, AttnArgs x) {
  constexpr uint32_t NB = HD / 32, ND = HD / 16, VST = HD + 16;   // row stride of K and V in LDS (bytes)
  constexpr uint32_t LPR = HD / 16, RPL = 64 / LPR;               // lanes to a row of K or V, rows to a load
  constexpr uint32_t KV = 32u * VST, DS = 32u * NB * 2u, WAVE = 2u * KV + 2u * DS;   // bytes: K or V, their scales, a wave's
  constexpr uint32_t BP = RT == 4 && NB > 1 ? 2 : 1;              // blocks to one set of weights
  constexpr uint32_t R = RT * NT;                                 // query rows
  constexpr uint32_t TERMS = RT == 16 ? 2 : 1;                    // of the lane's own column
  static_assert(RT == 16 || RT == 8 || RT == 4, "");
  constexpr uint32_t BUF = 4u * R * HD * 4u > 4u * WAVE ? 4u * R * HD * 4u : 4u * WAVE;
  __shared__ __attribute__((aligned(16))) uint8_t s_buf[BUF];
  __shared__ float s_ml[4][R][2];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t n = lane & 15u, g = lane >> 4;
  // the column's row, its term, and (RT 4) which of two blocks it has weights for
  const bool second = RT == 16 ? false : RT == 8 ? n >= 8u : (n & 4u) != 0u;
  const uint32_t col = RT == 16 ? n : RT == 8 ? n & 7u : second ? 7u - (n & 7u) : n & 7u, pb = BP == 1 ? 0u : n >> 3;
  constexpr int OTHER = RT == 8 ? 0x128 : 0x141;   // row_ror:8, row_half_mirror: the other term's column
  const uint32_t group = x.group, tb = x.tb;

  // the workgroup's unit: each XCD takes a run of them, so that blocks that read
  // the same rows share its L2 (the grid's width is a multiple of eight)
  const uint32_t kvh = blockIdx.y;
  const CutScan cut = scan_cut(b, tb, c.n_kv, x.places);
  const uint32_t run = (cut.all_units + 7u) / 8u, item = blockIdx.x % 8u * run + blockIdx.x / 8u;
  if (cut.bad || blockIdx.x / 8u >= run || item >= cut.all_units) return;
  Unit u;
  if (!find_cut<true>(b, cut, tb, item, u)) return;
  u = uniform(u);
  uint32_t ck = item - u.at, blk = 0;
  if (u.nb > 1) {
    blk = ck % u.nb;
    ck /= u.nb;
  }
  const int first_row = (int)u.r.len - (int)u.r.n + (int)(blk * tb);       // of the block's first token
  const uint32_t n_tok = min(tb, u.r.n - blk * tb);
  const int upto_i = block_upto(u.r, tb, blk);
  const uint32_t upto = upto_i < 0 ? 0u : (uint32_t)upto_i;
  const uint32_t n_vt = (upto + 31u) / 32u;
  const uint32_t ut = unit_tiles(u.r.len, u.nc);
  if (ck && ck * ut >= n_vt) return;                                       // behind what the block sees
  const uint32_t n_unit = (n_vt + ut - 1u) / ut;                           // of the block's that see anything
  const uint32_t slot0 = (u.slot + blk) * c.n_kv + kvh, slot_step = u.nb * c.n_kv, slot = slot0 + ck * slot_step;
  if (n_unit > 1 && u.slot + (u.nc - 1u) * u.nb + blk >= x.max_slots) return;   // more than the host allowed for
  const uint32_t end = min(n_vt, (ck + 1u) * ut), each = (min(ut, end - min(end, ck * ut)) + 3u) / 4u;
  const uint32_t vt0 = min(end, ck * ut + wave * each), vt1 = min(end, vt0 + each);

  // The table's entries for a tile's halves of 16 rows, scalars read a tile ahead
  // of their use (the last entry again behind the last row).  As constant memory:
  // the waits in the loop would make them vector loads.
  typedef const __attribute__((address_space(4))) int32_t const_i32;
  const uint32_t n_ent = (upto + (1u << b.shift) - 1u) >> b.shift;
  const_i32* table = (const_i32*)(uintptr_t)(b.table + (size_t)u.seq * b.stride);
  uint32_t ent0 = 0, ent1 = 0;
  auto read_entries = [&](uint32_t vt) {
    const uint32_t last = n_ent - 1u;
    ent0 = (uint32_t)table[uniform(min((vt * 32u) >> b.shift, last))];
    ent1 = (uint32_t)table[uniform(min((vt * 32u + 16u) >> b.shift, last))];
  };
  if (vt0 < vt1) read_entries(vt0);   // n_ent >= 1

  // the block's queries, on their way beside the pages' numbers
  float4u qv[NT][NB][2];
  int lim[NT];   // rows that each sees
#pragma unroll
  for (uint32_t ct = 0; ct < NT; ++ct) {
    const uint32_t r = min(ct * RT + col, n_tok * group - 1u), tk = r / group;
    lim[ct] = first_row + (int)tk + 1;
    const float* qr = x.a.q + ((size_t)(u.r.tok + blk * tb + tk) * x.a.n_head + kvh * group + (r - tk * group)) * HD + 8u * g;
#pragma unroll
    for (uint32_t bk = 0; bk < NB; ++bk)
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) qv[ct][bk][h] = *reinterpret_cast<const float4u*>(qr + 32u * bk + 4u * h);
  }

  // The first row's number of each half in a plane of rows, and whether there is
  // a page.
  auto row_of = [&](uint32_t row, uint32_t page, bool& ok) -> uint64_t {
    ok = page < b.n_pages && row < upto;
    return (((uint64_t)(ok ? page : 0u) * c.n_kv + kvh) << b.shift) + (row & ((1u << b.shift) - 1u));
  };
  uint64_t row0 = 0, row1 = 0;
  bool ok0 = false, ok1 = false;
  auto find_tile = [&](uint32_t vt) {
    row0 = row_of(vt * 32u, ent0, ok0);
    row1 = row_of(vt * 32u + 16u, ent1, ok1);
  };

  // A tile's bytes on their way to LDS, loaded for the next tile as soon as they
  // are there -- always, behind the last tile the same one again.  Lanes 0 .. 31
  // load a row's K scales, the others its V scales.
  u32x4 k16[NB], v16[NB];
  Scales<NB> d16;
  const uint32_t in_head = (lane / LPR) * HD + 16u * (lane % LPR);   // of a load's rows
  auto load = [&]() {
    const uint64_t apart = row1 - row0 - 16u;   // 0 but on pages of 16
    const int8_t *const kp = c.k_qs + row0 * HD, *const vp = c.v_qs + row0 * HD;
#pragma unroll
    for (uint32_t j = 0; j < NB; ++j) {
      uint64_t skip = j * RPL * HD;             // to this load's rows, uniform
      if (RPL < 32 && j * RPL >= 16u) skip += apart * HD;
      if constexpr (RPL == 32) {
        const uint64_t at = in_head + (lane < 32u ? 0u : apart * HD);
        k16[j] = *reinterpret_cast<const u32x4*>(kp + at);
        v16[j] = *reinterpret_cast<const u32x4*>(vp + at);
      } else {
        k16[j] = *reinterpret_cast<const u32x4*>(kp + skip + in_head);
        v16[j] = *reinterpret_cast<const u32x4*>(vp + skip + in_head);
      }
    }
    const uint16_t* const dp = (lane < 32u ? c.k_d : c.v_d) + row0 * NB;
    d16 = load_scales<NB>(dp + (lane & 16u ? apart + 16u : 0u) * NB + (lane & 15u) * NB);
  };
  if (vt0 < vt1) {
    find_tile(vt0);
    load();
    read_entries(vt0 + 1u);
  }

  // Q^T operands, to give scores in base 2 but for their rows' powers of two,
  // before a tile takes the registers
  half8v qb[TERMS][NT][NB];
  float f_row[NT];
#pragma unroll
  for (uint32_t ct = 0; ct < NT; ++ct) {
    const float scale = 1.4426950408889634f / sqrtf((float)HD);
    float amax = 0.0f;
#pragma unroll
    for (uint32_t bk = 0; bk < NB; ++bk)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        qv[ct][bk][j / 4][j % 4] *= scale;
        amax = fmaxf(amax, fabsf(qv[ct][bk][j / 4][j % 4]));
      }
    amax = xor32_pair(xor16_pair(amax, true), true);
    const int e = top_shift(amax);
    const float up = pow2f(e);
    f_row[ct] = pow2f(-e);
#pragma unroll
    for (uint32_t bk = 0; bk < NB; ++bk)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const float y = qv[ct][bk][j / 4][j % 4] * up;
        const _Float16 hi = (_Float16)y;
        if constexpr (TERMS == 2) {
          qb[0][ct][bk][j] = hi;
          qb[1][ct][bk][j] = (_Float16)(y - (float)hi);
        } else {
          qb[0][ct][bk][j] = second ? (_Float16)(y - (float)hi) : hi;
        }
      }
  }

  // the power of two of V's scales, in two f16 factors (2^15 is f16's largest)
  uint32_t top = 0;
  int kv = 0;
  float w_up = 0.0f;
  half2v d_up1 = {(_Float16)1.0f, (_Float16)1.0f}, d_up2 = d_up1;

  float4v o[NT][ND];
  float ref[NT], l_run[NT];
#pragma unroll
  for (uint32_t ct = 0; ct < NT; ++ct) {
    ref[ct] = -__builtin_inff();
    l_run[ct] = 0.0f;
#pragma unroll
    for (uint32_t d = 0; d < ND; ++d) o[ct][d] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  }
  uint8_t* const sk = s_buf + wave * WAVE;
  uint8_t* const sv = sk + KV;
  uint8_t* const sd = sv + KV;             // K's scales, then V's: [NB][32 rows]
  // a 32-dim block's scales of this lane's 8 rows, in pairs
  auto scales = [&](uint32_t which, uint32_t bk) { return *reinterpret_cast<const u32x4*>(sd + which * DS + 64u * bk + 16u * g); };

  for (uint32_t vt = vt0; vt < vt1; ++vt) {
    const bool whole = (int)(vt * 32u + 32u) <= first_row + 1 && ok0 && ok1;   // uniform
    const bool is0 = ok0, is1 = ok1;
#pragma unroll
    for (uint32_t j = 0; j < NB; ++j) {
      const uint32_t at = (j * RPL + lane / LPR) * VST + 16u * (lane % LPR);
      *reinterpret_cast<u32x4*>(sk + at) = k16[j];
      *reinterpret_cast<u32x4*>(sv + at) = v16[j];
    }
#pragma unroll
    for (uint32_t bk = 0; bk < NB; ++bk)
      *reinterpret_cast<uint16_t*>(sd + (lane >> 5) * DS + 64u * bk + 2u * (lane & 31u)) = d16.d[bk];
    // a scale above the largest so far, among the rows that somebody sees (as
    // bits, a negative or infinite one is above all, and looked at closer)
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t bk = 0; bk < NB; ++bk) mine = max(mine, (uint32_t)d16.d[bk]);
    if (lane < 32u) mine = 0u;
    if (__builtin_amdgcn_ballot_w64(mine > top) != 0) {
      asm volatile("" : "+v"(mine));   // a branch, not selects in every tile
      mine = lane < 32u || vt * 32u + (lane & 31u) >= upto || !(lane & 16u ? is1 : is0) ? 0u : top_scale(d16);
    }
    if (__builtin_amdgcn_ballot_w64(mine > top) != 0) {   // seldom after the first tile
      top = (uint32_t)__builtin_amdgcn_readfirstlane((int)lane_max_u32<64>(max(mine, top)));
      const int to_top = scale_shift(top) - 7, up = (int)kWeightUp, now = max(to_top, 0) + min(to_top + up, 0), now1 = min(now, 15);
      w_up = (float)max(up + min(to_top, 0), 0);
      const _Float16 up1 = (_Float16)pow2f(now1), up2 = (_Float16)pow2f(now - now1);
      d_up1 = half2v{up1, up1};
      d_up2 = half2v{up2, up2};
      float move = pow2f(now - kv);
      asm volatile("" : "+v"(move));
      kv = now;
#pragma unroll
      for (uint32_t ct = 0; ct < NT; ++ct)
#pragma unroll
        for (uint32_t d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[ct][d][i] *= move;
    }
    if (vt + 1u < vt1) find_tile(vt + 1u);
    load();
    read_entries(vt + 2u);
    wave_lds_order();

    float s[NT][8];
#pragma unroll
    for (uint32_t bk = 0; bk < NB; ++bk) {
      const u32x4 dk = scales(0, bk);
#pragma unroll
      for (uint32_t mt = 0; mt < 2; ++mt) {
        const uint8_t* kr = sk + (8u * (n >> 2) + 4u * mt + (n & 3u)) * VST + 8u * g + 32u * bk;
        const half8v kf = codes8_f16(*reinterpret_cast<const u32x2*>(kr));
        float d[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const half2v w = __builtin_bit_cast(half2v, (uint32_t)dk[2u * mt + i / 2u]);
          d[i] = (float)(i & 1u ? w.y : w.x);
        }
#pragma unroll
        for (uint32_t ct = 0; ct < NT; ++ct) {
          float4v t{};
#pragma unroll
          for (uint32_t e = 0; e < TERMS; ++e) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qb[e][ct][bk], t, 0, 0, 0);
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            s[ct][4u * mt + i] = __builtin_fmaf(d[i], t[i], bk == 0 ? 0.0f : s[ct][4u * mt + i]);
        }
      }
    }
    const int pos = (int)(vt * 32u + 8u * g);      // of this lane's 8 scores
    const bool here = g < 2u ? is0 : is1;
    half2v p0[NT][4], p1[NT][4];
#pragma unroll
    for (uint32_t ct = 0; ct < NT; ++ct) {
      float pm = -__builtin_inff();
      if constexpr (TERMS == 1) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) s[ct][j] += dpp_mov<OTHER>(s[ct][j]);   // the other term's column
      }
      if (!whole) {
        int p = pos;
        asm volatile("" : "+v"(p));   // a branch, not compares in every tile
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          asm volatile("" : "+v"(s[ct][j]));
          s[ct][j] = here && p + (int)j < lim[ct] ? s[ct][j] : -__builtin_inff();
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) pm = fmaxf(pm, s[ct][j]);
      pm = xor32_pair(xor16_pair(pm, true), true) * f_row[ct];   // a power of two: exact, as in the weights
      const bool move = pm - ref[ct] > w_up + kWeightLag;
      if (__builtin_amdgcn_ballot_w64(move) != 0) {
        const float to = move ? weight_ref(pm, w_up) : ref[ct];
        float alpha = move ? __builtin_amdgcn_exp2f(ref[ct] - to) : 1.0f;
        asm volatile("" : "+v"(alpha));   // a branch: not products and copies in every tile
        ref[ct] = to;
        l_run[ct] *= alpha;
#pragma unroll
        for (uint32_t d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[ct][d][i] *= alpha;
      }
      const float off = ref[ct] == -__builtin_inff() ? 0.0f : ref[ct];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        s[ct][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][j], f_row[ct], -off));
        l_run[ct] += s[ct][j];
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        uint32_t hi, lo;
        split_f16(s[ct][2 * k], s[ct][2 * k + 1], hi, lo);
        p0[ct][k] = __builtin_bit_cast(half2v, hi);
        p1[ct][k] = __builtin_bit_cast(half2v, lo);
      }
    }
    typedef __attribute__((address_space(3))) int2v lds_int2;
    const uint8_t* tr = sv + (8u * g + (n >> 1)) * VST + 8u * (n & 1u);
#pragma unroll
    for (uint32_t bi = 0; bi < NB; bi += BP) {
      // one operation on four pairs at a time: a packed result is not to be
      // read by the next instruction
      const u32x4 dv = *reinterpret_cast<const u32x4*>(sd + DS + 64u * (bi + pb) + 16u * g);
      half2v d[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) d[k] = __builtin_bit_cast(half2v, (uint32_t)dv[k]) * d_up1;
      if (kv > 15) {   // uniform: every scale below 2^-8
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          uint32_t y = __builtin_bit_cast(uint32_t, d[k]);
          asm volatile("" : "+v"(y));   // a branch, not selects
          d[k] = __builtin_bit_cast(half2v, y) * d_up2;
        }
      }
      u32x4 w[TERMS][NT];
#pragma unroll
      for (uint32_t ct = 0; ct < NT; ++ct) {
        half2v y[4], e[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) y[k] = p0[ct][k] * d[k];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) e[k] = __builtin_elementwise_fma(p0[ct][k], d[k], -y[k]);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) e[k] = __builtin_elementwise_fma(p1[ct][k], d[k], e[k]);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
          if constexpr (TERMS == 2) {
            w[0][ct][k] = __builtin_bit_cast(uint32_t, y[k]);
            w[1][ct][k] = __builtin_bit_cast(uint32_t, e[k]);
          } else {
            w[0][ct][k] = __builtin_bit_cast(uint32_t, second ? e[k] : y[k]);
          }
        }
        if (!whole) {   // a weight of 0 times a scale that is not finite
          int p = pos;
          asm volatile("" : "+v"(p));
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t lo = here && p + (int)(2u * k) < lim[ct] ? 0xffffu : 0u;
            const uint32_t hi = here && p + (int)(2u * k + 1u) < lim[ct] ? 0xffff0000u : 0u;
#pragma unroll
            for (uint32_t m = 0; m < TERMS; ++m) w[m][ct][k] &= lo | hi;
          }
        }
      }
#pragma unroll
      for (uint32_t h = 0; h < 2u * BP; ++h) {   // RT 4: the columns of the other block's weights give nothing
        const uint32_t dt = 2u * bi + h;
        const u32x2 vb = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(tr + 16u * dt)));
        const half8v vf = codes8_f16(vb);
#pragma unroll
        for (uint32_t ct = 0; ct < NT; ++ct)
#pragma unroll
          for (uint32_t m = 0; m < TERMS; ++m)
            o[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, __builtin_bit_cast(half8v, w[m][ct]), o[ct][dt], 0, 0, 0);
      }
    }
    wave_lds_order();   // read before the next tile's rows are written
  }
  const float down = pow2f(-kv);

  // the two terms' columns, the wave's sums, then the four waves'
  __syncthreads();   // every wave is done with its part of s_buf
  float* s_o = reinterpret_cast<float*>(s_buf);
#pragma unroll
  for (uint32_t ct = 0; ct < NT; ++ct) {
    const float l = xor32_pair(xor16_pair(l_run[ct], false), false);
#pragma unroll
    for (uint32_t d = 0; d < ND; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (TERMS == 1) o[ct][d][i] += dpp_mov<OTHER>(o[ct][d][i]);
        o[ct][d][i] *= down;
      }
      if (!second && (RT == 4 ? n >> 3 : 0u) == (BP == 2 ? d / 2u % 2u : 0u))
        *reinterpret_cast<float4v*>(s_o + ((wave * R + ct * RT + col) * HD + 16u * d + 4u * g)) = o[ct][d];
    }
    if (!second && (RT == 16 || n < 8u) && g == 0) {
      s_ml[wave][ct * RT + col][0] = l != l ? 0.0f : ref[ct];   // -inf only where nothing was seen
      s_ml[wave][ct * RT + col][1] = l;
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < n_tok * group * (HD / 4u); i += 256u) {
    const uint32_t r = i / (HD / 4u), d = i % (HD / 4u) * 4u;
    const size_t row = (size_t)(u.r.tok + blk * tb + r / group) * x.a.n_head + kvh * group + r % group;
    float4u gate{};
    if (n_unit <= 1 && x.a.gate) gate = *reinterpret_cast<const float4u*>(x.a.gate + row * HD + d);
    float m = s_ml[0][r][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, s_ml[w][r][0]);
    float l = 0.0f;
    float4v y{};
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const float rw = s_ml[w][r][0];
      if (rw == -__builtin_inff()) continue;
      const float e = __builtin_amdgcn_exp2f(rw - m);
      l += s_ml[w][r][1] * e;
      const float4v ow = *reinterpret_cast<const float4v*>(s_o + (w * R + r) * HD + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] += ow[j] * e;
    }
    if (n_unit <= 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = l == 0.0f ? 0.0f : y[j] / l;
      store_out(x.a, row * HD + d, y, gate);
    } else {
      *reinterpret_cast<float4v*>(x.o + ((size_t)slot * R + r) * HD + d) = y;
      if (d == 0) *reinterpret_cast<float2*>(x.ml + 2u * ((size_t)slot * R + r)) = float2{m, l};
    }
  }
}

// The partial sums of the rows whose block has more than one unit: W waves to a
// row (token, head), HD / 4 lanes to a partial.
template <int HD, int W>
__global__ __launch_bounds__(256) void paged_join_kernel(PagesDev c, PagedDev b, AttnArgs x, uint32_t rows_per_slot) {
  constexpr uint32_t L = HD / 4, G = 64 / L;
  __shared__ float4v s_acc[4][64];
  __shared__ float s_l[4];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, part = W == 1 ? 0u : wave;
  const uint32_t row = __builtin_amdgcn_readfirstlane((int)(W == 1 ? blockIdx.x * 4u + wave : blockIdx.x));
  const uint32_t t = row / x.a.n_head, head = row % x.a.n_head;
  if (t >= b.n_tok) return;
  const CutScan cut = scan_cut(b, x.tb, c.n_kv, x.places);
  Unit u;
  if (cut.bad || !find_cut<false>(b, cut, x.tb, t, u)) return;
  const uint32_t in_seq = t - u.r.tok, blk = in_seq / x.tb, kvh = head / x.group, r = (in_seq % x.tb) * x.group + head % x.group;
  const int upto = block_upto(u.r, x.tb, blk);
  const uint32_t ut = unit_tiles(u.r.len, u.nc), n = upto <= 0 ? 0u : (((uint32_t)upto + 31u) / 32u + ut - 1u) / ut;
  if (n <= 1 || u.slot + (u.nc - 1u) * u.nb + blk >= x.max_slots) return;   // stored already
  const size_t step = (size_t)u.nb * c.n_kv * rows_per_slot, first = ((size_t)(u.slot + blk) * c.n_kv + kvh) * rows_per_slot + r;
  const float* ml = x.ml + 2u * first;
  const float* po = x.o + first * HD + 4u * (lane % L);
  const size_t at = (size_t)row * HD + 4u * (lane % L);
  const float4u gate = x.a.gate ? *reinterpret_cast<const float4u*>(x.a.gate + at) : float4u{};
  float2 w[4];
  float4v y[4];
  auto load = [&](uint32_t i0) {
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t i = min(i0 + k * W * G, n - 1u);
      w[k] = *reinterpret_cast<const float2*>(ml + 2u * i * step);
      y[k] = *reinterpret_cast<const float4v*>(po + i * step * HD);
    }
  };
  load(part * G + lane / L);   // on its way beside the references
  float m = -__builtin_inff();
  for (uint32_t i = lane; i < n; i += 64u) m = fmaxf(m, ml[2u * i * step]);
  m = lane_reduce<64, true>(m);
  float l = 0.0f;
  float4v acc{};
  for (uint32_t i0 = part * G + lane / L; i0 < n; i0 += 4u * W * G) {
    if (i0 >= 4u * W * G) load(i0);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      if (i0 + k * W * G >= n || w[k].x == -__builtin_inff()) continue;
      const float e = __builtin_amdgcn_exp2f(w[k].x - m);
      l += w[k].y * e;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += y[k][j] * e;
    }
  }
  auto groups = [](float v) {   // sum over the wave's groups
    if constexpr (L <= 8) v += dpp_mov<0x128>(v);   // row_ror:8
    if constexpr (L <= 16) v = xor16_pair(v, false);
    if constexpr (L <= 32) v = xor32_pair(v, false);
    return v;
  };
  l = groups(l);
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = groups(acc[j]);
  if constexpr (W > 1) {
    s_acc[wave][lane] = acc;
    if (lane == 0) s_l[wave] = l;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (uint32_t k = 1; k < W; ++k) {
      l += s_l[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += s_acc[k][lane][j];
    }
  }
  if (lane >= L) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = l == 0.0f ? 0.0f : acc[j] / l;
  store_out(x.a, at, acc, gate);
}

// Workgroups of a kernel that run at once.
template <int HD, int NT, int RT>
uint32_t places_of() {
  static const uint32_t places = [] {
    int to_cu = 0, dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&to_cu, paged_attn_kernel<HD, NT, RT>, 256, 0) != hipSuccess || to_cu < 1 || cus < 1)
      return 512u;
    return (uint32_t)std::min(to_cu * cus, 4096);
  }();
  return places;
}

struct Sizes {
  uint32_t nt, rt, tb, places;
  uint64_t units, slots;
};
Sizes sizes_of(const PagesDev& c, const PagedDev& b, const PagedAttn& a) {
  Sizes z;
  const uint32_t group = a.n_head / c.n_kv;
  // Rows to a block by what a sequence has on average.  128 dims, 12 sequences of 2,000
  // to 20,000 rows, 4 kv heads, in forms of 8 and 16: 4 rows 32.8 and 33.1 us, 8 rows 41
  // and 35, 13 rows 48 and 41.6, 82 rows 104 and 71 (a token of 5 heads, 8 sequences of
  // 20,000 to 30,000 rows, 100 and 97); 64 dims, 6 rows 24.7 and 25.8, 12
  // rows 28.9 and 27.3.  256 dims, where 16 rows spill: 24 rows 111 and 122, 41 rows 220
  // and 140.  One token of 4 heads, 8 sequences of 20,000 to 30,000 rows: 4 rows 95 us, 8
  // rows 98.  Two column tiles, to 64 dims (at 64 they spill 23 registers, at 128 too
  // many: 82 rows 120 for 71), 12 sequences of 2,000 to 20,000 rows, 4 kv heads: 64 rows 41
  // and 41, 96 rows 56 and 52, 160 rows 81 and 78.  32 dims, in forms of 8, 16 and two
  // tiles of 16: 4 rows 17.4, 17.9 and 20.6 (of four rows 17.6), 8 rows 17.8, 18.1 and 21,
  // 16 rows 24, 19 and 22, 64 rows 46, 31 and 28, 160 rows 96, 61 and 50.
  const uint64_t rows = (uint64_t)b.n_tok * group;
  z.nt = c.hd <= 64 && rows > 64ull * b.n_seq ? 2u : 1u;
  z.rt = group <= 4u && b.n_tok <= b.n_seq ? 4u : rows > (c.hd == 256 ? 32ull : c.hd == 128 ? 4ull : 6ull) * b.n_seq ? 16u : 8u;
  z.tb = z.rt * z.nt / group;
  auto places = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    if constexpr (HD <= 64) {
      if (z.nt == 2) return places_of<HD, 2, 16>();
    }
    if (z.rt == 16) return places_of<HD, 1, 16>();
    return z.rt == 4 ? places_of<HD, 1, 4>() : places_of<HD, 1, 8>();
  };
  z.places = c.hd == 256   ? places(std::integral_constant<int, 256>{})
             : c.hd == 128 ? places(std::integral_constant<int, 128>{})
             : c.hd == 64  ? places(std::integral_constant<int, 64>{})
                           : places(std::integral_constant<int, 32>{});
  z.units = most_units(b, z.tb, c.n_kv, z.places);
  z.slots = most_slots(b, z.tb, c.n_kv, z.places);
  return z;
}

template <int HD, int NT, int RT>
void attn_hd(const PagesDev& c, const PagedDev& b, const AttnArgs& x, const Sizes& z, hipStream_t s) {
  const dim3 grid((uint32_t)((z.units + 7u) / 8u * 8u), c.n_kv);
  paged_attn_kernel<HD, NT, RT><<<grid, 256, 0, s>>>(c, b, x);
  if (z.slots == 0) return;
  const uint32_t rows = b.n_tok * x.a.n_head;
  // four waves to a row while rows are few (512 rows 27.0 us, with one wave 27.7;
  // 1,328 rows 33.0 and 30.7)
  if (rows <= 1024u)
    paged_join_kernel<HD, 4><<<rows, 256, 0, s>>>(c, b, x, RT * NT);
  else
    paged_join_kernel<HD, 1><<<(rows + 3u) / 4u, 256, 0, s>>>(c, b, x, RT * NT);
}

template <int HD>
void attn_nt(const PagesDev& c, const PagedDev& b, const AttnArgs& x, const Sizes& z, hipStream_t s) {
  if constexpr (HD <= 64) {
    if (z.nt == 2) return attn_hd<HD, 2, 16>(c, b, x, z, s);
  }
  if (z.rt == 16) return attn_hd<HD, 1, 16>(c, b, x, z, s);
  if (z.rt == 4) return attn_hd<HD, 1, 4>(c, b, x, z, s);
  attn_hd<HD, 1, 8>(c, b, x, z, s);
}

}  // namespace

size_t paged_attn_workspace(const PagesDev& c, const PagedDev& b, const PagedAttn& a) {
  const Sizes z = sizes_of(c, b, a);
  return (size_t)z.slots * c.n_kv * z.rt * z.nt * (c.hd + 2u) * sizeof(float);
}

hipError_t launch_paged_attn(const PagesDev& c, const PagedDev& b, const PagedAttn& a, void* ws, hipStream_t s) {
  const Sizes z = sizes_of(c, b, a);
  if (z.units > 0xfffff0u) return hipErrorInvalidValue;   // 2^32 threads: more than 2^25 query rows
  float* o = static_cast<float*>(ws);
  const AttnArgs x{a, a.n_head / c.n_kv, z.tb, (uint32_t)z.slots, z.places, o + (size_t)z.slots * c.n_kv * z.rt * z.nt * c.hd, o};
  switch (c.hd) {
    case 32: attn_nt<32>(c, b, x, z, s); break;
    case 64: attn_nt<64>(c, b, x, z, s); break;
    case 128: attn_nt<128>(c, b, x, z, s); break;
    case 256: attn_nt<256>(c, b, x, z, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace vxt
