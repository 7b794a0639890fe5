// attn_rows.hip -- attention of many query rows over one Q8_0 KV cache: a
// tree of drafted tokens, or a causal batch whose attention weights are
// summed per cache row (what eviction ranks by).
//
// Tree.  Node i (its K and V already in cache row pos + i) attends to rows
// [0, pos), its ancestors' rows and its own:
//   s = q . K / sqrt(hd),  p = softmax(s) over those rows,  out = sum p V.
// The ancestor sets are 256-bit masks, built in LDS by pointer doubling (each
// node ORs in its jump target's set and jumps twice as far: 8 rounds for any
// tree), and only by the workgroups whose rows reach past pos.
//
// Weighed batch.  Token m attends to rows [0, pos + m]; besides the output,
// weight[kv head][t] = sum over tokens and the group's heads of p.  p needs the
// row's whole sum first, so a second kernel forms the scores again, transposed
// (a wave holds 32 cache rows and walks the queries), from the queries'
// operands that the first one stored; sums in a fixed order, no atomics.
#include "kv_ops.hpp"

#include <algorithm>

namespace vxt {

namespace {

// Where the masks and jumps of a tree are built.
struct TreeLds {
  u32x4 anc[kTreeMax][2];
  int16_t jump[kTreeMax];
};

// anc[i] = the set of node i's ancestors and itself.  A parent outside
// [-1, i) counts as -1 (the node hangs on the last committed row).  One wave
// does it, with parents[lane + 64 u] in par[u]: in each round a node ORs in the
// set of the node its jump leads to and doubles the jump (itself, where it
// leads nowhere: a round is without branches), until no jump leads anywhere.
// The workgroup meets at a barrier after it.
__device__ __forceinline__ void tree_masks(const int (&par)[kTreeMax / 64], uint32_t n, TreeLds& t, uint32_t lane) {
  constexpr uint32_t PER = kTreeMax / 64;
  u32x4 m[PER][2];
  int jump[PER];
#pragma unroll
  for (uint32_t u = 0; u < PER; ++u) {
    const uint32_t i = lane + 64u * u;
    jump[u] = i >= n || par[u] < -1 || par[u] >= (int)i ? -1 : par[u];
#pragma unroll
    for (uint32_t w = 0; w < kTreeWords; ++w) m[u][w / 4u][w % 4u] = w == i / 32u ? 1u << (i & 31u) : 0u;
    t.jump[i] = (int16_t)jump[u];
    t.anc[i][0] = m[u][0];
    t.anc[i][1] = m[u][1];
  }
  wave_lds_order();
  for (;;) {
    int any = 0;
#pragma unroll
    for (uint32_t u = 0; u < PER; ++u) {
      if (64u * u >= n) break;   // uniform
      const uint32_t j = jump[u] < 0 ? lane + 64u * u : (uint32_t)jump[u];
      m[u][0] |= t.anc[j][0];
      m[u][1] |= t.anc[j][1];
      const int next = t.jump[j];
      jump[u] = jump[u] < 0 ? -1 : next;
      any |= jump[u] >= 0;
    }
    wave_lds_order();   // read before they are written
#pragma unroll
    for (uint32_t u = 0; u < PER; ++u) {
      if (64u * u >= n) break;
      t.anc[lane + 64u * u][0] = m[u][0];
      t.anc[lane + 64u * u][1] = m[u][1];
      t.jump[lane + 64u * u] = (int16_t)jump[u];
    }
    wave_lds_order();
    if (__builtin_amdgcn_ballot_w64(any != 0) == 0) break;
  }
}

// Which of the 32 rows from p0 a node sees (bit j: row p0 + j).
__device__ __forceinline__ uint32_t tree_sees(const uint32_t* anc, uint32_t p0, uint32_t pos) {
  if (p0 >= pos) {
    const uint32_t off = p0 - pos, w = off >> 5, sh = off & 31u;
    const uint32_t lo = w < kTreeWords ? anc[w] : 0u, hi = w + 1u < kTreeWords ? anc[w + 1u] : 0u;
    return sh ? (lo >> sh) | (hi << (32u - sh)) : lo;
  }
  const uint32_t k = pos - p0;
  return k >= 32u ? ~0u : (anc[0] << k) | ((1u << k) - 1u);
}

// ... a token at my_pos, causally.
__device__ __forceinline__ uint32_t causal_sees(uint32_t p0, uint32_t my_pos) {
  return my_pos < p0 ? 0u : my_pos - p0 >= 31u ? ~0u : (2u << (my_pos - p0)) - 1u;
}

// The first block of tq tokens from pos whose last token sees row `row`, which
// the last token of all sees.
__host__ __device__ __forceinline__ uint32_t causal_blocks(uint32_t row, uint32_t pos, uint32_t tq) {
  return row < pos + tq ? 0u : (row - pos) / tq;
}

struct RowsArgs {
  const float* q;
  const float* gate;   // gate and out: one segment only, else the join has them
  float* out;
  const int32_t* parents;
  uint32_t n_tok, pos, n_head, group, tq, blocks, seg_tiles, n_seg, split;   // split: a tree's first tile of the last segment
  float* ml;        // [n_tok * n_head][n_seg][2]: reference (base 2), sum
  float* o;         // [n_tok * n_head][n_seg][hd]
  uint4* frag;      // weigh: query operands, [n_kv][row tiles][2 terms][hd / 16][64 lanes]
  float* row_f;     // weigh: [n_kv][row tiles * 32] factor of the row's scores, a power of two
  float2* stat;     // weigh: [n_kv][row tiles * 32] reference and 1 / sum; +inf and 0 for a spare row, whose weight is 0
};

// Row stride of the V planes in LDS (f16): 16 words modulo 64, so the four
// rows x 16 words that a transposing read takes per half wave lie in
// different banks.
template <int HD>
constexpr uint32_t v_stride() { return HD == 32 ? 32u : HD + 32u; }

// Workgroup (kv head, block of tq tokens, segment of positions): RG waves of
// 32 query rows that share the tile of 32 positions.  Per tile:
//   S^T (positions x rows) = K Q^T, a fresh accumulator per 32-dim scale block,
//     K's codes exact in f16 and Q in two terms; S += d_k * block, in f32;
//   softmax against a reference per row that moves only when the maximum
//     passes it by 2^kWeightLag, so O is rescaled on few tiles;
//   O^T (dims x rows) += V^T P^T with V = code * scale as two exact f16 terms
//     (hi = q * d rounded, lo = fma(q, d, -hi)), the weights as two, hi hi +
//     hi lo + lo hi.  V lies in LDS as rows of positions and is read
//     transposed (ds_read_b64_tr_b16), in the order in which the scores'
//     accumulator holds the positions, so the weights go from accumulator to
//     operand without leaving their lane.
// V's scales are brought to [64, 128) at the top by a power of two found in a
// scan of the segment's scales ahead of the loop.
// The second product of a tile runs a tile late, beside the next one's softmax:
// matrix and vector unit work at once within a wave (without it each was busy
// 36 % of the time, one after the other, though two waves share a SIMD).
//
// Measured, heads of 128.  250 nodes over 30,011 rows, 32 / 8 heads: 332 us, 360
// in a long row of calls (the clock falls to 1.8 GHz), 372 TFLOP/s of the
// formula's products and 2.5 times that issued (two terms of Q, three products
// with V); matrix and vector unit busy 46 %, LDS 39 %.  64 nodes over 8,190 rows,
// 16 / 4 heads: 26 us, five tiles to a workgroup taking 12 of them, the rest the
// queries' way to operands, the scan and the sums' stores.  1,500 tokens
// causally, 16 / 4 heads: 44 us, eleven tiles to a workgroup.
template <int HD, int RG, bool TREE>
__global__ __launch_bounds__(64 * RG, (HD <= 64 && RG > 1) || (HD <= 128 && RG > 2) ? 2 : 1) void attn_rows_kernel(KvQ8Dev c, RowsArgs a) {
  constexpr uint32_t NT = 64 * RG, TP = 32, NST = HD / 16, NB = HD / 32;
  constexpr uint32_t KST = HD + 8, VST = v_stride<HD>();
  constexpr uint32_t NPC = TP * (HD / 16), PER = (NPC + NT - 1) / NT;   // pieces: 1 position x 16 dims
  struct alignas(16) Buf {
    _Float16 k[TP * KST], vh[TP * VST], vl[TP * VST];
    uint16_t kd[NB * TP], vd[NB * TP];   // scales as they are
    uint32_t odd[RG * PER];              // by who unpacked it: a V scale that is not finite among those
  };
  // the two tiles' buffers; before the first tile, the queries' staging, HQ dims at a time
  constexpr uint32_t HQ = HD < 64 ? HD : 64, QST = HQ + 4;
  constexpr size_t STAGE = (size_t)RG * 32u * QST * 4u;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[STAGE > 2u * sizeof(Buf) ? STAGE : 2u * sizeof(Buf)];
  Buf* const s_buf = reinterpret_cast<Buf*>(s_mem);
  __shared__ uint32_t s_top[RG];
  __shared__ TreeLds s_tree;         // dropped where TREE is false
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, h = lane >> 5, col = lane & 31u;
  uint32_t kvh = blockIdx.x, yb = blockIdx.y, seg = blockIdx.z;
  if constexpr (!TREE) {
    // the segments there are, one after the other: the first ones of all
    // blocks, then the second ones of those that have one, ...; the last
    // tokens' blocks, which have most rows to see, first
    kvh = blockIdx.x % c.n_kv;
    yb = blockIdx.x / c.n_kv;
    for (seg = 0; seg < a.n_seg; ++seg) {
      const uint32_t first = causal_blocks(seg * a.seg_tiles * 32u, a.pos, a.tq), n = a.blocks - first;
      if (yb < n) break;
      yb -= n;
    }
    if (seg == a.n_seg) return;   // not with the grid that goes with the plan
    yb = a.blocks - 1u - yb;
  }
  const uint32_t tb = yb * a.tq;
  const uint32_t t_end = min(a.n_tok, tb + a.tq);
  const uint32_t r = wave * 32u + col;
  const uint32_t tk = tb + r / a.group, g = r % a.group;
  const bool live = r < a.tq * a.group && tk < a.n_tok;
  const uint32_t tkc = live ? tk : tb;                  // spare rows shadow the block's first token
  const uint32_t head = kvh * a.group + g;
  const uint32_t my_pos = a.pos + tkc;
  const uint32_t last = TREE ? a.pos + a.n_tok - 1u : a.pos + t_end - 1u;
  const uint32_t full_end = TREE ? a.pos : a.pos + tb + 1u;   // every row of the block sees the positions below
  // A tree's last segment is what the others leave: the tiles with its nodes,
  // and as many before them as make up its length.
  const bool tail = TREE && seg + 1u == a.n_seg;
  const uint32_t tile0 = tail ? a.split : seg * a.seg_tiles;
  if (tile0 * TP > last) return;
  const uint32_t n_tiles = tail ? last / TP + 1u : min(TREE ? a.split : last / TP + 1u, tile0 + a.seg_tiles);
  const bool whole = TREE ? a.n_seg == 1u : last / TP < a.seg_tiles;   // the only segment: no partial sums
  const uint32_t row_q = c.n_kv * HD, row_d = c.n_kv * NB;

  // the first tile's bytes, then the queries, then the segment's V scales;
  // a position past the last one reads that again
  u32x4 kq[PER], vq[PER];
  uint32_t kdb[PER], vdb[PER];
  auto fetch = [&](uint32_t p0) {
#pragma unroll
    for (uint32_t u = 0; u < PER; ++u) {
      const uint32_t ch = min(tid + NT * u, NPC - 1u);
      const uint32_t p = min(p0 + ch / (HD / 16u), last), dg = ch % (HD / 16u);
      const size_t qo = (size_t)p * row_q + kvh * HD + 16u * dg, dof = (size_t)p * row_d + kvh * NB + dg / 2u;
      kq[u] = *reinterpret_cast<const u32x4*>(c.k_qs + qo);
      vq[u] = *reinterpret_cast<const u32x4*>(c.v_qs + qo);
      kdb[u] = c.k_d[dof];
      vdb[u] = c.v_d[dof];
    }
  };
  fetch(tile0 * TP);
  int par[TREE ? kTreeMax / 64 : 1];
  if constexpr (TREE) {
#pragma unroll
    for (uint32_t u = 0; u < kTreeMax / 64; ++u) par[u] = tail ? a.parents[min(lane + 64u * u, a.n_tok - 1u)] : -1;
  }

  // Q^T operand: lane holds row col's dims 16 st + 8 h .. + 7, two terms
  half8v q0[NST], q1[NST];
  float f_row;
  {
    // Through the wave's part of LDS: loaded in operand order, every lane would
    // be in a line of its own (four waves of 128 dims: 4,000 cycles).
    constexpr uint32_t LR = HQ / 4, RI = 64 / LR, NL = 32 / RI;
    float* sq = reinterpret_cast<float*>(s_mem) + wave * 32u * QST;
    const uint32_t by = 65536u / a.group + 1u;   // r / group = r * by >> 16 for r < 128, group <= 8
    float v[NST][8];
    float amax = 0.0f;
    float4v x[HD / HQ][NL];
#pragma unroll
    for (uint32_t i = 0; i < NL; ++i) {
      const uint32_t rl = wave * 32u + i * RI + lane / LR, t = (rl * by) >> 16, gl = rl - t * a.group;
      const bool in = rl < a.tq * a.group && tb + t < a.n_tok;
      const float* qr = a.q + ((size_t)(in ? tb + t : tb) * a.n_head + kvh * a.group + gl) * HD + 4u * (lane % LR);
#pragma unroll
      for (uint32_t p = 0; p < HD / HQ; ++p)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) x[p][i][j] = qr[HQ * p + j];
    }
#pragma unroll
    for (uint32_t p = 0; p < HD / HQ; ++p) {
#pragma unroll
      for (uint32_t i = 0; i < NL; ++i)
        *reinterpret_cast<float4v*>(sq + (i * RI + lane / LR) * QST + 4u * (lane % LR)) = x[p][i];
      wave_lds_order();
#pragma unroll
      for (uint32_t st = 0; st < HQ / 16u; ++st)
#pragma unroll
        for (uint32_t j = 0; j < 8; j += 4) {
          const float4v y = *reinterpret_cast<const float4v*>(sq + col * QST + 16u * st + 8u * h + j);
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            v[HQ / 16u * p + st][j + e] = y[e];
            amax = fmaxf(amax, fabsf(y[e]));
          }
        }
      wave_lds_order();   // read before the next dims are written
    }
    amax = xor32_pair(amax, true);
    // log2(e) / sqrt(hd) goes into the operand: what is left is a power of two,
    // so a score times it is exact, the same number in the maximum and the weight
    const float by2 = 1.4426950408889634f / sqrtf((float)HD);
    const int e = top_shift(amax * by2);
    const float up = by2 * pow2f(e);
    f_row = pow2f(-e);
#pragma unroll
    for (uint32_t st = 0; st < NST; ++st)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        float x = v[st][j] * up;
        asm("" : "+v"(x));   // one number: both terms are of the rounded product
        const _Float16 t0 = (_Float16)x;
        q0[st][j] = t0;
        q1[st][j] = (_Float16)(x - (float)t0);
      }
  }
  if (!TREE && seg == 0) {
    const uint32_t rt = yb * RG + wave, n_rt = a.blocks * RG;
    uint4* fr = a.frag + ((size_t)kvh * n_rt + rt) * (2u * NST * 64u) + lane;
#pragma unroll
    for (uint32_t st = 0; st < NST; ++st) {
      fr[st * 64u] = __builtin_bit_cast(uint4, q0[st]);
      fr[(NST + st) * 64u] = __builtin_bit_cast(uint4, q1[st]);
    }
    if (h == 0) {
      a.row_f[((size_t)kvh * n_rt + rt) * 32u + col] = f_row;
      if (!live || !whole) a.stat[((size_t)kvh * n_rt + rt) * 32u + col] = make_float2(__builtin_inff(), 0.0f);
    }
  }

  // the largest finite V scale of the segment, eight rows of a thread in flight
  {
    uint32_t top = 0;
    const uint32_t lo = tile0 * TP, end = min(last + 1u, n_tiles * TP);
    for (uint32_t p0 = lo + tid; p0 < end; p0 += 8u * NT) {
      Scales<NB> d[8];
#pragma unroll
      for (uint32_t u = 0; u < 8; ++u)
        d[u] = load_scales<NB>(c.v_d + (size_t)min(p0 + NT * u, end - 1u) * row_d + kvh * NB);
#pragma unroll
      for (uint32_t u = 0; u < 8; ++u) top = max(top, top_scale(d[u]));
    }
    top = lane_max_u32<64>(top);
    if (lane == 0) s_top[wave] = top;
  }
  if constexpr (TREE) {
    if (tail && wave == 0) tree_masks(par, a.n_tok, s_tree, lane);
  }
  __syncthreads();
  uint32_t top = s_top[0];
#pragma unroll
  for (uint32_t w = 1; w < RG; ++w) top = max(top, s_top[w]);
  const int kv = scale_shift(top);
  const float v_up = pow2f(kv);

  // Half `half` (8 dims) of the fetched piece u, of the tile from position p0,
  // into a buffer.  No branches: the code around it is scheduled as one.
  constexpr uint32_t ITEMS = 2u * PER;
  auto unpack = [&](Buf& s, uint32_t p0, uint32_t u, uint32_t half) {
    const uint32_t ch = min(tid + NT * u, NPC - 1u);   // spare threads repeat the last piece
    const uint32_t pp = ch / (HD / 16u), dg = ch % (HD / 16u);
    // a position past the last one adds nothing; where rows see different
    // positions, a scale that is not finite is kept out of the product and
    // left for the rows that see it to find
    const bool past = p0 + pp > last, bad = p0 + TP > full_end && (vdb[u] & 0x7c00u) == 0x7c00u;
    const float vd = past || bad ? 0.0f : f16_to_f32(vdb[u]) * v_up;
    if (half == 0) {   // two threads write the same
      s.kd[(dg / 2u) * TP + pp] = (uint16_t)kdb[u];
      s.vd[(dg / 2u) * TP + pp] = past ? 0 : (uint16_t)vdb[u];
      s.odd[wave * PER + u] = __builtin_amdgcn_ballot_w64(bad && !past) != 0 ? 1u : 0u;
    }
    const half2v vd2 = {(_Float16)vd, (_Float16)vd};
    u32x4 kk, hi, lo;
#pragma unroll
    for (uint32_t w = 0; w < 2; ++w) {
      half2v x[2], y[2];
      codes_f16(kq[u][2u * half + w], y[0], y[1]);
      codes_f16(vq[u][2u * half + w], x[0], x[1]);
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        const half2v p = x[e] * vd2;
        kk[2u * w + e] = __builtin_bit_cast(uint32_t, y[e]);
        hi[2u * w + e] = __builtin_bit_cast(uint32_t, p);
        lo[2u * w + e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x[e], vd2, -p));
      }
    }
    const uint32_t d = 16u * dg + 8u * half;
    *reinterpret_cast<u32x4*>(s.k + pp * KST + d) = kk;
    *reinterpret_cast<u32x4*>(s.vh + pp * VST + d) = hi;
    *reinterpret_cast<u32x4*>(s.vl + pp * VST + d) = lo;
  };

  float16x o[NB];
#pragma unroll
  for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
  float ref = -__builtin_inff(), l_run = 0.0f;

  // V operands of a tile.  A lane's address for the transposing reads: of 16
  // lanes, lane 4 i + j points at row i, dims 4 j; it gets dim lane % 16 of the
  // four rows.
  const uint32_t tr = (4u * h + ((lane & 15u) >> 2)) * VST + (col & 16u) + 4u * (lane & 3u);
  typedef __attribute__((address_space(3))) short4v lds_short4;
  auto read8 = [&](const _Float16* v, uint32_t at) {   // 4 + 4 positions of a dim
    const short4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(v + at));
    const short4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(v + at + 8u * VST));
    return __builtin_bit_cast(half8v, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // O^T += V^T P^T, a block of dims after the other, V read a unit ahead
  half8v ph[2], pl[2];   // the weights of the last tile, two terms
  auto weigh_values = [&](const Buf& s) {
    half8v vv[2][2];
    auto read_v = [&](uint32_t u) {   // unit u: block u % NB, positions 16 (u / NB) .. + 15
      const uint32_t at = tr + 16u * (u / NB) * VST + 32u * (u % NB);
      vv[u & 1u][0] = read8(s.vh, at);
      vv[u & 1u][1] = read8(s.vl, at);
    };
    read_v(0);
#pragma unroll
    for (uint32_t u = 0; u < 2u * NB; ++u) {
      if (u + 1u < 2u * NB) read_v(u + 1u);
      const uint32_t b = u % NB, x = u / NB;
      o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[u & 1u][0], ph[x], o[b], 0, 0, 0);
      o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[u & 1u][0], pl[x], o[b], 0, 0, 0);
      o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv[u & 1u][1], ph[x], o[b], 0, 0, 0);
    }
  };

  // no tile before the first: weights of zero, over values of zero
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) ph[i][j] = pl[i][j] = (_Float16)0.0f;
  {
    u32x4* z = reinterpret_cast<u32x4*>(s_buf[(tile0 & 1u) ^ 1u].vh);
    for (uint32_t i = tid; i < 2u * TP * VST / 8u; i += NT) z[i] = u32x4{0, 0, 0, 0};
  }
#pragma unroll
  for (uint32_t i = 0; i < ITEMS; ++i) unpack(s_buf[tile0 & 1u], tile0 * TP, i / 2u, i % 2u);
  fetch((tile0 + 1u) * TP);

  for (uint32_t T = tile0; T < n_tiles; ++T) {
    const uint32_t p0 = T * TP;
    const bool masked = p0 + TP > full_end;   // uniform: rows see different positions
    const Buf& s = s_buf[T & 1u];
    Buf& other = s_buf[(T & 1u) ^ 1u];   // V of the tile before, then the next tile
    lds_barrier();   // this tile is there
    // ahead of the CU's other workgroup while there are products to issue: its
    // vector work then fills in (trees of 250 nodes at 30,000: 395 -> 374 us)
    __builtin_amdgcn_s_setprio(1);
    // Scores: accumulator register i of this lane is position
    // p0 + 8 (i / 4) + 4 h + i % 4 of row col.  Step b: the products of block b
    // and the scaling of block b - 1's, for the vector unit to work while the
    // matrix unit does; operands are read a step ahead.
    float16x sacc, t[2];
    half8v kc[2][2];
    half4v dk[2][4];
    auto read_k = [&](uint32_t b) {
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e)
        kc[b & 1u][e] = *reinterpret_cast<const half8v*>(s.k + col * KST + 16u * (2u * b + e) + 8u * h);
    };
    read_k(0);
#pragma unroll
    for (uint32_t b = 0; b <= NB; ++b) {
      if (b < NB) {
        if (b + 1u < NB) read_k(b + 1u);
#pragma unroll
        for (int j = 0; j < 4; ++j) dk[b & 1u][j] = *reinterpret_cast<const half4v*>(s.kd + b * TP + 8u * j + 4u * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) t[b & 1u][i] = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
          t[b & 1u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kc[b & 1u][e], q0[2u * b + e], t[b & 1u], 0, 0, 0);
          t[b & 1u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kc[b & 1u][e], q1[2u * b + e], t[b & 1u], 0, 0, 0);
        }
      }
      if (b > 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sacc[i] = __builtin_fmaf((float)dk[(b - 1u) & 1u][i / 4][i % 4], t[(b - 1u) & 1u][i], b == 1 ? 0.0f : sacc[i]);
      }
      if (b < NB) {
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);    // the reads
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // an MFMA
          __builtin_amdgcn_sched_group_barrier(0x2, 5, 0);    // VALU
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    uint32_t mine = 0;
    if (masked) {
      mine = (TREE ? tree_sees(reinterpret_cast<const uint32_t*>(s_tree.anc[tkc]), p0, a.pos) : causal_sees(p0, my_pos)) >> (4u * h);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sacc[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1u ? sacc[i] : -__builtin_inff();
    }
    __builtin_amdgcn_sched_barrier(0);
    // The products with V of the tile before, and beside them this tile's
    // softmax.
    weigh_values(other);
    float pm = sacc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) pm = fmaxf(pm, sacc[i]);
    pm = xor32_pair(pm, true) * f_row;
    const bool move = pm - ref > kWeightUp + kWeightLag;
    const float to = move ? weight_ref(pm, kWeightUp) : ref;
    const float off = to == -__builtin_inff() ? 0.0f : to;   // no position yet: exp2(-inf) = 0
    float ps = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sacc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i], f_row, -off));
      ps += sacc[i];
    }
    u32x4 nh[2], nl[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t x, y;
        split_f16(sacc[8 * i + 2 * k], sacc[8 * i + 2 * k + 1], x, y);
        nh[i][k] = x;
        nl[i][k] = y;
      }
#pragma unroll
    for (uint32_t i = 0; i < 6u * NB; ++i) {
      if (i % 3u == 0) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);   // a unit's reads
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);      // an MFMA
      __builtin_amdgcn_sched_group_barrier(0x2, NB >= 4 ? 5 : 10, 0);   // VALU
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (__builtin_amdgcn_ballot_w64(move) != 0) {
      float alpha = move ? __builtin_amdgcn_exp2f(ref - to) : 1.0f;
      asm volatile("" : "+v"(alpha));   // a branch: not products and copies in every tile
      l_run *= alpha;
#pragma unroll
      for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] *= alpha;
    }
    ref = to;
    l_run += ps;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ph[i] = __builtin_bit_cast(half8v, nh[i]);
      pl[i] = __builtin_bit_cast(half8v, nl[i]);
    }
    if (masked) {
      uint32_t odd = 0, spoil = 0;
#pragma unroll
      for (uint32_t i = 0; i < RG * PER; ++i) odd |= s.odd[i];
      if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
        // a row that sees a V scale which is not finite: NaN in that block
#pragma unroll 1
        for (uint32_t b = 0; b < NB; ++b) {
          float bad = 0.0f;
#pragma unroll 1
          for (uint32_t i = 0; i < 16; ++i) {
            const uint32_t d = s.vd[b * TP + 8u * (i >> 2) + 4u * h + (i & 3u)];
            bad = (mine >> (8u * (i >> 2) + (i & 3u))) & 1u && (d & 0x7c00u) == 0x7c00u ? 1.0f : bad;
          }
          if (xor32_pair(bad, true) != 0.0f) spoil |= 1u << b;
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[b][i] = spoil >> b & 1u ? __builtin_nanf("") : o[b][i];
      }
    }
    lds_barrier();   // every wave is done with the tile before
#pragma unroll
    for (uint32_t i = 0; i < ITEMS; ++i) unpack(other, p0 + TP, i / 2u, i % 2u);   // behind the last tile: read by nobody
    fetch(p0 + 2u * TP);
    __builtin_amdgcn_sched_barrier(0);
  }
  weigh_values(s_buf[(n_tiles - 1u) & 1u]);

  l_run = xor32_pair(l_run, false);   // the row's other half of the positions
  if (!live) return;
  const float down = pow2f(-kv);
  if (whole) {
    // 16 bytes a lane, the gates all on their way first: one by one, and a
    // float at a time, the stores of a block took as long as ten tiles
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    const float inv = down / l_run;
    const size_t base = ((size_t)tk * a.n_head + head) * HD + 4u * h;
    float4u gv[4 * NB];
    if (a.gate) {
#pragma unroll
      for (uint32_t j = 0; j < 4u * NB; ++j) gv[j] = *reinterpret_cast<const float4u*>(a.gate + base + 8u * j);
    }
#pragma unroll
    for (uint32_t j = 0; j < 4u * NB; ++j) {
      float4u v;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        v[i] = o[j / 4u][4u * (j % 4u) + i] * inv;
        if (a.gate) v[i] *= 1.0f / (1.0f + expf(-gv[j][i]));
      }
      *reinterpret_cast<float4u*>(a.out + base + 8u * j) = v;
    }
    if (!TREE && h == 0)
      a.stat[((size_t)kvh * a.blocks * RG + yb * RG + wave) * 32u + col] = make_float2(l_run != l_run ? 0.0f : ref, 1.0f / l_run);
    return;
  }
  const size_t at = ((size_t)tk * a.n_head + head) * a.n_seg + seg;
  if (h == 0) {
    a.ml[2u * at] = l_run != l_run ? 0.0f : ref;   // -inf only where nothing was seen
    a.ml[2u * at + 1u] = l_run;
  }
  float* po = a.o + at * HD + 4u * h;
#pragma unroll
  for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float4v v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = o[b][4 * j + i] * down;
      *reinterpret_cast<float4v*>(po + 32u * b + 8u * j) = v;
    }
}

template <int HD, int W>
__global__ __launch_bounds__(256) void attn_join_kernel(JoinCall a) {
  __shared__ JoinLds<HD, W> s;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t row = W == 1 ? (blockIdx.x * 256u + threadIdx.x) / (HD / 4u) : blockIdx.x;
  if (row < a.n_rows) join_row<HD, W>(a, row, W == 1 ? 0u : wave, lane, s);
}

template <int HD>
hipError_t launch_join_hd(const JoinCall& j, hipStream_t s) {
  // Heads of 128, half a wave to a row against four, sixteen: 416
  // rows of 33 partials 8.1, 4.5, 6.9 us, 1,024 of 52 10.7, 7.2, 12.2, 8,000 of 8
  // 7.8, 21.9, 67.
  if (j.n_rows < 2048u && j.n_seg > 8u)
    hipLaunchKernelGGL((attn_join_kernel<HD, 4>), dim3(j.n_rows), dim3(256), 0, s, j);
  else
    hipLaunchKernelGGL((attn_join_kernel<HD, 1>), dim3((j.n_rows + 1024 / HD - 1) / (1024 / HD)), dim3(256), 0, s, j);
  return hipGetLastError();
}

// Column sums of the softmax: workgroup (kv head, 128 cache rows, `per` of the
// query row tiles that see them), 4 waves of 32 cache rows.  A wave keeps its
// rows' K as operands; the workgroup stages one query tile (32 rows, two terms)
// after the other in LDS, the next one's pieces on their way.  p = exp2(s f -
// reference) / sum, the two apart: log2 of the sum on top of a large reference
// would lose its bits.  1,500 tokens, 16 / 4 heads of 128: 20 us for 4.6 GFLOP of
// scores (twice that issued); 32 with a tile's pieces loaded when it was due and a
// third of the workgroups in a second round.
struct WeighArgs {
  const uint4* frag;
  const float* row_f;
  const float2* stat;
  uint32_t n_tok, pos, group, tq, rg, n_rt, per, n_split;
  float* part;        // [n_split][n_kv][rows], when n_split > 1: a block of rows has the first few
  float* weight;
  uint32_t* position;
  uint32_t plane, tok_pos;
};

// The first row tile of tokens that see cache row 128 y.
__host__ __device__ __forceinline__ uint32_t weigh_first(uint32_t y, uint32_t pos, uint32_t tq, uint32_t rg) {
  return 128u * y > pos ? (128u * y - pos) / tq * rg : 0u;
}
// Blocks of 128 cache rows that more than `done` row tiles see: the first ones.
__host__ __device__ __forceinline__ uint32_t weigh_blocks(uint32_t done, uint32_t pos, uint32_t n_tok, uint32_t tq, uint32_t rg, uint32_t n_rt) {
  if (done >= n_rt) return 0u;
  return (min(pos + (n_rt - done + rg - 1u) / rg * tq, pos + n_tok) + 127u) / 128u;
}

template <int HD>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_weigh_kernel(KvQ8Dev c, WeighArgs a) {
  constexpr uint32_t NST = HD / 16, NB = HD / 32, NF = 2u * NST * 64u, PER = NF / 256u;   // 16-byte pieces of a query tile
  __shared__ u32x4 s_q[2][NF];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, h = lane >> 5, col = lane & 31u;
  const uint32_t kvh = blockIdx.x % c.n_kv, rows = a.pos + a.n_tok;
  // the pieces there are: all blocks' first, those blocks' second that have one, ...
  uint32_t y = blockIdx.x / c.n_kv, z = 0;
  for (; z < a.n_split; ++z) {
    const uint32_t blocks = weigh_blocks(z * a.per, a.pos, a.n_tok, a.tq, a.rg, a.n_rt);
    if (y < blocks) break;
    y -= blocks;
  }
  if (z == a.n_split) return;   // not with the grid that goes with the plan
  const uint32_t p0 = y * 128u + wave * 32u;
  const uint32_t row_q = c.n_kv * HD, row_d = c.n_kv * NB;

  const uint32_t rt0 = weigh_first(y, a.pos, a.tq, a.rg) + z * a.per, rt1 = min(a.n_rt, rt0 + a.per);
  // a tile's operands and its rows' numbers, a tile ahead
  u32x4 x[PER];
  float f_next;
  float2 stat_next;
  auto fetch = [&](uint32_t rt) {
    const size_t at = (size_t)kvh * a.n_rt + min(rt, a.n_rt - 1u);
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) x[i] = reinterpret_cast<const u32x4*>(a.frag)[at * NF + 256u * i + tid];
    f_next = a.row_f[at * 32u + col];
    stat_next = a.stat[at * 32u + col];
  };
  fetch(rt0);

  half8v k8[NST];
  {
    const int8_t* kr = c.k_qs + (size_t)min(p0 + col, rows - 1u) * row_q + kvh * HD + 8u * h;
#pragma unroll
    for (uint32_t st = 0; st < NST; ++st) k8[st] = codes8_f16(*reinterpret_cast<const u32x2*>(kr + 16u * st));
  }
  _Float16 dk[NB][16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t p = min(p0 + 8u * (i >> 2) + 4u * h + (i & 3), rows - 1u);
    const Scales<NB> d = load_scales<NB>(c.k_d + (size_t)p * row_d + kvh * NB);
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) dk[b][i] = __builtin_bit_cast(_Float16, d.d[b]);
  }
  float sum[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[i] = 0.0f;

  const uint32_t by = 65536u / a.group + 1u;   // r / group = r * by >> 16 for r < 128, group <= 8
  for (uint32_t rt = rt0; rt < rt1; ++rt) {
    u32x4* const s = s_q[(rt - rt0) & 1u];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) s[256u * i + tid] = x[i];
    const float f = f_next;
    const float ref = stat_next.x;
    float inv = stat_next.y;
    lds_barrier();   // the tile is there; every wave is done with the one before the last
    fetch(rt + 1u);
    // rg is 1, 2 or 4
    const uint32_t tb = (rt >> (a.rg >> 1)) * a.tq, tb_end = min(a.n_tok, tb + a.tq);
    if (p0 >= a.pos + tb_end) continue;   // uniform: none of the tile's tokens sees the wave's rows
    float16x sacc, t[2];
#pragma unroll
    for (uint32_t b = 0; b <= NB; ++b) {   // the products of block b beside the scaling of block b - 1's
      if (b < NB) {
#pragma unroll
        for (int i = 0; i < 16; ++i) t[b & 1u][i] = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
          const uint32_t st = 2u * b + e;
          t[b & 1u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[st], __builtin_bit_cast(half8v, s[st * 64u + lane]), t[b & 1u], 0, 0, 0);
          t[b & 1u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8[st], __builtin_bit_cast(half8v, s[(NST + st) * 64u + lane]),
                                                            t[b & 1u], 0, 0, 0);
        }
      }
      if (b > 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sacc[i] = __builtin_fmaf((float)dk[b - 1u][i], t[(b - 1u) & 1u][i], b == 1 ? 0.0f : sacc[i]);
      }
    }
    if (p0 + 31u > a.pos + tb) {   // uniform: the tile's tokens see different rows of the wave's
      const uint32_t r = (rt & (a.rg - 1u)) * 32u + col, tk = tb + ((r * by) >> 16);
      // a spare row has a reference of +inf; it shadows the block's first token, rows that this does not see included
      const bool live = r < a.tq * a.group && tk < a.n_tok;
      const uint32_t mine = causal_sees(p0, a.pos + (live ? tk : tb)) >> (4u * h);
      // a sum of NaN goes to the rows that its token sees, and to no other
      const float nan = inv == inv ? 0.0f : inv;
      inv = inv == inv ? inv : 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sacc[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1u ? sacc[i] + nan : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(sacc[i], f, -ref)), inv, sum[i]);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float v = lane_reduce<32>(sum[i]);
    const uint32_t p = p0 + 8u * (i >> 2) + 4u * h + (i & 3);
    if (col == 0 && p < rows) {
      if (a.n_split > 1) {
        a.part[((size_t)z * c.n_kv + kvh) * rows + p] = v;
      } else {
        const size_t at = (size_t)kvh * a.plane + p;
        a.weight[at] = p < a.pos ? a.weight[at] + v : v;
        if (p >= a.pos) a.position[at] = a.tok_pos + (p - a.pos);
      }
    }
  }
}

__global__ __launch_bounds__(64) void attn_weigh_join_kernel(WeighArgs a, uint32_t n_kv) {
  const uint32_t rows = a.pos + a.n_tok, p = blockIdx.x * 64u + threadIdx.x, kvh = blockIdx.y;
  if (p >= rows) return;
  float v = 0.0f;
  const uint32_t n = (a.n_rt - weigh_first(p / 128u, a.pos, a.tq, a.rg) + a.per - 1u) / a.per;
  const size_t at = (size_t)kvh * a.plane + p;
  const float old = a.weight[at];
  for (uint32_t z0 = 0; z0 < n; z0 += 8u) {   // eight on their way, added in order
    float x[8];
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) x[u] = a.part[((size_t)min(z0 + u, n - 1u) * n_kv + kvh) * rows + p];
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) v += z0 + u < n ? x[u] : 0.0f;
  }
  a.weight[at] = p < a.pos ? old + v : v;
  if (p >= a.pos) a.position[at] = a.tok_pos + (p - a.pos);
}

// Workgroups of four waves that run at once, two to a CU.
constexpr uint32_t kRowsAtOnce = 512;

// How a call is cut: RG waves of rows per workgroup, tokens per workgroup,
// segments.  The segments are as many as run at once (one more would wait for a
// whole one), at most 64 to a row (the join reads them all).  One tile to a
// segment pays where there are few: alone on its CU a tile takes 1.5 to 4 us
// (64 to 256 dims), the join 3: six nodes at 150, heads of 64 10.3 us, with two
// tiles to a segment 10.7, with one segment of five 12.5; of 128 13.5, 15.0 and
// 19.8; of 256 18.1, 20.5 and 30.1.
struct RowsPlan {
  uint32_t rg, tq, blocks, seg_tiles, n_seg, split, n_rt, per, n_split, weigh_wgs;
  size_t ml, o, frag, row_f, stat, part, total;   // byte offsets in the workspace
};

// The least s in [lo, hi) with ok(s), ok being false and then true; hi if none.
template <class Ok>
uint32_t least(uint32_t lo, uint32_t hi, Ok ok) {
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2u;
    if (ok(mid)) hi = mid;
    else lo = mid + 1u;
  }
  return hi;
}

RowsPlan rows_plan(const KvQ8Dev& c, const RowsCall& r) {
  RowsPlan p{};
  const uint32_t group = r.n_head / c.n_kv;
  const size_t rows = (size_t)r.n_tok * group;
  p.rg = rows <= 32 && c.hd <= 128 ? 1u : rows <= 64 ? 2u : 4u;   // one wave of head_dim 256 would spill
  p.tq = 32u * p.rg / group;
  p.blocks = (r.n_tok + p.tq - 1) / p.tq;
  const uint32_t full = r.pos / 32u, all_tiles = (r.pos + r.n_tok - 1u) / 32u + 1u, grid = c.n_kv * p.blocks;
  const uint32_t want = std::max(1u, std::min(64u, kRowsAtOnce / grid));
  if (r.parents) {
    // a tile with nodes, and the masks, take about twice a tile's time
    const uint32_t odd = 2u * (all_tiles - full) + 2u;
    p.seg_tiles = std::max(1u, (full + odd + want - 1) / want);
    p.split = full - std::min(full, p.seg_tiles > odd ? p.seg_tiles - odd : 0u);
    p.n_seg = (p.split + p.seg_tiles - 1) / p.seg_tiles + 1u;
  } else {
    // the shortest segments with which all the blocks' run at once; a block has
    // as many as its last token's rows take
    p.seg_tiles = least((all_tiles + 63u) / 64u, (all_tiles + want - 1) / want, [&](uint32_t s) {
      uint64_t n = 0;
      for (uint32_t b = 0; b < p.blocks && n <= kRowsAtOnce; ++b)
        n += (uint64_t)c.n_kv * ((r.pos + std::min(r.n_tok, (b + 1) * p.tq) - 1u) / 32u / s + 1u);
      return n <= kRowsAtOnce;
    });
    p.n_seg = (all_tiles - 1u) / p.seg_tiles + 1u;
  }
  p.n_rt = p.blocks * p.rg;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off += (n + 255) & ~(size_t)255;
    return at;
  };
  const size_t all = (size_t)r.n_tok * r.n_head * p.n_seg;
  if (p.n_seg > 1) {
    p.ml = take(all * 8);
    p.o = take(all * c.hd * 4);
  }
  p.n_split = 1;
  if (!r.parents) {
    p.frag = take((size_t)c.n_kv * p.n_rt * 2 * (c.hd / 16) * 64 * 16);
    p.row_f = take((size_t)c.n_kv * p.n_rt * 32 * 4);
    p.stat = take((size_t)c.n_kv * p.n_rt * 32 * 8);
    // the fewest row tiles a workgroup with which all run at once, or all of them
    auto wgs = [&](uint32_t per) {
      uint64_t n = 0;
      for (uint32_t done = 0; done < p.n_rt && n <= kRowsAtOnce; done += per)
        n += (uint64_t)c.n_kv * weigh_blocks(done, r.pos, r.n_tok, p.tq, p.rg, p.n_rt);
      return n;
    };
    p.per = least(std::max(2u, (p.n_rt + 31u) / 32u), p.n_rt, [&](uint32_t per) { return wgs(per) <= kRowsAtOnce; });
    p.n_split = (p.n_rt - 1u) / p.per + 1u;
    p.weigh_wgs = 0;
    for (uint32_t z = 0; z < p.n_split; ++z) p.weigh_wgs += c.n_kv * weigh_blocks(z * p.per, r.pos, r.n_tok, p.tq, p.rg, p.n_rt);
    if (p.n_split > 1) p.part = take((size_t)p.n_split * c.n_kv * (r.pos + r.n_tok) * 4);
  }
  p.total = off;
  return p;
}

template <int HD, bool TREE>
hipError_t launch_rows_rg(const KvQ8Dev& c, const RowsArgs& a, const RowsPlan& p, hipStream_t s) {
  dim3 grid(c.n_kv, p.blocks, p.n_seg);
  if (!TREE) {
    uint32_t n = 0;
    for (uint32_t z = 0; z < p.n_seg; ++z) n += p.blocks - causal_blocks(z * p.seg_tiles * 32u, a.pos, p.tq);
    grid = dim3(c.n_kv * n);
  }
  switch (p.rg) {
    case 1:
      if constexpr (HD <= 128) hipLaunchKernelGGL((attn_rows_kernel<HD, 1, TREE>), grid, dim3(64), 0, s, c, a);
      break;
    case 2: hipLaunchKernelGGL((attn_rows_kernel<HD, 2, TREE>), grid, dim3(128), 0, s, c, a); break;
    default: hipLaunchKernelGGL((attn_rows_kernel<HD, 4, TREE>), grid, dim3(256), 0, s, c, a); break;
  }
  return hipGetLastError();
}

template <int HD>
hipError_t launch_rows_hd(const KvQ8Dev& c, const RowsCall& r, void* ws, hipStream_t s) {
  const bool tree = r.parents != nullptr;
  const RowsPlan p = rows_plan(c, r);
  char* base = static_cast<char*>(ws);
  const uint32_t group = r.n_head / c.n_kv;
  RowsArgs a{};
  a.q = r.q;
  a.gate = r.gate;
  a.out = r.out;
  a.parents = r.parents;
  a.n_tok = r.n_tok;
  a.pos = r.pos;
  a.n_head = r.n_head;
  a.group = group;
  a.tq = p.tq;
  a.blocks = p.blocks;
  a.seg_tiles = p.seg_tiles;
  a.n_seg = p.n_seg;
  a.split = p.split;
  a.ml = reinterpret_cast<float*>(base + p.ml);
  a.o = reinterpret_cast<float*>(base + p.o);
  if (!tree) {
    a.frag = reinterpret_cast<uint4*>(base + p.frag);
    a.row_f = reinterpret_cast<float*>(base + p.row_f);
    a.stat = reinterpret_cast<float2*>(base + p.stat);
  }
  hipError_t e = tree ? launch_rows_rg<HD, true>(c, a, p, s) : launch_rows_rg<HD, false>(c, a, p, s);
  if (e != hipSuccess) return e;
  if (p.n_seg > 1) {
    const JoinCall j{a.ml, a.o, r.gate, r.out, r.n_tok * r.n_head, r.n_head, p.n_seg, p.seg_tiles * 32u, r.pos,
                     tree ? 0u : 1u, a.stat, group, p.tq, p.rg, p.n_rt, r.n_tok};
    e = launch_join_hd<HD>(j, s);
  }
  if (e != hipSuccess || tree) return e;
  const WeighArgs w{a.frag, a.row_f, a.stat, r.n_tok, r.pos, group, p.tq, p.rg, p.n_rt, p.per, p.n_split,
                    reinterpret_cast<float*>(base + p.part), r.weight, r.position, r.plane, r.tok_pos};
  const uint32_t rows = r.pos + r.n_tok;
  hipLaunchKernelGGL(attn_weigh_kernel<HD>, dim3(p.weigh_wgs), dim3(256), 0, s, c, w);
  e = hipGetLastError();
  if (e != hipSuccess || p.n_split == 1) return e;
  hipLaunchKernelGGL(attn_weigh_join_kernel, dim3((rows + 63u) / 64u, c.n_kv), dim3(64), 0, s, w, c.n_kv);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_join(uint32_t hd, const JoinCall& j, hipStream_t s) {
  switch (hd) {
    case 32: return launch_join_hd<32>(j, s);
    case 64: return launch_join_hd<64>(j, s);
    case 128: return launch_join_hd<128>(j, s);
    case 256: return launch_join_hd<256>(j, s);
    default: return hipErrorInvalidValue;
  }
}

size_t attn_rows_workspace(const KvQ8Dev& c, const RowsCall& r) { return rows_plan(c, r).total; }

// Requires hd in {32, 64, 128, 256}, n_head % n_kv == 0, n_head / n_kv <= 8,
// pos + n_tok <= max_seq (and plane), a tree's parents, n_tok <= kTreeMax, or a
// batch's weights; ws holds attn_rows_workspace(c, r) bytes.
hipError_t launch_attn_rows(const KvQ8Dev& c, const RowsCall& r, void* ws, hipStream_t s) {
  const uint32_t group = r.n_head / c.n_kv;
  if (group == 0 || group > 8u || r.n_tok == 0 || !r.parents == !r.weight || (r.parents && r.n_tok > kTreeMax)) return hipErrorInvalidValue;
  switch (c.hd) {
    case 32: return launch_rows_hd<32>(c, r, ws, s);
    case 64: return launch_rows_hd<64>(c, r, ws, s);
    case 128: return launch_rows_hd<128>(c, r, ws, s);
    case 256: return launch_rows_hd<256>(c, r, ws, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace vxt
