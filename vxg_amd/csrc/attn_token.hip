// attn_token.hip -- attention of single tokens over a Q8_0 KV cache on MFMA,
// in two forms that a plain decode step does not have: with the weights of
// the cache's rows summed up (what eviction ranks by), and over blocks of rows
// that a cheap score selects.
//
// Block selection, per (token, kv head).  The summary of a block of B rows is
// the mean of its dequantised keys, as Q8_0 blocks (kv_block_mean_kernel).
// The group's queries, summed in 64 bits and rounded to f32, are quantised the
// same way; the score of a block is
//   f32( sum over 32-value blocks b of  d_q[b] * d_k[b] * (code dot)_b )
// with the sum in 64 bits, where every term is exact: neighbours first, then
// pairs of them, then fours (it rounds where the scales lie far apart).  The
// first n_first and the last n_local blocks (the token's own among them) are
// taken whatever they score, the rest of n_sel by score, the lowest index first
// among equals, NaN last.  The heads of the group attend to the rows of the
// selected blocks up to the token's own.
#include "kv_ops.hpp"

#include <algorithm>

namespace vxt {

namespace {

struct TokenArgs {
  const float* q;
  const float* gate;
  float* out;
  uint32_t n_head, group, seq, tiles, n_chunk, n_unit;   // token z sees rows [0, seq + z); tiles of 32 rows to a wave; tokens * chunks
  float* ml;         // [rows][n_chunk][2]
  float* o;          // [rows][n_chunk][hd]
  float* score;      // weigh: [n_head][stride] base-2 scores
  uint32_t stride;
  const uint32_t* sel;   // blocks: [tokens][n_kv][n_sel], ascending, kNoBlock behind the last
  uint32_t block, n_sel;
};

// Workgroup (kv head, chunk of a token's tiles): 4 waves, each on its own tiles
// of 32 rows.  Workgroups go round the eight XCDs by their number, each with an
// L2 of its own; the kv heads of a chunk take numbers of one XCD, because a
// row's scales of all heads lie in one cache line (60000 rows, 8 kv heads: the
// L2s fetched half as much again as the planes hold with a head per XCD).  The
// 16 columns of v_mfma_f32_16x16x32_f16 are the (at most 8) heads of the group
// in two f16 terms: column n is head n % 8, term n / 8.
//   S (positions x columns) = K Q^T per 32-dim block, K's codes exact, then
//     S += d_k * block and the two terms' columns added: the lanes of column n
//     and n + 8 both hold head n % 8's scores of 8 positions;
//   O^T (dims x columns) += V^T W with V's codes exact and W = weight * d_v, per
//     32-dim block, as the first or the second f16 term of the lane's column.
// A lane's 8 positions are those of its operand in the second product, so no
// weight leaves its lane.  K, V and the scales go through a wave's own LDS as
// rows: read from memory in operand order, neighbouring lanes would be in
// different rows, and a load of 64 separate lines holds the L1 for 64 cycles
// (400 tokens x 16 blocks of 64 rows, 16 heads x 128: 117 us that way).  V is
// read transposed (ds_read_b64_tr_b8).
// V's scales carry the power of two that brings the wave's largest up to
// [1/2, 1), the weights the one that makes up for a larger one, 2^13 at most, so
// that with weights of at most 2^15 the products stay below 2^15.  No scale is
// rounded, but for those 2^24 below a largest of 2^13 or more (to 2^-37 of it).
// Two terms each hold a product to 2^-36 of the largest weight times the largest
// scale (f16 ends at 2^-24).
// 60,001 rows, 8 kv heads of 128: 32 us, 4.1 TB/s of the planes.  400 tokens x 16
// blocks, 4 kv heads: 78 us, the vector unit busy 74 % (520 instructions to a
// tile and wave, 160 of them codes to f16, 80 the weights times the scales), 5.8
// TB/s of rows out of the L2s.
template <int HD, bool BLOCKS>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_token_kernel(KvQ8Dev c, TokenArgs a) {
  constexpr uint32_t NB = HD / 32, ND = HD / 16, VST = HD + 16;   // row stride of K and V in LDS (bytes)
  constexpr uint32_t LPR = HD / 16;                               // lanes to a row of K or V
  constexpr uint32_t KV = 32u * VST, DS = 32u * NB * 2u, WAVE = 2u * KV + 2u * DS;   // bytes: K or V, their scales, a wave's
  constexpr uint32_t BUF = 4u * 8u * HD * 4u > 4u * WAVE ? 4u * 8u * HD * 4u : 4u * WAVE;
  __shared__ __attribute__((aligned(16))) uint8_t s_buf[BUF];
  __shared__ float s_ml[4][8][2];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t n = lane & 15u, g = lane >> 4, r = n & 7u;
  const bool second = n >= 8u;
  const uint32_t slot = blockIdx.x / 8u, unit = slot / c.n_kv * 8u + blockIdx.x % 8u, kvh = slot % c.n_kv;
  if (unit >= a.n_unit) return;
  const uint32_t z = unit / a.n_chunk, ck = unit % a.n_chunk;
  const uint32_t seq = a.seq + z, group = a.group;
  const uint32_t row_q = c.n_kv * HD, row_d = c.n_kv * NB;
  const uint32_t bt = BLOCKS ? a.block / 32u : 1u;
  const uint32_t n_vt = BLOCKS ? a.n_sel * bt : (seq + 31u) / 32u;
  const uint32_t vt0 = (ck * 4u + wave) * a.tiles, vt1 = min(n_vt, vt0 + a.tiles);
  const uint32_t* sel = BLOCKS ? a.sel + ((size_t)z * c.n_kv + kvh) * a.n_sel : nullptr;

  // first row of tile vt, or seq where there is none
  auto tile_row = [&](uint32_t vt) -> uint32_t {
    if (vt >= vt1) return seq;
    if constexpr (BLOCKS) {
      const uint32_t blk = sel[vt / bt];
      return blk == kNoBlock ? seq : min(seq, blk * a.block + (vt % bt) * 32u);
    }
    return vt * 32u;
  };

  // A tile's bytes on their way to LDS, loaded for the next tile as soon as
  // they are there -- always, behind the last tile the same one again: a
  // conditional load would be waited for on the spot, to be copied.  The
  // tile's first row is uniform; positions past the last row read it again.
  // Lanes 0 .. 31 load a row's K scales, the others its V scales.
  u32x4 k16[NB], v16[NB];
  Scales<NB> d16;
  auto load = [&](uint32_t t0) {
    const size_t base = (size_t)t0 * row_q + kvh * HD;
    const uint32_t lim = seq - t0 - 1u;
#pragma unroll
    for (uint32_t j = 0; j < NB; ++j) {
      const uint32_t off = min(j * (64u / LPR) + lane / LPR, lim) * row_q + 16u * (lane % LPR);
      k16[j] = *reinterpret_cast<const u32x4*>(c.k_qs + base + off);
      v16[j] = *reinterpret_cast<const u32x4*>(c.v_qs + base + off);
    }
    const uint16_t* plane = lane < 32u ? c.k_d : c.v_d;
    d16 = load_scales<NB>(plane + (size_t)t0 * row_d + kvh * NB + min(lane & 31u, lim) * row_d);
  };
  uint32_t t0 = tile_row(vt0);
  if (t0 < seq) load(t0);

  // Q^T operand and the power of two of its rows
  half8v qb[NB];
  float f_row;
  {
    const float* qr = a.q + ((size_t)z * a.n_head + kvh * group + min(r, group - 1u)) * HD + 8u * g;
    float v[NB][8];
    float amax = 0.0f;
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) v[b][j] = qr[32u * b + j];
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[b][j]));
    amax = xor32_pair(xor16_pair(amax, true), true);
    const int e = top_shift(amax);
    const float up = pow2f(e);
    f_row = 1.4426950408889634f / sqrtf((float)HD) * pow2f(-e);
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const float x = v[b][j] * up;
        const _Float16 hi = (_Float16)x;
        qb[b][j] = second ? (_Float16)(x - (float)hi) : hi;
      }
  }
  // the largest finite V scale of the wave's tiles, eight tiles in flight
  uint32_t top = 0;
  for (uint32_t v0 = vt0; v0 < vt1; v0 += 8u) {
    Scales<NB> d[8];
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) {   // past the last tile (or block) the cache's last row
      const uint32_t row = min(tile_row(v0 + u) + (lane & 31u), seq - 1u);
      d[u] = load_scales<NB>(c.v_d + (size_t)row * row_d + kvh * NB);
    }
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) top = max(top, v0 + u < vt1 ? top_scale(d[u]) : 0u);
  }
  top = lane_max_u32<32>(top);
  // V's scales are brought up in f16, in two steps (2^15 is f16's largest power)
  const int to_top = scale_shift(top) - 7, up = (int)kWeightUp;
  const int kv = max(to_top, 0) + min(to_top + up, 0), kv1 = min(kv, 15);
  const float w_up = (float)max(up + min(to_top, 0), 0);
  const _Float16 up1 = (_Float16)pow2f(kv1), up2 = (_Float16)pow2f(kv - kv1);
  const half2v d_up1 = {up1, up1}, d_up2 = {up2, up2};

  float4v o[ND];
#pragma unroll
  for (uint32_t d = 0; d < ND; ++d) o[d] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  float ref = -__builtin_inff(), l_run = 0.0f;
  uint8_t* const sk = s_buf + wave * WAVE;
  uint8_t* const sv = sk + KV;
  uint8_t* const sd = sv + KV;             // K's scales, then V's: [32 rows][NB]
  // 8 rows' scales of this lane: value b of row j is f16 j * NB + b
  auto scales = [&](uint32_t which, u32x4 (&d)[NB]) {
#pragma unroll
    for (uint32_t i = 0; i < NB; ++i) d[i] = *reinterpret_cast<const u32x4*>(sd + which * DS + 16u * NB * g + 16u * i);
  };
  // f16 i of them
  auto word_of = [](const u32x4 (&d)[NB], uint32_t i) { return (uint32_t)d[i / 8][(i % 8) / 2]; };

  for (uint32_t vt = vt0; t0 < seq; ++vt) {
    const uint32_t t1 = tile_row(vt + 1u);
#pragma unroll
    for (uint32_t j = 0; j < NB; ++j) {
      const uint32_t at = (j * (64u / LPR) + lane / LPR) * VST + 16u * (lane % LPR);
      *reinterpret_cast<u32x4*>(sk + at) = k16[j];
      *reinterpret_cast<u32x4*>(sv + at) = v16[j];
    }
    *reinterpret_cast<Scales<NB>*>(sd + lane * 2u * NB) = d16;
    load(t1 < seq ? t1 : t0);
    wave_lds_order();
    float s[8];
    {
      u32x4 dk[NB];
      scales(0, dk);
#pragma unroll
      for (uint32_t mt = 0; mt < 2; ++mt) {
        const uint8_t* kr = sk + (8u * (n >> 2) + 4u * mt + (n & 3u)) * VST + 8u * g;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
          float4v t{};
          t = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8_f16(*reinterpret_cast<const u32x2*>(kr + 32u * b)), qb[b], t,
                                                     0, 0, 0);
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t at = (4u * mt + i) * NB + b;
            const half2v w = __builtin_bit_cast(half2v, word_of(dk, at));
            const float d = (float)(at & 1u ? w.y : w.x);
            s[4u * mt + i] = b == 0 ? d * t[i] : __builtin_fmaf(d, t[i], s[4u * mt + i]);
          }
        }
      }
    }
    float pm = -__builtin_inff();
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      s[j] += dpp_mov<0x128>(s[j]);   // row_ror:8: the other term's column
      s[j] *= f_row;
    }
    if (seq - t0 < 32u) {   // uniform: the last rows' tile
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        asm volatile("" : "+v"(s[j]));   // a branch, not selects in every tile
        s[j] = t0 + 8u * g + j < seq ? s[j] : -__builtin_inff();
      }
    }
    if (!BLOCKS && a.score && n < group) {   // n < group <= 8: first terms' lanes
      float* ps = a.score + (size_t)(kvh * group + n) * a.stride + t0 + 8u * g;
      *reinterpret_cast<float4v*>(ps) = float4v{s[0], s[1], s[2], s[3]};
      *reinterpret_cast<float4v*>(ps + 4) = float4v{s[4], s[5], s[6], s[7]};
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) pm = fmaxf(pm, s[j]);
    pm = xor32_pair(xor16_pair(pm, true), true);
    const bool move = pm - ref > w_up + kWeightLag;
    if (__builtin_amdgcn_ballot_w64(move) != 0) {
      const float to = move ? weight_ref(pm, w_up) : ref;
      float alpha = move ? __builtin_amdgcn_exp2f(ref - to) : 1.0f;
      asm volatile("" : "+v"(alpha));   // a branch: not products and copies in every tile
      ref = to;
      l_run *= alpha;
#pragma unroll
      for (uint32_t d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
    }
    const float off = ref == -__builtin_inff() ? 0.0f : ref;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      s[j] = __builtin_amdgcn_exp2f(s[j] - off);
      l_run += s[j];
    }
    // the weights as two f16 terms, then times a block's scales: the first
    // term of the product rounded, its error exact by an fma, plus the second
    // term's product
    half2v p0[4], p1[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      uint32_t hi, lo;
      split_f16(s[2 * k], s[2 * k + 1], hi, lo);
      p0[k] = __builtin_bit_cast(half2v, hi);
      p1[k] = __builtin_bit_cast(half2v, lo);
    }
    u32x4 dv[NB];
    scales(1, dv);
#pragma unroll
    for (uint32_t i = 0; i < NB; ++i)
#pragma unroll
      for (uint32_t w = 0; w < 4; ++w)
        dv[i][w] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (uint32_t)dv[i][w]) * d_up1);
    if (kv > 15) {   // uniform: every scale below 2^-8
#pragma unroll
      for (uint32_t i = 0; i < NB; ++i)
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
          uint32_t x = dv[i][w];
          asm volatile("" : "+v"(x));   // a branch, not selects
          dv[i][w] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, x) * d_up2);
        }
    }
    typedef __attribute__((address_space(3))) int2v lds_int2;
    const uint8_t* tr = sv + (8u * g + (n >> 1)) * VST + 8u * (n & 1u);
#pragma unroll
    for (uint32_t b = 0; b < NB; ++b) {
      // one operation on four pairs at a time: a packed result is not to be
      // read by the next instruction
      u32x4 w;
      half2v d[4], x[4], e[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t at = 2u * k * NB + b;   // rows 2 k and 2 k + 1
        d[k] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(word_of(dv, at + NB), word_of(dv, at),
                                                                NB == 1 ? 0x07060100u : b & 1u ? 0x07060302u : 0x05040100u));
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) x[k] = p0[k] * d[k];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) e[k] = __builtin_elementwise_fma(p0[k], d[k], -x[k]);
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) e[k] = __builtin_elementwise_fma(p1[k], d[k], e[k]);
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) w[k] = __builtin_bit_cast(uint32_t, second ? e[k] : x[k]);
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t dt = 2u * b + h;
        const u32x2 vb = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(tr + 16u * dt)));
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8_f16(vb), __builtin_bit_cast(half8v, w), o[dt], 0, 0, 0);
      }
    }
    wave_lds_order();   // read before the next tile's rows are written
    t0 = t1;
  }
  const float down = pow2f(-kv);

  // the two terms' columns, the wave's sums, then the four waves'
  l_run = xor32_pair(xor16_pair(l_run, false), false);
#pragma unroll
  for (uint32_t d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[d][i] = (o[d][i] + dpp_mov<0x128>(o[d][i])) * down;
  __syncthreads();   // every wave is done with its part of s_buf
  float* s_o = reinterpret_cast<float*>(s_buf);
  if (n < group) {
#pragma unroll
    for (uint32_t d = 0; d < ND; ++d)
      *reinterpret_cast<float4v*>(s_o + (wave * 8u + n) * HD + 16u * d + 4u * g) = o[d];
    if (g == 0) {
      s_ml[wave][n][0] = l_run != l_run ? 0.0f : ref;   // -inf only where nothing was seen
      s_ml[wave][n][1] = l_run;
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < group * HD; i += 256u) {
    const uint32_t h = i / HD, d = i % HD;
    float m = s_ml[0][h][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, s_ml[w][h][0]);
    float l = 0.0f, x = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const float rw = s_ml[w][h][0];
      const float e = rw == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(rw - m);
      l += s_ml[w][h][1] * e;
      x += s_o[(w * 8u + h) * HD + d] * e;
    }
    const size_t row = (size_t)z * a.n_head + kvh * group + h;
    if (a.n_chunk == 1) {
      float v = x / l;
      if (a.gate) v *= 1.0f / (1.0f + expf(-a.gate[row * HD + d]));
      a.out[row * HD + d] = v;
    } else {
      a.o[(row * a.n_chunk + ck) * HD + d] = x;
    }
    if (d == 0 && a.ml) {
      a.ml[2u * (row * a.n_chunk + ck)] = m;
      a.ml[2u * (row * a.n_chunk + ck) + 1u] = l;
    }
  }
}

// The end of a weighed token in one launch, workgroups of 16 waves.  The first
// n_head join a head's chunks (join_row).  The others, a kv head's 2048 rows
// each, add the weights:
//   weight[kv head][t] += sum over the group's heads of exp2(s - reference) / sum,
// taking the heads' references and sums from the chunks' partials themselves, a
// wave to a head.  60,001 rows, 32 / 8 heads: 7 us, a chain of
// loads (partials, then scores) and not their bytes.
struct FinishArgs {
  JoinCall j;
  const float* score;
  uint32_t stride, group, pos, plane, tok_pos, n_part;   // n_part: workgroups to a kv head
  float* weight;
  uint32_t* position;
};
template <int HD>
__global__ __launch_bounds__(1024) void attn_token_finish_kernel(FinishArgs a) {
  __shared__ JoinLds<HD, 16> s_join;
  __shared__ float s_ref[8], s_inv[8];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t n_join = a.j.n_seg > 1 ? a.j.n_rows : 0u;
  if (blockIdx.x < n_join) {
    join_row<HD, 16>(a.j, blockIdx.x, wave, lane, s_join);
    return;
  }
  const uint32_t kvh = (blockIdx.x - n_join) / a.n_part, t0 = (blockIdx.x - n_join) % a.n_part * 2048u;
  if (wave < a.group) {
    const float* p = a.j.ml + 2u * (size_t)(kvh * a.group + wave) * a.j.n_seg;
    float m = -__builtin_inff();
    for (uint32_t c = lane; c < a.j.n_seg; c += 64u) m = fmaxf(m, p[2u * c]);
    m = lane_reduce<64, true>(m);
    float l = 0.0f;
    for (uint32_t c = lane; c < a.j.n_seg; c += 64u)
      l += p[2u * c] == -__builtin_inff() ? 0.0f : p[2u * c + 1u] * __builtin_amdgcn_exp2f(p[2u * c] - m);
    l = lane_reduce<64>(l);
    if (lane == 0) {
      s_ref[wave] = m;
      s_inv[wave] = 1.0f / l;
    }
  }
  float s[8][2], old[2];
#pragma unroll
  for (uint32_t u = 0; u < 2; ++u) {
    const uint32_t t = min(t0 + u * 1024u + tid, a.pos);
#pragma unroll
    for (uint32_t h = 0; h < 8; ++h) s[h][u] = a.score[(size_t)(kvh * a.group + min(h, a.group - 1u)) * a.stride + t];
    old[u] = a.weight[(size_t)kvh * a.plane + t];
  }
  __syncthreads();
#pragma unroll
  for (uint32_t u = 0; u < 2; ++u) {
    const uint32_t t = t0 + u * 1024u + tid;
    if (t > a.pos) break;
    float v = 0.0f;
#pragma unroll
    for (uint32_t h = 0; h < 8; ++h)
      if (h < a.group) v = __builtin_fmaf(__builtin_amdgcn_exp2f(s[h][u] - s_ref[h]), s_inv[h], v);
    const size_t at = (size_t)kvh * a.plane + t;
    a.weight[at] = t < a.pos ? old[u] + v : v;
    if (t == a.pos) a.position[at] = a.tok_pos;
  }
}

// ---- block selection ----------------------------------------------------------

// Mean keys of whole blocks: workgroup (block, kv head), a thread per value of
// the head (rows split over the rest of the 256), sums in 64 bits.  Six blocks
// of 64 rows, 4 kv heads of 128: 4.7 us, one round of loads and the launch.
template <int HD>
__global__ __launch_bounds__(256) void kv_block_mean_kernel(KvQ8Dev c, int8_t* __restrict__ mean_qs,
                                                            uint16_t* __restrict__ mean_d, uint32_t block,
                                                            uint32_t blk0) {
  constexpr uint32_t P = 256 / HD;   // row parts
  __shared__ double s_sum[P][HD];
  const uint32_t d = threadIdx.x % HD, part = threadIdx.x / HD, kvh = blockIdx.y, blk = blk0 + blockIdx.x;
  const uint32_t per = c.n_kv * HD;
  const size_t row0 = (size_t)blk * block + part * (block / P);
  double sum = 0.0;
  const int8_t* q = c.k_qs + row0 * per + kvh * HD + d;
  const uint16_t* s = c.k_d + row0 * (per / 32u) + (kvh * HD + d) / 32u;
#pragma unroll 8
  for (uint32_t t = 0; t < block / P; ++t)
    sum += (double)((float)q[(size_t)t * per] * f16_to_f32(s[(size_t)t * (per / 32u)]));   // the product is exact in f32
  s_sum[part][d] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (uint32_t p = 0; p < P; ++p) sum += s_sum[p][d];
  uint32_t dh;
  const int v = q8_lane((float)(sum / (double)block), dh);   // every lane takes part
  if (part != 0) return;
  mean_qs[(size_t)blk * per + kvh * HD + d] = (int8_t)v;
  if ((d & 31u) == 0) mean_d[(size_t)blk * (per / 32u) + (kvh * HD + d) / 32u] = (uint16_t)dh;
}

struct SelectArgs {
  const float* q;
  const int8_t* mean_qs;
  const uint16_t* mean_d;
  uint32_t n_head, n_kv, pos, block, n_sel, n_first, n_local;
  uint32_t* sel;        // workspace [tokens][n_kv][n_sel]
  uint32_t* sel_user;   // null or [tokens][n_kv][stride], stride >= n_sel
  uint32_t stride;
};

// A pair's or a quad's other half of a 64-bit sum, by DPP.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint64_t y = (uint64_t)dpp_u32<CTRL>((uint32_t)(x >> 32)) << 32 | dpp_u32<CTRL>((uint32_t)x);
  return v + __builtin_bit_cast(double, y);
}

// Workgroup (kv head, token) of NT threads: the group's query as Q8_0 blocks,
// every block's score as a key in LDS (HD / 16 lanes to a block's mean, four
// means of a lane in flight, the first of them ahead of the query), the n_sel
// largest, written in ascending order.  One token over 1,876 blocks, 8 kv heads:
// 11.6 us, four counting passes over the keys between barriers; 400 tokens over
// 190 blocks: 11 us.
template <int HD, int NT>
__global__ __launch_bounds__(NT) void kv_select_kernel(SelectArgs a) {
  constexpr uint32_t LPB = HD / 16, NB = HD / 32, NW = NT / 64, U = 4;
  extern __shared__ uint32_t s_key[];
  __shared__ __attribute__((aligned(16))) uint32_t s_hist[4][256];
  __shared__ __attribute__((aligned(16))) int8_t s_q[HD];
  __shared__ float s_qd[NB];
  __shared__ uint32_t s_cnt[NW];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t kvh = blockIdx.x, z = blockIdx.y, group = a.n_head / a.n_kv;
  const uint32_t own = (a.pos + z) / a.block, nb = own + 1u;
  uint32_t* out = a.sel + ((size_t)z * a.n_kv + kvh) * a.n_sel;
  uint32_t* user = a.sel_user ? a.sel_user + ((size_t)z * a.n_kv + kvh) * a.stride : nullptr;
  if (nb <= a.n_sel) {   // every block
    for (uint32_t i = tid; i < a.n_sel; i += NT) out[i] = i < nb ? i : kNoBlock;
    if (user)
      for (uint32_t i = tid; i < a.stride; i += NT) user[i] = i < nb ? i : kNoBlock;
    return;
  }
  if (user)   // a call with fewer blocks than the caller's n_sel
    for (uint32_t i = a.n_sel + tid; i < a.stride; i += NT) user[i] = kNoBlock;

  const uint32_t sub = lane % LPB, per = a.n_kv * HD;
  constexpr uint32_t BW = NT / LPB;   // blocks at a time
  const int8_t* mq = a.mean_qs + kvh * HD + 16u * sub;
  const uint16_t* md = a.mean_d + kvh * NB + sub / 2u;
  // the last n_local blocks need no mean, and have none yet
  const uint32_t last = own >= a.n_local ? own - a.n_local : 0u;
  u32x4 k[U];
  uint32_t kd[U];
  auto load = [&](uint32_t b0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t b = min(b0 + u * BW + tid / LPB, last);
      k[u] = *reinterpret_cast<const u32x4*>(mq + (size_t)b * per);
      kd[u] = md[(size_t)b * (per / 32u)];
    }
  };
  load(0);
  for (uint32_t i = tid; i < 1024u; i += NT) s_hist[i / 256u][i % 256u] = 0u;
  if (tid < ((HD + 63u) & ~63u)) {   // whole waves
    const uint32_t d = min(tid, HD - 1u);
    const float* q = a.q + ((size_t)z * a.n_head + kvh * group) * HD + d;
    float x[8];
#pragma unroll
    for (uint32_t h = 0; h < 8; ++h) x[h] = q[(size_t)min(h, group - 1u) * HD];
    double sum = 0.0;
#pragma unroll
    for (uint32_t h = 0; h < 8; ++h) sum += h < group ? (double)x[h] : 0.0;
    uint32_t dh;
    const int v = q8_lane((float)sum, dh);
    if (tid < HD) {
      s_q[tid] = (int8_t)v;
      if ((tid & 31u) == 0) s_qd[tid / 32u] = f16_to_f32(dh);
    }
  }
  __syncthreads();
  int qw[4];
  __builtin_memcpy(qw, s_q + 16u * sub, 16);
  const float qd = s_qd[sub / 2u];
  for (uint32_t b0 = 0; b0 < nb; b0 += U * BW) {
    uint32_t key[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      int dot = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) dot = __builtin_amdgcn_sdot4((int)k[u][w], qw[w], dot, false);
      dot += (int)dpp_u32<0xB1>((uint32_t)dot);                     // the pair of a 32-value block
      double s = (double)(qd * f16_to_f32(kd[u])) * (double)dot;   // the scales' product is exact in f32
      if constexpr (LPB >= 4) s = dpp_add<0x4E>(s);
      if constexpr (LPB >= 8) s = dpp_add<0x141>(s);
      if constexpr (LPB >= 16) s = dpp_add<0x140>(s);
      key[u] = rank_key((float)s);
    }
    if (b0 + U * BW < nb) load(b0 + U * BW);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t b = b0 + u * BW + tid / LPB;
      if (sub == 0 && b < nb) s_key[b] = b < a.n_first || own - b < a.n_local ? kKeep : key[u];
    }
  }
  __syncthreads();
  const uint2 kth = kth_largest<NT>(nb, a.n_sel, [&](uint32_t i) { return s_key[i]; }, s_hist, tid);
  // in order: each wave a stretch of the blocks; the larger ones and the first
  // equal ones of the waves before it come first
  const uint32_t per_w = ((nb + NW - 1u) / NW + 63u) & ~63u, i0 = wave * per_w, i1 = min(nb, i0 + per_w);
  uint32_t eq = 0, gt = 0;
  for (uint32_t i = i0; i < i1; i += 64u) {
    const uint32_t v = i + lane < i1 ? s_key[i + lane] : 0u;
    gt += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(v > kth.x));
    eq += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(i + lane < i1 && v == kth.x));
  }
  if (lane == 0) s_cnt[wave] = gt | eq << 16;   // at most kSelectMax each
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (uint32_t w = 0; w < NW; ++w) before += w < wave ? s_cnt[w] : 0u;
  uint32_t eq_at = before >> 16, at = (before & 0xffffu) + min(eq_at, kth.y);
  for (uint32_t i = i0; i < i1; i += 64u) {
    const bool in = i + lane < i1;
    const uint32_t v = in ? s_key[i + lane] : 0u;
    const uint64_t me = __builtin_amdgcn_ballot_w64(in && v == kth.x);
    const bool take = in && (v > kth.x || (v == kth.x && eq_at + ones_below(me, lane) < kth.y));
    const uint64_t mt = __builtin_amdgcn_ballot_w64(take);
    const uint32_t place = at + ones_below(mt, lane);
    if (take && place < a.n_sel) {
      out[place] = i + lane;
      if (user) user[place] = i + lane;
    }
    eq_at += (uint32_t)__popcll(me);
    at += (uint32_t)__popcll(mt);
  }
}

struct TokenPlan {
  uint32_t tiles, n_chunk, stride;
  size_t ml, o, score, sel, total;
};

// Tiles to a wave: as many as leave the chip three waves per SIMD, a quarter
// of a token's at most (the workgroup has four).  60,000 rows, 32 heads of 128:
// 35.7 us at two waves per SIMD, 31.3 at three, 32.4 at four, whose chunks
// cost the join another 0.7.
TokenPlan token_plan(const KvQ8Dev& c, const TokenCall& r) {
  TokenPlan p{};
  const bool blocks = r.mean_qs != nullptr, weigh = r.weight != nullptr;
  const uint64_t n_vt = blocks ? (uint64_t)r.n_sel * (r.block / 32u) : ((uint64_t)r.pos + 32u) / 32u;
  const uint64_t all = n_vt * c.n_kv * r.n_tok;
  p.tiles = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((n_vt + 3u) / 4u, all / (3u * 1024u)));
  p.n_chunk = (uint32_t)((n_vt + 4ull * p.tiles - 1) / (4ull * p.tiles));
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off += (n + 255) & ~(size_t)255;
    return at;
  };
  const size_t rows = (size_t)r.n_tok * r.n_head * p.n_chunk;
  if (p.n_chunk > 1 || weigh) p.ml = take(rows * 8);
  if (p.n_chunk > 1) p.o = take(rows * c.hd * 4);
  p.stride = (r.pos + 32u) / 32u * 32u;
  if (weigh) p.score = take((size_t)r.n_head * p.stride * 4);
  if (blocks) p.sel = take((size_t)r.n_tok * c.n_kv * r.n_sel * 4);
  p.total = off;
  return p;
}

template <int HD>
hipError_t launch_token_hd(const KvQ8Dev& c, const TokenCall& r, void* ws, hipStream_t s) {
  const TokenPlan p = token_plan(c, r);
  const bool blocks = r.mean_qs != nullptr, weigh = r.weight != nullptr;
  char* base = static_cast<char*>(ws);
  TokenArgs a{};
  a.q = r.q;
  a.gate = r.gate;
  a.out = r.out;
  a.n_head = r.n_head;
  a.group = r.n_head / c.n_kv;
  a.seq = r.pos + 1u;
  a.tiles = p.tiles;
  a.n_chunk = p.n_chunk;
  if (p.n_chunk > 1 || weigh) a.ml = reinterpret_cast<float*>(base + p.ml);
  if (p.n_chunk > 1) a.o = reinterpret_cast<float*>(base + p.o);
  a.n_unit = r.n_tok * p.n_chunk;
  const dim3 grid((a.n_unit + 7u) / 8u * 8u * c.n_kv);
  hipError_t e;
  if (blocks) {
    uint32_t* sel = reinterpret_cast<uint32_t*>(base + p.sel);
    const SelectArgs sa{r.q, r.mean_qs, r.mean_d, r.n_head, c.n_kv, r.pos, r.block, r.n_sel, r.n_first, r.n_local,
                        sel, r.sel, r.sel_stride};
    const uint32_t nb = (r.pos + r.n_tok - 1u) / r.block + 1u;
    // 256 threads against 1024, whole calls, 8 kv heads: one token over 256
    // blocks 15.2 and 15.4 us, 512 17.1 and 15.9, 1876 27.8 and 20.7; 64 tokens
    // over 512 26.5 and 27.4, 1024 30.6 and 30.5, 1876 37.8 and 35.6.
    if (nb <= (r.n_tok < 16u ? 256u : 1024u))
      hipLaunchKernelGGL((kv_select_kernel<HD, 256>), dim3(c.n_kv, r.n_tok), dim3(256), nb * 4u, s, sa);
    else
      hipLaunchKernelGGL((kv_select_kernel<HD, 1024>), dim3(c.n_kv, r.n_tok), dim3(1024), nb * 4u, s, sa);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.sel = sel;
    a.block = r.block;
    a.n_sel = r.n_sel;
    hipLaunchKernelGGL((attn_token_kernel<HD, true>), grid, dim3(256), 0, s, c, a);
  } else {
    a.score = reinterpret_cast<float*>(base + p.score);
    a.stride = p.stride;
    hipLaunchKernelGGL((attn_token_kernel<HD, false>), grid, dim3(256), 0, s, c, a);
  }
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const JoinCall j{a.ml, a.o, r.gate, r.out, r.n_tok * r.n_head, r.n_head, p.n_chunk, 0, 0, 0, nullptr, 0, 0, 0, 0, 0};
  if (weigh) {
    const uint32_t n_part = r.pos / 2048u + 1u;
    const FinishArgs f{j, a.score, p.stride, a.group, r.pos, r.plane, r.tok_pos, n_part, r.weight, r.position};
    hipLaunchKernelGGL(attn_token_finish_kernel<HD>, dim3((p.n_chunk > 1 ? r.n_head : 0u) + n_part * c.n_kv), dim3(1024),
                       0, s, f);
    return hipGetLastError();
  }
  if (p.n_chunk > 1) e = launch_attn_join(HD, j, s);
  return e;
}

}  // namespace

size_t attn_token_workspace(const KvQ8Dev& c, const TokenCall& r) { return token_plan(c, r).total; }

// Requires hd in {32, 64, 128, 256}, n_head % n_kv == 0, n_head / n_kv <= 8,
// pos + n_tok <= max_seq; weigh: one token; blocks: block 32, 64 or 128,
// n_first + n_local <= n_sel, n_local >= 1, at most kSelectMax blocks, means of
// every whole block below the tokens.  ws holds attn_token_workspace bytes.
hipError_t launch_attn_token(const KvQ8Dev& c, const TokenCall& r, void* ws, hipStream_t s) {
  const uint32_t group = r.n_head / c.n_kv;
  if (group == 0 || group > 8u || r.n_tok == 0 || (r.weight && r.n_tok != 1)) return hipErrorInvalidValue;
  switch (c.hd) {
    case 32: return launch_token_hd<32>(c, r, ws, s);
    case 64: return launch_token_hd<64>(c, r, ws, s);
    case 128: return launch_token_hd<128>(c, r, ws, s);
    case 256: return launch_token_hd<256>(c, r, ws, s);
    default: return hipErrorInvalidValue;
  }
}

// Means of blocks blk0 .. blk0 + n - 1.
hipError_t launch_block_means(const KvQ8Dev& c, int8_t* mean_qs, uint16_t* mean_d, uint32_t block, uint32_t blk0,
                              uint32_t n, hipStream_t s) {
  const dim3 grid(n, c.n_kv);
  switch (c.hd) {
    case 32: hipLaunchKernelGGL(kv_block_mean_kernel<32>, grid, dim3(256), 0, s, c, mean_qs, mean_d, block, blk0); break;
    case 64: hipLaunchKernelGGL(kv_block_mean_kernel<64>, grid, dim3(256), 0, s, c, mean_qs, mean_d, block, blk0); break;
    case 128: hipLaunchKernelGGL(kv_block_mean_kernel<128>, grid, dim3(256), 0, s, c, mean_qs, mean_d, block, blk0); break;
    case 256: hipLaunchKernelGGL(kv_block_mean_kernel<256>, grid, dim3(256), 0, s, c, mean_qs, mean_d, block, blk0); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace vxt
