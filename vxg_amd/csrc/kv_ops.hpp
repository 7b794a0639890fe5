// kv_ops.hpp -- what the operators over the Q8_0 KV cache share: the call
// descriptors and the device pieces (int8 codes as MFMA operands, two-term
// f16 splits, the k largest keys of a list).
//
// Numbers.  A cache value is code * scale: an int8 is exact in f16, so the
// products with it need the other operand only.  That operand (a query, a
// softmax weight, a dequantised value) goes in as two f16 terms, hi + lo, 22
// bits, after a power of two has moved the largest magnitude near the top of
// f16's range; what lies 2^15 or more below the largest loses bits, and is right
// to 2^-38 of it (2^-36 for a weight times a scale, the operand of
// attn_token.hip).  A V scale that lies 2^21 below a largest one of 128 or more
// is right to 2^-31 of that in attn_rows.hip; every other scale is exact.  Sums
// run in f32.  The results are within a few 1e-7 of the same formulas in 64
// bits, relative to an output's norm.
#pragma once

#include "common.hpp"

namespace vxt {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16x __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef int int2v __attribute__((ext_vector_type(2)));

constexpr uint32_t kTreeMax = 256;        // nodes of a drafted tree
constexpr uint32_t kTreeWords = kTreeMax / 32;
constexpr uint32_t kNoBlock = 0xffffffffu;
constexpr uint32_t kSelectMax = 14336;    // blocks to select from: their keys lie in 56 KB of LDS

// A call of the many-row attention kernel (attn_rows.hip).  Row r of a
// workgroup's block is token tb + r / group, query head kvh * group + r % group.
struct RowsCall {
  const float* q;            // [n_tok][n_head * hd], prepared
  const float* gate;         // null or like q
  float* out;                // like q
  const int32_t* parents;    // tree: [n_tok], device
  uint32_t n_tok, pos, n_head;
  // weigh only: null otherwise
  float* weight;             // [n_kv][plane]
  uint32_t* position;        // [n_kv][plane]
  uint32_t plane, tok_pos;
};

// A call of the one-token attention kernel (attn_token.hip).
struct TokenCall {
  const float* q;            // [n_tok][n_head * hd]
  const float* gate;
  float* out;
  uint32_t n_tok, pos, n_head;
  float* weight;             // weigh only
  uint32_t* position;
  uint32_t plane, tok_pos;
  // blocks only
  const int8_t* mean_qs;
  const uint16_t* mean_d;
  uint32_t block, n_sel, n_first, n_local;
  uint32_t* sel;             // null or [n_tok][n_kv][sel_stride]
  uint32_t sel_stride;       // >= n_sel
};

// The join of a row's partial sums (attn_rows.hip).  n_seg partials a row,
// causal: those up to its token's position, seg_len rows each.
struct JoinCall {
  const float* ml;     // [n_rows][n_seg][2]: reference (base 2; -inf: nothing seen), sum
  const float* o;      // [n_rows][n_seg][hd]
  const float* gate;   // null or [n_rows][hd]
  float* out;          // [n_rows][hd]
  uint32_t n_rows, n_head, n_seg, seg_len, pos, causal;
  float2* stat;        // null, or where a row's reference and 1 / sum go, by row tile (attn_rows.hip)
  uint32_t group, tq, rg, n_rt, n_tok;
};
hipError_t launch_attn_join(uint32_t hd, const JoinCall& j, hipStream_t s);

// ---- conversions ------------------------------------------------------------

// Four int8 codes as two words of f16 pairs, exact: with the sign bit turned
// a code is code + 128 in 0 .. 255, the low byte of the f16 whose high byte is
// 0x64 (1024 + that), and 1152 comes off again.
__device__ __forceinline__ void codes_f16(uint32_t w, half2v& a, half2v& b) {
  const uint32_t u = w ^ 0x80808080u;
  const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
  a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
  b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
}

__device__ __forceinline__ half8v codes8_f16(u32x2 w) {
  half2v a, b, c, d;
  codes_f16(w.x, a, b);
  codes_f16(w.y, c, d);
  return half8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Softmax weights are operands 2^kWeightUp times as large as they are to the
// row's maximum when the reference, 2^-kWeightUp of that, last moved; it moves
// when the maximum has passed that by 2^kWeightLag: at most 2^15.  f16 ends at
// 2^-24, so a weight is right to 2^-38 of the largest, half a step, and has its 22
// bits from 2^-15 of it on.  A lag of 2^8, with weights 2^7 times as large, would
// be right to 2^-32, for 2 % of the time or so: 250 nodes over 30,011 rows 341 us
// with it and 346 without, a prompt of 1,500 42.1 and 42.9, 400 tokens over 16
// blocks of 64 rows 77.2 and 77.1.
constexpr float kWeightUp = 13.0f, kWeightLag = 2.0f;

// The reference of a row (base 2) whose maximum is now `top`: `up` below it, or
// the maximum itself where that much is lost in its rounding (from 2^26 on); no
// score up to `top` is more than `up` + kWeightLag above it.
__device__ __forceinline__ float weight_ref(float top, float up) {
  const float r = top - up;
  return top - r <= up + kWeightLag ? r : top;
}

// Two f32 as f16 pairs hi and lo with hi + lo the value to 22 bits, each
// rounded to nearest: truncated, all of a sum's terms would err downward.  The
// remainders a - hi are fma(hi, -1, a) with a -1 that the compiler does not
// know: one v_fma_mix_f32 each, not a conversion and a subtraction.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  float minus = -1.0f;
  asm("" : "+s"(minus));
  const half2v h = __builtin_convertvector((float2v{a, b}), half2v);
  const float2v r = {__builtin_fmaf((float)h.x, minus, a), __builtin_fmaf((float)h.y, minus, b)};
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, half2v));
}

// 2^e as an f32, -126 <= e <= 127.
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent that brings a magnitude `amax` to [2^14, 2^15) (as near as
// +-120 goes); 0 for a zero, infinite or NaN one.
__device__ __forceinline__ int top_shift(float amax) {
  const uint32_t b = __float_as_uint(amax) & 0x7fffffffu;
  if (b == 0 || b >= 0x7f800000u) return 0;
  const int e = 14 - ((int)(b >> 23) - 127);
  return e > 120 ? 120 : e < -120 ? -120 : e;
}

// The exponent that brings the largest of a set of f16 scales (bits) to
// [64, 128); 0 when there is none.
__device__ __forceinline__ int scale_shift(uint32_t top_bits) {
  if (top_bits == 0) return 0;
  const float f = f16_to_f32(top_bits);
  return 6 - ((int)(__float_as_uint(f) >> 23) - 127);
}

// A scale's magnitude bits for a maximum: the non-finite ones count as none.
__device__ __forceinline__ uint32_t finite_scale(uint32_t d) {
  const uint32_t m = d & 0x7fffu;
  return m < 0x7c00u ? m : 0u;
}

// Orders a wave's LDS operations among its own lanes: the hardware runs them
// in order, so this only waits for them and keeps the compiler from moving
// one past another.
__device__ __forceinline__ void wave_lds_order() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// N consecutive f16 as raw bits, from a 2-byte aligned address.
template <int N>
struct __attribute__((aligned(N == 1 ? 2 : 2 * N))) Scales {
  uint16_t d[N];
};
template <int N>
__device__ __forceinline__ Scales<N> load_scales(const uint16_t* p) {
  Scales<N> s;
  __builtin_memcpy(&s, p, 2 * N);
  return s;
}
// The largest finite one's magnitude bits.
template <int N>
__device__ __forceinline__ uint32_t top_scale(const Scales<N>& s) {
  uint32_t top = 0;
#pragma unroll
  for (int b = 0; b < N; ++b) top = max(top, finite_scale(s.d[b]));
  return top;
}

// ---- wave64 sums and scans of unsigned words, by DPP ---------------------------

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {   // 0 where no lane is read
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}

// Maximum over aligned groups of N lanes (16 <= N <= 64), in every lane.
template <int N>
__device__ __forceinline__ uint32_t lane_max_u32(uint32_t v) {
  v = max(v, dpp_u32<0xB1>(v));    // quad_perm [1,0,3,2]
  v = max(v, dpp_u32<0x4E>(v));    // quad_perm [2,3,0,1]
  v = max(v, dpp_u32<0x141>(v));   // row_half_mirror
  v = max(v, dpp_u32<0x140>(v));   // row_mirror
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  if constexpr (N >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  return v;
}

// Sum over lanes 0 .. this one; lane 63 holds the wave's.
__device__ __forceinline__ uint32_t lane_scan_u32(uint32_t v) {
  v += dpp_u32<0x111>(v);          // row_shr:1, 2, 4, 8
  v += dpp_u32<0x112>(v);
  v += dpp_u32<0x114>(v);
  v += dpp_u32<0x118>(v);
  v += dpp_u32<0x142, 0xa>(v);     // row_bcast:15 into rows 1 and 3
  v += dpp_u32<0x143, 0xc>(v);     // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ uint32_t lane63(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }

// ---- Q8_0 blocks --------------------------------------------------------------

// f32 -> f16 bits, round to nearest even with f16 subnormals kept and
// overflow to infinity: what fp16.rs:33-77 computes with integer steps, here
// v_cvt_f16_f32 (default round-to-nearest-even mode, f16 denormals on).
// Inputs are never NaN (the callers pass a maximum of magnitudes that skips
// NaN).
__device__ __forceinline__ uint32_t f32_to_f16_bits(float val) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)val);
}

// KvQ8Block::quantize of one value per lane, each aligned 32-lane group
// holding one block (every lane of the wave must call it): amax of |x| with
// NaN ignored, dh = f16 bits of amax / 127, q = round_ties_even(x / f32(dh))
// clamped to +-127, NaN -> 0.
__device__ __forceinline__ int q8_lane(float x, uint32_t& dh) {
#pragma clang fp contract(off)
  const float a = fabsf(x);
  float amax = a == a ? a : 0.0f;
  amax = lane_reduce<32, true>(amax);
  dh = f32_to_f16_bits(amax / 127.0f);
  const float df = f16_to_f32_exact(dh);
  const float inv = df > 0.0f ? 1.0f / df : 0.0f;
  const float r = rintf(x * inv);
  return r != r ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

// ---- the k largest of a list --------------------------------------------------

// f32 as an unsigned key of the same order: NaN lowest, -0 as +0.  No value's
// key is kKeep.
constexpr uint32_t kKeep = 0xffffffffu;
__device__ __forceinline__ uint32_t rank_key(float f) {
  uint32_t b = __float_as_uint(f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;
  if (b == 0x80000000u) b = 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The bin in which the need-th largest falls: `c` are this lane's counts of
// bins lane * B .. lane * B + B - 1.  Returns that bin, what is needed of it and
// what it holds, uniform in the wave.
template <int B>
__device__ __forceinline__ void find_bin(const uint32_t (&c)[B], uint32_t need, uint32_t& bin, uint32_t& of, uint32_t& in) {
  uint32_t sum = 0;
#pragma unroll
  for (int j = 0; j < B; ++j) sum += c[j];
  const uint32_t upto = lane_scan_u32(sum);
  uint32_t above = lane63(upto) - upto;   // in higher lanes' bins
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t b = 0, o = 0, n = 0;
  bool here = false;
#pragma unroll
  for (int j = B - 1; j >= 0; --j) {
    if (above < need && need <= above + c[j]) {
      here = true;
      b = lane * B + j;
      o = need - above;
      n = c[j];
    }
    above += c[j];
  }
  const uint64_t m = __builtin_amdgcn_ballot_w64(here);
  const int l = __builtin_ctzll(m ? m : 1ull);
  bin = (uint32_t)__builtin_amdgcn_readlane((int)b, l);
  of = (uint32_t)__builtin_amdgcn_readlane((int)o, l);
  in = (uint32_t)__builtin_amdgcn_readlane((int)n, l);
}

// The k-th largest of key(0 .. n - 1), 1 <= k <= n: its value and how many of
// the keys equal to it are among the k largest.  Four passes of eight bits,
// counted in LDS (four tables, cleared by the caller before a barrier); every
// wave finds the bin for itself, so a pass has one barrier.
template <int NT, typename Key>
__device__ __forceinline__ uint2 kth_largest(uint32_t n, uint32_t k, Key key, uint32_t (&hist)[4][256], uint32_t tid) {
  uint32_t prefix = 0, need = k;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    for (uint32_t i = tid; i < n; i += NT) {
      const uint32_t v = key(i);
      if (pass == 0 || (v >> (shift + 8)) == prefix) atomicAdd(&hist[pass][(v >> shift) & 255u], 1u);
    }
    __syncthreads();
    const u32x4 h = *reinterpret_cast<const u32x4*>(&hist[pass][4u * (tid & 63u)]);
    const uint32_t c[4] = {h.x, h.y, h.z, h.w};
    uint32_t bin, in;
    find_bin<4>(c, need, bin, need, in);
    prefix = prefix << 8 | bin;
  }
  return make_uint2(prefix, need);
}

// Exclusive prefix of per-wave counts: s has one word per wave.
template <int NW>
__device__ __forceinline__ uint32_t wave_prefix(uint32_t mine, uint32_t* s, uint32_t wave, uint32_t lane) {
  if (lane == 0) s[wave] = mine;
  __syncthreads();
  uint32_t sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < NW; ++w) sum += w < wave ? s[w] : 0u;
  __syncthreads();
  return sum;
}

__device__ __forceinline__ uint32_t ones_below(uint64_t mask, uint32_t lane) {
  return (uint32_t)__popcll(mask & ((1ull << lane) - 1ull));
}

// ---- the join of a row's partial sums ------------------------------------------

template <int HD, int W>
struct alignas(16) JoinLds {
  float acc[W][W > 1 ? HD : 4];
  float l[W];
};

// Reference M = the largest, factors exp2(ref - M), out = sum O / sum l, times
// the sigmoid gate.  HD / 4 lanes to a row's dims, 16 bytes each.  W == 1: a row
// to each such group of lanes.  Else W waves to a row: group g of them adds
// partials g, g + groups, ..., then the wave's groups' sums are added, then the
// waves'.  The gate and the first partials are on their way before M is known.
template <int HD, int W>
__device__ __forceinline__ void join_row(const JoinCall& a, uint32_t row, uint32_t wave, uint32_t lane, JoinLds<HD, W>& s) {
#pragma clang fp contract(off)
  typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
  constexpr uint32_t L = HD / 4, G = W == 1 ? 1u : 64u / L, STEP = W * G;
  const uint32_t d0 = 4u * (lane % L), first = W == 1 ? 0u : wave * G + lane / L;
  const uint32_t tk = row / a.n_head, head = row % a.n_head;
  uint32_t ns = a.n_seg;
  if (a.causal) {
    // a block of tokens whose rows fit one segment has its output already
    if ((a.pos + min(a.n_tok, (tk / a.tq + 1u) * a.tq) - 1u) / a.seg_len == 0) return;
    ns = min(ns, (a.pos + tk) / a.seg_len + 1u);
  }
  const float* ml = a.ml + 2u * (size_t)row * a.n_seg;
  const float* po = a.o + (size_t)row * a.n_seg * HD + d0;
  constexpr uint32_t U = W == 16 ? 4 : 8;   // partials in flight
  float2 r[U];
  float4v x[U];
  auto load = [&](uint32_t s0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t i = min(s0 + u * STEP, ns - 1u);
      r[u] = *reinterpret_cast<const float2*>(ml + 2u * i);
      x[u] = *reinterpret_cast<const float4v*>(po + (size_t)i * HD);
    }
  };
  load(first);
  float4u gv{};
  if (a.gate) gv = *reinterpret_cast<const float4u*>(a.gate + (size_t)row * HD + d0);
  float m = -__builtin_inff();
  for (uint32_t i = W == 1 ? lane % L : lane; i < ns; i += W == 1 ? L : 64u) m = fmaxf(m, ml[2u * i]);
  m = lane_reduce<W == 1 ? L : 64, true>(m);
  float l = 0.0f;
  float4v acc{};
  for (uint32_t s0 = first; s0 < ns; s0 += U * STEP) {
    if (s0 != first) load(s0);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (s0 + u * STEP >= ns || r[u].x == -__builtin_inff()) continue;   // nothing, or nothing the row sees
      const float e = __builtin_amdgcn_exp2f(r[u].x - m);
      l += r[u].y * e;
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += x[u][j] * e;
    }
  }
  if constexpr (W > 1) {
    auto groups = [](float v) {   // sum over the wave's groups
      if constexpr (L <= 8) v += dpp_mov<0x128>(v);   // row_ror:8
      if constexpr (L <= 16) v = xor16_pair(v, false);
      if constexpr (L <= 32) v = xor32_pair(v, false);
      return v;
    };
    l = groups(l);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = groups(acc[j]);
    if (lane < L) *reinterpret_cast<float4v*>(&s.acc[wave][d0]) = acc;
    if (lane == 0) s.l[wave] = l;
    __syncthreads();
    if (wave != 0 || lane >= L) return;
#pragma unroll
    for (uint32_t k = 1; k < W; ++k) {
      l += s.l[k];
      const float4v y = *reinterpret_cast<const float4v*>(&s.acc[k][d0]);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += y[j];
    }
  }
  float4u v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = acc[j] / l;
    if (a.gate) v[j] *= 1.0f / (1.0f + expf(-gv[j]));
  }
  *reinterpret_cast<float4u*>(a.out + (size_t)row * HD + d0) = v;
  if (a.stat && d0 == 0) {
    const uint32_t kvh = head / a.group, i = (tk % a.tq) * a.group + head % a.group;
    const uint32_t rt = (tk / a.tq) * a.rg + i / 32u;
    a.stat[((size_t)kvh * a.n_rt + rt) * 32u + (i & 31u)] = make_float2(l != l ? 0.0f : m, 1.0f / l);
  }
}

}  // namespace vxt
