// kv_ops.hpp -- what the operators over the Q8_0 KV cache share: the call
// descriptors and the device pieces (int8 codes as MFMA operands, two-term
// f16 splits, the k largest keys of a list).
//
// Numbers.  A cache value is code * scale: an int8 is exact in f16, so the
// products with it need the other operand only.  That operand (a query, a
// softmax weight, a dequantised value) goes in as two f16 terms, hi + lo, 22
// bits, after a power of two has moved its largest magnitude near the top of
// f16's range; what lies 2^17 or more below the largest loses bits, never
// more than 2^-39 of the largest.  Sums run in f32.  The results are within a
// few 1e-7 of the same formulas in 64 bits.
#pragma once

#include "common.hpp"

namespace vxt {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
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
  float* lse;          // null, or where reference + log2(sum) goes, by row tile (attn_rows.hip)
  uint32_t group, tq, rg, n_rt;
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

// Two f32 as f16 pairs hi and lo with hi + lo the value to 22 bits
// (truncating conversions: the first term's error is the second's business).
// The remainders a - hi as one v_fma_mix_f32 each, which the compiler makes a
// conversion and a subtraction of.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
  float ra, rb;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(ra, rb));
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

template <int N>
__device__ __forceinline__ uint32_t lane_max_u32(uint32_t v) {
#pragma unroll
  for (int s = 1; s < N; s <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, s, 64));
  return v;
}

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

struct KthLds {
  uint32_t hist[256];
  uint32_t out[2];
};

// The k-th largest of key(0 .. n - 1), 1 <= k <= n: its value and how many of
// the keys equal to it are among the k largest.  Four passes of eight bits,
// the counts in LDS; every one of the NT threads calls it and gets both.
template <int NT, typename Key>
__device__ __forceinline__ uint2 kth_largest(uint32_t n, uint32_t k, Key key, KthLds& s, uint32_t tid) {
  uint32_t prefix = 0, need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (uint32_t i = tid; i < 256u; i += NT) s.hist[i] = 0u;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += NT) {
      const uint32_t v = key(i);
      if (shift == 24 || (v >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s.hist[(v >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid < 64u) {
      // lane l counts bins 4 l .. 4 l + 3; `above` is what lies in higher bins
      uint32_t c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j] = s.hist[4u * tid + j];
        sum += c[j];
      }
      uint32_t above = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_down((int)above, d, 64);
        if (tid + d < 64u) above += o;
      }
      above -= sum;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        if (above < need && need <= above + c[j]) {
          s.out[0] = prefix | ((4u * tid + j) << shift);
          s.out[1] = need - above;
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix = s.out[0];
    need = s.out[1];
    __syncthreads();
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

}  // namespace vxt
