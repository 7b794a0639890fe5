// kv_pages.hip -- rows of a paged Q8_0 KV cache written and read back.
//
// Write (paged_prep_kernel).  Per token and head, in 64 bits:
//   x = input + bias;  x *= w / sqrt(sum x^2 / hd + eps);
//   pair i turned by  pos[axis(i)] * base^(-2 i / rope_dim);
// rounded once to f32 (the query's result), and for K and V quantised from there
// as KvQ8Block::quantize does (llm_prefill.rs:27-42) into the token's row.  With
// f32 steps the codes of a value next to a border would hang on the order of a
// sum, and the angle of position 100,000 would be off by 4e-3; a 64-bit multiply
// and add takes a wave as long as a 32-bit one here.  1,900 tokens of 16 + 4 heads of
// 128, gated, bf16: 21 us, 55 MB; some 170 vector operations a head (11 us of issue
// over the chip) and, before the first, 6 us for the chain token range - row - page
// and the angles.  A token: 4.2 us.
//
// Read (paged_read_kernel).  value = code * scale, of the same rows.  Bound by memory:
// 60,000 rows of 8 heads of 128 as f32, 622 MB: 117 us (5.3 TB/s) with other pages each
// time, 94 with the same ones, which the last-level cache holds in part.
#include "kv_pages.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace vxt {

namespace {

constexpr uint32_t kPrepWaves = 8, kPrepTokens = 8;

// N consecutive values, bf16 or f32, from an address aligned to one of them.
template <bool BF16, int N>
__device__ __forceinline__ void load_x(const void* p, size_t i, float (&x)[N]) {
  if constexpr (BF16) {
    uint16_t w[N];
    __builtin_memcpy(w, static_cast<const uint16_t*>(p) + i, 2 * N);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = bf16_to_f32(w[j]);
  } else {
    __builtin_memcpy(x, static_cast<const float*>(p) + i, 4 * N);
  }
}

// The value of the lane that `xor`s 32, 16 or 1, as two 32-bit exchanges.
template <int XOR>
__device__ __forceinline__ double lane_xor(double v, uint32_t lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  auto other = [&](uint32_t w) {
    if constexpr (XOR == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xf, 0xf, false);   // quad_perm [1,0,3,2]
    const auto r = XOR == 32 ? __builtin_amdgcn_permlane32_swap(w, w, false, false) : __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return (lane & XOR) ? (uint32_t)r[0] : (uint32_t)r[1];
  };
  return __builtin_bit_cast(double, (uint64_t)other((uint32_t)(b >> 32)) << 32 | other((uint32_t)b));
}

// Sum over the wave, in every lane.
__device__ __forceinline__ double wave_sum64(double v, uint32_t lane) {
  v += lane_xor<1>(v, lane);
  auto step = [&](auto ctrl) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, decltype(ctrl)::value, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), decltype(ctrl)::value, 0xf, 0xf, false);
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  step(std::integral_constant<int, 0x4E>{});    // quad_perm [2,3,0,1]
  step(std::integral_constant<int, 0x141>{});   // row_half_mirror
  step(std::integral_constant<int, 0x140>{});   // row_mirror
  v += lane_xor<16>(v, lane);
  return v + lane_xor<32>(v, lane);
}

// 1 / sqrt(a), a > 0 and finite, to an ulp or two: the hardware's, squared twice
// as exact by two steps.  0 and what is not finite as the library has them, where
// some lane of the wave needs that.
__device__ __forceinline__ double rsqrt64(double a) {
  double y = __builtin_amdgcn_rsq(a);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double e = __builtin_fma(-a * y, y, 1.0);
    y = __builtin_fma(y * 0.5, e, y);
  }
  if (__builtin_amdgcn_ballot_w64(!(a > 0x1p-900 && a < 0x1p900)) != 0) {
    asm volatile("" : "+v"(a));   // a branch, not both and a choice
    y = a > 0x1p-900 && a < 0x1p900 ? y : 1.0 / sqrt(a);
  }
  return y;
}

// KvQ8Block::quantize of a wave's 64 * E values, E to a lane: a block is 32 / E
// lanes.  (The steps of q8_lane.)
template <int E>
__device__ __forceinline__ void q8_values(const float (&x)[E], int (&q)[E], uint32_t& dh) {
#pragma clang fp contract(off)
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) amax = fmaxf(amax, fabsf(x[j]));   // NaN is passed over
  amax = lane_reduce<32 / E, true>(amax);
  dh = f32_to_f16_bits(amax / 127.0f);
  const float df = f16_to_f32_exact(dh);
  const float inv = df > 0.0f ? 1.0f / df : 0.0f;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const float r = rintf(x[j] * inv);
    q[j] = r != r ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
  }
}

// A workgroup to `T` tokens (or gridDim.y of them, which share the heads), a wave to
// one head of one token at a time (query heads, then kv heads), the next one's
// values on their way; lane l holds values E l .. E l + E - 1.  The tokens' angles are evaluated first, by all threads.
template <int HD, bool BF16>
__global__ __launch_bounds__(kPrepWaves * 64) void paged_prep_kernel(PagesDev c, PagedDev b, PagedPrep a, PagedRope rope, uint32_t T) {
#pragma clang fp contract(off)
  constexpr int E = HD >= 64 ? HD / 64 : 1;
  __shared__ double s_cs[kPrepTokens][HD];       // cos, sin of pair i at 2 i, 2 i + 1
  __shared__ double s_x[kPrepWaves][HD];         // a head, where pairs lie across lanes unevenly
  __shared__ int32_t s_row[kPrepTokens];
  __shared__ uint32_t s_page[kPrepTokens];       // kNoSeq: none; s_row of a token of nobody: INT_MIN
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t t0 = blockIdx.x * T, n_t = min(T, b.n_tok - t0), n_waves = blockDim.x >> 6;
  const uint32_t n_q = a.q_raw ? a.n_head : 0u, units = n_q + c.n_kv;
  const uint32_t d0 = min(lane * E, (uint32_t)HD - E);   // HD 32: lanes 32 on repeat
  const bool live = HD >= 64 || lane < HD;

  struct Vals {
    float x[E], y[E];   // a query head and its gate, or a kv head's K and V
  };
  // a wave's heads, token by token: (j, h), every n_waves-th
  auto step = [&](uint32_t& j, uint32_t& h) {
    h += n_waves * gridDim.y;
    while (h >= units) {
      h -= units;
      ++j;
    }
  };
  // Behind the last token the last one's first head.  Rows of nobody are loaded too, as
  // are positions: whose a token is takes two loads in a chain to find.
  auto load = [&](uint32_t j, uint32_t h, Vals& w) {
    if (j >= n_t) {
      j = n_t - 1u;
      h = 0;
    }
    const uint32_t t = t0 + j;
    const bool is_q = h < n_q;
    const uint32_t off = is_q ? h * (a.gated ? 2u : 1u) * HD : (h - n_q) * HD;
    const size_t at = (size_t)t * (is_q ? a.q_stride : a.kv_stride) + off + d0;
    load_x<BF16>(is_q ? a.q_raw : a.k_cur, at, w.x);
    load_x<BF16>(is_q ? a.q_raw : a.v_cur, at + (is_q && a.gated ? HD : 0), w.y);
  };
  Vals cur, nxt;
  uint32_t j = 0, h = blockIdx.y * n_waves + wave, j1, h1;
  while (h >= units) {
    h -= units;
    ++j;
  }
  load(j, h, cur);
  float wq[E], wk[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    wq[e] = a.q_norm ? a.q_norm[d0 + e] : 1.0f;
    wk[e] = a.k_norm ? a.k_norm[d0 + e] : 1.0f;
  }

  auto angles = [&]() {
    for (uint32_t i = tid; i < n_t * a.half; i += blockDim.x) {
      const uint32_t k = i / a.half, p = i % a.half;
      const int32_t at = a.rope_pos ? a.rope_pos[(size_t)rope.axis[p] * b.n_tok + t0 + k] : s_row[k];
      double sn, cs;
      sincos((double)at * rope.f[p], &sn, &cs);
      s_cs[k][2u * p] = cs;
      s_cs[k][2u * p + 1u] = sn;
    }
  };
  const bool given = a.rope_pos != nullptr;   // positions that need no row
  if (given) angles();
  for (uint32_t i = n_waves - 1u - wave; i < n_t; i += n_waves) {   // by the waves that have the fewest angles
    const uint32_t t = t0 + i, seq = find_seq(b.tok_start, b.n_seq, t);
    int32_t row = INT32_MIN;
    uint32_t page = kNoSeq;
    if (seq != kNoSeq) {
      const SeqRange r = seq_range(b, seq);
      row = row_of_token(r, t);
      if (row < 0 || !page_of(b, seq, row, page)) page = kNoSeq;
    }
    if (lane == 0) {
      s_row[i] = row;
      s_page[i] = page;
    }
  }
  __syncthreads();
  if (!given) {
    angles();
    __syncthreads();
  }
  // how a head's pairs lie: in a lane or with one to exchange, or anyhow
  const bool near = a.neox ? 2u * a.half == HD : E > 1 || a.half * 2u == HD;

  for (; j < n_t; j = j1, h = h1) {
    j1 = j;
    h1 = h;
    step(j1, h1);
    load(j1, h1, nxt);
    const uint32_t t = t0 + j;
    const bool is_q = h < n_q;
    const int32_t row = __builtin_amdgcn_readfirstlane(s_row[j]);
    if (row != INT32_MIN) {   // uniform
      const uint32_t off = is_q ? h * (a.gated ? 2u : 1u) * HD : (h - n_q) * HD;
      const float* bias = is_q ? a.q_bias : a.k_bias;
      const float* bias2 = is_q ? a.q_bias : a.v_bias;
      double x[E], y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = (double)cur.x[e];
        y[e] = (double)cur.y[e];
        if (bias) x[e] += (double)bias[off + d0 + e];
        if (bias2) y[e] += (double)bias2[off + d0 + e + (is_q && a.gated ? HD : 0)];
      }
      if (is_q ? a.q_norm : a.k_norm) {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) sum = __builtin_fma(x[e], x[e], sum);
        const double scale = rsqrt64(wave_sum64(live ? sum : 0.0, lane) / HD + (double)a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * scale * (double)(is_q ? wq[e] : wk[e]);
      }
      if (a.half && near) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (a.neox) {   // pairs (d, d + HD / 2): the lane half a head away
            constexpr int FAR = HD >= 64 ? 32 : 16;
            const double o = lane_xor<FAR>(x[e], lane);
            const uint32_t p = (d0 + e) % (HD / 2);
            const double cs = s_cs[j][2u * p], sn = s_cs[j][2u * p + 1u];
            x[e] = lane & FAR ? o * sn + x[e] * cs : x[e] * cs - o * sn;
          } else if constexpr (E == 1) {
            const double o = lane_xor<1>(x[0], lane);
            const double cs = s_cs[j][d0 & ~1u], sn = s_cs[j][d0 | 1u];
            x[0] = lane & 1u ? o * sn + x[0] * cs : x[0] * cs - o * sn;
          } else if (!(e & 1) && (d0 + e) / 2u < a.half) {
            const double cs = s_cs[j][d0 + e], sn = s_cs[j][d0 + e + 1u], x0 = x[e], x1 = x[e + 1];
            x[e] = x0 * cs - x1 * sn;
            x[e + 1] = x0 * sn + x1 * cs;
          }
        }
      } else if (a.half) {
        double* sx = s_x[wave];
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (live) sx[d0 + e] = x[e];
        wave_lds_order();
        for (uint32_t i = lane; i < a.half; i += 64u) {
          const double cs = s_cs[j][2u * i], sn = s_cs[j][2u * i + 1u];
          const uint32_t i0 = a.neox ? i : 2u * i, i1 = a.neox ? i + a.half : 2u * i + 1u;
          const double x0 = sx[i0], x1 = sx[i1];
          sx[i0] = x0 * cs - x1 * sn;
          sx[i1] = x0 * sn + x1 * cs;
        }
        wave_lds_order();
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = sx[d0 + e];
        wave_lds_order();   // the next head is written there again
      }
      float xf[E], yf[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        xf[e] = (float)x[e];
        yf[e] = (float)y[e];
      }
      if (is_q) {
        const size_t at = ((size_t)t * a.n_head + h) * HD + d0;
        if (live) __builtin_memcpy(a.q_out + at, xf, sizeof(xf));
        if (live && a.gated) __builtin_memcpy(a.gate_out + at, yf, sizeof(yf));
      } else {
        const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)s_page[j]);
        int kq[E], vq[E];
        uint32_t kd, vd;
        q8_values(xf, kq, kd);
        q8_values(yf, vq, vd);
        if (page != kNoSeq && live) {
          const uint32_t in_page = (uint32_t)row & ((1u << b.shift) - 1u), kvh = h - n_q;
          const size_t at = page_at(b.shift, c.n_kv, page, kvh, in_page, HD) + d0;
          int8_t k8[E], v8[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            k8[e] = (int8_t)kq[e];
            v8[e] = (int8_t)vq[e];
          }
          __builtin_memcpy(c.k_qs + at, k8, E);
          __builtin_memcpy(c.v_qs + at, v8, E);
          if (d0 % 32u == 0) {
            const size_t d_at = page_at(b.shift, c.n_kv, page, kvh, in_page, HD / 32) + d0 / 32u;
            c.k_d[d_at] = (uint16_t)kd;
            c.v_d[d_at] = (uint16_t)vd;
          }
        }
      }
    }
    cur = nxt;
  }
}

// A workgroup to 4 T consecutive tokens, a wave to every fourth: their sequence and
// pages found once (a lane to a token's page number), then row by row, V values of
// K and of V to a lane, which it stores as 16 bytes.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(256) void paged_read_kernel(PagesDev c, PagedDev b, void* k_out, void* v_out, uint32_t stride, uint32_t T) {
  constexpr uint32_t V = BF16 ? 8 : 4, U = 4;   // values to a lane and step, steps at once
  const uint32_t lane = threadIdx.x & 63u, per = c.n_kv * c.hd, hd_shift = __builtin_ctz(c.hd);
  uint32_t t = blockIdx.x * 4u * T + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t end = min((blockIdx.x + 1u) * 4u * T, b.n_tok);
  const size_t head = (size_t)c.hd << b.shift;   // a head's values of a page
  while (t < end) {
    const uint32_t seq = find_seq(b.tok_start, b.n_seq, t);
    if (seq == kNoSeq) {
      t += 4u;
      continue;
    }
    const SeqRange r = seq_range(b, seq);
    const uint32_t n = (min(end, r.tok + r.n) - t + 3u) / 4u;   // of its tokens: t lies in the range, T <= 64
    const int32_t mine = row_of_token(r, t + 4u * min(lane, n - 1u));
    uint32_t pg = kNoSeq;
    if (mine >= 0 && !page_of(b, seq, mine, pg)) pg = kNoSeq;
    for (uint32_t i = 0; i < n; ++i, t += 4u) {
      const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)pg, (int)i);
      const uint32_t in_page = (uint32_t)__builtin_amdgcn_readlane(mine, (int)i) & ((1u << b.shift) - 1u);
      const bool there = page != kNoSeq;
      const size_t row = ((size_t)(there ? page : 0u) * c.n_kv << b.shift) + in_page;   // of head 0
      for (uint32_t d0 = lane * V; d0 < per; d0 += 64u * V * U) {
        uint32_t kw[U][V / 4], vw[U][V / 4];
        uint16_t kd[U], vd[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint32_t d = min(d0 + u * 64u * V, per - V);
          const size_t at = row * c.hd + (size_t)(d >> hd_shift) * head + (d & (c.hd - 1u));
          __builtin_memcpy(kw[u], __builtin_assume_aligned(c.k_qs + at, V), V);
          __builtin_memcpy(vw[u], __builtin_assume_aligned(c.v_qs + at, V), V);
          kd[u] = c.k_d[at / 32u];
          vd[u] = c.v_d[at / 32u];
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint32_t d = d0 + u * 64u * V;
          if (d >= per) break;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const float s = there ? f16_to_f32(which ? vd[u] : kd[u]) : 0.0f;
            float f[V];
#pragma unroll
            for (uint32_t e = 0; e < V; ++e) {
              const uint32_t w = which ? vw[u][e / 4] : kw[u][e / 4];
              f[e] = there ? (float)(int8_t)(w >> (8u * (e % 4u))) * s : 0.0f;
            }
            const size_t o = (size_t)t * stride + d;
            void* out = which ? v_out : k_out;
            if constexpr (VEC) {
              u32x4 q;
#pragma unroll
              for (uint32_t e = 0; e < 4; ++e) q[e] = BF16 ? bf16x2_pack(f[2 * e % V], f[(2 * e + 1) % V]) : __float_as_uint(f[e]);
              __builtin_nontemporal_store(q, reinterpret_cast<u32x4*>(static_cast<char*>(out) + o * (BF16 ? 2u : 4u)));
            } else {
#pragma unroll
              for (uint32_t e = 0; e < V; ++e) {
                if constexpr (BF16)
                  static_cast<uint16_t*>(out)[o + e] = f32_to_bf16(f[e]);
                else
                  static_cast<float*>(out)[o + e] = f[e];
              }
            }
          }
        }
      }
    }
  }
}

template <int HD>
void prep_hd(const PagesDev& c, const PagedDev& b, const PagedPrep& a, const PagedRope& rope, bool bf16, hipStream_t s) {
  // A workgroup's tokens share what comes before its first head (1,900 tokens: one
  // token each 27.0 us, two 25.5, three 25.6, eight 32.6, with the read-back); below a
  // thousand one each, and their heads over several workgroups (64 tokens of 40
  // heads: one workgroup each 9.0 us, five 6.0; eight tokens to one 40).
  const uint32_t T = std::max(1u, std::min(kPrepTokens, b.n_tok / 512u)), units = ((a.q_raw ? a.n_head : 0u) + c.n_kv) * T;
  const uint32_t wgs = (b.n_tok + T - 1u) / T, per_wg = std::min(units, kPrepWaves);
  const dim3 grid(wgs, std::max(1u, std::min(512u / wgs, (units + per_wg - 1u) / per_wg))), block(64u * per_wg);
  if (bf16)
    paged_prep_kernel<HD, true><<<grid, block, 0, s>>>(c, b, a, rope, T);
  else
    paged_prep_kernel<HD, false><<<grid, block, 0, s>>>(c, b, a, rope, T);
}

}  // namespace

hipError_t launch_paged_prep(const PagesDev& c, const PagedDev& b, PagedPrep a, uint32_t rope_dim, float base,
                             const uint8_t* axis, bool bf16, hipStream_t s) {
  const uint32_t dim = rope_dim < c.hd ? rope_dim : c.hd;
  a.half = dim / 2u;
  PagedRope rope{};
  for (uint32_t i = 0; i < a.half; ++i) {
    rope.f[i] = std::pow((double)base, -2.0 * i / dim);
    rope.axis[i] = axis ? axis[i] : 0;
  }
  switch (c.hd) {
    case 32: prep_hd<32>(c, b, a, rope, bf16, s); break;
    case 64: prep_hd<64>(c, b, a, rope, bf16, s); break;
    case 128: prep_hd<128>(c, b, a, rope, bf16, s); break;
    case 256: prep_hd<256>(c, b, a, rope, bf16, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_paged_read(const PagesDev& c, const PagedDev& b, void* k_out, void* v_out, uint32_t stride, bool bf16,
                             hipStream_t s) {
  const size_t esz = bf16 ? 2 : 4;
  const bool vec = (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0 && (b.n_tok == 1 || stride * esz % 16 == 0);
  // Two tokens to a wave share what finding them costs (17,000 of 40 sequences 12.9
  // us, one 14.2, four 13.7); where the results are more than the 256 MB cache
  // holds, one, so that what is written at a time lies together (60,000 f32 rows of
  // 1,024 values, two caches in turn: one 111 us, two 123, eight 132; the same cache each
  // time 94, 92 and 95).
  const uint32_t T = (uint64_t)b.n_tok * c.n_kv * c.hd * 2u * esz >= 1u << 28 ? 1u : 2u, grid = (b.n_tok + 4u * T - 1u) / (4u * T);
  if (bf16 && vec)
    paged_read_kernel<true, true><<<grid, 256, 0, s>>>(c, b, k_out, v_out, stride, T);
  else if (bf16)
    paged_read_kernel<true, false><<<grid, 256, 0, s>>>(c, b, k_out, v_out, stride, T);
  else if (vec)
    paged_read_kernel<false, true><<<grid, 256, 0, s>>>(c, b, k_out, v_out, stride, T);
  else
    paged_read_kernel<false, false><<<grid, 256, 0, s>>>(c, b, k_out, v_out, stride, T);
  return hipGetLastError();
}

}  // namespace vxt
