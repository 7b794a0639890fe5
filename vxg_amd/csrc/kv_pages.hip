// kv_pages.hip -- rows of a paged Q8_0 KV cache written and read back.
//
// Write (paged_prep_kernel).  Per token and head, in 64 bits:
//   x = input + bias;  x *= w / sqrt(sum x^2 / hd + eps);
//   pair i turned by  pos[axis(i)] * base^(-2 i / rope_dim);
// rounded once to f32 (the query's result), and for K and V quantised from there
// as KvQ8Block::quantize does (llm_prefill.rs:27-42) into the token's row.  With
// f32 steps the codes of a value next to a border would hang on the order of a
// sum, and the angle of position 100,000 would be off by 4e-3; a 64-bit multiply
// and add takes a wave as long as a 32-bit one here.
//
// Read (paged_read_kernel).  value = code * scale, of the same rows.
#include "kv_pages.hpp"

#include <cmath>

namespace vxt {

namespace {

constexpr uint32_t kPrepWaves = 16;

template <bool BF16>
__device__ __forceinline__ float load_x(const void* p, size_t i) {
  if constexpr (BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) v += __shfl_xor(v, o);
  return v;
}

// One workgroup per token, a wave for every head (query heads, then kv heads);
// lane l holds values l, l + 64, ... of its head.
template <int HD, bool BF16>
__global__ __launch_bounds__(kPrepWaves * 64) void paged_prep_kernel(PagesDev c, PagedDev b, PagedPrep a, PagedRope rope) {
#pragma clang fp contract(off)
  constexpr int J = HD >= 64 ? HD / 64 : 1;
  __shared__ double s_x[kPrepWaves][HD];
  __shared__ double s_cs[HD];           // cos, sin of pair i at 2 i, 2 i + 1
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, t = blockIdx.x, n_waves = blockDim.x >> 6;
  const uint32_t seq = find_seq(b.tok_start, b.n_seq, t);
  if (seq == kNoSeq) return;            // uniform
  const SeqRange r = seq_range(b, seq);
  const int32_t row = row_of_token(r, t);
  uint32_t page = 0;
  const bool kept = row >= 0 && page_of(b, seq, row, page);
  const uint32_t in_page = (uint32_t)row & ((1u << b.shift) - 1u);
  for (uint32_t i = tid; i < a.half; i += blockDim.x) {
    const int32_t at = a.rope_pos ? a.rope_pos[(size_t)rope.axis[i] * b.n_tok + t] : row;
    double sn, cs;
    sincos((double)at * rope.f[i], &sn, &cs);
    s_cs[2u * i] = cs;
    s_cs[2u * i + 1u] = sn;
  }
  __syncthreads();
  const uint32_t n_q = a.q_raw ? a.n_head : 0u;
  for (uint32_t u = wave; u < n_q + c.n_kv; u += n_waves) {
    const bool is_q = u < n_q;
    const uint32_t kvh = u - n_q;
    const uint32_t off = is_q ? u * (a.gated ? 2u : 1u) * HD : kvh * HD;
    const void* src = is_q ? a.q_raw : a.k_cur;
    const float* bias = is_q ? a.q_bias : a.k_bias;
    const size_t at = (size_t)t * (is_q ? a.q_stride : a.kv_stride) + off;
    double x[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t d = lane + 64u * j;
      x[j] = 0.0;
      if (d < HD) {
        x[j] = (double)load_x<BF16>(src, at + d);
        if (bias) x[j] += (double)bias[off + d];
        if (is_q && a.gated) {
          double g = (double)load_x<BF16>(src, at + HD + d);
          if (bias) g += (double)bias[off + HD + d];
          a.gate_out[((size_t)t * a.n_head + u) * HD + d] = (float)g;
        }
      }
    }
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (w) {
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < J; ++j) sum += x[j] * x[j];
      const double scale = 1.0 / sqrt(wave_sum64(sum) / HD + (double)a.eps);
#pragma unroll
      for (int j = 0; j < J; ++j) x[j] = x[j] * scale * (double)w[min(lane + 64u * j, HD - 1u)];
    }
    if (a.half) {
      double* sx = s_x[wave];
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (lane + 64u * j < HD) sx[lane + 64u * j] = x[j];
      wave_lds_order();
      for (uint32_t i = lane; i < a.half; i += 64u) {
        const double cs = s_cs[2u * i], sn = s_cs[2u * i + 1u];
        const uint32_t i0 = a.neox ? i : 2u * i, i1 = a.neox ? i + a.half : 2u * i + 1u;
        const double x0 = sx[i0], x1 = sx[i1];
        sx[i0] = x0 * cs - x1 * sn;
        sx[i1] = x0 * sn + x1 * cs;
      }
      wave_lds_order();
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (lane + 64u * j < HD) x[j] = sx[lane + 64u * j];
      wave_lds_order();
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t d = lane + 64u * j;
      if (is_q) {
        if (d < HD) a.q_out[((size_t)t * a.n_head + u) * HD + d] = (float)x[j];
        continue;
      }
      double v = d < HD ? (double)load_x<BF16>(a.v_cur, at + d) : 0.0;
      if (a.v_bias && d < HD) v += (double)a.v_bias[off + d];
      uint32_t kd, vd;
      const int kq = q8_lane((float)x[j], kd), vq = q8_lane((float)v, vd);
      if (!kept || d >= HD) continue;
      const size_t q_at = page_at(b.shift, c.n_kv, page, kvh, in_page, HD) + d;
      c.k_qs[q_at] = (int8_t)kq;
      c.v_qs[q_at] = (int8_t)vq;
      if ((d & 31u) == 0) {
        const size_t d_at = page_at(b.shift, c.n_kv, page, kvh, in_page, HD / 32) + d / 32u;
        c.k_d[d_at] = (uint16_t)kd;
        c.v_d[d_at] = (uint16_t)vd;
      }
    }
  }
}

// One workgroup per token, a lane for 4 values of K and of V.
template <bool BF16>
__global__ __launch_bounds__(256) void paged_read_kernel(PagesDev c, PagedDev b, void* k_out, void* v_out, uint32_t stride) {
  const uint32_t t = blockIdx.x, per = c.n_kv * c.hd;
  const uint32_t seq = find_seq(b.tok_start, b.n_seq, t);
  if (seq == kNoSeq) return;
  const SeqRange r = seq_range(b, seq);
  const int32_t row = row_of_token(r, t);
  uint32_t page = 0;
  const bool there = row >= 0 && page_of(b, seq, row, page);
  const uint32_t in_page = (uint32_t)row & ((1u << b.shift) - 1u);
  for (uint32_t i = threadIdx.x; i < per; i += blockDim.x) {
    const uint32_t kvh = i / c.hd, d = i % c.hd;
    float k = 0.0f, v = 0.0f;
    if (there) {
      const size_t q_at = page_at(b.shift, c.n_kv, page, kvh, in_page, c.hd) + d, d_at = page_at(b.shift, c.n_kv, page, kvh, in_page, c.hd / 32) + d / 32u;
      k = (float)c.k_qs[q_at] * f16_to_f32(c.k_d[d_at]);
      v = (float)c.v_qs[q_at] * f16_to_f32(c.v_d[d_at]);
    }
    const size_t o = (size_t)t * stride + i;
    if constexpr (BF16) {
      static_cast<uint16_t*>(k_out)[o] = f32_to_bf16(k);
      static_cast<uint16_t*>(v_out)[o] = f32_to_bf16(v);
    } else {
      static_cast<float*>(k_out)[o] = k;
      static_cast<float*>(v_out)[o] = v;
    }
  }
}

template <int HD>
void prep_hd(const PagesDev& c, const PagedDev& b, const PagedPrep& a, const PagedRope& rope, bool bf16, hipStream_t s) {
  const uint32_t units = (a.q_raw ? a.n_head : 0u) + c.n_kv;
  const dim3 grid(b.n_tok), block(64u * (units < kPrepWaves ? units : kPrepWaves));
  if (bf16)
    paged_prep_kernel<HD, true><<<grid, block, 0, s>>>(c, b, a, rope);
  else
    paged_prep_kernel<HD, false><<<grid, block, 0, s>>>(c, b, a, rope);
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
  if (bf16)
    paged_read_kernel<true><<<b.n_tok, 256, 0, s>>>(c, b, k_out, v_out, stride);
  else
    paged_read_kernel<false><<<b.n_tok, 256, 0, s>>>(c, b, k_out, v_out, stride);
  return hipGetLastError();
}

}  // namespace vxt
