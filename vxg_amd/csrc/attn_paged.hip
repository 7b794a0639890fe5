// attn_paged.hip -- attention of a batch's new tokens over the pages of a Q8_0
// KV cache.  Token j of a sequence's n new ones, in row len - n + j, attends to
// rows [0, len - n + j]:
//   out = sum_t softmax(q . K_t / sqrt(hd)) V_t, times 1 / (1 + exp(-gate)).
// A token that sees no row (none, or on pages that are out of range) gets 0.
#include "kv_pages.hpp"

namespace vxt {

namespace {

// A workgroup to a (token, query head), 256 rows at a time: a thread to a row's
// score, then a thread to a dim of the sum, references in base 2.
template <int HD>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagesDev c, PagedDev b, PagedAttn a) {
  __shared__ float s_q[HD], s_p[256], s_red[4];
  __shared__ uint32_t s_page[256];
  const uint32_t tid = threadIdx.x, t = blockIdx.x / a.n_head, head = blockIdx.x % a.n_head;
  const uint32_t kvh = head / (a.n_head / c.n_kv);
  const uint32_t seq = find_seq(b.tok_start, b.n_seq, t);
  if (seq == kNoSeq) return;
  const SeqRange r = seq_range(b, seq);
  const int upto = row_of_token(r, t) + 1;
  const float* q = a.q + ((size_t)t * a.n_head + head) * HD;
  for (uint32_t d = tid; d < HD; d += 256u) s_q[d] = q[d] * (1.4426950408889634f / sqrtf((float)HD));
  float m = -__builtin_inff(), l = 0.0f, acc = 0.0f;
  const uint32_t n_part = 256u / HD ? 256u / HD : 1u, part = tid / HD, dim = tid % HD;   // HD 256: one part
  for (int t0 = 0; t0 < upto; t0 += 256) {
    __syncthreads();
    const int row = t0 + (int)tid;
    uint32_t page = 0;
    float s = -__builtin_inff();
    const uint32_t rin = (uint32_t)row & ((1u << b.shift) - 1u);
    s_page[tid] = kNoSeq;
    if (row < upto && page_of(b, seq, row, page)) {
      s_page[tid] = page;
      const int8_t* k = c.k_qs + page_at(b.shift, c.n_kv, page, kvh, rin, HD);
      const uint16_t* kd = c.k_d + page_at(b.shift, c.n_kv, page, kvh, rin, HD / 32);
      s = 0.0f;
      for (uint32_t blk = 0; blk < HD / 32; ++blk) {
        float x = 0.0f;
        for (uint32_t d = 0; d < 32; ++d) x += s_q[32u * blk + d] * (float)k[32u * blk + d];
        s += x * f16_to_f32(kd[blk]);
      }
    }
    float top = lane_reduce<64, true>(s);
    if ((tid & 63u) == 0) s_red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])), m);
    const float off = top == -__builtin_inff() ? 0.0f : top;
    const float p = __builtin_amdgcn_exp2f(s - off), again = __builtin_amdgcn_exp2f(m - off);
    s_p[tid] = p;
    float sum = lane_reduce<64>(p);
    __syncthreads();
    if ((tid & 63u) == 0) s_red[tid >> 6] = sum;
    __syncthreads();
    l = l * again + (s_red[0] + s_red[1] + s_red[2] + s_red[3]);
    m = top;
    acc *= again;
    for (uint32_t i = part; i < 256u; i += n_part) {
      if (s_page[i] == kNoSeq) continue;
      const uint32_t ri = (uint32_t)(t0 + (int)i) & ((1u << b.shift) - 1u);
      const float v = (float)c.v_qs[page_at(b.shift, c.n_kv, s_page[i], kvh, ri, HD) + dim] *
                      f16_to_f32(c.v_d[page_at(b.shift, c.n_kv, s_page[i], kvh, ri, HD / 32) + dim / 32u]);
      acc += s_p[i] * v;
    }
  }
  __syncthreads();
  s_p[tid] = acc;
  __syncthreads();
  if (tid >= HD) return;
  float x = 0.0f;
  for (uint32_t k = 0; k < n_part; ++k) x += s_p[k * HD + tid];
  x = l == 0.0f ? 0.0f : x / l;
  const size_t o = ((size_t)t * a.n_head + head) * HD + tid;
  if (a.gate) x *= 1.0f / (1.0f + expf(-a.gate[o]));
  if (a.out_bf16)
    static_cast<uint16_t*>(a.out)[o] = f32_to_bf16(x);
  else
    static_cast<float*>(a.out)[o] = x;
}

}  // namespace

size_t paged_attn_workspace(const PagesDev&, const PagedDev&, const PagedAttn&) { return 0; }

hipError_t launch_paged_attn(const PagesDev& c, const PagedDev& b, const PagedAttn& a, void*, hipStream_t s) {
  const uint32_t grid = b.n_tok * a.n_head;
  switch (c.hd) {
    case 32: paged_attn_kernel<32><<<grid, 256, 0, s>>>(c, b, a); break;
    case 64: paged_attn_kernel<64><<<grid, 256, 0, s>>>(c, b, a); break;
    case 128: paged_attn_kernel<128><<<grid, 256, 0, s>>>(c, b, a); break;
    case 256: paged_attn_kernel<256><<<grid, 256, 0, s>>>(c, b, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace vxt
