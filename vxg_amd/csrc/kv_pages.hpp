// kv_pages.hpp -- the paged Q8_0 KV cache and a batch of sequences on it, as
// the kernels see them (VxtKvPagesQ8, VxtPagedBatch).
//
// A page's rows of one kv head lie together ([page][n_kv][rows][hd]): what a
// workgroup of one head reads is whole runs of rows * hd bytes, and the scales
// of 16 rows of 128 values fill a cache line, where rows of all heads
// interleaved would leave a head pieces of hd bytes.
#pragma once

#include "kv_ops.hpp"
#include "paged_rows.hpp"

namespace vxt {

struct PagesDev {
  int8_t* k_qs;
  uint16_t* k_d;
  int8_t* v_qs;
  uint16_t* v_d;
  uint32_t n_kv, hd;
};

constexpr uint32_t kNoSeq = 0xffffffffu;

// Axes of the positions that a head's pairs turn by, and their frequencies.
struct PagedRope {
  double f[128];
  uint8_t axis[128];
};

// The preparation of a batch's tokens (VxtGqaParams); x f32 or bf16.
struct PagedPrep {
  const void *q_raw, *k_cur, *v_cur;   // q_raw null: K and V alone
  const float *q_norm, *k_norm, *q_bias, *k_bias, *v_bias;
  const int32_t* rope_pos;             // null (the row) or [axes][n_tok]
  float *q_out, *gate_out;
  uint32_t q_stride, kv_stride, n_head, gated, half, neox;
  float eps;
};

struct PagedAttn {
  const float *q, *gate;
  void* out;
  uint32_t n_head, out_bf16;
};

// A verification of drafted tokens (verify.hip).
struct VerifyCall {
  const void *logits, *draft;     // [n_tok][stride], draft may be null
  uint32_t vocab, stride, bf16, vec;   // vec: rows of whole aligned 16-byte pieces
  const uint32_t* tokens;
  const int32_t* tok_start;
  uint32_t n_seq, n_tok;
  const float *temperature, *u_accept, *u_next;
  const int32_t* seq_len;
  int32_t* new_len;
  uint32_t *n_accept, *next;
};

// The sequence of token t (uniform), by every lane of a wave: two rounds over
// starts that do not fall (n_seq <= 4096); kNoSeq if it is none's.
__device__ __forceinline__ uint32_t find_seq(const int32_t* tok_start, uint32_t n_seq, uint32_t t) {
  if (!tok_start) return t < n_seq ? t : kNoSeq;
  const uint32_t lane = threadIdx.x & 63u, step = (n_seq + 63u) / 64u;
  const int32_t at = (int32_t)t;
  // how many of `first`, `first` + `by`, ... start at or before t
  auto upto = [&](uint32_t first, uint32_t by, uint32_t n) {
    const uint32_t i = first + lane * by;
    return (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(lane < n && i < n_seq && tok_start[min(i, n_seq)] <= at));
  };
  uint32_t n = upto(0, step, 64u);
  if (n == 0) return kNoSeq;
  uint32_t s = (n - 1u) * step;
  if (step > 1) {
    n = upto(s, 1u, step);
    s += n ? n - 1u : 0u;
  }
  s = (uint32_t)__builtin_amdgcn_readfirstlane((int)s);
  return tok_start[s] <= at && at < tok_start[s + 1] ? s : kNoSeq;
}

}  // namespace vxt
