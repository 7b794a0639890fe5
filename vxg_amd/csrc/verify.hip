// verify.hip -- drafted tokens judged by the model's probabilities and given
// random numbers, so that what comes out is distributed as the model's own
// samples.
//
// A sequence's tokens are its last committed one and the drafts behind it; row
// t's logits are the model's for what follows token t, with draft model's q
// beside them (or none: q is 1 for the draft).  In order, the draft x after row t
// is accepted iff  u q(x) < p(x).  After the first refusal, at row a, the next
// token is drawn from  r = max(p_a - q_a, 0)  (p_a without x where there is no q),
// after no refusal from p of the last row: the first id whose running sum of r
// passes u' times the whole.  p, q: softmax at the sequence's temperature;
// temperature 0: all on the lowest of the largest logits.
//
// Numbers.  Weights exp((l - max) / T), their sums and the products are 64 bits:
// the running sums of 150,000 probabilities in 32 bits are off by 1e-7, which is
// as much as many of them hold, and ids would depend on the order of a sum.
// Sums run in a fixed order, without atomics on values.
#include "kv_pages.hpp"

namespace vxt {

namespace {

constexpr uint32_t kPart = 2048;    // logits of a row to a wave: 32 a lane
constexpr uint32_t kSlice = 8192;   // logits of a row to a workgroup's sum of r

// A part of a row: the largest logit, its lowest id, the sum of weights to it.
struct PartStat {
  float m;
  uint32_t id;
  double sum;
};

struct RowStat {
  float m;
  uint32_t id;
  double inv;   // 1 / sum of weights; 0 where nothing has any
};

// What the draws of a sequence need: its row, and both distributions' sums.
struct SeqState {
  uint32_t row, mode;   // kDone, kPlain (p), kOver (max(p - q, 0)), kWithout (p without token x)
  uint32_t x, pad;
  RowStat p, q;
};
enum : uint32_t { kDone = 0, kPlain = 1, kOver = 2, kWithout = 3 };

struct Sums {
  double r, p;
};

// Weight of a logit against the largest, at 1 / T: 1 for the largest itself
// (also an infinite one), 0 for -inf and NaN.
__device__ __forceinline__ double weight(float x, float m, double inv_t) {
  if (x == m) return m == -__builtin_inff() ? 0.0 : 1.0;
  if (!(x > -__builtin_inff()) || m == __builtin_inff()) return 0.0;
  return exp(((double)x - (double)m) * inv_t);
}

__device__ __forceinline__ float logit(const void* row, uint32_t i, uint32_t bf16) {
  const float x = bf16 ? bf16_to_f32(static_cast<const uint16_t*>(row)[i]) : static_cast<const float*>(row)[i];
  return x == x ? x : -__builtin_inff();
}

__device__ __forceinline__ const void* row_of(const VerifyCall& v, const void* base, uint32_t t) {
  return static_cast<const char*>(base) + (size_t)t * v.stride * (v.bf16 ? 2u : 4u);
}

__device__ __forceinline__ double lane_sum64(double x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
  return x;
}

__device__ __forceinline__ uint32_t lane_min(uint32_t x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x = min(x, (uint32_t)__shfl_xor((int)x, o));
  return x;
}

// 1 / temperature of a sequence; 0 stands for greedy.
__device__ __forceinline__ double inverse_t(const VerifyCall& v, uint32_t seq) {
  const float t = v.temperature ? v.temperature[seq] : 1.0f;
  return t > 0.0f ? 1.0 / (double)t : 0.0;
}
__device__ __forceinline__ bool greedy(const VerifyCall& v, uint32_t seq) {
  return v.temperature && !(v.temperature[seq] > 0.0f);
}

// Stat of each part of each row: a wave to a part.  Rows [0, n_tok) are the
// model's, then the draft model's.
__global__ __launch_bounds__(256) void verify_stat_kernel(VerifyCall v, PartStat* stat, uint32_t n_part, uint32_t n_wg) {
  const uint32_t row = blockIdx.x / n_wg, part = (blockIdx.x % n_wg) * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
  const bool is_draft = row >= v.n_tok;
  const uint32_t t = is_draft ? row - v.n_tok : row;
  const uint32_t seq = find_seq(v.tok_start, v.n_seq, t);
  if (seq == kNoSeq || part >= n_part) return;
  if (is_draft) {
    const SeqRange r = token_range(v.tok_start, v.n_tok, seq);
    if (t + 1u >= r.tok + r.n) return;   // judges nothing
  }
  const void* x = row_of(v, is_draft ? v.draft : v.logits, t);
  float f[32];
  float m = -__builtin_inff();
#pragma unroll
  for (uint32_t i = 0; i < 32; ++i) {
    const uint32_t at = part * kPart + i * 64u + lane;
    f[i] = at < v.vocab ? logit(x, at, v.bf16) : -__builtin_inff();
    m = fmaxf(m, f[i]);
  }
  m = lane_reduce<64, true>(m);
  const double inv_t = inverse_t(v, seq);
  double sum = 0.0;
  uint32_t id = 0xffffffffu;
#pragma unroll
  for (uint32_t i = 0; i < 32; ++i) {
    sum += weight(f[i], m, inv_t);
    if (f[i] == m) id = min(id, part * kPart + i * 64u + lane);
  }
  sum = lane_sum64(sum);
  id = lane_min(id);
  if (lane == 0) stat[(size_t)row * n_part + part] = PartStat{m, id, sum};
}

// A row's parts joined, by every lane of a wave.
__device__ __forceinline__ RowStat join_parts(const PartStat* stat, uint32_t n_part, double inv_t) {
  const uint32_t lane = threadIdx.x & 63u;
  float m = -__builtin_inff();
  for (uint32_t i = lane; i < n_part; i += 64u) m = fmaxf(m, stat[i].m);
  m = lane_reduce<64, true>(m);
  double sum = 0.0;
  uint32_t id = 0xffffffffu;
  for (uint32_t i = lane; i < n_part; i += 64u) {
    const PartStat s = stat[i];
    sum += s.sum * weight(s.m, m, inv_t);
    if (s.m == m) id = min(id, s.id);
  }
  sum = lane_sum64(sum);
  id = lane_min(id);
  return RowStat{m, m == -__builtin_inff() ? 0u : id, sum > 0.0 ? 1.0 / sum : 0.0};
}

__device__ __forceinline__ double prob(float x, const RowStat& s, double inv_t) { return weight(x, s.m, inv_t) * s.inv; }

// Workgroup (sequence, slice of the vocabulary): every one judges the drafts
// for itself, then sums r over its slice.
__global__ __launch_bounds__(256) void verify_judge_kernel(VerifyCall v, const PartStat* stat, uint32_t n_part,
                                                           SeqState* state, Sums* sums, uint32_t n_slice) {
  __shared__ uint32_t s_first;
  __shared__ Sums s_sum[4];
  const uint32_t seq = blockIdx.x / n_slice, slice = blockIdx.x % n_slice, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u;
  const SeqRange r = token_range(v.tok_start, v.n_tok, seq);
  const uint32_t t0 = r.tok, drafts = r.n ? r.n - 1u : 0u;
  const bool cold = greedy(v, seq);
  const double inv_t = inverse_t(v, seq);
  if (tid == 0) s_first = drafts;
  __syncthreads();
  for (uint32_t j = wave; j < drafts; j += 4u) {
    const uint32_t t = t0 + j, x = v.tokens[t + 1u];
    const RowStat p = join_parts(stat + (size_t)t * n_part, n_part, inv_t);
    bool good;
    if (cold) {
      good = x == p.id;
    } else {
      double q_x = 1.0;
      if (v.draft) {
        const RowStat q = join_parts(stat + (size_t)(v.n_tok + t) * n_part, n_part, inv_t);
        q_x = x < v.vocab ? prob(logit(row_of(v, v.draft, t), x, v.bf16), q, inv_t) : 0.0;
      }
      const double p_x = x < v.vocab ? prob(logit(row_of(v, v.logits, t), x, v.bf16), p, inv_t) : 0.0;
      good = (double)v.u_accept[t + 1u] * q_x < p_x;
    }
    if (!good && lane == 0) atomicMin(&s_first, j);
  }
  __syncthreads();
  const uint32_t n_ok = s_first, row = t0 + n_ok;
  if (r.n == 0) {   // a sequence without tokens
    if (slice == 0 && tid == 0) {
      v.n_accept[seq] = 0u;
      v.next[seq] = 0xffffffffu;
      if (v.new_len) v.new_len[seq] = v.seq_len[seq];
      state[seq] = SeqState{0u, kDone, 0u, 0u, {}, {}};
    }
    return;
  }
  SeqState st{};
  st.row = row;
  st.p = join_parts(stat + (size_t)row * n_part, n_part, inv_t);
  st.mode = cold ? kDone : n_ok == drafts ? kPlain : v.draft ? kOver : kWithout;
  if (st.mode == kOver) st.q = join_parts(stat + (size_t)(v.n_tok + row) * n_part, n_part, inv_t);
  if (st.mode == kWithout) st.x = v.tokens[row + 1u];
  if (slice == 0 && tid == 0) {
    v.n_accept[seq] = n_ok;
    if (cold) v.next[seq] = st.p.id;
    if (v.new_len) v.new_len[seq] = v.seq_len[seq] - (int32_t)(drafts - n_ok);
    state[seq] = st;
  }
  if (cold) return;
  const void *pr = row_of(v, v.logits, row), *qr = v.draft ? row_of(v, v.draft, row) : nullptr;
  Sums sum{0.0, 0.0};
  for (uint32_t i = tid; i < kSlice; i += 256u) {
    const uint32_t at = slice * kSlice + i;
    if (at >= v.vocab) break;
    const double p = prob(logit(pr, at, v.bf16), st.p, inv_t);
    double over = p;
    if (st.mode == kOver) over = fmax(p - prob(logit(qr, at, v.bf16), st.q, inv_t), 0.0);
    if (st.mode == kWithout && at == st.x) over = 0.0;
    sum.p += p;
    sum.r += over;
  }
  sum.r = lane_sum64(sum.r);
  sum.p = lane_sum64(sum.p);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (tid == 0)
    sums[(size_t)seq * n_slice + slice] = Sums{s_sum[0].r + s_sum[1].r + s_sum[2].r + s_sum[3].r,
                                              s_sum[0].p + s_sum[1].p + s_sum[2].p + s_sum[3].p};
}

// A workgroup to a sequence: the slice in which the running sum passes the
// target, then the 256 ids of one of its waves, then the id.
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyCall v, const SeqState* state, const Sums* sums,
                                                          uint32_t n_slice) {
  constexpr uint32_t N = kSlice / 256;   // waves' pieces of a slice, in the order of their ids
  __shared__ double s_piece[N];
  const uint32_t seq = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u;
  SeqState st = state[seq];
  if (st.mode == kDone) return;
  const double inv_t = inverse_t(v, seq);
  const Sums* sl = sums + (size_t)seq * n_slice;
  double whole = 0.0;
  for (uint32_t i = 0; i < n_slice; ++i) whole += sl[i].r;
  if (!(whole > 0.0)) {   // nothing over: p itself
    st.mode = kPlain;
    whole = 0.0;
    for (uint32_t i = 0; i < n_slice; ++i) whole += sl[i].p;
  }
  if (!(whole > 0.0)) {
    if (tid == 0) v.next[seq] = 0u;
    return;
  }
  const double target = (double)v.u_next[seq] * whole;
  auto of_slice = [&](uint32_t i) { return st.mode == kPlain ? sl[i].p : sl[i].r; };
  uint32_t slice = 0;
  double before = 0.0, run = 0.0;
  bool found = false;
  for (uint32_t i = 0; i < n_slice && !found; ++i) {
    const double w = of_slice(i);
    if (w > 0.0) {
      slice = i;
      before = run;
    }
    run += w;
    found = run > target;
  }
  const void *pr = row_of(v, v.logits, st.row), *qr = v.draft ? row_of(v, v.draft, st.row) : nullptr;
  auto r_of = [&](uint32_t at) {
    if (at >= v.vocab || (st.mode == kWithout && at == st.x)) return 0.0;
    const double p = prob(logit(pr, at, v.bf16), st.p, inv_t);
    return st.mode == kOver ? fmax(p - prob(logit(qr, at, v.bf16), st.q, inv_t), 0.0) : p;
  };
  for (uint32_t i = wave; i < N; i += 4u) {
    double w = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) w += r_of(slice * kSlice + i * 256u + lane * 4u + j);
    w = lane_sum64(w);
    if (lane == 0) s_piece[i] = w;
  }
  __syncthreads();
  if (wave != 0) return;
  uint32_t piece = 0;
  found = false;
  run = before;
  for (uint32_t i = 0; i < N && !found; ++i) {
    if (s_piece[i] > 0.0) {
      piece = i;
      before = run;
    }
    run += s_piece[i];
    found = run > target;
  }
  double r[4], mine = 0.0;
  const uint32_t at = slice * kSlice + piece * 256u + lane * 4u;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    r[j] = r_of(at + j);
    mine += r[j];
  }
  double upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const double x = __shfl_up(upto, o);
    if ((int)lane >= o) upto += x;
  }
  double sum = before + (upto - mine);
  uint32_t id = 0xffffffffu, last = 0u;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    sum += r[j];
    if (r[j] > 0.0) {
      last = at + j;
      if (sum > target) id = min(id, at + j);
    }
  }
  id = lane_min(id);
  last = ~lane_min(~last);
  if (lane == 0) v.next[seq] = id == 0xffffffffu ? last : id;
}

size_t up256(size_t n) { return (n + 255u) & ~(size_t)255u; }

}  // namespace

size_t verify_workspace(const VerifyCall& v) {
  const size_t n_part = (v.vocab + kPart - 1u) / kPart, n_slice = (v.vocab + kSlice - 1u) / kSlice;
  return up256(v.n_tok * (v.draft ? 2u : 1u) * n_part * sizeof(PartStat)) + up256(v.n_seq * sizeof(SeqState)) +
         up256(v.n_seq * n_slice * sizeof(Sums));
}

hipError_t launch_verify(const VerifyCall& v, void* ws, hipStream_t s) {
  const uint32_t n_part = (v.vocab + kPart - 1u) / kPart, n_slice = (v.vocab + kSlice - 1u) / kSlice, n_wg = (n_part + 3u) / 4u;
  const uint32_t rows = v.n_tok * (v.draft ? 2u : 1u);
  PartStat* stat = static_cast<PartStat*>(ws);
  char* at = static_cast<char*>(ws) + up256((size_t)rows * n_part * sizeof(PartStat));
  SeqState* state = reinterpret_cast<SeqState*>(at);
  Sums* sums = reinterpret_cast<Sums*>(at + up256(v.n_seq * sizeof(SeqState)));
  verify_stat_kernel<<<rows * n_wg, 256, 0, s>>>(v, stat, n_part, n_wg);
  verify_judge_kernel<<<v.n_seq * n_slice, 256, 0, s>>>(v, stat, n_part, state, sums, n_slice);
  verify_draw_kernel<<<v.n_seq, 256, 0, s>>>(v, state, sums, n_slice);
  return hipGetLastError();
}

}  // namespace vxt
