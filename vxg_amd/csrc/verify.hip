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
// 2^y is 2^n (1 + f c_1 + .. + f^10 c_10), n the nearest whole number, with the
// polynomial through Chebyshev's nodes on [-1/2, 1/2]: right to 6e-16.  Sums run
// in a fixed order, without atomics on values.
//
// Three launches: a stat of each stretch of each row (the only one that reads
// much: 16 bytes a lane, eight loads in flight, about 20 vector operations a
// logit); the drafts judged and r summed by pieces of 512 ids, by a workgroup to
// each slice of a sequence's vocabulary; the draw, a wave to a sequence.
#include "kv_pages.hpp"

namespace vxt {

namespace {

constexpr uint32_t kPart = 2048;     // logits of a row that a wave holds at once: 32 a lane
constexpr uint32_t kPiece = 512;     // logits of a sum of r: 8 a lane
constexpr uint32_t kJudgeWaves = 16;
constexpr uint32_t kSlice = kPiece * kJudgeWaves;

// A stretch of a row: the largest logit, its lowest id (greedy only), the sum of
// weights to it.
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

// What the draw of a sequence needs: its row, and both distributions' sums.
struct SeqState {
  uint32_t row, mode;   // kDone, kPlain (p), kOver (max(p - q, 0)), kWithout (p without token x)
  uint32_t x, pad;
  RowStat p, q;
};
enum : uint32_t { kDone = 0, kPlain = 1, kOver = 2, kWithout = 3 };

struct Sums {
  double r, p;
};

constexpr float kNone = -__builtin_inff();   // no probability

// ---- 64-bit numbers --------------------------------------------------------------

// 2^y, 0 from y = -2000 down and for NaN; y <= 0.
__device__ __forceinline__ double exp2_64(double y) {
  y = __builtin_fmax(y, -2000.0);
  const double n = __builtin_rint(y), f = y - n;
  double p = 0x1.e5ea1aaa76421p-28;
  p = __builtin_fma(p, f, 0x1.b6571e1b18f3cp-24);
  p = __builtin_fma(p, f, 0x1.62bfe44904923p-20);
  p = __builtin_fma(p, f, 0x1.ffcb76784ab99p-17);
  p = __builtin_fma(p, f, 0x1.430913038349fp-13);
  p = __builtin_fma(p, f, 0x1.5d87fe908faf3p-10);
  p = __builtin_fma(p, f, 0x1.3b2ab6fba381dp-7);
  p = __builtin_fma(p, f, 0x1.c6b08d7044117p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff82c591p-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa39f7p-1);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// Weight of a logit x <= m against m, c = log2(e) / T: 1 for m itself, 0 for
// -inf; m -inf or infinite is the caller's.
__device__ __forceinline__ double weight(float x, float m, double c) { return exp2_64(((double)x - (double)m) * c); }
// The same for any m: beside an infinite one nothing else has weight.
__device__ __forceinline__ double weight_any(float x, float m, double c) {
  if (m == __builtin_inff()) return x == m ? 1.0 : 0.0;
  return m == kNone ? 0.0 : weight(x, m, c);
}

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over the wave, in every lane (the pairs of lane_reduce).
__device__ __forceinline__ double lane_sum64(double v) {
  v += dpp_f64<0xB1>(v);    // quad_perm [1,0,3,2]
  v += dpp_f64<0x4E>(v);    // quad_perm [2,3,0,1]
  v += dpp_f64<0x141>(v);   // row_half_mirror
  v += dpp_f64<0x140>(v);   // row_mirror
#pragma unroll
  for (int far = 0; far < 2; ++far) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)b, hi = (uint32_t)(b >> 32);
    const auto l = far ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto h = far ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = __builtin_bit_cast(double, (uint64_t)(uint32_t)h[0] << 32 | (uint32_t)l[0]) +
        __builtin_bit_cast(double, (uint64_t)(uint32_t)h[1] << 32 | (uint32_t)l[1]);
  }
  return v;
}

// Sum over lanes 0 .. this one.
__device__ __forceinline__ double lane_scan64(double v, uint32_t lane) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const double x = __shfl_up(v, o);
    if ((int)lane >= o) v += x;
  }
  return v;
}

__device__ __forceinline__ uint32_t lane_min(uint32_t x) { return ~lane_max_u32<64>(~x); }

// ---- logits -----------------------------------------------------------------------

__device__ __forceinline__ float logit(const void* row, uint32_t i, uint32_t bf16) {
  const float x = bf16 ? bf16_to_f32(static_cast<const uint16_t*>(row)[i]) : static_cast<const float*>(row)[i];
  return x == x ? x : kNone;
}

__device__ __forceinline__ const void* row_of(const VerifyCall& v, const void* base, uint32_t t) {
  return static_cast<const char*>(base) + (size_t)t * v.stride * (v.bf16 ? 2u : 4u);
}

// G * E logits of a row for each lane: runs of E = 8 (bf16: 16 bytes) or 4 (f32)
// from `at`, 64 E apart; none behind the vocabulary's end.
template <bool BF16, int N>
__device__ __forceinline__ void load_logits(const VerifyCall& v, const void* row, uint32_t at, uint32_t apart, float (&f)[N]) {
  constexpr uint32_t E = BF16 ? 8 : 4;
#pragma unroll
  for (uint32_t g = 0; g < N / E; ++g) {
    const uint32_t i = at + g * apart;
    if (v.vec && i + E <= v.vocab) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const char*>(row) + (size_t)i * (BF16 ? 2u : 4u));
#pragma unroll
      for (uint32_t j = 0; j < E; ++j) {
        if constexpr (BF16)
          f[g * E + j] = bf16_to_f32(j & 1u ? w[j / 2] >> 16 : w[j / 2] & 0xffffu);
        else
          f[g * E + j] = __uint_as_float(w[j]);
      }
    } else {
#pragma unroll
      for (uint32_t j = 0; j < E; ++j) f[g * E + j] = i + j < v.vocab ? logit(row, i + j, BF16) : kNone;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = __builtin_fmaxf(f[j], kNone);   // NaN: none
}

// log2(e) / temperature of a sequence; greedy: not above 0.
__device__ __forceinline__ float temperature_of(const VerifyCall& v, uint32_t seq) { return v.temperature ? v.temperature[seq] : 1.0f; }
__device__ __forceinline__ double scale_of(float t) { return 0x1.71547652b82fep+0 / (double)t; }

// ---- 1. a stat of each stretch -------------------------------------------------------
// Rows [0, n_tok) are the model's, then the draft model's.  A wave takes `parts`
// parts of a row, a lane's logits against the lane's own largest.
template <bool BF16>
__global__ __launch_bounds__(256) void verify_stat_kernel(VerifyCall v, PartStat* stat, uint32_t n_stat, uint32_t n_wg, uint32_t parts) {
  constexpr uint32_t E = BF16 ? 8 : 4;
  const uint32_t row = blockIdx.x / n_wg, which = (blockIdx.x % n_wg) * 4u + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
  const bool is_draft = row >= v.n_tok;
  const uint32_t t = is_draft ? row - v.n_tok : row;
  const uint32_t seq = find_seq(v.tok_start, v.n_seq, t);
  if (seq == kNoSeq || which >= n_stat) return;
  if (is_draft) {
    const SeqRange r = token_range(v.tok_start, v.n_tok, seq);
    if (t + 1u >= r.tok + r.n) return;   // judges nothing
  }
  const float temp = temperature_of(v, seq);
  const double c = scale_of(temp);
  const bool cold = !(temp > 0.0f);
  const void* x = row_of(v, is_draft ? v.draft : v.logits, t);
  float m = kNone;
  double sum = 0.0;
  uint32_t id = 0xffffffffu;
  for (uint32_t p = 0; p < parts; ++p) {
    const uint32_t at = (which * parts + p) * kPart + lane * E;
    if ((which * parts + p) * kPart >= v.vocab) break;
    float f[32];
    load_logits<BF16>(v, x, at, 64u * E, f);
    float top = f[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, f[i]);
    if (cold) {   // uniform
#pragma unroll
      for (uint32_t i = 0; i < 32; ++i)
        if (f[i] > m) {
          m = f[i];
          id = at + i / E * 64u * E + i % E;
        }
      continue;
    }
    if (top > m) {
      sum *= weight_any(m, top, c);
      m = top;
    }
    double part = 0.0;
#pragma unroll
    for (int i = 0; i < 32; ++i) part += weight(f[i], m, c);
    if (m == __builtin_inff()) {   // only infinite ones have weight
      part = 0.0;
#pragma unroll
      for (int i = 0; i < 32; ++i) part += f[i] == m ? 1.0 : 0.0;
    }
    sum += m == kNone ? 0.0 : part;
  }
  const float top = lane_reduce<64, true>(m);
  id = lane_min(m == top ? id : 0xffffffffu);
  if (!cold) sum = lane_sum64(sum * weight_any(m, top, c));
  if (lane == 0) stat[(size_t)row * n_stat + which] = PartStat{top, id, sum};
}

// A row's stats joined, by every lane of a wave.
__device__ __forceinline__ RowStat join_parts(const PartStat* stat, uint32_t n_stat, bool cold, double c) {
  const uint32_t lane = threadIdx.x & 63u;
  const PartStat mine = stat[min(lane, n_stat - 1u)];
  float m = mine.m;
  for (uint32_t i = lane + 64u; i < n_stat; i += 64u) m = fmaxf(m, stat[i].m);
  m = lane_reduce<64, true>(m);
  double sum = 0.0;
  uint32_t id = 0xffffffffu;
  for (uint32_t i = lane; i < n_stat; i += 64u) {
    const PartStat s = i == lane ? mine : stat[i];
    if (!cold) sum += s.sum * weight_any(s.m, m, c);
    if (s.m == m) id = min(id, s.id);
  }
  if (cold) id = lane_min(id);
  if (!cold) sum = lane_sum64(sum);
  return RowStat{m, m == kNone ? 0u : id, sum > 0.0 ? 1.0 / sum : 0.0};
}

__device__ __forceinline__ double prob(float x, const RowStat& s, double c) { return s.inv == 0.0 ? 0.0 : weight_any(x, s.m, c) * s.inv; }

// r (and p) of 8 logits of the row that a sequence draws from.
template <bool BF16>
__device__ __forceinline__ void left_over(const VerifyCall& v, const SeqState& st, double c, uint32_t at, double (&p)[8], double (&r)[8]) {
  constexpr uint32_t E = BF16 ? 8 : 4;
  float f[8], q[8];
  load_logits<BF16>(v, row_of(v, v.logits, st.row), at, E, f);
  if (st.mode == kOver) load_logits<BF16>(v, row_of(v, v.draft, st.row), at, E, q);
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    p[j] = f[j] == kNone ? 0.0 : prob(f[j], st.p, c);
    r[j] = p[j];
    if (st.mode == kOver) r[j] = __builtin_fmax(p[j] - (q[j] == kNone ? 0.0 : prob(q[j], st.q, c)), 0.0);
    if (st.mode == kWithout && at + j == st.x) r[j] = 0.0;
  }
}

// ---- 2. the drafts judged, r summed ---------------------------------------------------
// Workgroup (sequence, slice of the vocabulary): every one judges the drafts for
// itself, a wave to a draft, then sums r over its slice, a wave to a piece.
template <bool BF16>
__global__ __launch_bounds__(kJudgeWaves * 64) void verify_judge_kernel(VerifyCall v, const PartStat* stat, uint32_t n_stat,
                                                                        SeqState* state, Sums* sums, uint32_t n_slice) {
  __shared__ RowStat s_p[kJudgeWaves], s_q[kJudgeWaves];
  __shared__ uint32_t s_good[kJudgeWaves];
  const uint32_t seq = blockIdx.x / n_slice, slice = blockIdx.x % n_slice, tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const SeqRange r = token_range(v.tok_start, v.n_tok, seq);
  const uint32_t t0 = r.tok, drafts = r.n ? r.n - 1u : 0u;
  const float temp = temperature_of(v, seq);
  const bool cold = !(temp > 0.0f);
  const double c = scale_of(temp);
  if (r.n == 0) {   // a sequence without tokens
    if (slice == 0 && tid == 0) {
      v.n_accept[seq] = 0u;
      v.next[seq] = 0xffffffffu;
      if (v.new_len) v.new_len[seq] = v.seq_len[seq];
      state[seq] = SeqState{0u, kDone, 0u, 0u, {}, {}};
    }
    return;
  }
  uint32_t n_ok = 0, at = 0;   // accepted; the refused (or last) row among those that the waves hold
  for (uint32_t j0 = 0;; j0 += kJudgeWaves) {
    const uint32_t j = j0 + wave;
    if (j <= drafts) {
      const uint32_t t = t0 + j, x = j < drafts ? v.tokens[t + 1u] : 0u;
      const float u = j < drafts ? v.u_accept[t + 1u] : 0.0f;
      const bool in = j < drafts && x < v.vocab, with_q = v.draft && j < drafts;
      const float lp = in ? logit(row_of(v, v.logits, t), x, BF16) : kNone;
      const float lq = in && with_q ? logit(row_of(v, v.draft, t), x, BF16) : kNone;
      const RowStat p = join_parts(stat + (size_t)t * n_stat, n_stat, cold, c);
      RowStat q{};
      if (with_q && !cold) q = join_parts(stat + (size_t)(v.n_tok + t) * n_stat, n_stat, cold, c);
      bool good = in && x == p.id;
      if (!cold) {
        const double p_x = lp == kNone ? 0.0 : prob(lp, p, c), q_x = !with_q ? 1.0 : lq == kNone ? 0.0 : prob(lq, q, c);
        good = in && (double)u * q_x < p_x;
      }
      if (lane == 0) {
        s_p[wave] = p;
        s_q[wave] = q;
        s_good[wave] = good;
      }
    }
    __syncthreads();
    const uint32_t held = min(kJudgeWaves, drafts - j0 + 1u);   // rows, the last of all among them or not
    at = 0;
    while (at < held && j0 + at < drafts && s_good[at]) ++at;
    n_ok = j0 + at;
    if (at < held) break;   // refused, or the last row
    __syncthreads();        // read before the next rows are written
  }
  SeqState st;
  st.row = t0 + n_ok;
  st.x = 0u;
  st.pad = 0u;
  st.p = s_p[at];
  st.q = s_q[at];
  st.mode = cold ? kDone : n_ok == drafts ? kPlain : v.draft ? kOver : kWithout;
  if (st.mode == kWithout) st.x = v.tokens[st.row + 1u];
  if (slice == 0 && tid == 0) {
    v.n_accept[seq] = n_ok;
    if (cold) v.next[seq] = st.p.id;
    if (v.new_len) v.new_len[seq] = v.seq_len[seq] - (int32_t)(drafts - n_ok);
    state[seq] = st;
  }
  if (cold) return;
  const uint32_t piece = slice * kJudgeWaves + wave;
  if (piece * kPiece >= v.vocab) return;
  double p8[8], r8[8];
  left_over<BF16>(v, st, c, piece * kPiece + lane * 8u, p8, r8);
  Sums sum{0.0, 0.0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    sum.r += r8[j];
    sum.p += p8[j];
  }
  sum.r = lane_sum64(sum.r);
  sum.p = lane_sum64(sum.p);
  if (lane == 0) sums[(size_t)seq * n_slice * kJudgeWaves + piece] = sum;
}

// ---- 3. the draw --------------------------------------------------------------------
// The first of a wave's runs at whose end the sum, from `before` on, is over
// `target`; where none is, the last that holds anything.  `before`: the sum in
// front of it.
__device__ __forceinline__ uint32_t pick_lane(double mine, double target, double& before, uint32_t lane) {
  const double upto = before + lane_scan64(mine, lane);
  const uint64_t over = __builtin_amdgcn_ballot_w64(upto > target && mine > 0.0), some = __builtin_amdgcn_ballot_w64(mine > 0.0);
  const uint32_t l = over ? (uint32_t)__builtin_ctzll(over) : some ? 63u - (uint32_t)__builtin_clzll(some) : 0u;
  before = __shfl(upto - mine, (int)l);
  return l;
}

// A wave to a sequence: the piece in which the running sum passes the target,
// then the id.
template <bool BF16>
__global__ __launch_bounds__(64) void verify_draw_kernel(VerifyCall v, const SeqState* state, const Sums* sums, uint32_t n_slice) {
  const uint32_t seq = blockIdx.x, lane = threadIdx.x;
  const uint32_t n_piece = (v.vocab + kPiece - 1u) / kPiece, per = (n_piece + 63u) / 64u;
  SeqState st = state[seq];
  const float temp = temperature_of(v, seq);
  const Sums* mine = sums + (size_t)seq * n_slice * kJudgeWaves;
  const uint32_t first = lane * per;
  if (st.mode == kDone) return;
  const double c = scale_of(temp);
  Sums sum{0.0, 0.0};
  for (uint32_t i = first; i < first + per && i < n_piece; ++i) {
    const Sums x = mine[i];
    sum.r += x.r;
    sum.p += x.p;
  }
  double whole = lane_sum64(sum.r);
  if (!(whole > 0.0)) {   // nothing over: p itself
    st.mode = kPlain;
    sum.r = sum.p;
    whole = lane_sum64(sum.p);
  }
  if (!(whole > 0.0)) {
    if (lane == 0) v.next[seq] = 0u;
    return;
  }
  const double target = (double)v.u_next[seq] * whole;
  double before = 0.0;
  const uint32_t l = pick_lane(sum.r, target, before, lane);
  uint32_t piece = l * per;
  double run = before;
  for (uint32_t i = l * per; i < l * per + per && i < n_piece; ++i) {   // uniform
    const Sums x = mine[i];
    const double w = st.mode == kPlain ? x.p : x.r;
    if (w > 0.0) {
      piece = i;
      before = run;
    }
    run += w;
    if (run > target && w > 0.0) break;
  }
  double p8[8], r8[8], all = 0.0;
  left_over<BF16>(v, st, c, piece * kPiece + lane * 8u, p8, r8);
#pragma unroll
  for (int j = 0; j < 8; ++j) all += r8[j];
  const uint32_t at = pick_lane(all, target, before, lane);
  if (lane != at) return;
  uint32_t id = 0;
  bool found = false;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    before += r8[j];
    if (!found && r8[j] > 0.0) {
      id = piece * kPiece + lane * 8u + j;
      found = before > target;
    }
  }
  v.next[seq] = id;
}

size_t up256(size_t n) { return (n + 255u) & ~(size_t)255u; }

struct Layout {
  uint32_t rows, parts, n_stat, n_slice;   // parts of a row to a wave; stats of a row
  size_t state, sums, bytes;
};

// A wave takes more parts of a row where there are rows for four thousand waves.
Layout layout_of(const VerifyCall& v) {
  Layout l;
  const uint32_t n_part = (v.vocab + kPart - 1u) / kPart;
  l.rows = v.n_tok * (v.draft ? 2u : 1u);
  const uint64_t waves = (uint64_t)l.rows * n_part;
  l.parts = (uint32_t)(waves < 4096u ? 1u : waves / 4096u < 8u ? waves / 4096u : 8u);
  l.n_stat = (n_part + l.parts - 1u) / l.parts;
  l.n_slice = (v.vocab + kSlice - 1u) / kSlice;
  l.state = up256((size_t)l.rows * l.n_stat * sizeof(PartStat));
  l.sums = l.state + up256(v.n_seq * sizeof(SeqState));
  l.bytes = l.sums + up256((size_t)v.n_seq * l.n_slice * kJudgeWaves * sizeof(Sums));
  return l;
}

template <bool BF16>
void verify(const VerifyCall& v, const Layout& l, char* ws, hipStream_t s) {
  PartStat* stat = reinterpret_cast<PartStat*>(ws);
  SeqState* state = reinterpret_cast<SeqState*>(ws + l.state);
  Sums* sums = reinterpret_cast<Sums*>(ws + l.sums);
  const uint32_t n_wg = (l.n_stat + 3u) / 4u;
  verify_stat_kernel<BF16><<<l.rows * n_wg, 256, 0, s>>>(v, stat, l.n_stat, n_wg, l.parts);
  verify_judge_kernel<BF16><<<v.n_seq * l.n_slice, kJudgeWaves * 64, 0, s>>>(v, stat, l.n_stat, state, sums, l.n_slice);
  verify_draw_kernel<BF16><<<v.n_seq, 64, 0, s>>>(v, state, sums, l.n_slice);
}

}  // namespace

size_t verify_workspace(const VerifyCall& v) { return layout_of(v).bytes; }

hipError_t launch_verify(const VerifyCall& v, void* ws, hipStream_t s) {
  if (v.bf16)
    verify<true>(v, layout_of(v), static_cast<char*>(ws), s);
  else
    verify<false>(v, layout_of(v), static_cast<char*>(ws), s);
  return hipGetLastError();
}

}  // namespace vxt
