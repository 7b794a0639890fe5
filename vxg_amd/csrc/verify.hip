// verify.hip -- drafted tokens settled by the model's probabilities and given
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
// 2^y is 2^n (1 + f c_1 + .. + f^9 c_9), n the nearest whole number, with the
// polynomial through Chebyshev's nodes on [-1/2, 1/2]: right to 4e-14, a step of
// an f32 random number over a million.  A weight below 2^-1000 of the largest is no
// probability, where a draft is accepted as where r is made.  Sums run in a fixed
// order, without atomics on values.
//
// Launches: a stat of each stretch of each row, which reads everything once (16 logits
// a lane and the next 16 on their way, about 20 vector operations of 64 bits a
// logit).  With a draft model two more: the drafts settled (accepted or refused) and r
// summed by pieces of 512 ids, by a workgroup to each slice of a sequence's
// vocabulary, which reads one row of each distribution again; the draw, a wave to a
// sequence.  Without one, one more: r is p but for the refused token, so the sums by
// parts of 1,024 that the first has anyway will do, and a workgroup to a sequence
// settles and draws (three launches 33.2 us at the third figure below).
// 48 sequences of up to six rows of 151,936 in f32 and as many drafts', 168 MB: 41 +
// 22 + 6 us, where a copy at 5.06 TB/s would take 33 (30 without the drafts' rows of the
// sequences at temperature 0, which are read and not used); the vector unit is busy
// for 60 % of the first and half of the second.  One of five rows, 18 us: the
// launches.  16 of up to nine rows of 248,320 in bf16, 35 MB: 20 + 12 us; half of the
// first is the vector unit (850 operations a wave, of which 380 are the logits'), the
// second a chain of loads.
#include "kv_pages.hpp"

#include <algorithm>

namespace vxt {

namespace {

constexpr uint32_t kPart = 1024;     // logits of a row that a wave holds at once: 16 a lane
constexpr uint32_t kPiece = 512;     // logits of a sum of r: 8 a lane
constexpr uint32_t kSettleWaves = 16;

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
  uint32_t x;
  float temp;
  RowStat p, q;
};
enum : uint32_t { kDone = 0, kPlain = 1, kOver = 2, kWithout = 3 };

constexpr float kNone = -__builtin_inff();   // no probability

// ---- 64-bit numbers --------------------------------------------------------------

// The polynomial's coefficients as scalars that the compiler does not know: as
// constants each would be moved into vector registers first.
struct Pow2 {
  double c[9];
};
__device__ __forceinline__ Pow2 pow2_coefficients() {
  Pow2 k = {{0x1.62e42fefa39efp-1, 0x1.ebfbdff823cedp-3, 0x1.c6b08d7047e52p-5, 0x1.3b2ab7181b759p-7, 0x1.5d87fe86fe981p-10,
             0x1.4308ac85aabcbp-13, 0x1.ffcb9515834efp-17, 0x1.63d13635db944p-20, 0x1.b63880bfc2ac3p-24}};
#pragma unroll
  for (int i = 0; i < 9; ++i) asm("" : "+s"(k.c[i]));
  return k;
}
// 2^f, -1/2 <= f <= 1/2.
__device__ __forceinline__ double pow2_part(double f, const Pow2& k) {
  double p = __builtin_fma(k.c[8], f, k.c[7]);
#pragma unroll
  for (int i = 6; i >= 0; --i) p = __builtin_fma(p, f, k.c[i]);
  return __builtin_fma(p, f, 1.0);
}

// 2^y, 0 from y = -2000 down and for NaN; y <= 0.
__device__ __forceinline__ double exp2_64(double y) {
  y = __builtin_fmax(y, -2000.0);
  const double n = __builtin_rint(y);
  return __builtin_amdgcn_ldexp(pow2_part(y - n, pow2_coefficients()), (int)n);
}

// Weight of a logit x <= m against m, c = log2(e) / T: 1 for m itself, 0 for
// -inf and NaN; m -inf or infinite is the caller's.
__device__ __forceinline__ double weight(float x, float m, double c) { return exp2_64(((double)x - (double)m) * c); }
// The same for any m: beside an infinite one nothing else has weight.
__device__ __forceinline__ double weight_any(float x, float m, double c) {
  if (m == __builtin_inff()) return x == m ? 1.0 : 0.0;
  return m == kNone ? 0.0 : weight(x, m, c);
}

// The weights of several logits to one m.  Those below 2^-1000 count as that much,
// or, exactly, as 0: with x kept above lo no exponent leaves its range, and
// n = 2^52 (3/2) + y - 2^52 (3/2) is the nearest whole number, whose low word goes
// to the exponent, with no conversion (they take four times as long as an
// addition).  ok: there is such an f32 lo, to 1 in the exponent (no temperature far
// off 1, m finite).
struct Weigher {
  float m, lo;
  bool ok;
};
__device__ __forceinline__ Weigher weigher(float m, float temp, double c) {
  const float lo = m - (float)((1000.0 / 0x1.71547652b82fep+0) * (double)temp);
  const double far = ((double)lo - (double)m) * c;
  return Weigher{m, lo, far > -1001.0 && far < -999.0};
}
__device__ __forceinline__ double weigh(float x, const Weigher& w, double md, double c, const Pow2& k) {
  const double d = (double)__builtin_fmaxf(x, w.lo) - md;
  const double t = __builtin_fma(d, c, 0x1.8p52), n = t - 0x1.8p52;
  const uint64_t b = __builtin_bit_cast(uint64_t, pow2_part(__builtin_fma(d, c, -n), k));
  uint32_t hi = (uint32_t)(b >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, t) << 20);
  asm("" : "+v"(hi));   // one 32-bit operation, not two of 64
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)b);
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

// N logits of a row for each lane of a wave: runs of E = 4 (bf16: 8), 16 bytes,
// from `at`, `apart` from one to the next; `end`: behind the last of the wave's.
// One branch for all of them, uniform, so that every load is on its way before the
// first is waited for; none behind the vocabulary's end.
template <bool BF16, int N>
__device__ __forceinline__ void load_logits(const VerifyCall& v, const void* row, uint32_t at, uint32_t apart, uint32_t end, float (&f)[N]) {
  constexpr uint32_t E = BF16 ? 8 : 4;
  if (v.vec && end <= v.vocab) {
    u32x4 w[N / E];
#pragma unroll
    for (uint32_t g = 0; g < N / E; ++g)
      w[g] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(static_cast<const char*>(row) + (size_t)(at + g * apart) * (BF16 ? 2u : 4u)));
#pragma unroll
    for (uint32_t g = 0; g < N / E; ++g)
#pragma unroll
      for (uint32_t j = 0; j < E; ++j) {
        if constexpr (BF16)
          f[g * E + j] = bf16_to_f32(j & 1u ? w[g][j / 2] >> 16 : w[g][j / 2] & 0xffffu);
        else
          f[g * E + j] = __uint_as_float(w[g][j]);
      }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      const uint32_t k = at + i / E * apart + i % E;
      const uint32_t in = min(k, v.vocab - 1u);
      const float x = BF16 ? bf16_to_f32(static_cast<const uint16_t*>(row)[in]) : static_cast<const float*>(row)[in];
      f[i] = k < v.vocab ? x : kNone;
    }
  }
}

// log2(e) / temperature of a sequence; greedy: not above 0.
__device__ __forceinline__ float temperature_of(const VerifyCall& v, uint32_t seq) { return v.temperature ? v.temperature[seq] : 1.0f; }
__device__ __forceinline__ double scale_of(float t) { return 0x1.71547652b82fep+0 / (double)t; }

// ---- 1. a stat of each stretch -------------------------------------------------------
// Rows [0, n_tok) are the model's, then the draft model's.  A wave takes `parts`
// parts of a row, the next one's logits on their way; the workgroup's four waves are
// one stat.  KEEP: each part's sum is kept, to the largest logit that the wave had met
// by then, with the part's own largest (as bits, in `id`).
template <bool BF16, bool KEEP>
__global__ __launch_bounds__(256, 5) void verify_stat_kernel(VerifyCall v, PartStat* stat, uint32_t n_stat, uint32_t parts, PartStat* kept) {
  constexpr uint32_t E = BF16 ? 8 : 4;
  __shared__ PartStat s_part[4];
  const uint32_t row = blockIdx.x / n_stat, wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
  const uint32_t which = (blockIdx.x % n_stat) * 4u + wave;
  const bool is_draft = row >= v.n_tok;
  const uint32_t t = is_draft ? row - v.n_tok : row;
  const void* x = row_of(v, is_draft ? v.draft : v.logits, t);
  const uint32_t first = which * parts * kPart, end = min(first + parts * kPart, v.vocab);
  float f[16], ahead[16];
  auto load = [&](uint32_t p) { load_logits<BF16>(v, x, p + lane * E, 64u * E, p + kPart, ahead); };
  const uint32_t seq = find_seq(v.tok_start, v.n_seq, t);
  if (seq == kNoSeq) return;
  if (is_draft) {
    const SeqRange r = token_range(v.tok_start, v.n_tok, seq);
    if (t + 1u >= r.tok + r.n) return;   // settles nothing
  }
  if (first < end) load(first);
  const float temp = temperature_of(v, seq);
  const double c = scale_of(temp);
  const bool cold = !(temp > 0.0f);
  const Pow2 k = pow2_coefficients();
  float m = kNone;
  double sum = 0.0;
  uint32_t id = 0xffffffffu;
  Weigher w{kNone, 0.0f, false};
  for (uint32_t p = first; p < end; p += kPart) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = ahead[i];
    if (p + kPart < end) load(p + kPart);
    if (cold) {   // uniform
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (f[i] > m) {
          m = f[i];
          id = p + lane * E + i / E * 64u * E + i % E;
        }
      continue;
    }
    float top = kNone;   // NaN is passed over
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, f[i]);
    top = lane_reduce<64, true>(top);
    if (__builtin_amdgcn_ballot_w64(top > m) != 0) {   // uniform, and seldom after the first
      if (__builtin_amdgcn_ballot_w64(m != kNone) != 0) sum *= weight_any(m, top, c);
      m = top;
      w = weigher(m, temp, c);
    }
    double part = 0.0;
    if (__builtin_amdgcn_ballot_w64(!w.ok) == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) part += weigh(f[i], w, (double)m, c, k);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) part += weight_any(f[i], m, c);
    }
    if constexpr (KEEP) {
      part = lane_sum64(part);
      if (lane == 0) kept[(size_t)row * ((v.vocab + kPart - 1u) / kPart) + p / kPart] = PartStat{m, __float_as_uint(top), part};
    }
    sum += part;
  }
  const float top = cold ? lane_reduce<64, true>(m) : m;
  if (cold) id = lane_min(m == top ? id : 0xffffffffu);
  if (!cold && !KEEP) sum = lane_sum64(sum);
  if (lane == 0) s_part[wave] = PartStat{top, id, sum};
  __syncthreads();
  if (threadIdx.x != 0) return;
  PartStat all = s_part[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) all.m = fmaxf(all.m, s_part[w].m);
  all.id = 0xffffffffu;
  all.sum = 0.0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (s_part[w].m == all.m) all.id = min(all.id, s_part[w].id);
    if (!cold) all.sum += s_part[w].sum * weight_any(s_part[w].m, all.m, c);
  }
  stat[blockIdx.x] = all;
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

// p of a logit.
__device__ __forceinline__ double prob(float x, const RowStat& s, double c) {
  const bool none = s.inv == 0.0 || ((double)x - (double)s.m) * c < -1000.0;
  const double p = weight_any(x, s.m, c) * s.inv;
  return none ? 0.0 : p;
}

// The lane's 8 logits of a piece of the row that a sequence draws from.
struct Piece {
  float f[8], q[8];
};
template <bool BF16>
__device__ __forceinline__ void load_piece(const VerifyCall& v, const SeqState& st, uint32_t piece, uint32_t lane, Piece& o) {
  constexpr uint32_t E = BF16 ? 8 : 4;
  const uint32_t at = piece * kPiece + lane * 8u, end = piece * kPiece + kPiece;
  load_logits<BF16>(v, row_of(v, v.logits, st.row), at, E, end, o.f);
  if (st.mode == kOver) load_logits<BF16>(v, row_of(v, v.draft, st.row), at, E, end, o.q);
}

// r of them.
__device__ __forceinline__ void left_over(const SeqState& st, double c, const Pow2& k, uint32_t piece, uint32_t lane, const Piece& in,
                                          double (&r)[8]) {
  auto probs = [&](const float (&x)[8], const RowStat& s, double (&to)[8]) {
    const Weigher w = weigher(s.m, st.temp, c);
    if (w.ok && s.inv > 0.0) {   // uniform
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = x[j] > w.lo ? weigh(x[j], w, (double)s.m, c, k) * s.inv : 0.0;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = prob(x[j], s, c);
    }
  };
  probs(in.f, st.p, r);
  if (st.mode == kOver) {
    double less[8];
    probs(in.q, st.q, less);
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = __builtin_fmax(r[j] - less[j], 0.0);
  }
  if (st.mode == kWithout) {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      if (piece * kPiece + lane * 8u + j == st.x) r[j] = 0.0;
  }
}

// The sum of r over a piece, in every lane.
__device__ __forceinline__ double piece_sum(const SeqState& st, double c, const Pow2& k, uint32_t piece, uint32_t lane, const Piece& in) {
  double r[8];
  left_over(st, c, k, piece, lane, in, r);
  return lane_sum64(((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7])));
}

// ---- 2. the drafts settled, r summed ---------------------------------------------------

// A workgroup of kSettleWaves settles a sequence's drafts, a wave to a draft, and
// (`tell`) says how many are accepted; false if nothing is to be drawn.  Where the
// token ranges fall, no sequence has tokens.
struct SettleLds {
  RowStat p[kSettleWaves], q[kSettleWaves];
  uint32_t flags[kSettleWaves];   // 1: the wave's draft is accepted; 2: it has seen ranges that fall
};
template <bool BF16>
__device__ __forceinline__ bool settle(const VerifyCall& v, const PartStat* stat, uint32_t n_stat, uint32_t seq, double c, bool tell,
                                       SettleLds& s, SeqState& st) {
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const SeqRange r = token_range(v.tok_start, v.n_tok, seq);
  const uint32_t t0 = r.tok, drafts = r.n ? r.n - 1u : 0u;
  const float temp = temperature_of(v, seq);
  const bool cold = !(temp > 0.0f);
  st = SeqState{0u, kDone, 0u, temp, {}, {}};
  auto nothing = [&]() {   // a sequence without tokens
    if (tell) {
      v.n_accept[seq] = 0u;
      v.next[seq] = 0xffffffffu;
      if (v.new_len) v.new_len[seq] = v.seq_len[seq];
    }
    return false;
  };
  if (r.n == 0) return nothing();
  // a thread to a sequence's start and end (launch_verify: there are enough), from the
  // last wave on, which seldom has a row
  const uint32_t i = (kSettleWaves - 1u - wave) * 64u + lane;
  int32_t from = 0, upto = 0;
  if (v.tok_start && i < v.n_seq) {
    from = v.tok_start[i];
    upto = v.tok_start[i + 1u];
  }
  uint32_t n_ok = 0, at = 0;   // accepted; the refused (or last) row among those that the waves hold
  for (uint32_t j0 = 0;; j0 += kSettleWaves) {
    const uint32_t j = j0 + wave;
    uint32_t flags = 0;
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
        const double p_x = prob(lp, p, c), q_x = !with_q ? 1.0 : prob(lq, q, c);
        good = in && (double)u * q_x < p_x;
      }
      if (lane == 0) {
        s.p[wave] = p;
        s.q[wave] = q;
      }
      flags = good ? 1u : 0u;
    }
    if (__builtin_amdgcn_ballot_w64(clamp_u32(upto, v.n_tok) < clamp_u32(from, v.n_tok)) != 0) flags |= 2u;
    if (lane == 0) s.flags[wave] = flags;
    __syncthreads();
    const uint32_t all = s.flags[lane % kSettleWaves];
    // where ranges fall, some rows above have no statistics of this call
    if (__builtin_amdgcn_ballot_w64((all & 2u) != 0) != 0) return nothing();
    at = (uint32_t)__builtin_ctzll(~__builtin_amdgcn_ballot_w64((all & 1u) != 0) | 1ull << min(kSettleWaves, drafts - j0));
    n_ok = j0 + at;
    if (at < kSettleWaves) break;   // refused, or the last row
    __syncthreads();        // read before the next rows are written
  }
  st.row = t0 + n_ok;
  st.p = s.p[at];
  st.q = s.q[at];
  st.mode = cold ? kDone : n_ok == drafts ? kPlain : v.draft ? kOver : kWithout;
  if (st.mode == kWithout) st.x = v.tokens[st.row + 1u];
  if (tell) {
    v.n_accept[seq] = n_ok;
    if (cold) v.next[seq] = st.p.id;
    if (v.new_len) v.new_len[seq] = v.seq_len[seq] - (int32_t)(drafts - n_ok);
  }
  return !cold;
}

// With a draft model: workgroup (sequence, slice of the vocabulary); every one settles
// the drafts for itself, then sums r over its slice, a wave to a piece.
template <bool BF16>
__global__ __launch_bounds__(kSettleWaves * 64) void verify_settle_kernel(VerifyCall v, const PartStat* stat, uint32_t n_stat,
                                                                          SeqState* state, double* sums, uint32_t n_slice, uint32_t pieces) {
  __shared__ SettleLds s_settle;
  const uint32_t seq = blockIdx.x / n_slice, slice = blockIdx.x % n_slice, lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double c = scale_of(temperature_of(v, seq));
  const bool tell = slice == 0 && threadIdx.x == 0;
  SeqState st;
  const bool live = settle<BF16>(v, stat, n_stat, seq, c, tell, s_settle, st);
  if (tell) state[seq] = st;
  if (!live) return;
  const Pow2 k = pow2_coefficients();
  const uint32_t n_piece = (v.vocab + kPiece - 1u) / kPiece;
  const uint32_t first = slice * pieces * kSettleWaves + wave, end = min(first + pieces * kSettleWaves, n_piece);
  Piece in, ahead;
  if (first < end) load_piece<BF16>(v, st, first, lane, ahead);
  for (uint32_t piece = first; piece < end; piece += kSettleWaves) {
    in = ahead;
    if (piece + kSettleWaves < end) load_piece<BF16>(v, st, piece + kSettleWaves, lane, ahead);
    const double sum = piece_sum(st, c, k, piece, lane, in);
    if (lane == 0) sums[(size_t)seq * n_piece + piece] = sum;
  }
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

// By a wave: the run of PIECES pieces (`n` sums, by lanes' stretches) in which the
// running sum passes the target, then the id.  Where r is 0 throughout, again(st)
// makes the sums again, of p.
template <bool BF16, uint32_t PIECES, class Again>
__device__ __forceinline__ void draw(const VerifyCall& v, uint32_t seq, SeqState st, double c, const Pow2& k, const double* sums, uint32_t n,
                                     uint32_t lane, Again again) {
  const uint32_t n_piece = (v.vocab + kPiece - 1u) / kPiece, per = (n + 63u) / 64u;
  const uint32_t first = lane * per, end = min(first + per, n);
  double sum = 0.0;
  for (uint32_t i = first; i < end; ++i) sum += sums[i];
  double whole = lane_sum64(sum);
  if (!(whole > 0.0)) {
    st.mode = kPlain;
    again(st);
    __threadfence_block();
    sum = 0.0;
    for (uint32_t i = first; i < end; ++i) sum += sums[i];
    whole = lane_sum64(sum);
  }
  if (!(whole > 0.0)) {
    if (lane == 0) v.next[seq] = 0u;
    return;
  }
  const double target = (double)v.u_next[seq] * whole;
  double before = 0.0;
  const uint32_t l = pick_lane(sum, target, before, lane);
  uint32_t at = l * per;
  double run = before;
  for (uint32_t i = l * per; i < min(l * per + per, n); ++i) {   // uniform
    const double w = sums[i];
    if (w > 0.0) {
      at = i;
      before = run;
    }
    run += w;
    if (run > target && w > 0.0) break;
  }
  uint32_t piece = at * PIECES;
  double r[8], all = 0.0;
  Piece in;
  load_piece<BF16>(v, st, piece, lane, in);
  left_over(st, c, k, piece, lane, in, r);
#pragma unroll
  for (int j = 0; j < 8; ++j) all += r[j];
  if constexpr (PIECES == 2) {
    if (piece + 1u < n_piece) {   // the first of two, if the target lies in it or the second holds nothing
      double r2[8], all2 = 0.0;
      load_piece<BF16>(v, st, piece + 1u, lane, in);
      left_over(st, c, k, piece + 1u, lane, in, r2);
#pragma unroll
      for (int j = 0; j < 8; ++j) all2 += r2[j];
      const double here = lane_sum64(all);
      if (!(here > 0.0 && before + here > target) && lane_sum64(all2) > 0.0) {
        ++piece;
        before += here;
        all = all2;
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = r2[j];
      }
    }
  }
  const uint32_t who = pick_lane(all, target, before, lane);
  if (lane != who) return;
  uint32_t id = 0;
  bool found = false;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    before += r[j];
    if (!found && r[j] > 0.0) {
      id = piece * kPiece + lane * 8u + j;
      found = before > target;
    }
  }
  v.next[seq] = id;
}

template <bool BF16>
__global__ __launch_bounds__(64) void verify_draw_kernel(VerifyCall v, const SeqState* state, double* sums) {
  const uint32_t seq = blockIdx.x, lane = threadIdx.x, n_piece = (v.vocab + kPiece - 1u) / kPiece, per = (n_piece + 63u) / 64u;
  const SeqState st = state[seq];
  if (st.mode == kDone) return;
  const double c = scale_of(temperature_of(v, seq));
  const Pow2 k = pow2_coefficients();
  double* mine = sums + (size_t)seq * n_piece;
  draw<BF16, 1>(v, seq, st, c, k, mine, n_piece, lane, [&](const SeqState& plain) {
    for (uint32_t i = 0; i < n_piece; ++i) {
      Piece in;
      load_piece<BF16>(v, plain, i, lane, in);
      const double w = piece_sum(plain, c, k, i, lane, in);
      if (lane == i / per) mine[i] = w;
    }
  });
}

// Without a draft model r is p, but for the refused token: the parts' sums that the
// first kernel kept, and that token's part made again.  A workgroup to a sequence
// settles, brings the sums to the row's largest, and draws.
template <bool BF16>
__global__ __launch_bounds__(kSettleWaves * 64) void verify_pick_kernel(VerifyCall v, const PartStat* stat, uint32_t n_stat,
                                                                        const PartStat* kept, double* sums) {
  __shared__ SettleLds s_settle;
  const uint32_t seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, n_part = (v.vocab + kPart - 1u) / kPart;
  const double c = scale_of(temperature_of(v, seq));
  SeqState st;
  if (!settle<BF16>(v, stat, n_stat, seq, c, tid == 0, s_settle, st)) return;
  const Pow2 k = pow2_coefficients();
  double* mine = sums + (size_t)seq * n_part;
  const PartStat* from = kept + (size_t)st.row * n_part;
  const Weigher w = weigher(st.p.m, st.temp, c);
  // what left_over would add up to; nothing exactly where it finds nothing
  auto p_of = [&](uint32_t i) {
    const PartStat s = from[i];
    const float top = __uint_as_float(s.id);
    const bool some = w.ok && st.p.inv > 0.0 ? top > w.lo : prob(top, st.p, c) > 0.0;
    return some ? s.sum * weight_any(s.m, st.p.m, c) * st.p.inv : 0.0;
  };
  const uint32_t again = st.mode == kWithout && st.x < v.vocab ? st.x / kPart : 0xffffffffu;
  for (uint32_t i = tid; i < n_part; i += kSettleWaves * 64u)
    if (i != again) mine[i] = p_of(i);
  if (again < n_part && tid >= (kSettleWaves - 1u) * 64u) {   // by the last wave
    const uint32_t n_piece = (v.vocab + kPiece - 1u) / kPiece;
    double sum = 0.0;
    for (uint32_t piece = 2u * again; piece < min(2u * again + 2u, n_piece); ++piece) {
      Piece in;
      load_piece<BF16>(v, st, piece, lane, in);
      sum += piece_sum(st, c, k, piece, lane, in);
    }
    if (lane == 0) mine[again] = sum;
  }
  __syncthreads();
  if (tid >= 64u) return;
  draw<BF16, 2>(v, seq, st, c, k, mine, n_part, lane, [&](const SeqState&) {
    for (uint32_t i = lane; i < n_part; i += 64u) mine[i] = p_of(i);
  });
}

size_t up256(size_t n) { return (n + 255u) & ~(size_t)255u; }

struct Layout {
  uint32_t rows, parts, n_stat;   // parts of a row to a wave; stats of a row
  uint32_t n_slice, pieces;       // slices of a sequence's sum; pieces of one to a wave
  size_t state, sums, kept, bytes;
};

uint32_t per(uint32_t n, uint32_t of) { return (n + of - 1u) / of; }

// Workgroups that a launch is brought down to by giving each more: 48 sequences of
// up to six rows of 151,936, 1024 / 2048 / 8000 of the first kind 72 / 70 / 81 us a
// call, 256 / 512 / 1024 of the second 69.8 / 74 / 78.
constexpr uint32_t kStatWgs = 2048, kSettleWgs = 256;

Layout layout_of(const VerifyCall& v) {
  Layout l;
  l.rows = v.n_tok * (v.draft ? 2u : 1u);
  const uint64_t most = (uint64_t)l.rows * per(v.vocab, 4u * kPart);
  l.parts = (uint32_t)(most < kStatWgs ? 1u : std::min<uint64_t>(most / kStatWgs, 8u));
  l.n_stat = per(v.vocab, 4u * l.parts * kPart);
  const uint32_t n_piece = per(v.vocab, kPiece), slices = per(n_piece, kSettleWaves);
  l.pieces = per(slices, per(kSettleWgs, v.n_seq));
  l.n_slice = per(slices, l.pieces);
  l.state = up256((size_t)l.rows * l.n_stat * sizeof(PartStat));
  l.sums = l.state + up256(v.n_seq * sizeof(SeqState));
  l.kept = l.sums + up256((size_t)v.n_seq * n_piece * sizeof(double));
  l.bytes = l.kept + (v.draft ? 0 : (size_t)l.rows * per(v.vocab, kPart) * sizeof(PartStat));
  return l;
}

template <bool BF16>
void verify(const VerifyCall& v, const Layout& l, char* ws, hipStream_t s) {
  PartStat* stat = reinterpret_cast<PartStat*>(ws);
  SeqState* state = reinterpret_cast<SeqState*>(ws + l.state);
  double* sums = reinterpret_cast<double*>(ws + l.sums);
  PartStat* kept = reinterpret_cast<PartStat*>(ws + l.kept);
  if (!v.draft) {
    verify_stat_kernel<BF16, true><<<l.rows * l.n_stat, 256, 0, s>>>(v, stat, l.n_stat, l.parts, kept);
    verify_pick_kernel<BF16><<<v.n_seq, kSettleWaves * 64, 0, s>>>(v, stat, l.n_stat, kept, sums);
    return;
  }
  verify_stat_kernel<BF16, false><<<l.rows * l.n_stat, 256, 0, s>>>(v, stat, l.n_stat, l.parts, kept);
  verify_settle_kernel<BF16><<<v.n_seq * l.n_slice, kSettleWaves * 64, 0, s>>>(v, stat, l.n_stat, state, sums, l.n_slice, l.pieces);
  verify_draw_kernel<BF16><<<v.n_seq, 64, 0, s>>>(v, state, sums);
}

}  // namespace

size_t verify_workspace(const VerifyCall& v) { return layout_of(v).bytes; }

hipError_t launch_verify(const VerifyCall& v, void* ws, hipStream_t s) {
  if (v.n_seq > kSettleWaves * 64u) return hipErrorInvalidValue;
  if (v.bf16)
    verify<true>(v, layout_of(v), static_cast<char*>(ws), s);
  else
    verify<false>(v, layout_of(v), static_cast<char*>(ws), s);
  return hipGetLastError();
}

}  // namespace vxt
