// kv_evict.hip -- rows of a Q8_0 KV cache moved about: eviction by
// accumulated attention weight, and the accepted path of a drafted tree.
//
// Eviction, per kv head: of seq rows the `keep` stay that come first in the
// order (protected, weight, lower row): a row is protected when its position
// is below n_first or among the last n_recent; NaN weighs least.  A kept row
// below `keep` stays where it is; the kept rows at and above `keep` go, in
// ascending order, into the rows that the evicted ones left below it, also
// ascending.  So a cache in place has as many rows copied as are evicted below
// `keep`, no source is a destination, and no order of the copies matters.
#include "kv_ops.hpp"
#include "narrow.hpp"

#include <algorithm>

namespace vxt {

namespace {

struct EvictArgs {
  const float* weight;        // [n_kv][plane]
  const uint32_t* position;
  uint32_t plane, seq, keep, n_first, recent_from, words;
  // what stays, per kv head and word of 64 rows: a bit per row, and how many
  // rows are left free below `keep`, and kept from there on, in earlier words
  uint64_t* kept;             // [n_kv][words]
  uint32_t* holes;            // [n_kv][words], of the word's stretch alone
  uint32_t* movers;           // [n_kv][words], likewise
  // a selection over several workgroups: stretches of `stretch` rows
  uint32_t stretch, n_str;    // n_str 1: the whole of a head
  uint2* total;               // [n_kv][n_str] free rows, movers
  uint32_t* hist;             // [n_kv][kWideBins]
  uint32_t* n_list;           // [n_kv]
  uint2* list;                // [n_kv][seq] key, ~row: the keys of the bin in which the last kept one falls
  uint4* cut;                 // [n_kv] that bin, how many of it stay; then key, ~row of the last kept
};

// A row's rank among the rows of its head.
__device__ __forceinline__ uint32_t row_key(const EvictArgs& a, const float* w, const uint32_t* pos, uint32_t i) {
  const uint32_t p = pos[i];
  const float x = w[i];
  return p < a.n_first || p >= a.recent_from ? kKeep : rank_key(x);
}

constexpr uint32_t kSelThreads = 1024, kSelWaves = kSelThreads / 64, kList = 4096;

// Selection by one workgroup to a kv head.  Each wave has a stretch of the
// rows, lane l of step j row i0 + 64 j + l, so a ballot is a word of `kept` and
// ranks are in row order.  A lane keeps its STEPS keys in registers: the rows
// are read once.
//
// The keep-th largest key: the protected rows are counted, then the range of
// the others' keys is narrowed by counts over 512 equal bins of it -- the
// counts spread over the bins whatever the weights' magnitudes, where bins of
// the leading bits would pile up in a few exponents and the LDS adds of a wave
// run one after the other.  Once the range holds no more than kList keys they
// are gathered in LDS, and the further rounds (at most four in all, for 32
// bits) go over those.  2,112 rows, 4 heads: 6.2 us, barriers and one load.
template <int STEPS>
__global__ __launch_bounds__(kSelThreads) void kv_evict_select_kernel(EvictArgs a) {
  __shared__ uint32_t s_hist[4][kBins];   // bin b at word 64 (b % 8) + b / 8: a lane's eight bins in eight reads
  __shared__ uint32_t s_list[kList];
  __shared__ uint32_t s_w[3][kSelWaves];
  __shared__ uint32_t s_n;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t kvh = blockIdx.x;
  const float* w = a.weight + (size_t)kvh * a.plane;
  const uint32_t* pos = a.position + (size_t)kvh * a.plane;
  const uint32_t per_w = ((a.seq + kSelWaves - 1u) / kSelWaves + 63u) & ~63u;
  const uint32_t i0 = min(a.seq, wave * per_w), i1 = min(a.seq, i0 + per_w);
  const uint32_t steps = (i1 - i0 + 63u) / 64u;
  uint32_t keys[STEPS];
#pragma unroll
  for (uint32_t j = 0; j < (uint32_t)STEPS; ++j)   // of a row past the stretch: never counted, see `in`
    keys[j] = row_key(a, w, pos, min(i0 + 64u * j + lane, a.seq - 1u));
  auto each = [&](auto f) {
    uint32_t row0 = i0 + lane;
    asm volatile("" : "+v"(row0));   // the rows anew in each pass, not in registers across them
#pragma unroll
    for (uint32_t j = 0; j < (uint32_t)STEPS; ++j) f(keys[j], row0 + 64u * j, j);
  };

  // protected rows, and the range of the others' keys (its low end as a maximum)
  uint32_t lo = 0, hi = 0, n_safe = 0;
  each([&](uint32_t k, uint32_t row, uint32_t) {
    const bool in = row < i1, safe = in && k == kKeep;
    n_safe += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(safe));
    lo = in && !safe ? max(lo, ~k) : lo;
    hi = in && !safe ? max(hi, k) : hi;
  });
  lo = lane_max_u32<64>(lo);
  hi = lane_max_u32<64>(hi);
  if (lane == 0) {
    s_w[0][wave] = n_safe;
    s_w[1][wave] = lo;
    s_w[2][wave] = hi;
  }
  for (uint32_t i = tid; i < 4u * kBins; i += kSelThreads) s_hist[i / kBins][i % kBins] = 0u;
  if (tid == 0) s_n = 0u;
  __syncthreads();
  n_safe = 0;
#pragma unroll
  for (uint32_t v = 0; v < kSelWaves; ++v) {
    n_safe += s_w[0][v];
    lo = max(lo, s_w[1][v]);
    hi = max(hi, s_w[2][v]);
  }
  lo = ~lo;
  // kept: key > at, or key == at and among the first `need` of the n_eq such
  uint32_t at = kKeep, need = a.keep, n_eq = n_safe;
  if (n_safe < a.keep) {
    need = a.keep - n_safe;
    n_eq = a.seq - n_safe;
    bool listed = false;
    uint32_t round = 0;
    const Range r = narrow({lo, hi - lo}, need, n_eq, [&](Range in, uint32_t shift, uint32_t& want, uint32_t& held) {
      if (round > 0 && !listed && held <= kList) {   // uniform
        each([&](uint32_t k, uint32_t row, uint32_t) {
          if (row < i1 && k - in.lo <= in.width) s_list[atomicAdd(&s_n, 1u)] = k;
        });
        listed = true;
        __syncthreads();
      }
      auto count = [&](uint32_t k) {   // kKeep lies above every range
        const uint32_t b = (k - in.lo) >> shift;
        if (k - in.lo <= in.width) atomicAdd(&s_hist[round][(b & 7u) * 64u + (b >> 3)], 1u);
      };
      if (listed) {
        for (uint32_t i = tid; i < s_n; i += kSelThreads) count(s_list[i]);
      } else {
        each([&](uint32_t k, uint32_t row, uint32_t) {
          if (row < i1) count(k);
        });
      }
      __syncthreads();
      uint32_t c[8], bin;
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = s_hist[round][j * 64u + lane];
      find_bin<8>(c, want, bin, want, held);
      ++round;
      return bin;
    });
    at = lo = r.lo;
    if (need == n_eq && lo != 0) {   // every key from lo on: no ranks needed (from 0 on: all ranks are taken)
      at = lo - 1u;
      need = n_eq = 0;
    }
  }

  // equal keys ahead of this wave's stretch
  uint32_t e = 0;
  if (need < n_eq) {   // uniform
    each([&](uint32_t k, uint32_t row, uint32_t) {
      e += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(row < i1 && k == at));
    });
    e = wave_prefix<kSelWaves>(e, s_w[0], wave, lane);
  }
  uint64_t* kept = a.kept + (size_t)kvh * a.words + i0 / 64u;
  const bool ranks = need > 0;
  each([&](uint32_t k, uint32_t row, uint32_t j) {
    const bool in = row < i1;
    uint64_t m = __builtin_amdgcn_ballot_w64(in && k > at);
    if (ranks) {   // uniform
      const uint64_t me = __builtin_amdgcn_ballot_w64(in && k == at);
      m |= __builtin_amdgcn_ballot_w64(in && k == at && e + ones_below(me, lane) < need);
      e += (uint32_t)__popcll(me);
    }
    if (j < steps && lane == 0) kept[j] = m;
  });
  __syncthreads();   // every word is there, and visible within the workgroup
  // free rows and movers ahead of each word
  kept = a.kept + (size_t)kvh * a.words;
  uint32_t h0 = 0, m0 = 0;
  for (uint32_t b = 0; b < a.words; b += kSelThreads) {
    const uint32_t i = b + tid;
    const uint64_t m = i < a.words ? kept[i] : 0ull;
    const uint32_t below = i * 64u >= a.keep ? 0u : min(64u, a.keep - i * 64u);   // rows of the word below `keep`
    const uint64_t low = below >= 64u ? ~0ull : (1ull << below) - 1ull;
    const uint32_t h = i < a.words ? (uint32_t)__popcll(~m & low) : 0u, v = (uint32_t)__popcll(m & ~low);
    const uint32_t hs = lane_scan_u32(h), vs = lane_scan_u32(v);
    __syncthreads();
    if (lane == 63u) {
      s_w[0][wave] = hs;
      s_w[1][wave] = vs;
    }
    __syncthreads();
    uint32_t hp = h0, vp = m0;
#pragma unroll
    for (uint32_t x = 0; x < kSelWaves; ++x) {
      hp += x < wave ? s_w[0][x] : 0u;
      vp += x < wave ? s_w[1][x] : 0u;
      h0 += s_w[0][x];
      m0 += s_w[1][x];
    }
    if (i < a.words) {
      a.holes[(size_t)kvh * a.words + i] = hp + hs - h;
      a.movers[(size_t)kvh * a.words + i] = vp + vs - v;
    }
  }
}

// ---- selection over many workgroups ---------------------------------------------
// Four launches, workgroup (stretch, kv head) but for the third:
//   count   the keys' upper 12 bits, in LDS and from there into hist;
//   gather  the bin in which the keep-th largest falls, and its keys as
//           (key, ~row) -- no two alike -- into the head's list, in any order;
//   cut     a workgroup to a head: the last kept of the list;
//   words   what stays, row by row against the cut, and the words' counts.
// Nothing but integers is added by atomics: no order of theirs shows.
// 65,000 rows, 8 heads: 2 to 4 us the clearing, 7.7, 7.8, 3.9 and 4.9 us, each a
// launch, one round of loads (4 MB in all) and its counts; one workgroup to a
// head, with 64 keys to a lane, took 69.
constexpr uint32_t kWideBins = 4096, kWideThreads = 256, kWideRows = 8, kBatch = kWideThreads * kWideRows, kStretches = 256;

__global__ __launch_bounds__(kWideThreads) void kv_evict_clear_kernel(EvictArgs a) {
  const uint32_t i = blockIdx.x * kWideThreads + threadIdx.x;
  if (i < kWideBins) a.hist[(size_t)blockIdx.y * kWideBins + i] = 0u;
  if (i == 0) a.n_list[blockIdx.y] = 0u;
}

// The keys of rows i0 + lane of the batch: thread t of 256 has rows 64 apart,
// a wave 8 words.  Rows from `end` on repeat the one before it.
__device__ __forceinline__ void load_keys(const EvictArgs& a, uint32_t kvh, uint32_t i0, uint32_t end, uint32_t (&keys)[kWideRows]) {
  const float* w = a.weight + (size_t)kvh * a.plane;
  const uint32_t* pos = a.position + (size_t)kvh * a.plane;
#pragma unroll
  for (uint32_t j = 0; j < kWideRows; ++j) keys[j] = row_key(a, w, pos, min(i0 + 64u * j, end - 1u));
}

__global__ __launch_bounds__(kWideThreads) void kv_evict_count_kernel(EvictArgs a) {
  __shared__ uint32_t s_hist[kWideBins];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, kvh = blockIdx.y;
  const uint32_t b0 = blockIdx.x * a.stretch, end = min(a.seq - b0, a.stretch) + b0;
  for (uint32_t i = tid; i < kWideBins; i += kWideThreads) s_hist[i] = 0u;
  __syncthreads();
  for (uint32_t b = b0; b < end; b += min(end - b, kBatch)) {
    uint32_t keys[kWideRows];
    const uint32_t i0 = b + (tid >> 6) * (64u * kWideRows) + lane;
    load_keys(a, kvh, i0, end, keys);
#pragma unroll
    for (uint32_t j = 0; j < kWideRows; ++j)
      if (i0 + 64u * j < end) atomicAdd(&s_hist[keys[j] >> 20], 1u);
  }
  __syncthreads();
  uint32_t c[kWideBins / kWideThreads];
#pragma unroll
  for (uint32_t j = 0; j < kWideBins / kWideThreads; ++j) c[j] = s_hist[tid + j * kWideThreads];
#pragma unroll
  for (uint32_t j = 0; j < kWideBins / kWideThreads; ++j)
    if (c[j]) atomicAdd(&a.hist[(size_t)kvh * kWideBins + tid + j * kWideThreads], c[j]);
}

__global__ __launch_bounds__(kWideThreads) void kv_evict_gather_kernel(EvictArgs a) {
  constexpr uint32_t W = kWideThreads / 64, PER = kWideBins / kWideThreads;
  __shared__ uint32_t s_sum[W], s_bin[2], s_at;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, kvh = blockIdx.y;
  const uint32_t b0 = blockIdx.x * a.stretch, end = min(a.seq - b0, a.stretch) + b0;
  uint32_t keys[kWideRows];
  load_keys(a, kvh, b0 + wave * (64u * kWideRows) + lane, end, keys);
  // bins from the top: thread t has the 16 below kWideBins - 16 t
  const u32x4* h = reinterpret_cast<const u32x4*>(a.hist + (size_t)kvh * kWideBins + (kWideThreads - 1u - tid) * PER);
  uint32_t c[PER], sum = 0;
#pragma unroll
  for (uint32_t j = 0; j < PER / 4u; ++j) {
    const u32x4 x = h[j];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) c[4u * j + e] = x[e];
  }
#pragma unroll
  for (uint32_t j = 0; j < PER; ++j) sum += c[j];
  uint32_t above = lane_scan_u32(sum);
  if (lane == 63u) s_sum[wave] = above;
  __syncthreads();
  above -= sum;
#pragma unroll
  for (uint32_t v = 0; v < W; ++v) above += v < wave ? s_sum[v] : 0u;
#pragma unroll
  for (int j = PER - 1; j >= 0; --j) {
    if (above < a.keep && a.keep <= above + c[j]) {   // one bin of one thread: keep <= seq
      s_bin[0] = (kWideThreads - 1u - tid) * PER + j;
      s_bin[1] = a.keep - above;
    }
    above += c[j];
  }
  __syncthreads();
  const uint32_t bin = s_bin[0];
  if (blockIdx.x == 0 && tid == 0) a.cut[kvh] = make_uint4(bin, s_bin[1], 0u, 0u);
  uint2* list = a.list + (size_t)kvh * a.seq;
  for (uint32_t b = b0; b < end; b += min(end - b, kBatch)) {
    const uint32_t i0 = b + wave * (64u * kWideRows) + lane;
    if (b != b0) load_keys(a, kvh, i0, end, keys);
    uint32_t n = 0;
#pragma unroll
    for (uint32_t j = 0; j < kWideRows; ++j) n += i0 + 64u * j < end && keys[j] >> 20 == bin ? 1u : 0u;
    const uint32_t upto = lane_scan_u32(n);
    if (lane == 63u) s_sum[wave] = upto;
    __syncthreads();
    if (tid == 0) {
      uint32_t all = 0;
#pragma unroll
      for (uint32_t v = 0; v < W; ++v) all += s_sum[v];
      s_at = all ? atomicAdd(&a.n_list[kvh], all) : 0u;
    }
    __syncthreads();
    uint32_t at = s_at + upto - n;
#pragma unroll
    for (uint32_t v = 0; v < W; ++v) at += v < wave ? s_sum[v] : 0u;
#pragma unroll
    for (uint32_t j = 0; j < kWideRows; ++j)
      if (i0 + 64u * j < end && keys[j] >> 20 == bin) list[at++] = make_uint2(keys[j], ~(i0 + 64u * j));
    __syncthreads();   // s_sum and s_at are read
  }
}

// The need-th largest (key, ~row) of the list: the range of the keys is narrowed
// by counts over 512 equal bins of it, then, where not all rows of the last kept
// key stay, that of the rows.  A list too long for LDS is read from memory, its
// keys' range first (most rows with the same weight would all count in one bin,
// one after the other), until what the range holds fits.  65,000 rows to 16,000,
// 8 heads, whole calls on the same planes: 45 us with weights far apart, 101 with
// one weight, 74 with all within a sixteenth of each other; 273 and 99 without
// any of that.
__global__ __launch_bounds__(kSelThreads) void kv_evict_cut_kernel(EvictArgs a) {
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint2 s_list[kList];
  __shared__ uint32_t s_w[2][kSelWaves], s_n;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, kvh = blockIdx.x;
  const uint4 bin0 = a.cut[kvh];
  const uint2* list = a.list + (size_t)kvh * a.seq;
  uint32_t n = a.n_list[kvh], need = bin0.y, n_eq = n;
  bool listed = n <= kList;   // uniform
  if (listed)
    for (uint32_t i = tid; i < n; i += kSelThreads) s_list[i] = list[i];
  if (tid == 0) s_n = 0u;
  auto each = [&](auto f) {
    if (listed) {
      for (uint32_t i = tid; i < n; i += kSelThreads) f(s_list[i]);
    } else {
      for (uint32_t i = tid; i < n; i += 8u * kSelThreads) {   // eight on their way
        uint2 e[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) e[u] = list[min(i + u * kSelThreads, n - 1u)];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u)
          if (i + u * kSelThreads < n) f(e[u]);
      }
    }
  };
  // value(entry, x): does it count, and its x; n_eq of them lie in the range
  auto search = [&](Range all, auto value) {
    return narrow(all, need, n_eq, [&](Range in, uint32_t shift, uint32_t& want, uint32_t& held) {
      if (!listed && held <= kList) {   // uniform; once: what is left goes to LDS, in any order
        each([&](uint2 e) {
          uint32_t x;
          if (value(e, x) && x - in.lo <= in.width) s_list[atomicAdd(&s_n, 1u)] = e;
        });
        listed = true;
        n = held;
      }
      __syncthreads();   // the last round's counts are read, the list is there
      if (tid < kBins) s_hist[tid] = 0u;
      __syncthreads();
      each([&](uint2 e) {
        uint32_t x;
        if (value(e, x) && x - in.lo <= in.width) {
          const uint32_t b = (x - in.lo) >> shift;
          atomicAdd(&s_hist[(b & 7u) * 64u + (b >> 3)], 1u);
        }
      });
      __syncthreads();
      uint32_t c[8], bin;
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = s_hist[j * 64u + lane];
      find_bin<8>(c, want, bin, want, held);
      return bin;
    }).lo;
  };
  uint32_t lo = bin0.x << 20, hi = lo + 0xfffffu;
  if (!listed) {
    uint32_t least = 0, most = 0;   // the least as a maximum
    each([&](uint2 e) {
      least = max(least, ~e.x);
      most = max(most, e.x);
    });
    least = lane_max_u32<64>(least);
    most = lane_max_u32<64>(most);
    if (lane == 0) {
      s_w[0][wave] = least;
      s_w[1][wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t v = 0; v < kSelWaves; ++v) {
      least = max(least, s_w[0][v]);
      most = max(most, s_w[1][v]);
    }
    lo = ~least;
    hi = most;
  }
  const uint32_t key = search({lo, hi - lo}, [](uint2 e, uint32_t& x) { x = e.x; return true; });
  uint32_t row = 0u;   // ~row of the last kept: at least this
  if (need != n_eq)
    row = search({~(a.seq - 1u), a.seq - 1u}, [key](uint2 e, uint32_t& x) { x = e.y; return e.x == key; });
  if (tid == 0) a.cut[kvh] = make_uint4(bin0.x, bin0.y, key, row);
}

__global__ __launch_bounds__(kWideThreads) void kv_evict_words_kernel(EvictArgs a) {
  constexpr uint32_t W = kBatch / 64;
  __shared__ uint64_t s_m[W];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, kvh = blockIdx.y;
  const uint32_t b0 = blockIdx.x * a.stretch, end = min(a.seq - b0, a.stretch) + b0;
  const uint4 cut = a.cut[kvh];
  const size_t head = (size_t)kvh * a.words;
  uint32_t h0 = 0, m0 = 0;   // wave 0's, uniform
  for (uint32_t b = b0; b < end; b += min(end - b, kBatch)) {
    uint32_t keys[kWideRows];
    const uint32_t i0 = b + wave * (64u * kWideRows) + lane;
    load_keys(a, kvh, i0, end, keys);
#pragma unroll
    for (uint32_t j = 0; j < kWideRows; ++j) {
      const uint32_t i = i0 + 64u * j;
      const uint64_t m = __builtin_amdgcn_ballot_w64(i < end && (keys[j] > cut.z || (keys[j] == cut.z && ~i >= cut.w)));
      if (lane == 0) s_m[wave * kWideRows + j] = m;
    }
    __syncthreads();
    if (wave == 0) {
      const uint32_t i = b / 64u + lane;
      const bool in = lane < W && i * 64u < end;
      const uint64_t m = in ? s_m[lane] : 0ull;
      const uint32_t below = i * 64u >= a.keep ? 0u : min(64u, a.keep - i * 64u);   // rows of the word below `keep`
      const uint64_t low = below >= 64u ? ~0ull : (1ull << below) - 1ull;
      const uint32_t h = in ? (uint32_t)__popcll(~m & low) : 0u, v = (uint32_t)__popcll(m & ~low);
      const uint32_t hs = lane_scan_u32(h), vs = lane_scan_u32(v);
      if (in) {
        a.kept[head + i] = m;
        a.holes[head + i] = h0 + hs - h;
        a.movers[head + i] = m0 + vs - v;
      }
      h0 += lane63(hs);
      m0 += lane63(vs);
    }
    __syncthreads();
  }
  if (tid == 0) a.total[(size_t)kvh * a.n_str + blockIdx.x] = make_uint2(h0, m0);
}

struct MoveArgs {
  KvQ8Dev from, to;
  EvictArgs e;
  uint32_t in_place;
  float* w_to;
  uint32_t* p_to;
  uint32_t plane_to;
};

// The row of set bit n of m.
__device__ __forceinline__ uint32_t nth_bit(uint64_t m, uint32_t n) {
  uint32_t at = 0;
#pragma unroll
  for (uint32_t s = 32; s > 0; s >>= 1) {
    const uint32_t c = (uint32_t)__popcll((m >> at) & ((1ull << s) - 1ull));
    if (n >= c) {
      n -= c;
      at += s;
    }
  }
  return at;
}

// kMoveRows rows of one kv head to a workgroup.  First a thread to a row finds its
// source: a kept row is its own, a free one's is the mover of its rank among
// the free ones, found by bisection of the movers' counts, of which every
// 2^s-th word's lie in LDS.  Then the rows that move, HD / 8 lanes to a row,
// each a 16-byte piece of K or V; the scales, the weight and the position by
// some of them.
// 64 rows to a workgroup: 5.5 us where 64 rows of 2,112 go, 6.5 with 128.  Of
// 65,000 rows to 16,000 (8 heads of 128) 19.6 us, 22.3 with the heads' workgroups
// spread over the XCDs: 3.5 TB/s of the codes, scales and their copies, the
// reads 128 bytes here and there.
constexpr uint32_t kCoarse = 1024, kMoveRows = 64, kMoveAhead = 4;
template <int HD>
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs a) {
  constexpr uint32_t L = HD / 8, NB = HD / 32, U = kMoveAhead, R = 256 / L;
  __shared__ uint32_t s_mov[kCoarse], s_base[2][kStretches], s_w[2][4];
  __shared__ uint2 s_move[kMoveRows];   // row, source
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t n_kv = a.from.n_kv, sub = tid % L, keep = a.e.keep, words = a.e.words;
  // The heads of the same rows on one XCD (workgroups go round the eight of
  // them): a row's scales of all heads are one or two lines.
  const uint32_t k = blockIdx.x / 8u % n_kv, b0 = blockIdx.x / 8u / n_kv * 8u + blockIdx.x % 8u, bn = gridDim.x / n_kv;
  if (b0 > (keep - 1u) / kMoveRows) return;
  const uint32_t row_q = n_kv * HD, row_d = n_kv * NB;
  const uint64_t* kept = a.e.kept + (size_t)k * words;
  const uint32_t* holes = a.e.holes + (size_t)k * words;
  const uint32_t* movers = a.e.movers + (size_t)k * words;
  const uint32_t per = a.e.stretch / 64u;   // words of a stretch
  // counts ahead of each stretch
  if (a.e.n_str > 1u) {
    const uint2 c = tid < a.e.n_str ? a.e.total[(size_t)k * a.e.n_str + tid] : make_uint2(0u, 0u);
    const uint32_t hs = lane_scan_u32(c.x), vs = lane_scan_u32(c.y);
    if (lane == 63u) {
      s_w[0][wave] = hs;
      s_w[1][wave] = vs;
    }
    __syncthreads();
    uint32_t hp = hs - c.x, vp = vs - c.y;
#pragma unroll
    for (uint32_t v = 0; v < 4; ++v) {
      hp += v < wave ? s_w[0][v] : 0u;
      vp += v < wave ? s_w[1][v] : 0u;
    }
    s_base[0][tid] = hp;
    s_base[1][tid] = vp;
  } else if (tid == 0) {
    s_base[0][0] = s_base[1][0] = 0u;
  }
  __syncthreads();
  auto moved = [&](uint32_t i) { return movers[i] + s_base[1][i / per]; };
  uint32_t shift = 0;
  while ((words - 1u) >> shift >= kCoarse) ++shift;
  const uint32_t coarse = ((words - 1u) >> shift) + 1u;
  for (uint32_t i = tid; i < coarse; i += 256u) s_mov[i] = moved(i << shift);
  __syncthreads();
  auto source = [&](uint32_t r) -> uint32_t {
    const uint64_t m = kept[r / 64u];
    if (m >> (r & 63u) & 1ull) return r;
    const uint32_t rank = holes[r / 64u] + s_base[0][r / 64u / per] + ones_below(~m, r & 63u);
    uint32_t lo = 0, hi = coarse;          // the last word whose count is <= rank
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) / 2u;
      if (s_mov[mid] <= rank) lo = mid;
      else hi = mid;
    }
    lo <<= shift;
    hi = min(words, lo + (1u << shift));
    while (hi - lo > 1u) {
      const uint32_t mid = (lo + hi) / 2u;
      if (moved(mid) <= rank) lo = mid;
      else hi = mid;
    }
    uint64_t x = kept[lo];
    if (lo * 64u < keep) x &= keep - lo * 64u >= 64u ? 0ull : ~0ull << (keep - lo * 64u);
    return lo * 64u + nth_bit(x, rank - moved(lo));
  };
  const bool is_v = sub >= L / 2u;
  const int8_t* fq = (is_v ? a.from.v_qs : a.from.k_qs) + k * HD + 16u * (sub % (L / 2u));
  int8_t* tq = (is_v ? a.to.v_qs : a.to.k_qs) + k * HD + 16u * (sub % (L / 2u));
  const bool has_d = sub < 2u * NB, d_v = sub >= NB;
  const uint16_t* fd = (d_v ? a.from.v_d : a.from.k_d) + k * NB + sub % NB;
  uint16_t* td = (d_v ? a.to.v_d : a.to.k_d) + k * NB + sub % NB;
  const uint32_t* wf = reinterpret_cast<const uint32_t*>(sub == L - 1u ? reinterpret_cast<const float*>(a.e.position) : a.e.weight) + (size_t)k * a.e.plane;
  uint32_t* wt = (sub == L - 1u ? a.p_to : reinterpret_cast<uint32_t*>(a.w_to)) + (size_t)k * a.plane_to;
  const bool has_w = sub >= L - 2u;
  for (uint32_t b = b0; b <= (keep - 1u) / kMoveRows; b += bn) {
    const uint32_t r = tid < kMoveRows ? b * kMoveRows + tid : keep;
    const uint32_t src = r < keep ? source(r) : 0u;
    const bool go = r < keep && !(a.in_place && src == r);
    const uint64_t m = __builtin_amdgcn_ballot_w64(go);
    if (lane == 0) s_w[0][wave] = (uint32_t)__popcll(m);
    __syncthreads();
    uint32_t at = ones_below(m, lane), n = 0;
#pragma unroll
    for (uint32_t v = 0; v < 4; ++v) {
      at += v < wave ? s_w[0][v] : 0u;
      n += s_w[0][v];
    }
    if (go) s_move[at] = make_uint2(r, src);
    __syncthreads();
    for (uint32_t i0 = tid / L; i0 < n; i0 += R * U) {
      uint2 s[U];
      u32x4 x[U];
      uint16_t y[U];
      uint32_t z[U];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {   // behind the last: it again
        s[u] = s_move[min(i0 + u * R, n - 1u)];
        x[u] = *reinterpret_cast<const u32x4*>(fq + (size_t)s[u].y * row_q);
        if (has_d) y[u] = fd[(size_t)s[u].y * row_d];
        if (has_w) z[u] = wf[s[u].y];
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        if (i0 + u * R >= n) break;
        *reinterpret_cast<u32x4*>(tq + (size_t)s[u].x * row_q) = x[u];
        if (has_d) td[(size_t)s[u].x * row_d] = y[u];
        if (has_w) wt[s[u].x] = z[u];
      }
    }
    __syncthreads();   // s_w and s_move are read
  }
}

// Rows pos + path[1 + j] -> pos + j for j < path[0].  A thread owns one
// 16-byte column of K or V, or one scale, and walks the path: an ascending
// path has path[1 + j] >= j, so what a step writes no later step reads.
__global__ __launch_bounds__(256) void kv_keep_path_kernel(KvQ8Dev c, const uint32_t* __restrict__ path,
                                                           uint32_t n_nodes, uint32_t pos) {
  const uint32_t per = c.n_kv * c.hd, nq = per / 16u, nd = per / 32u;
  const uint32_t col = blockIdx.x * 256u + threadIdx.x;
  if (col >= 2u * (nq + nd)) return;
  const uint32_t count = min(path[0], n_nodes);
  uint32_t prev = 0;
  for (uint32_t j = 0; j < count; ++j) {
    const uint32_t i = path[1u + j];
    if (i >= n_nodes || i < j || (j > 0 && i <= prev)) return;   // not ascending: the path ends here
    prev = i;
    if (i == j) continue;
    const size_t from = (size_t)pos + i, to = (size_t)pos + j;
    if (col < 2u * nq) {
      int8_t* p = (col < nq ? c.k_qs : c.v_qs) + 16u * (col % nq);
      *reinterpret_cast<u32x4*>(p + to * per) = *reinterpret_cast<const u32x4*>(p + from * per);
    } else {
      const uint32_t d = col - 2u * nq;
      uint16_t* p = (d < nd ? c.k_d : c.v_d) + d % nd;
      p[to * nd] = p[from * nd];
    }
  }
}

}  // namespace

namespace {

// One workgroup to a head up to here (with 4, 8 or 16 keys to a lane), several
// from there on.  An eviction to 64 rows, 2 or 8 heads of 128 alike: of 4,000
// rows 12 us; of 8,000 14.4 (with 16 keys to a lane 18.4); of 16,000 18.8, over
// several workgroups 24.2, at any size up to there.
constexpr uint32_t kWideFrom = 16u * kSelThreads;

struct EvictPlan {
  uint32_t words, stretch, n_str;
  size_t holes, movers, total, hist, n_list, cut, list, bytes;   // offsets into the workspace; kept is at 0
};

EvictPlan evict_plan(uint32_t n_kv, uint32_t seq) {
  EvictPlan p{};
  p.words = seq / 64u + (seq % 64u != 0);
  p.stretch = 64u * p.words;
  p.n_str = 1;
  size_t at = 0;
  auto room = [&](size_t n) {
    const size_t here = at;
    at += (n + 15u) / 16u * 16u;
    return here;
  };
  const size_t n = (size_t)n_kv * p.words;
  room(8 * n);
  p.holes = room(4 * n);
  p.movers = room(4 * n);
  if (seq > kWideFrom) {
    const uint32_t each = (p.words + kStretches - 1) / kStretches * 64u;
    p.stretch = std::max(kBatch, each);
    p.n_str = (seq - 1u) / p.stretch + 1u;
    p.total = room(8ull * n_kv * p.n_str);
    p.hist = room(4ull * n_kv * kWideBins);
    p.n_list = room(4ull * n_kv);
    p.cut = room(16ull * n_kv);
    p.list = room(8ull * n_kv * seq);
  }
  p.bytes = at;
  return p;
}

}  // namespace

size_t kv_evict_workspace(uint32_t n_kv, uint32_t seq) { return evict_plan(n_kv, seq).bytes; }

// Requires 1 <= keep <= seq <= from.max_seq, keep <= to.max_seq, equal n_kv and
// hd, planes of at least seq (from) and keep (to) rows; to either is `from`
// itself or overlaps none of it.  ws holds kv_evict_workspace(n_kv, seq) bytes.
hipError_t launch_kv_evict(const KvQ8Dev& from, const KvQ8Dev& to, const float* weight, const uint32_t* position,
                           uint32_t plane, float* w_to, uint32_t* p_to, uint32_t plane_to, uint32_t seq,
                           uint32_t keep, uint32_t n_first, uint32_t recent_from, void* ws, hipStream_t s) {
  const EvictPlan p = evict_plan(from.n_kv, seq);
  uint8_t* w8 = static_cast<uint8_t*>(ws);
  const EvictArgs e{weight, position, plane, seq, keep, n_first, recent_from, p.words,
                    reinterpret_cast<uint64_t*>(w8), reinterpret_cast<uint32_t*>(w8 + p.holes),
                    reinterpret_cast<uint32_t*>(w8 + p.movers), p.stretch, p.n_str,
                    reinterpret_cast<uint2*>(w8 + p.total), reinterpret_cast<uint32_t*>(w8 + p.hist),
                    reinterpret_cast<uint32_t*>(w8 + p.n_list), reinterpret_cast<uint2*>(w8 + p.list),
                    reinterpret_cast<uint4*>(w8 + p.cut)};
  const dim3 heads(from.n_kv), threads(kSelThreads), wide(p.n_str, from.n_kv), wt(kWideThreads);
  if (p.n_str > 1) {
    hipLaunchKernelGGL(kv_evict_clear_kernel, dim3(kWideBins / kWideThreads, from.n_kv), wt, 0, s, e);
    hipLaunchKernelGGL(kv_evict_count_kernel, wide, wt, 0, s, e);
    hipLaunchKernelGGL(kv_evict_gather_kernel, wide, wt, 0, s, e);
    hipLaunchKernelGGL(kv_evict_cut_kernel, heads, threads, 0, s, e);
    hipLaunchKernelGGL(kv_evict_words_kernel, wide, wt, 0, s, e);
  } else if (seq <= 4u * kSelThreads) {
    hipLaunchKernelGGL(kv_evict_select_kernel<4>, heads, threads, 0, s, e);
  } else if (seq <= 8u * kSelThreads) {
    hipLaunchKernelGGL(kv_evict_select_kernel<8>, heads, threads, 0, s, e);
  } else {
    hipLaunchKernelGGL(kv_evict_select_kernel<16>, heads, threads, 0, s, e);
  }
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  const MoveArgs m{from, to, e, to.k_qs == from.k_qs ? 1u : 0u, w_to, p_to, plane_to};
  const dim3 grid(std::min(512u, (keep - 1u) / kMoveRows / 8u + 1u) * 8u * from.n_kv);
  switch (from.hd) {
    case 32: hipLaunchKernelGGL(kv_move_kernel<32>, grid, dim3(256), 0, s, m); break;
    case 64: hipLaunchKernelGGL(kv_move_kernel<64>, grid, dim3(256), 0, s, m); break;
    case 128: hipLaunchKernelGGL(kv_move_kernel<128>, grid, dim3(256), 0, s, m); break;
    case 256: hipLaunchKernelGGL(kv_move_kernel<256>, grid, dim3(256), 0, s, m); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_kv_keep_path(const KvQ8Dev& c, const uint32_t* path, uint32_t n_nodes, uint32_t pos, hipStream_t s) {
  const uint32_t per = c.n_kv * c.hd, cols = 2u * (per / 16u + per / 32u);
  hipLaunchKernelGGL(kv_keep_path_kernel, dim3((cols + 255u) / 256u), dim3(256), 0, s, c, path, n_nodes, pos);
  return hipGetLastError();
}

}  // namespace vxt
