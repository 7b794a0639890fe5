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
  uint32_t* holes;            // [n_kv][words]
  uint32_t* movers;           // [n_kv][words]
};

constexpr uint32_t kSelThreads = 1024, kSelWaves = kSelThreads / 64, kBins = 512, kList = 4096;

// Workgroup (kv head).  Each wave has a stretch of the rows, lane l of step j
// row i0 + 64 j + l, so a ballot is a word of `kept` and ranks are in row order.
// With STEPS > 0 a lane keeps its keys in registers (STEPS of them, the rows
// read once); STEPS 0 reads them again in every pass, for any number of rows.
//
// The keep-th largest key: the protected rows are counted, then the range of
// the others' keys is narrowed by counts over 512 equal bins of it -- the
// counts spread over the bins whatever the weights' magnitudes, where bins of
// the leading bits would pile up in a few exponents and the LDS adds of a wave
// run one after the other.  Once the range holds no more than kList keys they
// are gathered in LDS, and the further rounds (at most four in all, for 32
// bits) go over those.
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
  auto load = [&](uint32_t j) {   // of a row past the stretch: never counted, see `in`
    const uint32_t i = min(i0 + 64u * j + lane, a.seq - 1u), p = pos[i];
    const float x = w[i];
    return p < a.n_first || p >= a.recent_from ? kKeep : rank_key(x);
  };
  uint32_t keys[STEPS > 0 ? STEPS : 1];
  if constexpr (STEPS > 0) {
#pragma unroll
    for (uint32_t j = 0; j < (uint32_t)STEPS; ++j) {
      keys[j] = load(j);
      if (j % 16u == 15u) __builtin_amdgcn_sched_barrier(0);   // no more than 32 loads in flight: their registers
    }
  }
  auto each = [&](auto f) {
    if constexpr (STEPS > 0) {
      uint32_t row0 = i0 + lane;
      asm volatile("" : "+v"(row0));   // the rows anew in each pass, not in registers across them
#pragma unroll
      for (uint32_t j = 0; j < (uint32_t)STEPS; ++j) {
        f(keys[j], row0 + 64u * j, j);
        if (STEPS > 16 && j % 4u == 3u) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      for (uint32_t j = 0; j < steps; ++j) f(load(j), i0 + 64u * j + lane, j);
    }
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
    bool listed = false;
    for (int round = 0; round < 4; ++round) {
      const uint32_t width = hi - lo;
      const uint32_t shift = width >= kBins ? 23u - (uint32_t)__clz((int)width) : 0u;   // width >> shift < 512
      auto count = [&](uint32_t k) {   // kKeep lies above every range
        const uint32_t b = (k - lo) >> shift;
        if (k - lo <= width) atomicAdd(&s_hist[round][(b & 7u) * 64u + (b >> 3)], 1u);
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
      find_bin<8>(c, need, bin, need, n_eq);
      lo += bin << shift;
      hi = min(hi, lo + ((1u << shift) - 1u));
      at = lo;
      if (shift == 0) break;
      if (need == n_eq && lo != 0) break;   // the whole bin stays
      if (!listed && n_eq <= kList) {       // uniform
        each([&](uint32_t k, uint32_t row, uint32_t) {
          if (row < i1 && k - lo <= hi - lo) s_list[atomicAdd(&s_n, 1u)] = k;
        });
        listed = true;
        __syncthreads();
      }
    }
    if (need == n_eq && lo != 0) {   // every key from lo on: no ranks needed
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

// Rows r of one kv head, HD / 8 lanes to a row, each a 16-byte piece of K or V;
// the scales, the weight and the position by some of them.  A kept row is its
// own source, a free one's is the mover of its rank among the free ones: found
// by bisection of the movers' counts, of which every 2^s-th word's lie in LDS.
constexpr uint32_t kCoarse = 1024;
template <int HD>
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs a) {
  constexpr uint32_t L = HD / 8, NB = HD / 32, U = 4, R = 256 / L;
  __shared__ uint32_t s_mov[kCoarse];
  const uint32_t n_kv = a.from.n_kv, sub = threadIdx.x % L, k = blockIdx.y, keep = a.e.keep, words = a.e.words;
  const uint32_t row_q = n_kv * HD, row_d = n_kv * NB;
  const uint64_t* kept = a.e.kept + (size_t)k * words;
  const uint32_t* holes = a.e.holes + (size_t)k * words;
  const uint32_t* movers = a.e.movers + (size_t)k * words;
  uint32_t shift = 0;
  while ((words - 1u) >> shift >= kCoarse) ++shift;
  const uint32_t coarse = ((words - 1u) >> shift) + 1u;
  for (uint32_t i = threadIdx.x; i < coarse; i += 256u) s_mov[i] = movers[(size_t)i << shift];
  __syncthreads();
  auto source = [&](uint32_t r) -> uint32_t {
    const uint64_t m = kept[r / 64u];
    if (m >> (r & 63u) & 1ull) return r;
    const uint32_t rank = holes[r / 64u] + ones_below(~m, r & 63u);
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
      if (movers[mid] <= rank) lo = mid;
      else hi = mid;
    }
    uint64_t x = kept[lo];
    if (lo * 64u < keep) x &= keep - lo * 64u >= 64u ? 0ull : ~0ull << (keep - lo * 64u);
    return lo * 64u + nth_bit(x, rank - movers[lo]);
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
  for (uint32_t r0 = blockIdx.x * R * U + threadIdx.x / L; r0 < keep; r0 += gridDim.x * R * U) {
    uint32_t s[U];
    bool live[U];
    u32x4 x[U];
    uint16_t y[U];
    uint32_t z[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * R;
      live[u] = r < keep;
      s[u] = live[u] ? source(r) : 0u;
      if (a.in_place && s[u] == r) live[u] = false;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (!live[u]) continue;
      x[u] = *reinterpret_cast<const u32x4*>(fq + (size_t)s[u] * row_q);
      if (has_d) y[u] = fd[(size_t)s[u] * row_d];
      if (has_w) z[u] = wf[s[u]];
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * R;
      if (!live[u]) continue;
      *reinterpret_cast<u32x4*>(tq + (size_t)r * row_q) = x[u];
      if (has_d) td[(size_t)r * row_d] = y[u];
      if (has_w) wt[r] = z[u];
    }
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

size_t kv_evict_workspace(uint32_t n_kv, uint32_t seq) { return (size_t)n_kv * ((seq + 63u) / 64u) * 16u; }

// Requires 1 <= keep <= seq <= from.max_seq, keep <= to.max_seq, equal n_kv and
// hd, planes of at least seq (from) and keep (to) rows; to either is `from`
// itself or overlaps none of it.  ws holds kv_evict_workspace(n_kv, seq) bytes.
hipError_t launch_kv_evict(const KvQ8Dev& from, const KvQ8Dev& to, const float* weight, const uint32_t* position,
                           uint32_t plane, float* w_to, uint32_t* p_to, uint32_t plane_to, uint32_t seq,
                           uint32_t keep, uint32_t n_first, uint32_t recent_from, void* ws, hipStream_t s) {
  const uint32_t words = (seq + 63u) / 64u;
  const size_t n = (size_t)from.n_kv * words;
  uint64_t* kept = static_cast<uint64_t*>(ws);
  uint32_t* holes = reinterpret_cast<uint32_t*>(kept + n);
  const EvictArgs e{weight, position, plane, seq, keep, n_first, recent_from, words, kept, holes, holes + n};
  const dim3 heads(from.n_kv), threads(kSelThreads);
  if (seq <= 4u * kSelThreads)
    hipLaunchKernelGGL(kv_evict_select_kernel<4>, heads, threads, 0, s, e);
  else if (seq <= 16u * kSelThreads)
    hipLaunchKernelGGL(kv_evict_select_kernel<16>, heads, threads, 0, s, e);
  else if (seq <= 64u * kSelThreads)
    hipLaunchKernelGGL(kv_evict_select_kernel<64>, heads, threads, 0, s, e);
  else
    hipLaunchKernelGGL(kv_evict_select_kernel<0>, heads, threads, 0, s, e);
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  const MoveArgs m{from, to, e, to.k_qs == from.k_qs ? 1u : 0u, w_to, p_to, plane_to};
  const uint32_t per_wg = 4u * 256u / (from.hd / 8u);
  const dim3 grid(std::min(2048u, (keep + per_wg - 1) / per_wg), from.n_kv);
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
