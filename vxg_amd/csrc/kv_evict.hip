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
  uint32_t plane, seq, keep, n_first, recent_from;
  uint32_t* src;              // [n_kv][keep]: the row that goes to row r
  uint32_t* hole;             // [n_kv][keep]
  uint32_t* mover;            // [n_kv][keep]
};

constexpr uint32_t kSelThreads = 1024, kSelWaves = kSelThreads / 64, kBins = 2048;

// Workgroup (kv head).  Each wave has a stretch of the rows, lane l of step j
// row i0 + 64 j + l, so ranks in row order come from ballots.  With STEPS > 0 a
// lane keeps its keys in registers (STEPS of them, the rows read once);
// STEPS 0 reads them again in every pass, for any number of rows.
//
// The keep-th largest key: the protected rows are counted, then the range of
// the others' keys is narrowed by counts over 2048 equal bins of it -- the
// counts spread over the bins whatever the weights' magnitudes, where bins of
// the leading bits would pile up in a few exponents and the LDS adds of a wave
// run one after the other.  At most three rounds, for 32 bits.
template <int STEPS>
__global__ __launch_bounds__(kSelThreads) void kv_evict_select_kernel(EvictArgs a) {
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_w[3][kSelWaves];
  __shared__ uint32_t s_out[3];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t kvh = blockIdx.x;
  const float* w = a.weight + (size_t)kvh * a.plane;
  const uint32_t* pos = a.position + (size_t)kvh * a.plane;
  const uint32_t per_w = ((a.seq + kSelWaves - 1u) / kSelWaves + 63u) & ~63u;
  const uint32_t i0 = min(a.seq, wave * per_w), i1 = min(a.seq, i0 + per_w);
  const uint32_t steps = STEPS > 0 ? STEPS : (per_w + 63u) / 64u;
  auto load = [&](uint32_t j) {   // of a row past the stretch: never counted, see `in`
    const uint32_t i = min(i0 + 64u * j + lane, a.seq - 1u), p = pos[i];
    const float x = w[i];
    return p < a.n_first || p >= a.recent_from ? kKeep : rank_key(x);
  };
  uint32_t kept_keys[STEPS > 0 ? STEPS : 1];
  if constexpr (STEPS > 0) {
#pragma unroll
    for (uint32_t j = 0; j < (uint32_t)STEPS; ++j) {
      kept_keys[j] = load(j);
      if (j % 16u == 15u) __builtin_amdgcn_sched_barrier(0);   // no more than 32 loads in flight: their registers
    }
  }
  auto each = [&](auto f) {
    if constexpr (STEPS > 0) {
      uint32_t row0 = i0 + lane;
      asm volatile("" : "+v"(row0));   // the rows anew in each pass, not in registers across them
#pragma unroll
      for (uint32_t j = 0; j < (uint32_t)STEPS; ++j) {
        f(kept_keys[j], row0 + 64u * j);
        if (STEPS > 16 && j % 4u == 3u) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      for (uint32_t j = 0; j < steps; ++j) f(load(j), i0 + 64u * j + lane);
    }
  };

  // protected rows, and the range of the others' keys
  uint32_t lo = 0xffffffffu, hi = 0, n_safe = 0;
  each([&](uint32_t k, uint32_t row) {
    const bool in = row < i1, safe = in && k == kKeep;
    n_safe += safe ? 1u : 0u;
    lo = in && !safe ? min(lo, k) : lo;
    hi = in && !safe ? max(hi, k) : hi;
  });
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    n_safe += (uint32_t)__shfl_xor((int)n_safe, s, 64);
    lo = min(lo, (uint32_t)__shfl_xor((int)lo, s, 64));
    hi = max(hi, (uint32_t)__shfl_xor((int)hi, s, 64));
  }
  if (lane == 0) {
    s_w[0][wave] = n_safe;
    s_w[1][wave] = lo;
    s_w[2][wave] = hi;
  }
  __syncthreads();
  n_safe = 0;
#pragma unroll
  for (uint32_t v = 0; v < kSelWaves; ++v) {
    n_safe += s_w[0][v];
    lo = min(lo, s_w[1][v]);
    hi = max(hi, s_w[2][v]);
  }
  // kept: key > above, or key == at and among the first `need` of those
  uint32_t at = kKeep, need = a.keep;
  if (n_safe < a.keep) {
    need = a.keep - n_safe;
    for (;;) {
      const uint32_t width = hi - lo;
      const uint32_t shift = width >= kBins ? 21u - (uint32_t)__clz((int)width) : 0u;   // width >> shift < 2048
      __syncthreads();
      for (uint32_t i = tid; i < kBins; i += kSelThreads) s_hist[i] = 0u;
      __syncthreads();
      each([&](uint32_t k, uint32_t row) {
        if (row < i1 && k - lo <= width) atomicAdd(&s_hist[(k - lo) >> shift], 1u);   // kKeep lies above every range
      });
      __syncthreads();
      // thread t counts bins 2 t and 2 t + 1; `above`: what lies in higher bins
      const uint32_t c0 = s_hist[2u * tid], c1 = s_hist[2u * tid + 1u];
      uint32_t above = c0 + c1;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_down((int)above, d, 64);
        if (lane + d < 64u) above += o;
      }
      if (lane == 0) s_w[0][wave] = above;
      above -= c0 + c1;
      __syncthreads();
#pragma unroll
      for (uint32_t v = 0; v < kSelWaves; ++v) above += v > wave ? s_w[0][v] : 0u;
      if (above < need && need <= above + c1) {
        s_out[0] = 2u * tid + 1u;
        s_out[1] = need - above;
        s_out[2] = c1;
      } else if (above + c1 < need && need <= above + c1 + c0) {
        s_out[0] = 2u * tid;
        s_out[1] = need - above - c1;
        s_out[2] = c0;
      }
      __syncthreads();
      lo += s_out[0] << shift;
      need = s_out[1];
      at = lo;
      if (shift == 0) break;
      const uint32_t top = lo + ((1u << shift) - 1u);
      hi = min(hi, top);
    }
  }

  // per wave: equal keys, larger ones, and those of them below row `keep`
  uint32_t eq = 0, eq_lo = 0, gt_lo = 0, gt_hi = 0;
  each([&](uint32_t k, uint32_t row) {
    const bool in = row < i1;
    const uint64_t me = __builtin_amdgcn_ballot_w64(in && k == at), mg = __builtin_amdgcn_ballot_w64(in && k > at);
    const uint64_t ml = __builtin_amdgcn_ballot_w64(row < a.keep);
    eq += (uint32_t)__popcll(me);
    eq_lo += (uint32_t)__popcll(me & ml);
    gt_lo += (uint32_t)__popcll(mg & ml);
    gt_hi += (uint32_t)__popcll(mg & ~ml);
  });
  __syncthreads();   // s_w and s_out are free again
  const uint32_t eq0 = wave_prefix<kSelWaves>(eq, s_w[0], wave, lane);
  const uint32_t take = min(eq, need > eq0 ? need - eq0 : 0u), take_lo = min(take, eq_lo);   // in row order
  const uint32_t rows_lo = min(i1, a.keep) - min(i0, a.keep);
  const uint32_t holes = rows_lo - gt_lo - take_lo, movers = gt_hi + take - take_lo;
  uint32_t h = wave_prefix<kSelWaves>(holes, s_w[0], wave, lane);
  uint32_t m = wave_prefix<kSelWaves>(movers, s_w[0], wave, lane);
  if (wave == kSelWaves - 1u && lane == 0) s_out[0] = h + holes;   // as many as movers

  uint32_t* src = a.src + (size_t)kvh * a.keep;
  uint32_t* hole = a.hole + (size_t)kvh * a.keep;
  uint32_t* mover = a.mover + (size_t)kvh * a.keep;
  uint32_t e = eq0;
  each([&](uint32_t k, uint32_t row) {
    const bool in = row < i1;
    const uint64_t me = __builtin_amdgcn_ballot_w64(in && k == at);
    const bool kept = in && (k > at || (k == at && e + ones_below(me, lane) < need));
    const bool is_hole = in && !kept && row < a.keep, moves = kept && row >= a.keep;
    const uint64_t mh = __builtin_amdgcn_ballot_w64(is_hole), mm = __builtin_amdgcn_ballot_w64(moves);
    if (is_hole) hole[h + ones_below(mh, lane)] = row;
    else if (moves) mover[m + ones_below(mm, lane)] = row;
    else if (kept) src[row] = row;
    e += (uint32_t)__popcll(me);
    h += (uint32_t)__popcll(mh);
    m += (uint32_t)__popcll(mm);
  });
  __syncthreads();   // the lists are complete, and visible within the workgroup
  const uint32_t n = s_out[0];
  for (uint32_t i = tid; i < n; i += kSelThreads) src[hole[i]] = mover[i];
}

struct MoveArgs {
  KvQ8Dev from, to;
  const uint32_t* src;
  uint32_t keep, in_place;
  const float* w_from;
  const uint32_t* p_from;
  float* w_to;
  uint32_t* p_to;
  uint32_t plane_from, plane_to;
};

// Row r of kv head k from row src[k][r]: HD / 8 lanes to a row and head, each a
// 16-byte piece of K or V; the scales, the weight and the position by some of
// them.  Four rows of a lane in flight.
template <int HD>
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs a) {
  constexpr uint32_t L = HD / 8, NB = HD / 32, U = 4;
  const uint32_t n_kv = a.from.n_kv, sub = threadIdx.x % L;
  const uint32_t row_q = n_kv * HD, row_d = n_kv * NB;
  const uint64_t n = (uint64_t)a.keep * n_kv, step = (uint64_t)gridDim.x * (256u / L);
  const uint64_t first = (uint64_t)blockIdx.x * (256u / L) + threadIdx.x / L;
  const bool is_v = sub >= L / 2u;
  const int8_t* fq = is_v ? a.from.v_qs : a.from.k_qs;
  int8_t* tq = is_v ? a.to.v_qs : a.to.k_qs;
  const uint32_t qo = 16u * (sub % (L / 2u));
  const bool has_d = sub < 2u * NB, d_v = sub >= NB;
  const uint16_t* fd = d_v ? a.from.v_d : a.from.k_d;
  uint16_t* td = d_v ? a.to.v_d : a.to.k_d;
  for (uint64_t i0 = first; i0 < n; i0 += U * step) {
    uint32_t r[U], k[U], s[U];
    bool live[U];
    u32x4 x[U];
    uint32_t y[U], z[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint64_t i = i0 + u * step;
      live[u] = i < n;
      const uint64_t ic = live[u] ? i : n - 1u;
      r[u] = (uint32_t)(ic / n_kv);
      k[u] = (uint32_t)(ic % n_kv);
      s[u] = a.src[(size_t)k[u] * a.keep + r[u]];
      if (a.in_place && s[u] == r[u]) live[u] = false;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (!live[u]) continue;
      x[u] = *reinterpret_cast<const u32x4*>(fq + (size_t)s[u] * row_q + k[u] * HD + qo);
      if (has_d) y[u] = fd[(size_t)s[u] * row_d + k[u] * NB + sub % NB];
      if (sub == L - 1u) z[u] = a.p_from[(size_t)k[u] * a.plane_from + s[u]];
      if (sub == L - 2u) z[u] = __float_as_uint(a.w_from[(size_t)k[u] * a.plane_from + s[u]]);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (!live[u]) continue;
      *reinterpret_cast<u32x4*>(tq + (size_t)r[u] * row_q + k[u] * HD + qo) = x[u];
      if (has_d) td[(size_t)r[u] * row_d + k[u] * NB + sub % NB] = (uint16_t)y[u];
      if (sub == L - 1u) a.p_to[(size_t)k[u] * a.plane_to + r[u]] = z[u];
      if (sub == L - 2u) a.w_to[(size_t)k[u] * a.plane_to + r[u]] = __uint_as_float(z[u]);
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

size_t kv_evict_workspace(uint32_t n_kv, uint32_t keep) { return (size_t)n_kv * keep * 12u; }

// Requires 1 <= keep <= seq <= from.max_seq, keep <= to.max_seq, equal n_kv and
// hd, planes of at least seq (from) and keep (to) rows; to either is `from`
// itself or overlaps none of it.
hipError_t launch_kv_evict(const KvQ8Dev& from, const KvQ8Dev& to, const float* weight, const uint32_t* position,
                           uint32_t plane, float* w_to, uint32_t* p_to, uint32_t plane_to, uint32_t seq,
                           uint32_t keep, uint32_t n_first, uint32_t recent_from, void* ws, hipStream_t s) {
  uint32_t* src = static_cast<uint32_t*>(ws);
  const size_t n = (size_t)from.n_kv * keep;
  const EvictArgs e{weight, position, plane, seq, keep, n_first, recent_from, src, src + n, src + 2 * n};
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
  const MoveArgs m{from, to, src, keep, to.k_qs == from.k_qs ? 1u : 0u, weight, position, w_to, p_to, plane, plane_to};
  const uint32_t per_wg = 256u / (from.hd / 8u);
  const dim3 grid((uint32_t)std::min<size_t>(2048, (n + 4 * per_wg - 1) / (4 * per_wg)));
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
