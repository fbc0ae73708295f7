// The rows that a bounded cache keeps, for gfx950, chosen by the attention
// weight they have received (wptv_attention_weights).
//
// Of a batch row's first lengths[b] rows, all when they are at most `keep`;
// else the first `first`, the last `recent`, and of the others the
// keep - first - recent of the largest weight, equal weights the lowest rows
// first (a NaN counts as the largest weight, -0 as 0), listed in row order.
// One workgroup a (layer, batch row):
//   choose_kept_regs  up to 16384 rows: the weights' keys in registers, the
//                     smallest one kept by kth_largest, the rows listed after
//                     one scan of the threads' counts
//   choose_kept_long  longer texts: the same over the weights in memory, each
//                     wavefront listing a stretch of the rows by ballots
// A serial chain of barriers bounds them, not the bytes: 24 layers of 16 texts of up
// to 4096 rows 13.6 us, one text of each 9.5, of 40000 rows 42; 4 of 320 rows 5.2.
#include "select_common.h"
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

__device__ __forceinline__ uint32_t weight_key(float f) { return f != f ? ~0u : order_key(f + 0.f); }

// Thread t holds the keys of 4 nv consecutive rows, nv = ceil(candidates / 4
// THREADS) <= V, so that the kept rows are counted and listed in row order.
template <int THREADS, int V>
__global__ __launch_bounds__(THREADS) void choose_kept_regs(const float* __restrict__ weights, int64_t wsl,
                                                            int64_t wsb, int B, int N,
                                                            const int64_t* __restrict__ lengths, int keep, int first,
                                                            int recent, int64_t* __restrict__ kept,
                                                            int64_t* __restrict__ counts) {
  constexpr int kWaves = THREADS / 64;
  static_assert(4 * V * THREADS < 65536, "packed counts hold 16 bits");
  __shared__ SelectShared<THREADS> select;
  __shared__ int waves[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int layer = blockIdx.x / B, b = blockIdx.x % B;
  const int64_t len64 = lengths[b];
  const int len = len64 < 0 ? 0 : len64 < N ? (int)len64 : N;
  int64_t* out = kept + (int64_t)blockIdx.x * keep;
  if (layer == 0 && tid == 0) counts[b] = len < keep ? len : keep;
  if (len <= keep) {
    for (int i = tid; i < keep; i += THREADS) out[i] = i < len ? i : -1;
    return;
  }
  const int take = keep - first - recent, candidates = len - first - recent;  // take < candidates
  for (int i = tid; i < first; i += THREADS) out[i] = i;
  for (int i = tid; i < recent; i += THREADS) out[keep - recent + i] = len - recent + i;
  if (take == 0) return;
  const float* s = weights + layer * wsl + b * wsb + first;
  const int nv = (candidates + 4 * THREADS - 1) / (4 * THREADS);
  const int base = tid * 4 * nv, valid = candidates - base;
  uint32_t key[4 * V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (v >= nv) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) key[4 * v + e] = 4 * v + e < valid ? weight_key(s[base + 4 * v + e]) : 0u;
  }
  auto each = [&](auto&& f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (v >= nv) break;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * v + e < valid) f(4 * v + e, key[4 * v + e]);
    }
  };
  const uint32_t tau = kth_largest<THREADS, (THREADS > 256)>(each, take, select);  // few keys a bin of a short text
  // rows above tau, and the first of those equal to it: one scan of both counts
  int mine = 0;
  each([&](int, uint32_t x) { mine += x > tau ? 1 : x == tau ? 65536 : 0; });
  const int upto = wave_scan_i32(mine);
  if (lane == 63) waves[w] = upto;
  __syncthreads();
  int before = upto - mine, above = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) before += waves[i];
    above += waves[i] & 65535;
  }
  const int equal = take - above;  // rows equal to tau that are kept
  int gt = before & 65535, eq = before >> 16;
  each([&](int i, uint32_t x) {
    if (x > tau || (x == tau && eq < equal)) out[first + gt + min(eq, equal)] = first + base + i;
    gt += x > tau ? 1 : 0;
    eq += x == tau ? 1 : 0;
  });
}

constexpr int kLongThreads = 1024, kLongWaves = kLongThreads / 64;
constexpr int kLongLoads = 8;  // rows a thread asks for at once

__global__ __launch_bounds__(kLongThreads) void choose_kept_long(const float* __restrict__ weights, int64_t wsl,
                                                                 int64_t wsb, int B, int N,
                                                                 const int64_t* __restrict__ lengths, int keep,
                                                                 int first, int recent, int64_t* __restrict__ kept,
                                                                 int64_t* __restrict__ counts) {
  __shared__ SelectShared<kLongThreads> select;
  __shared__ int above[kLongWaves], equals[kLongWaves];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int layer = blockIdx.x / B, b = blockIdx.x % B;
  const int64_t len64 = lengths[b];
  const int len = len64 < 0 ? 0 : len64 < N ? (int)len64 : N;
  int64_t* out = kept + (int64_t)blockIdx.x * keep;
  if (layer == 0 && tid == 0) counts[b] = len < keep ? len : keep;
  if (len <= keep) {
    for (int i = tid; i < keep; i += kLongThreads) out[i] = i < len ? i : -1;
    return;
  }
  const int take = keep - first - recent, candidates = len - first - recent;  // take < candidates
  for (int i = tid; i < first; i += kLongThreads) out[i] = i;
  for (int i = tid; i < recent; i += kLongThreads) out[keep - recent + i] = len - recent + i;
  if (take == 0) return;
  const float* s = weights + layer * wsl + b * wsb + first;
  // f(row, key) of rows begin + step i, several asked for at once
  auto rows = [&](int begin, int end, int step, auto&& f) {
    for (int n = begin; n < end; n += kLongLoads * step) {
      float x[kLongLoads];
#pragma unroll
      for (int i = 0; i < kLongLoads; ++i) x[i] = n + i * step < end ? s[n + i * step] : 0.f;
#pragma unroll
      for (int i = 0; i < kLongLoads; ++i)
        if (n + i * step < end) f(n + i * step, weight_key(x[i]));
    }
  };
  auto each = [&](auto&& f) { rows(tid, candidates, kLongThreads, f); };
  const uint32_t tau = kth_largest<kLongThreads, true>(each, take, select);
  // each wavefront counts, then lists, a stretch of consecutive rows
  const int stretch = ((candidates + kLongWaves - 1) / kLongWaves + 63) / 64 * 64;
  const int begin = min(w * stretch, candidates), end = min(begin + stretch, candidates);
  int gt = 0, eq = 0;
  rows(begin + lane, end, 64, [&](int, uint32_t x) {
    gt += x > tau ? 1 : 0;
    eq += x == tau ? 1 : 0;
  });
  gt = (int)wave_sum_u32(gt);
  eq = (int)wave_sum_u32(eq);
  if (lane == 0) {
    above[w] = gt;
    equals[w] = eq;
  }
  __syncthreads();
  int all = 0;
  gt = eq = 0;
  for (int i = 0; i < kLongWaves; ++i) {
    all += above[i];
    if (i < w) {
      gt += above[i];
      eq += equals[i];
    }
  }
  const int equal = take - all;  // rows equal to tau that are kept, the first ones
  const uint64_t below = (1ull << lane) - 1ull;
  for (int n0 = begin; n0 < end; n0 += kLongLoads * 64) {
    float x[kLongLoads];
#pragma unroll
    for (int i = 0; i < kLongLoads; ++i) x[i] = n0 + 64 * i + lane < end ? s[n0 + 64 * i + lane] : 0.f;
#pragma unroll
    for (int i = 0; i < kLongLoads; ++i) {
      const int n = n0 + 64 * i + lane;
      const uint32_t u = weight_key(x[i]);
      const uint64_t more = __builtin_amdgcn_ballot_w64(n < end && u > tau);
      const uint64_t same = __builtin_amdgcn_ballot_w64(n < end && u == tau);
      const int e = eq + __builtin_popcountll(same & below);
      if (n < end && (u > tau || (u == tau && e < equal)))
        out[first + gt + __builtin_popcountll(more & below) + min(e, equal)] = first + n;
      gt += __builtin_popcountll(more);
      eq += __builtin_popcountll(same);
    }
  }
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_choose_kept(const float* weights, int64_t weights_stride_l, int64_t weights_stride_b,
                                const int64_t* lengths, int L, int B, int N, int keep, int first, int recent,
                                int64_t* kept, int64_t* counts, hipStream_t stream) {
  if (L <= 0 || B < 0 || N < 0) return fail(WPTV_E_INVALID, "choose_kept: bad shape L=%d B=%d N=%d", L, B, N);
  if (first < 0 || recent < 0 || keep <= 0 || (int64_t)first + recent > keep)
    return fail(WPTV_E_INVALID, "choose_kept: keep=%d rows must hold the first %d and the last %d", keep, first, recent);
  if ((int64_t)L * B > INT32_MAX || N > (1 << 30))
    return fail(WPTV_E_UNSUPPORTED, "choose_kept: L=%d B=%d N=%d is too large", L, B, N);
  if (B == 0) return WPTV_OK;
  if ((N && !weights) || !lengths || !kept || !counts)
    return fail(WPTV_E_INVALID, "choose_kept: a required pointer is NULL");
#define WPTV_KEPT(THREADS, V)                                                                                    \
  choose_kept_regs<THREADS, V><<<L * B, THREADS, 0, stream>>>(weights, weights_stride_l, weights_stride_b, B, N, \
                                                              lengths, keep, first, recent, kept, counts)
  if (N <= 1024)
    WPTV_KEPT(256, 1);
  else if (N <= 4096)
    WPTV_KEPT(512, 2);
  else if (N <= 16384)
    WPTV_KEPT(1024, 4);
  else
    choose_kept_long<<<L * B, kLongThreads, 0, stream>>>(weights, weights_stride_l, weights_stride_b, B, N, lengths,
                                                         keep, first, recent, kept, counts);
#undef WPTV_KEPT
  return launched("choose_kept");
}
