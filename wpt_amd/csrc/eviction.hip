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
//   choose_kept       longer texts: a radix select over the weights in memory,
//                     most significant byte first, then one pass that lists the
//                     kept rows by wavefront ballots
#include "select_common.h"
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

constexpr int kST = 256;

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
  const uint32_t tau = kth_largest<THREADS>(each, take, select);
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

__global__ __launch_bounds__(kST) void choose_kept(const float* __restrict__ weights, int64_t wsl, int64_t wsb, int B,
                                                   int N, const int64_t* __restrict__ lengths, int keep, int first,
                                                   int recent, int64_t* __restrict__ kept,
                                                   int64_t* __restrict__ counts) {
  __shared__ int hist[256];
  __shared__ int sel[2];
  __shared__ int wcount[2][kST / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int layer = blockIdx.x / B, b = blockIdx.x % B;
  int64_t len64 = lengths[b];
  const int len = len64 < 0 ? 0 : len64 < N ? (int)len64 : N;
  int64_t* out = kept + (int64_t)blockIdx.x * keep;
  if (layer == 0 && tid == 0) counts[b] = len < keep ? len : keep;
  if (len <= keep) {
    for (int i = tid; i < keep; i += kST) out[i] = i < len ? i : -1;
    return;
  }
  const float* s = weights + layer * wsl + b * wsb;
  const int end = len - recent;          // candidates: rows first .. end - 1
  const int take = keep - first - recent;  // fewer than the candidates
  uint32_t tau = ~0u;
  int need_eq = 0;
  if (take > 0) {
    uint32_t prefix = 0, mask = 0;
    int remaining = take;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      hist[tid] = 0;
      __syncthreads();
      for (int n = first + tid; n < end; n += kST) {
        const uint32_t u = weight_key(s[n]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int above = 0, digit = 255;
        while (above + hist[digit] < remaining) above += hist[digit--];
        sel[0] = digit;
        sel[1] = remaining - above;
      }
      __syncthreads();
      prefix |= (uint32_t)sel[0] << shift;
      mask |= 255u << shift;
      remaining = sel[1];
    }
    tau = prefix;
    need_eq = remaining;
  }
  // one pass in row order: rows equal to the smallest kept weight are counted
  // so that the first need_eq of them are kept
  const uint64_t below = (1ull << lane) - 1ull;
  int base = 0, base_eq = 0;
  for (int start = 0; start < len; start += kST) {
    const int n = start + tid;
    const bool candidate = n >= first && n < end;
    const uint32_t u = candidate ? weight_key(s[n]) : 0u;
    const bool eq = candidate && take > 0 && u == tau;
    const uint64_t be = __builtin_amdgcn_ballot_w64(eq);
    if (lane == 0) wcount[0][w] = __builtin_popcountll(be);
    __syncthreads();
    int pe = base_eq;
    for (int i = 0; i < w; ++i) pe += wcount[0][i];
    pe += __builtin_popcountll(be & below);
    const bool in = n < len && (!candidate || (take > 0 && (u > tau || (eq && pe < need_eq))));
    const uint64_t bi = __builtin_amdgcn_ballot_w64(in);
    if (lane == 0) wcount[1][w] = __builtin_popcountll(bi);
    __syncthreads();
    int p = base;
    for (int i = 0; i < w; ++i) p += wcount[1][i];
    p += __builtin_popcountll(bi & below);
    if (in) out[p] = n;
    for (int i = 0; i < kST / 64; ++i) {
      base_eq += wcount[0][i];
      base += wcount[1][i];
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_choose_kept(const float* weights, int64_t weights_stride_l, int64_t weights_stride_b,
                                const int64_t* lengths, int L, int B, int N, int keep, int first, int recent,
                                int64_t* kept, int64_t* counts, hipStream_t stream) {
  if (L < 0 || B < 0 || N < 0) return fail(WPTV_E_INVALID, "choose_kept: bad shape L=%d B=%d N=%d", L, B, N);
  if (first < 0 || recent < 0 || keep <= 0 || (int64_t)first + recent > keep)
    return fail(WPTV_E_INVALID, "choose_kept: keep=%d rows must hold the first %d and the last %d", keep, first, recent);
  if ((int64_t)L * B > INT32_MAX) return fail(WPTV_E_UNSUPPORTED, "choose_kept: L=%d B=%d is too large", L, B);
  if (L == 0 || B == 0) return WPTV_OK;
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
    choose_kept<<<L * B, kST, 0, stream>>>(weights, weights_stride_l, weights_stride_b, B, N, lengths, keep, first,
                                           recent, kept, counts);
#undef WPTV_KEPT
  return launched("choose_kept");
}
