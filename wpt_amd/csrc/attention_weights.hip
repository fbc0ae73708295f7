// The attention weight that each cached row has received, for gfx950: the
// measure a bounded cache evicts by.
//
// For table row n of batch row b, over the first counts[b] queries t of the
// reading that see it (n <= positions[b, t]) and their H heads,
//   weights[b, n] += sum exp(scale q[b, t, h] . k[b, n] - lse[b, t, h]),
// each term the softmax weight the verify attention gave the row (lse is its
// log-sum-exp, the sink included).  Rows from start[b] on, the reading's own,
// begin at zero: a draft that was taken back leaves nothing behind.  Rows past
// the last counted position are not touched.
//
// No atomics: a wavefront owns its rows and takes the queries in order, so the
// sums do not depend on the launch.
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

constexpr int kKeys = 64;   // table rows of a workgroup of the generic kernel
constexpr int kGT = 256;
constexpr int kMaxWidth = 256;

// The counted queries of batch row b, and the last row they see (-1: none).
__device__ __forceinline__ int counted(const int64_t* counts, int b, int T) {
  if (!counts) return T;
  const int64_t n = counts[b];
  return n < 0 ? 0 : n < T ? (int)n : T;
}

template <typename E, int CMAX>
__global__ __launch_bounds__(kGT) void attention_weights_generic(
    const E* __restrict__ q, const E* __restrict__ k, int64_t ksb, int64_t ksn, const int64_t* __restrict__ positions,
    const float* __restrict__ lse, const int64_t* __restrict__ counts, const int64_t* __restrict__ start, int T, int H,
    int c, int N, float scale, int nkb, float* __restrict__ weights, int64_t wsb) {
  __shared__ float keys[kKeys][CMAX + 1];
  __shared__ float sums[kGT / 64][kKeys];
  const int b = blockIdx.x / nkb, n0 = (blockIdx.x % nkb) * kKeys;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tn = counted(counts, b, T);
  const int64_t* pos = positions + (int64_t)b * T;
  int64_t last = -1;
  for (int t = 0; t < tn; ++t) last = pos[t] > last ? pos[t] : last;
  if (n0 > last) return;  // uniform: no counted query sees these rows
  for (int i = tid; i < kKeys * c; i += kGT) {
    const int key = i / c, e = i % c;
    const int n = n0 + key < N ? n0 + key : N - 1;
    keys[key][e] = load_f32(k + (int64_t)b * ksb + (int64_t)n * ksn + e);
  }
  __syncthreads();
  const int n = n0 + lane;
  float sum = 0.f;
  for (int r = wave; r < tn * H; r += kGT / 64) {
    const int64_t row = (int64_t)b * T * H + r;
    const E* qr = q + row * c;
    float d = 0.f;
    for (int e = 0; e < c; ++e) d = fmaf(load_f32(qr + e), keys[lane][e], d);
    const float w = expf(d * scale - lse[row]);
    if (n <= pos[r / H]) sum += w;
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && n < N && n <= last) {
    float* out = weights + (int64_t)b * wsb + n;
    const float before = start && n >= start[b] ? 0.f : *out;
    sum = 0.f;
    for (int i = 0; i < kGT / 64; ++i) sum += sums[i][lane];
    *out = before + sum;
  }
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_attention_weights_workspace(int B, int T, int H, int c, int N, int dtype, int* splits,
                                                size_t* bytes) {
  if (!splits || !bytes) return fail(WPTV_E_INVALID, "attention_weights_workspace: splits and bytes must be given");
  if (B < 0 || T < 0 || H <= 0 || c <= 0 || N <= 0)
    return fail(WPTV_E_INVALID, "attention_weights: bad shape B=%d T=%d H=%d c=%d N=%d", B, T, H, c, N);
  if (dtype != WPTV_F32 && dtype != WPTV_BF16) return fail(WPTV_E_UNSUPPORTED, "attention_weights: dtype %d", dtype);
  if (c > kMaxWidth)
    return fail(WPTV_E_UNSUPPORTED, "attention_weights: head width at most %d (got %d)", kMaxWidth, c);
  if ((int64_t)T * H > INT32_MAX || (int64_t)B * ((N + kKeys - 1) / kKeys) > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "attention_weights: B=%d T=%d H=%d N=%d is too large", B, T, H, N);
  if (*splits < 0) return fail(WPTV_E_INVALID, "attention_weights: splits = %d", *splits);
  *splits = 1;
  *bytes = 0;
  return WPTV_OK;
}

extern "C" int wptv_attention_weights(const void* q, const void* k, int64_t k_stride_b, int64_t k_stride_n, int dtype,
                                      const int64_t* positions, const float* lse, const int64_t* counts,
                                      const int64_t* start, int B, int T, int H, int c, int N, float scale, int splits,
                                      float* weights, int64_t weights_stride_b, void* workspace,
                                      size_t workspace_bytes, hipStream_t stream) {
  size_t need = 0;
  const int status = wptv_attention_weights_workspace(B, T, H, c, N, dtype, &splits, &need);
  if (status != WPTV_OK) return status;
  if (B == 0 || T == 0) return WPTV_OK;
  if (!q || !k || !positions || !lse || !weights)
    return fail(WPTV_E_INVALID, "attention_weights: a required pointer is NULL");
  if (k_stride_n < c || (B > 1 && weights_stride_b < N))
    return fail(WPTV_E_INVALID, "attention_weights: rows overlap (k row stride %lld, weights stride %lld)",
                (long long)k_stride_n, (long long)weights_stride_b);
  if (workspace_bytes < need || (need && !workspace))
    return fail(WPTV_E_INVALID, "attention_weights: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const int nkb = (N + kKeys - 1) / kKeys;
#define WPTV_WEIGHTS(E, CMAX)                                                                                        \
  attention_weights_generic<E, CMAX><<<B * nkb, kGT, 0, stream>>>(                                                   \
      static_cast<const E*>(q), static_cast<const E*>(k), k_stride_b, k_stride_n, positions, lse, counts, start, T, H, \
      c, N, scale, nkb, weights, weights_stride_b)
  if (dtype == WPTV_BF16) {
    if (c <= 128) WPTV_WEIGHTS(unsigned short, 128); else WPTV_WEIGHTS(unsigned short, 256);
  } else {
    if (c <= 128) WPTV_WEIGHTS(float, 128); else WPTV_WEIGHTS(float, 256);
  }
#undef WPTV_WEIGHTS
  return launched("attention_weights");
}
