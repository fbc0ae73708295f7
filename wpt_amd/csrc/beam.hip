// Beam search's selection for gfx950: the next beams of every text over its
// beams and the vocabulary.
//
// A text's candidates are its W beams continued by each of V tokens, of value
//   total[w] + (x[w, v] - L[w]),  L[w] = log sum_v exp x[w, v]
// in 64 bits; the K largest are the next beams, equal values to the lowest
// w V + v.  The scores need not be normalised nor sorted as a whole: within a
// beam the value grows with x, so a beam's candidates are its K largest
// scores, and the next beams are among the W lists of K.  Two launches:
//   beam_rows   one workgroup a (text, beam): L and the K largest scores, ties
//               to the lowest token (keys of the score's order and the token)
//   beam_merge  one wavefront a text: a lane a beam, K times the best head of
//               the W lists
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

constexpr int kMaxBeams = 64;  // beams of a text: a lane each
constexpr int kMaxStops = 16;
constexpr int kRowThreads = 256;
constexpr float kNegInf = -__builtin_inff();

struct Stops {
  int n;
  int token[kMaxStops];
};

// A score's place among a beam's: larger scores first, then lower tokens.
// -0 counts as 0; no key of a token is 0.
__device__ __forceinline__ uint64_t score_key(float x, int v) {
  return ((uint64_t)order_key(x + 0.f) << 32) | (uint32_t)~v;
}

__device__ __forceinline__ uint64_t order_key64(double f) {
  const uint64_t u = (uint64_t)__double_as_longlong(f + 0.);
  return (u >> 63) ? ~u : (u | (1ull << 63));
}

__device__ __forceinline__ double key64_value(uint64_t k) {
  return __longlong_as_double((long long)((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}

template <typename E>
__global__ __launch_bounds__(kRowThreads) void beam_rows(const E* __restrict__ scores, int64_t sn, int64_t sw, int W,
                                                         int V, int K, double* __restrict__ lse,
                                                         uint64_t* __restrict__ lists) {
  __shared__ float red[kRowThreads / 64];
  __shared__ double sums[kRowThreads / 64];
  __shared__ uint64_t keys[kRowThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const E* x = scores + (row / W) * sn + (row % W) * sw;
  float m = kNegInf;
  for (int v = tid; v < V; v += kRowThreads) m = fmaxf(m, load_f32(x + v));
  m = wave_max(m);
  if (lane == 0) red[wave] = m;
  __syncthreads();
  for (int i = 0; i < kRowThreads / 64; ++i) m = fmaxf(m, red[i]);
  // NaN, +inf, or nothing above -inf: the sum becomes NaN or 0, and L no number
  const float at = m == kNegInf ? 0.f : m;
  double s = 0.;
  for (int v = tid; v < V; v += kRowThreads) s += (double)expf(load_f32(x + v) - at);
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) sums[wave] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.;
    for (int i = 0; i < kRowThreads / 64; ++i) s += sums[i];
    lse[row] = (double)at + log(s);
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t best = 0;
    for (int v = tid; v < V; v += kRowThreads) {
      const uint64_t key = score_key(load_f32(x + v), v);
      if (key < last && key > best) best = key;
    }
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o, 64);
      if (other > best) best = other;
    }
    __syncthreads();
    if (lane == 0) keys[wave] = best;
    __syncthreads();
    for (int i = 0; i < kRowThreads / 64; ++i)
      if (keys[i] > best) best = keys[i];
    if (tid == 0) lists[row * K + k] = best;  // 0 where the vocabulary holds fewer
    last = best;
  }
}

__global__ __launch_bounds__(64) void beam_merge(const double* __restrict__ lse, const uint64_t* __restrict__ lists,
                                                 const float* __restrict__ totals,
                                                 const unsigned char* __restrict__ ended, Stops stops, int W, int V,
                                                 int K, float* __restrict__ new_totals, int64_t* __restrict__ parents,
                                                 int64_t* __restrict__ tokens, unsigned char* __restrict__ new_ended) {
  const int lane = threadIdx.x;
  const int64_t row0 = (int64_t)blockIdx.x * W, row = row0 + lane;
  const bool mine = lane < W;
  double total = 0., base = 0.;
  bool over = false, alive = false;
  if (mine) {
    total = (double)totals[row];
    base = lse[row];
    over = ended && ended[row];
    alive = isfinite(total) && (over || isfinite(base));
  }
  const int stop = stops.n ? stops.token[0] : 0;
  // The head'th best candidate of this lane's beam: (value, ~(w V + v)), 0 for none.
  auto candidate = [&](int head, uint64_t& value, uint32_t& order) {
    value = 0;
    order = 0;
    if (!mine || head >= K) return;
    double f = (double)kNegInf;
    int64_t v = head;
    if (alive && over) {
      if (head == 0) {
        f = total;
        v = stop;
      } else {
        v = head - 1 + (head - 1 >= stop ? 1 : 0);
      }
    } else if (alive) {
      const uint64_t key = lists[row * K + head];
      if (key == 0) return;
      f = total + ((double)key_value((uint32_t)(key >> 32)) - base);
      v = (uint32_t)~(uint32_t)key;
    }
    if (v >= V) return;
    value = order_key64(f);
    order = ~(uint32_t)(lane * (int64_t)V + v);
  };
  int head = 0;
  uint64_t value;
  uint32_t order;
  candidate(head, value, order);
  for (int k = 0; k < K; ++k) {
    uint64_t bv = value;
    uint32_t bo = order;
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t ov = __shfl_xor((unsigned long long)bv, o, 64);
      const uint32_t oo = __shfl_xor(bo, o, 64);
      if (ov > bv || (ov == bv && oo > bo)) {
        bv = ov;
        bo = oo;
      }
    }
    if (mine && value == bv && order == bo) {  // one lane: the orders differ
      const uint32_t flat = ~bo;
      const int v = (int)(flat - (uint32_t)lane * (uint32_t)V);
      const int64_t at = (int64_t)blockIdx.x * K + k;
      new_totals[at] = (float)key64_value(bv);
      parents[at] = lane;
      tokens[at] = v;
      bool stopped = over;
      for (int i = 0; i < stops.n; ++i) stopped = stopped || stops.token[i] == v;
      new_ended[at] = stopped ? 1 : 0;
      candidate(++head, value, order);
    }
  }
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_beam_workspace(int n, int W, int V, int K, size_t* bytes) {
  if (!bytes) return fail(WPTV_E_INVALID, "beam_workspace: bytes is NULL");
  if (n < 0 || W <= 0 || V <= 0 || K <= 0 || (int64_t)K > (int64_t)W * V)
    return fail(WPTV_E_INVALID, "beam_workspace: bad shape n=%d W=%d V=%d K=%d", n, W, V, K);
  if (W > kMaxBeams || K > kMaxBeams)
    return fail(WPTV_E_UNSUPPORTED, "beam_workspace: at most %d beams a text (W=%d, K=%d)", kMaxBeams, W, K);
  if ((int64_t)W * V > INT32_MAX || (int64_t)n * W > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "beam_workspace: n=%d W=%d V=%d is too large", n, W, V);
  *bytes = (size_t)n * W * (sizeof(double) + (size_t)K * sizeof(uint64_t));
  return WPTV_OK;
}

extern "C" int wptv_beam_step(const void* scores, int64_t scores_stride_n, int64_t scores_stride_w, int scores_dtype,
                              const float* totals, const unsigned char* ended, const int64_t* stops, int n_stops,
                              int n, int W, int V, int K, float* new_totals, int64_t* parents, int64_t* tokens,
                              unsigned char* new_ended, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  size_t need = 0;
  const int status = wptv_beam_workspace(n, W, V, K, &need);
  if (status != WPTV_OK) return status;
  if (scores_dtype != WPTV_F32 && scores_dtype != WPTV_BF16)
    return fail(WPTV_E_UNSUPPORTED, "beam_step: scores of dtype %d are neither fp32 nor bf16", scores_dtype);
  if (n_stops < 0 || n_stops > kMaxStops || (n_stops && !stops))
    return fail(WPTV_E_INVALID, "beam_step: 0 to %d stop tokens (got %d)", kMaxStops, n_stops);
  if (ended && !n_stops) return fail(WPTV_E_INVALID, "beam_step: an ended beam goes on with a stop token; none is given");
  Stops s{n_stops, {}};
  for (int i = 0; i < n_stops; ++i) {
    if (stops[i] < 0 || stops[i] >= V)
      return fail(WPTV_E_INVALID, "beam_step: stop token %lld lies outside the vocabulary of %d", (long long)stops[i], V);
    s.token[i] = (int)stops[i];
  }
  if (n == 0) return WPTV_OK;
  if (!scores || !totals || !new_totals || !parents || !tokens || !new_ended || !workspace)
    return fail(WPTV_E_INVALID, "beam_step: a required pointer is NULL");
  if (workspace_bytes < need)
    return fail(WPTV_E_INVALID, "beam_step: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  double* lse = static_cast<double*>(workspace);
  uint64_t* lists = reinterpret_cast<uint64_t*>(lse + (size_t)n * W);
  if (scores_dtype == WPTV_F32)
    beam_rows<float><<<n * W, kRowThreads, 0, stream>>>(static_cast<const float*>(scores), scores_stride_n,
                                                        scores_stride_w, W, V, K, lse, lists);
  else
    beam_rows<unsigned short><<<n * W, kRowThreads, 0, stream>>>(static_cast<const unsigned short*>(scores),
                                                                 scores_stride_n, scores_stride_w, W, V, K, lse,
                                                                 lists);
  const int launch = launched("beam_rows");
  if (launch != WPTV_OK) return launch;
  beam_merge<<<n, 64, 0, stream>>>(lse, lists, totals, ended, s, W, V, K, new_totals, parents, tokens, new_ended);
  return launched("beam_merge");
}
