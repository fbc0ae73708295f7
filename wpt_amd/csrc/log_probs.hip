// The log-probability of written tokens under the model's scores, the entropy of
// the distribution they came from and its likeliest tokens, for gfx950
// (wptv_log_probs).
//
//   z = x / temperature, d = (x - high) / temperature, high = max x
//   log sum exp z - high / temperature = log S, S = sum exp d
//   logprob = d[token] - log S, entropy = log S - (sum d exp d) / S
//
// The terms at the maximum, each exactly 1, are counted and the others summed by
// themselves, log S = log n + log1p(rest / n): a token that is all but certain
// keeps the digits of its small log-probability.
#include "select_common.h"
#include "wptv_common.h"

#include <climits>
#include <cmath>

namespace wptv {
namespace {

constexpr int kMaxTop = 64;

__device__ __forceinline__ uint32_t score_key(float f) { return f != f ? ~0u : order_key(f + 0.f); }

struct Outputs {
  float* logprobs;
  float* entropy;
  int64_t* ids;
  float* best;
};

// One workgroup a row, its scores read again for every pass.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void log_probs_row(const T* __restrict__ scores, int64_t ssb, int64_t sst,
                                                         const int64_t* __restrict__ tokens, float inverse, int per_row,
                                                         int V, int top, Outputs out) {
  constexpr int kWaves = THREADS / 64;
  __shared__ SelectShared<THREADS> select;
  __shared__ float part[3][kWaves];
  __shared__ int many[kWaves], ncand;
  __shared__ uint32_t keys[kMaxTop];
  __shared__ int at[kMaxTop];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t m = blockIdx.x;
  const T* s = scores + m / per_row * ssb + m % per_row * sst;
  float high = -__builtin_inff();
  for (int i = tid; i < V; i += THREADS) high = fmaxf(high, load_f32<T>(s + i));
  high = wave_max(high);
  if (lane == 0) part[0][w] = high;
  if (tid == 0) ncand = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) high = fmaxf(high, part[0][i]);
  float rest = 0.f, weighted = 0.f;
  int highest = 0;
  for (int i = tid; i < V; i += THREADS) {
    const float x = load_f32<T>(s + i);
    const float d = (x - high) * inverse, e = exp2f(d * kLog2e);
    if (x == high) {
      ++highest;
    } else {
      rest += e;
      weighted += e == 0.f ? 0.f : e * d;
    }
  }
  rest = wave_sum(rest);
  weighted = wave_sum(weighted);
  highest = (int)wave_sum_u32(highest);
  __syncthreads();
  if (lane == 0) {
    part[1][w] = rest;
    part[2][w] = weighted;
    many[w] = highest;
  }
  __syncthreads();
  rest = weighted = 0.f;
  highest = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    rest += part[1][i];
    weighted += part[2][i];
    highest += many[i];
  }
  const bool none = !(fabsf(high) < __builtin_inff());  // +inf, or nothing above -inf
  const float n = (float)highest;
  const float log_sum = none ? __builtin_nanf("") : logf(n) + log1pf(rest / n);
  if (tid == 0) {
    const int64_t token = tokens[m];
    out.logprobs[m] =
        token >= 0 && token < V ? (load_f32<T>(s + token) - high) * inverse - log_sum : 0.f;
    out.entropy[m] = log_sum - weighted / (n + rest);
  }
  if (top == 0) return;
  auto each = [&](auto&& f) {
    for (int i = tid; i < V; i += THREADS) f(i, score_key(load_f32<T>(s + i)));
  };
  const uint32_t tau = kth_largest<THREADS, true>(each, top, select);
  int above = 0, equal = 0;
  each([&](int, uint32_t x) {
    above += x > tau;
    equal += x == tau;
  });
  above = (int)wave_sum_u32(above);
  equal = (int)wave_sum_u32(equal);
  __syncthreads();
  if (lane == 0) {
    many[w] = above;
    part[0][w] = __int_as_float(equal);
  }
  __syncthreads();
  above = equal = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    above += many[i];
    equal += __float_as_int(part[0][i]);
  }
  uint32_t last = 0u;  // the complement of the last place kept of those equal to tau
  if (equal > top - above)
    last = kth_largest<THREADS, true>(
        [&](auto&& f) {
          each([&](int i, uint32_t x) {
            if (x == tau) f(i, ~(uint32_t)i);
          });
        },
        top - above, select);
  each([&](int i, uint32_t x) {
    if (x > tau || (x == tau && ~(uint32_t)i >= last)) {
      const int c = atomicAdd(&ncand, 1);  // in any order: ranked below
      keys[c] = x;
      at[c] = i;
    }
  });
  __syncthreads();
  if (tid < top) {
    const uint32_t mine = keys[tid];
    const int i = at[tid];
    int before = 0;
    for (int c = 0; c < top; ++c) before += keys[c] > mine || (keys[c] == mine && at[c] < i) ? 1 : 0;
    out.ids[m * top + before] = i;
    out.best[m * top + before] = (load_f32<T>(s + i) - high) * inverse - log_sum;
  }
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_log_probs_workspace(int B, int T, int V, int top, size_t* bytes) {
  if (B < 0 || T < 0 || V <= 0 || top < 0 || !bytes)
    return fail(WPTV_E_INVALID, "log_probs: bad shape B=%d T=%d V=%d top=%d", B, T, V, top);
  if (top > V) return fail(WPTV_E_INVALID, "log_probs: the top %d of %d tokens", top, V);
  if (top > kMaxTop) return fail(WPTV_E_UNSUPPORTED, "log_probs: %d alternatives above %d", top, kMaxTop);
  if (V > (1 << 24) || (int64_t)B * T > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "log_probs: B=%d T=%d V=%d is too large", B, T, V);
  *bytes = 0;
  return WPTV_OK;
}

extern "C" int wptv_log_probs(const void* scores, int64_t scores_stride_b, int64_t scores_stride_t, int scores_dtype,
                              const int64_t* tokens, float temperature, int B, int T, int V, int top, float* logprobs,
                              float* entropy, int64_t* ids, float* best, void* workspace, size_t workspace_bytes,
                              hipStream_t stream) {
  size_t need = 0;
  const int status = wptv_log_probs_workspace(B, T, V, top, &need);
  if (status != WPTV_OK) return status;
  if (!(temperature > 0.f) || std::isinf(temperature))
    return fail(WPTV_E_INVALID, "log_probs: the temperature must be positive and finite; got %g", temperature);
  if (scores_dtype != WPTV_F32 && scores_dtype != WPTV_BF16)
    return fail(WPTV_E_UNSUPPORTED, "log_probs: dtype %d is neither fp32 nor bf16", scores_dtype);
  if ((int64_t)B * T == 0) return WPTV_OK;
  if (!scores || !tokens || !logprobs || !entropy || (top > 0 && (!ids || !best)))
    return fail(WPTV_E_INVALID, "log_probs: a required pointer is NULL");
  if (need && (!workspace || workspace_bytes < need))
    return fail(WPTV_E_INVALID, "log_probs: the workspace holds %zu bytes; %zu are needed", workspace ? workspace_bytes : 0,
                need);
  const float inverse = 1.f / temperature;
  const Outputs out{logprobs, entropy, ids, best};
  if (scores_dtype == WPTV_BF16)
    log_probs_row<unsigned short, 512><<<B * T, 512, 0, stream>>>(static_cast<const unsigned short*>(scores),
                                                                  scores_stride_b, scores_stride_t, tokens, inverse, T,
                                                                  V, top, out);
  else
    log_probs_row<float, 512><<<B * T, 512, 0, stream>>>(static_cast<const float*>(scores), scores_stride_b,
                                                         scores_stride_t, tokens, inverse, T, V, top, out);
  return launched("log_probs");
}
