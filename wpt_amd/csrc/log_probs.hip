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

// The workgroup's row (b, t) of scores.
template <typename T>
__device__ __forceinline__ const T* row_of(const T* scores, int64_t ssb, int64_t sst, int per_row) {
  const unsigned b = blockIdx.x / (unsigned)per_row, t = blockIdx.x - b * (unsigned)per_row;
  return scores + b * ssb + t * sst;
}

// The maximum over a wavefront without LDS; every lane must be active.
__device__ __forceinline__ float wave_max_dpp(float x) {
  x = row16_max(x);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// What a stretch of a row's scores comes to: their maximum, how many hold it, the
// others' sums of exp d and d exp d with d = (x - high) / temperature.
struct Part {
  float high, many, rest, weighted;
};

// The log-probabilities of a row from its part; NaN where it has no distribution.
struct Level {
  float high, inverse, log_sum;
  __device__ __forceinline__ Level(const Part& part, float inverse_) : high(part.high), inverse(inverse_) {
    const bool none = !(fabsf(high) < __builtin_inff());  // +inf, or nothing above -inf
    log_sum = none ? __builtin_nanf("") : logf(part.many) + log1pf(part.rest / part.many);
  }
  __device__ __forceinline__ float of(float x) const { return (x - high) * inverse - log_sum; }
};

// given: the score of the token, if one was written.
__device__ __forceinline__ void store_row(const Part& part, const Level& level, bool written, float given, int64_t m,
                                          const Outputs& out) {
  out.logprobs[m] = written ? level.of(given) : 0.f;
  out.entropy[m] = level.log_sum - part.weighted / (part.many + part.rest);
}

// ---- a stretch of a row in registers -----------------------------------------

// 16 bytes of scores, wherever they start.
template <typename T>
struct Chunk;

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <>
struct Chunk<float> {
  static constexpr int N = 4;
  typedef u32x4 Loose __attribute__((aligned(4)));
  static __device__ __forceinline__ float at(const u32x4& v, int i) { return __uint_as_float(v[i]); }
  // The first `skip` scores -inf.
  static __device__ __forceinline__ u32x4 cut(u32x4 v, int skip) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < skip ? 0xff800000u : v[i];
    return v;
  }
};

template <>
struct Chunk<unsigned short> {
  static constexpr int N = 8;
  typedef u32x4 Loose __attribute__((aligned(2)));
  static __device__ __forceinline__ float at(const u32x4& v, int i) {
    return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
  static __device__ __forceinline__ u32x4 cut(u32x4 v, int skip) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = 2 * i < skip ? (v[i] & 0xffff0000u) | 0xff80u : v[i];
      v[i] = 2 * i + 1 < skip ? (v[i] & 0xffffu) | 0xff800000u : v[i];
    }
    return v;
  }
};

// A chunk as it is held, for one pass over the scores: without this the compiler
// would keep every score widened to FP32 from one pass to the next, and many
// chunks' at a time, in twice the registers.
__device__ __forceinline__ u32x4 held(u32x4 v) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" : "+v"(v));
  return v;
}

constexpr int kCandidates = 256, kMaxParts = 8;

// A score's key and place as one number: larger scores, then lower places, the
// larger number.
__device__ __forceinline__ uint64_t ranked(uint32_t key, int at) { return (uint64_t)key << 32 | ~(uint32_t)at; }
__device__ __forceinline__ int place_of(uint64_t r) { return (int)~(uint32_t)r; }
__device__ __forceinline__ float score_of(uint64_t r) { return key_value((uint32_t)(r >> 32)); }

// How many of the `count` numbers are larger than mine.
__device__ __forceinline__ int larger(const uint64_t* all, int count, uint64_t mine) {
  int before = 0;
  for (int c = 0; c < count; c += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) before += c + u < count && all[min(c + u, count - 1)] > mine ? 1 : 0;
  }
  return before;
}

constexpr int kGroups = 128;  // groups of neighbouring threads whose maxima bound the selection

template <int THREADS>
struct TopShared {
  SelectShared<THREADS> select;
  uint32_t group[kGroups];
  uint64_t best[kCandidates];
  int count, sums[2][THREADS / 64];
};

template <>
struct TopShared<0> {};

// One workgroup a row, or a part of one (blockIdx.y of gridDim.y): its scores are
// read once and stay in registers, CHUNKS times 16 bytes a thread.  What bounds it
// is that stream and the arithmetic on it (2048 rows of 32768 bf16 scores 31 us, 4.3
// TB/s, the exponentials and sums alone about 20), and for few rows the chain of its
// steps: the maximum, a barrier, the sums and the candidates, a barrier, the ranks
// (160 rows of them with 20 alternatives 10.5 us, without 7.5).
//
// The selection (TOP): the `top`-th largest of the maxima of 128 groups of threads
// is reached by `top` scores at least, so that only scores from there on are
// candidates, a few more than `top` of them, found in few threads; they are ranked
// by counting.  When more than kCandidates reach it (many equal scores), the border
// is selected exactly (kth_largest), equal scores by their place.
template <typename T, int THREADS, int CHUNKS, bool TOP>
__global__ __launch_bounds__(THREADS) void log_probs_held(const T* __restrict__ scores, int64_t ssb, int64_t sst,
                                                          const int64_t* __restrict__ tokens, float inverse,
                                                          int per_row, int V, int stretch, int top, Outputs out,
                                                          Part* __restrict__ parts, uint64_t* __restrict__ best) {
  using C = Chunk<T>;
  constexpr int kWaves = THREADS / 64, kStep = THREADS * C::N;
  __shared__ float sums[4][kWaves];
  __shared__ TopShared<TOP ? THREADS : 0> shared;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t m = blockIdx.x;
  const T* s = row_of(scores, ssb, sst, per_row);
  const int from = blockIdx.y * stretch, count = min(stretch, V - from);  // at least 8, and `top`
  // chunk c of a thread starts at its place in the stretch, or 16 bytes before the stretch's end if that comes
  // first: what it then holds of the chunk before it, `skip` scores, counts as -inf
  const float lowest = -__builtin_inff();
  auto start = [&](int c) { return min(c * kStep + tid * C::N, count - C::N); };
  // The forms double in size: chunks of the upper half that lie past the end are passed over (in a graph, us: 1302 rows
  // of 16568 in bf16, four chunks of eight and a few scores, 24.3 -> 17.2, with 31 alternatives 37.1 -> 29.2; 201 of
  // 50257 in FP32, thirteen of sixteen, 17.7 -> 16.8; rows that fill them as before).
  auto some = [&](int c) { return c < (CHUNKS + 1) / 2 || c * kStep < count; };
  u32x4 v[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    if (some(c)) v[c] = *reinterpret_cast<const typename C::Loose*>(s + from + start(c));
  // the token's own score, asked for beside the others
  const int64_t token = tokens[m];
  const bool written = token >= 0 && token < V;
  const float given = load_f32<T>(s + (written ? token : 0));
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    if (some(c) && (c + 1) * kStep > count) v[c] = C::cut(v[c], c * kStep + tid * C::N - start(c));
  float own = lowest;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if (!some(c)) continue;
    const u32x4 chunk = held(v[c]);
#pragma unroll
    for (int i = 0; i < C::N; ++i) own = fmaxf(own, C::at(chunk, i));
  }
  float high = wave_max_dpp(own);
  if (lane == 0) sums[0][w] = high;
  if constexpr (TOP) {
    float group = own;  // of THREADS / kGroups lanes
    group = fmaxf(group, __int_as_float(dpp_move<kDppXor1>(__float_as_int(group))));
    if constexpr (THREADS >= 512) group = fmaxf(group, __int_as_float(dpp_move<kDppXor2>(__float_as_int(group))));
    if constexpr (THREADS >= 1024)
      group = fmaxf(group, __int_as_float(dpp_move<kDppHalfMirror>(__float_as_int(group))));
    if (tid % (THREADS / kGroups) == 0) shared.group[tid / (THREADS / kGroups)] = score_key(group);
    if (tid == 0) shared.count = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) high = fmaxf(high, sums[0][i]);

  // (x - high) / temperature in units of log 2, for exp2
  const float unit = inverse * kLog2e;
  float rest = 0.f, weighted = 0.f, many = 0.f;
  auto add = [&](float t, float e) {
    rest += e;
    weighted = fmaf(e, fmaxf(t, -1e4f), weighted);  // -inf adds 0; a NaN shows in `rest`
  };
  if (own == high) {  // the maximum is here: its terms apart
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (!some(c)) continue;
      const u32x4 chunk = held(v[c]);
#pragma unroll
      for (int i = 0; i < C::N; ++i) {
        const float x = C::at(chunk, i), t = (x - high) * unit;
        if (x == high)
          many += 1.f;
        else
          add(t, __builtin_amdgcn_exp2f(t));
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (!some(c)) continue;
      const u32x4 chunk = held(v[c]);
#pragma unroll
      for (int i = 0; i < C::N; ++i) {
        const float t = (C::at(chunk, i) - high) * unit;
        add(t, __builtin_amdgcn_exp2f(t));
      }
    }
  }
  const bool nan = rest != rest;  // one of the thread's own scores is one
  rest = wave_sum_dpp(rest);
  weighted = wave_sum_dpp(weighted);
  many = wave_sum_dpp(many);
  if (lane == 0) {
    sums[1][w] = rest;
    sums[2][w] = weighted;
    sums[3][w] = many;
  }

  auto each = [&](auto&& f) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (!some(c)) continue;
      const u32x4 chunk = held(v[c]);
      int first = tid * C::N;
      asm volatile("" : "+v"(first));  // as the chunks: the places are not kept from pass to pass
      first += c * kStep;
      const int begin = min(first, count - C::N);
#pragma unroll
      for (int i = 0; i < C::N; ++i)
        if (begin + i >= first) f(begin + i, score_key(C::at(chunk, i)));
    }
  };
  auto note = [&](int at, uint32_t x) {
    if constexpr (TOP) {
      const int c = atomicAdd(&shared.count, 1);  // in any order: ranked below
      if (c < kCandidates) shared.best[c] = ranked(x, at);
    }
  };
  if constexpr (TOP) {
    // the top-th largest of the groups' maxima, a bit at a time, by every wavefront for itself
    const uint32_t one = shared.group[lane], two = shared.group[64 + lane];
    uint32_t border = 0u;
    constexpr int kLastBit = sizeof(T) == 2 ? 16 : 0;  // bf16 keys differ in their upper half
    for (int bit = 31; bit >= kLastBit; --bit) {
      const uint32_t trial = border | (1u << bit);
      const int reach = __builtin_popcountll(__builtin_amdgcn_ballot_w64(one >= trial)) +
                        __builtin_popcountll(__builtin_amdgcn_ballot_w64(two >= trial));
      if (reach >= top) border = trial;
    }
    if (nan || score_key(own) >= border) {
      // as a comparison of scores: one below every score's key gives a NaN, which nothing is less than, as a NaN
      // is less than nothing
      const float least = key_value(border);
      constexpr int kHeld = CHUNKS * C::N, kWord = kHeld < 32 ? kHeld : 32;
#pragma unroll
      for (int word = 0; word < kHeld / kWord; ++word) {
        uint32_t reach = 0u;
#pragma unroll
        for (int c = word * kWord / C::N; c < (word + 1) * kWord / C::N; ++c) {
          if (!some(c)) continue;
          const u32x4 chunk = held(v[c]);
#pragma unroll
          for (int i = 0; i < C::N; ++i)
            reach |= C::at(chunk, i) < least ? 0u : 1u << (c * C::N + i) % kWord;
        }
        for (; reach; reach &= reach - 1u) {  // few: read again
          const int b = word * kWord + __builtin_ctz(reach), c = b / C::N;
          const int first = c * kStep + tid * C::N, at = min(first, count - C::N) + b % C::N;
          if (at >= first) note(at, score_key(load_f32<T>(s + from + at)));
        }
      }
    }
  }
  __syncthreads();
  int found = 0;
  if constexpr (TOP) {
    found = shared.count;
    if (found > kCandidates) {
      const uint32_t tau = kth_largest<THREADS, true>(each, top, shared.select);
      int above = 0, equal = 0;
      each([&](int, uint32_t x) {
        above += x > tau;
        equal += x == tau;
      });
      above = (int)wave_sum_u32(above);
      equal = (int)wave_sum_u32(equal);
      __syncthreads();
      if (lane == 0) {
        shared.sums[0][w] = above;
        shared.sums[1][w] = equal;
      }
      if (tid == 0) shared.count = 0;
      __syncthreads();
      above = equal = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        above += shared.sums[0][i];
        equal += shared.sums[1][i];
      }
      uint32_t last = 0u;  // the complement of the last place kept of those equal to tau
      if (equal > top - above)
        last = kth_largest<THREADS, true>(
            [&](auto&& f) {
              each([&](int at, uint32_t x) {
                if (x == tau) f(at, ~(uint32_t)at);
              });
            },
            top - above, shared.select);
      each([&](int at, uint32_t x) {
        if (x > tau || (x == tau && ~(uint32_t)at >= last)) note(at, x);
      });
      __syncthreads();
      found = shared.count;  // top of them
    }
  }
  if (64 * w >= (found > 0 ? found : 1)) return;  // the first wavefronts rank and store
  Part part = {high, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    part.rest += sums[1][i];
    part.weighted += sums[2][i];
    part.many += sums[3][i];
  }
  part.weighted *= kLn2;
  const Level level(part, inverse);
  const int64_t place = m * gridDim.y + blockIdx.y;
  if (tid == 0) {
    if (gridDim.y == 1)
      store_row(part, level, written, given, m, out);
    else
      parts[place] = part;
  }
  if constexpr (TOP) {
    if (tid < found) {
      const uint64_t mine = shared.best[tid];
      const int before = larger(shared.best, found, mine);
      if (before < top) {
        if (gridDim.y == 1) {
          out.ids[m * top + before] = place_of(mine);
          out.best[m * top + before] = level.of(score_of(mine));
        } else {
          best[place * top + before] = ranked((uint32_t)(mine >> 32), from + place_of(mine));
        }
      }
    }
  }
}

// One workgroup a row: its parts' sums brought to the common maximum and added in
// order, their best ranked together.
template <typename T>
__global__ __launch_bounds__(256) void log_probs_join(const T* __restrict__ scores, int64_t ssb, int64_t sst,
                                                      const int64_t* __restrict__ tokens, float inverse, int per_row,
                                                      int V, int count, int top, Outputs out,
                                                      const Part* __restrict__ parts,
                                                      const uint64_t* __restrict__ best) {
  __shared__ uint64_t all[kMaxParts * kMaxTop];
  const int tid = threadIdx.x, total = count * top;
  const int64_t m = blockIdx.x;
  const T* s = row_of(scores, ssb, sst, per_row);
  const int64_t token = tokens[m];
  const bool written = token >= 0 && token < V;
  const float given = load_f32<T>(s + (written ? token : 0));
  for (int i = tid; i < total; i += 256) all[i] = best[m * total + i];
  Part part = {-__builtin_inff(), 0.f, 0.f, 0.f};
  for (int i = 0; i < count; ++i) part.high = fmaxf(part.high, parts[m * count + i].high);
  for (int i = 0; i < count; ++i) {
    const Part one = parts[m * count + i];
    if (one.high == part.high) {
      part.many += one.many;
      part.rest += one.rest;
      part.weighted += one.weighted;
    } else {  // exp d = exp(d of the part) exp(shift); a part of -inf adds 0, a NaN shows in `rest`
      const float shift = (one.high - part.high) * inverse, scale = expf(shift), mass = one.many + one.rest;
      const bool empty = one.high == -__builtin_inff();
      part.rest += empty ? one.rest : scale * mass;
      part.weighted += empty || scale == 0.f ? 0.f : scale * (one.weighted + shift * mass);
    }
  }
  const Level level(part, inverse);
  if (tid == 0) store_row(part, level, written, given, m, out);
  __syncthreads();
  for (int i = tid; i < total; i += 256) {
    const int before = larger(all, total, all[i]);
    if (before < top) {
      out.ids[m * top + before] = place_of(all[i]);
      out.best[m * top + before] = level.of(score_of(all[i]));
    }
  }
}

// ---- rows of a few scores, and rows longer than the registers of eight workgroups ----

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
  const T* s = row_of(scores, ssb, sst, per_row);
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
  const Part row = {high, (float)highest, rest, weighted};
  const Level level(row, inverse);
  if (tid == 0) {
    const int64_t token = tokens[m];
    const bool written = token >= 0 && token < V;
    store_row(row, level, written, load_f32<T>(s + (written ? token : 0)), m, out);
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
    out.best[m * top + before] = level.of(load_f32<T>(s + i));
  }
}

// How rows are read: the threads and 16-byte chunks of a workgroup, and the parts
// a row is cut into (0: from memory, rows shorter than a chunk and rows longer
// than kMaxParts of the largest workgroup).
struct Form {
  int threads, chunks, parts, stretch;
};

constexpr int kRowThreads = 512;  // of the form from memory

Form row_form(int64_t rows, int V, int top, int dtype) {
  const int per = dtype == WPTV_BF16 ? 8 : 4;
  const int64_t units = compute_units();
  if (V < per) return Form{0, 0, 0, 0};
  if (V <= 256 * 2 * per) return Form{256, 2, 1, V};
  if (V <= 512 * 4 * per) return Form{512, 4, 1, V};
  // few rows: as many threads as there are, or the rows in parts over the compute units; more rows hide each other's
  // steps, which smaller workgroups do better.  bf16, 20 alternatives, us, 1024 threads and 512: 160 rows of 32768
  // 13.0, 16.3, 512 24.4, 21.8; 8 rows of 131072 in four parts 16.5, in one 35
  if (V <= 512 * 8 * per) return rows <= units ? Form{1024, 4, 1, V} : Form{512, 8, 1, V};
  const int few = 1024 * 4 * per, many = 1024 * 16 * per;
  int parts = (V + few - 1) / few;
  if (parts <= kMaxParts && rows * parts <= units) return Form{1024, 4, parts, ((V + parts - 1) / parts + 7) / 8 * 8};
  if (V <= 1024 * 8 * per) return Form{1024, 8, 1, V};
  // without alternatives in parts that three or four workgroups a compute unit take beside each other; with them each
  // part's choice costs what that gives.  bf16, us, parts and one or two of the largest workgroup: 1024 rows of 128000
  // 59, 81, of 152000 70, 103, 160 rows of 128000 19.2, 21.1; with 20 alternatives 102, 107, 160 rows 30.1, 27.6; 1024
  // rows of 65536, in eight chunks, 34.8 both
  parts = (V + 512 * 8 * per - 1) / (512 * 8 * per);
  if (top == 0 && parts <= kMaxParts) return Form{512, 8, parts, ((V + parts - 1) / parts + 7) / 8 * 8};
  parts = (V + many - 1) / many;
  if (parts > kMaxParts) return Form{0, 0, 0, 0};
  return Form{1024, 16, parts, parts == 1 ? V : ((V + parts - 1) / parts + 7) / 8 * 8};
}

size_t part_bytes(int64_t rows, const Form& form, int top) {
  return form.parts > 1 ? (size_t)rows * form.parts * (sizeof(Part) + (size_t)top * 8) : 0;
}

template <typename T>
int run_log_probs(const T* scores, int64_t ssb, int64_t sst, const int64_t* tokens, float inverse, int rows,
                  int per_row, int V, int top, const Form& form, const Outputs& out, void* workspace, hipStream_t stream) {
  if (form.parts == 0) {
    log_probs_row<T, kRowThreads><<<rows, kRowThreads, 0, stream>>>(scores, ssb, sst, tokens, inverse, per_row, V, top,
                                                                    out);
    return launched("log_probs");
  }
  Part* parts = static_cast<Part*>(workspace);
  const int64_t places = (int64_t)rows * form.parts;
  uint64_t* best = reinterpret_cast<uint64_t*>(parts + places);
#define WPTV_HELD(THREADS, CHUNKS)                                                                                \
  (top ? log_probs_held<T, THREADS, CHUNKS, true> : log_probs_held<T, THREADS, CHUNKS, false>)                    \
      <<<dim3(rows, form.parts), THREADS, 0, stream>>>(scores, ssb, sst, tokens, inverse, per_row, V,             \
                                                       form.stretch, top, out, parts, best)
  if (form.threads == 256)
    WPTV_HELD(256, 2);
  else if (form.threads == 512 && form.chunks == 4)
    WPTV_HELD(512, 4);
  else if (form.threads == 512)
    WPTV_HELD(512, 8);
  else if (form.chunks == 4)
    WPTV_HELD(1024, 4);
  else if (form.chunks == 8)
    WPTV_HELD(1024, 8);
  else
    WPTV_HELD(1024, 16);
#undef WPTV_HELD
  const int status = launched("log_probs");
  if (status != WPTV_OK || form.parts == 1) return status;
  log_probs_join<T><<<rows, 256, 0, stream>>>(scores, ssb, sst, tokens, inverse, per_row, V, form.parts, top, out,
                                             parts, best);
  return launched("log_probs (join)");
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
  const size_t bf16 = part_bytes((int64_t)B * T, row_form((int64_t)B * T, V, top, WPTV_BF16), top);
  const size_t fp32 = part_bytes((int64_t)B * T, row_form((int64_t)B * T, V, top, WPTV_F32), top);
  *bytes = bf16 > fp32 ? bf16 : fp32;
  return WPTV_OK;
}

extern "C" int wptv_log_probs(const void* scores, int64_t scores_stride_b, int64_t scores_stride_t, int scores_dtype,
                              const int64_t* tokens, float temperature, int B, int T, int V, int top, float* logprobs,
                              float* entropy, int64_t* ids, float* best, void* workspace, size_t workspace_bytes,
                              hipStream_t stream) {
  size_t need = 0;
  const int status = wptv_log_probs_workspace(B, T, V, top, &need);
  if (status != WPTV_OK) return status;
  if (!(temperature > 0.f) || std::isinf(temperature) || std::isinf(1.f / temperature))
    return fail(WPTV_E_INVALID, "log_probs: the temperature must be positive and finite; got %g", temperature);
  if (scores_dtype != WPTV_F32 && scores_dtype != WPTV_BF16)
    return fail(WPTV_E_UNSUPPORTED, "log_probs: dtype %d is neither fp32 nor bf16", scores_dtype);
  if ((int64_t)B * T == 0) return WPTV_OK;
  if (!scores || !tokens || !logprobs || !entropy || (top > 0 && (!ids || !best)))
    return fail(WPTV_E_INVALID, "log_probs: a required pointer is NULL");
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(WPTV_E_INVALID, "log_probs: the workspace holds %zu bytes; %zu are needed",
                workspace ? workspace_bytes : 0, need);
  const float inverse = 1.f / temperature;
  const Outputs out{logprobs, entropy, ids, best};
  const Form form = row_form((int64_t)B * T, V, top, scores_dtype);
  const int64_t threads = (int64_t)B * T * (form.parts ? form.threads : kRowThreads);
  if (threads > UINT32_MAX)  // a dimension of a grid
    return fail(WPTV_E_UNSUPPORTED, "log_probs: %lld rows of %d scores are %lld threads, above 2^32 - 1",
                (long long)B * T, V, (long long)threads);
  return scores_dtype == WPTV_BF16
             ? run_log_probs(static_cast<const unsigned short*>(scores), scores_stride_b, scores_stride_t, tokens,
                             inverse, B * T, T, V, top, form, out, workspace, stream)
             : run_log_probs(static_cast<const float*>(scores), scores_stride_b, scores_stride_t, tokens, inverse,
                             B * T, T, V, top, form, out, workspace, stream);
}
