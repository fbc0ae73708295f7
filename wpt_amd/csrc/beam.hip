// Beam search's selection for gfx950: the next beams of every text over its
// beams and the vocabulary.
//
// A text's candidates are its W beams continued by each of V tokens, of value
//   total[w] + (x[w, v] - L[w]),  L[w] = log sum_v exp x[w, v]
// in 64 bits; the K largest are the next beams, equal values to the lowest
// w V + v.  Within a beam the value does not fall with x, so nothing has to be
// normalised before it is selected: each score is read once.
//   beam_parts  a wavefront a part of a beam's scores, all of it in registers:
//               the part's maximum, its sum of exponentials, and its K largest
//               scores, ties to the lowest token
//   beam_merge  a workgroup a text: the parts' FP32 sums joined to L, and the K
//               best of the parts' lists; where two beams' candidates are closer
//               than those sums tell apart, L again in 64 bits from the scores
//   beam_text   both, for a text whose parts fit one workgroup
// The K largest of a part: the K-th largest of the lanes' maxima bounds them
// from below, and few scores reach it (in scores without order about K of 4096);
// those are gathered in LDS, 64 at a time sorted across the lanes and merged
// into the best so far.  No barrier, and any scores are served: where many reach
// the bound the part is read again.
//
// 64 texts of 5 beams over 50257 FP32 scores: 16.4 us and 6.2 (64 MB at 3.9 TB/s; the
// loads of all parts are in flight at once and their arithmetic follows); 32 texts of
// 8 beams over 32768 bf16 scores: 7.1 and 7.0; one text of 4 beams over 8192: 9.1 in one
// launch, the latency of its steps.
#include "wptv_common.h"

#include <climits>
#include <cmath>
#include <type_traits>

namespace wptv {
namespace {

constexpr int kMaxBeams = 64;  // beams of a text: a lane each of a sorted list
constexpr int kMaxStops = 16;
constexpr int kPartWaves = 4;  // wavefronts of a beam_parts workgroup
constexpr int kGathered = 256;  // keys a wavefront gathers
constexpr float kNegInf = -__builtin_inff();

struct Stops {
  int n;
  int token[kMaxStops];
};

// The maximum over the 64 lanes of a wavefront, in every lane (NaNs passed over).
__device__ __forceinline__ float wave_max_dpp(float x) {
  x = row16_max(x);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

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

// ---- sorting across the lanes --------------------------------------------------

// A key of N words, the most significant first; 0 sorts last.
template <int N>
struct Key {
  uint32_t w[N];
};

template <int N>
__device__ __forceinline__ bool above(const Key<N>& a, const Key<N>& b) {
  if constexpr (N == 1) {
    return a.w[0] > b.w[0];
  } else {
    const uint64_t x = ((uint64_t)a.w[0] << 32) | a.w[1], y = ((uint64_t)b.w[0] << 32) | b.w[1];
    if constexpr (N == 2) return x > y;
    return x > y || (x == y && a.w[2] > b.w[2]);
  }
}

// A move within a 16-lane row that every lane takes part in (no old value to keep).
template <int CTRL>
__device__ __forceinline__ uint32_t row_move(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}

// x of lane ^ M, without LDS traffic; every lane must be active.
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  if constexpr (M >= 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane_xor<M - 32>((threadIdx.x & 32) ? r[0] : r[1]);
  } else if constexpr (M >= 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane_xor<M - 16>((threadIdx.x & 16) ? r[0] : r[1]);
  } else if constexpr (M == 15) {
    return row_move<kDppMirror>(x);
  } else if constexpr (M == 8) {
    return row_move<0x128>(x);  // row_ror:8
  } else if constexpr (M == 7) {
    return row_move<kDppHalfMirror>(x);
  } else if constexpr (M == 4) {
    return lane_xor<3>(row_move<kDppHalfMirror>(x));
  } else if constexpr (M == 3) {
    return row_move<0x1B>(x);  // a quad reversed
  } else if constexpr (M == 2) {
    return row_move<kDppXor2>(x);
  } else if constexpr (M == 1) {
    return row_move<kDppXor1>(x);
  } else {
    static_assert(M == 0, "a lane exchange of this list");
    return x;
  }
}

// One compare-exchange with lane ^ M: the lanes with bit BIT clear keep the
// larger key.
template <int M, int BIT, int N>
__device__ __forceinline__ void exchange(Key<N>& k) {
  Key<N> other;
#pragma unroll
  for (int i = 0; i < N; ++i) other.w[i] = lane_xor<M>(k.w[i]);
  const bool larger = (threadIdx.x & BIT) == 0;
  if constexpr (N == 1) {
    k.w[0] = larger ? max(k.w[0], other.w[0]) : min(k.w[0], other.w[0]);
  } else {
    const bool mine = above(k, other) == larger;
#pragma unroll
    for (int i = 0; i < N; ++i) k.w[i] = mine ? k.w[i] : other.w[i];
  }
}

template <int BIT, int N>
__device__ __forceinline__ void merge_down(Key<N>& k) {
  if constexpr (BIT > 0) {
    exchange<BIT, BIT>(k);
    merge_down<BIT / 2>(k);
  }
}

// Falling order within each LAST lanes.
template <int LAST = 64, int SIZE = 2, int N>
__device__ __forceinline__ void wave_sort(Key<N>& k) {
  exchange<SIZE - 1, SIZE / 2>(k);
  merge_down<SIZE / 4>(k);
  if constexpr (SIZE < LAST) wave_sort<LAST, SIZE * 2>(k);
}

// Falling order of keys that only the first `many` lanes hold (the others 0).
template <int N>
__device__ __forceinline__ void wave_sort_first(Key<N>& k, int many) {
  if (many <= 16)
    wave_sort<16>(k);
  else
    wave_sort(k);
}

// best = the 64 largest of best and of `reversed`, a falling list read
// backwards; both falling afterwards.
template <int N>
__device__ __forceinline__ void merge_lists(Key<N>& best, const Key<N>& reversed) {
  if (above(reversed, best)) best = reversed;
  merge_down<32>(best);
}

template <int N>
__device__ __forceinline__ Key<N> backwards(const Key<N>& k) {
  Key<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.w[i] = lane_xor<63>(k.w[i]);
  return r;
}

// x of lane + 1 (the last lane's: no use).
__device__ __forceinline__ uint32_t next_lane(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x130, 0xf, 0xf, false);  // wave_shl:1
}

template <int N>
__device__ __forceinline__ Key<N> key_of_lane(const Key<N>& k, int lane) {
  Key<N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.w[i] = __builtin_amdgcn_readlane(k.w[i], lane);
  return r;
}

// ---- the parts -------------------------------------------------------------------

// 16 bytes of scores, at any element's address.
template <typename E>
struct Scores16;
template <>
struct Scores16<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Scores16<unsigned short> {
  typedef unsigned short type __attribute__((ext_vector_type(8), aligned(2)));
};

// The lanes before this one in mask.
__device__ __forceinline__ int below_me(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

struct PartSum {
  float top, sum;  // the largest score, and the sum of exp(x - top) (of exp x where nothing is above -inf)
};

// The sum and the list (K keys, 0 where it holds fewer) of part `part` of the V
// scores at p, by one wavefront.  held: kGathered keys of LDS.
template <typename E, int ITEMS>
__device__ __forceinline__ void part_list(const E* p, int V, int part, int K, uint64_t* held, PartSum* result,
                                          uint64_t* list) {
  typedef typename Scores16<E>::type Vec;
  constexpr int kVec = 16 / sizeof(E), kLoads = ITEMS / kVec;
  const int lane = threadIdx.x & 63;
  const int v0 = part * 64 * ITEMS + lane * kVec;  // this lane's first token; 64 kVec a load
  // a load that would pass the row's end is moved back to it, and the tokens that
  // another lane holds left out
  const int last_load = V > kVec ? V - kVec : 0;
  auto token = [&](int i) { return min(v0 + i / kVec * 64 * kVec, last_load) + i % kVec; };
  float x[ITEMS];
  if ((part + 1) * 64 * ITEMS <= V) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const Vec got = *reinterpret_cast<const Vec*>(p + v0 + i * 64 * kVec);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const E one = got[e];
        x[i * kVec + e] = load_f32(&one);
      }
    }
  } else {
    Vec got[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (V >= kVec) {
        got[i] = *reinterpret_cast<const Vec*>(p + token(i * kVec));
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) got[i][e] = p[min(e, V - 1)];
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int v = token(i);
      const E one = got[i / kVec][i % kVec];
      x[i] = v < V && v >= v0 + i / kVec * 64 * kVec ? load_f32(&one) : kNegInf;
    }
  }
  float most = kNegInf;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) most = fmaxf(most, x[i]);  // a NaN is passed over here and found in the sum
  const float top = wave_max_dpp(most);
  const float at = top == kNegInf ? 0.f : top;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) sum[i % 4] += __builtin_amdgcn_exp2f((x[i] - at) * kLog2e);
  const float total = wave_sum_dpp((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (lane == 0) *result = PartSum{top, total};

  if (top == kNegInf) {  // the part's first tokens
    const int v = part * 64 * ITEMS + lane;
    if (lane < K) list[lane] = v < V ? score_key(kNegInf, v) : 0;
    return;
  }
  // At least K scores reach the K-th largest of the lanes' maxima.
  Key<1> maxima{{order_key(most + 0.f)}};
  wave_sort(maxima);
  const uint32_t kth = key_of_lane(maxima, K - 1).w[0];
  const float bound = key_value(kth);
  int count = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint64_t mask = __builtin_amdgcn_ballot_w64(x[i] >= bound);
    if (mask == 0) continue;
    const int at = count + below_me(mask);
    if (x[i] >= bound && at < kGathered) {
      const int v = token(i);
      held[at] = v < V && v >= v0 + i / kVec * 64 * kVec ? score_key(x[i], v) : 0;
    }
    count += __builtin_popcountll(mask);
  }
  Key<2> best{{0, 0}}, last{{0, 0}};  // the part's list, and its K-th key
  bool some = false;
  auto sort_in = [&](int first, int end) {  // held[first .. end - 1], at most 64
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t mine = first + lane < end ? held[first + lane] : 0;
    Key<2> k{{(uint32_t)(mine >> 32), (uint32_t)mine}};
    wave_sort_first(k, end - first);
    if (some)
      merge_lists(best, backwards(k));
    else
      best = k;
    some = true;
    last = key_of_lane(best, K - 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  if (count <= kGathered) {
    for (int first = 0; first < count; first += 64) sort_in(first, count);
  } else {
    // Many scores equal the bound, or one lane holds many large ones.  The part
    // again from memory: first, of the lanes whose maximum is the bound, each
    // one's first token with it (the first of these, K less the lanes above the
    // bound, are enough ties), then every score that is left, against the best
    // so far.
    auto each = [&](auto&& f) {  // f(token, score) of this lane, in the order of the tokens
#pragma unroll 2
      for (int i = 0; i < kLoads; ++i) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int v = v0 + i * 64 * kVec + e;
          f(v, v < V ? load_f32(p + v) : kNegInf);
        }
      }
    };
    uint32_t first = 0;  // ~token
    each([&](int v, float f) { first = f == bound ? max(first, ~(uint32_t)v) : first; });
    Key<1> firsts{{most == bound ? first : 0u}};
    wave_sort(firsts);
    const int more = __builtin_popcountll(__builtin_amdgcn_ballot_w64(most > bound));
    const uint32_t tie = key_of_lane(firsts, K - 1 - more).w[0];
    count = 0;
    each([&](int v, float f) {
      const uint64_t key = score_key(f, v);
      const bool in = v < V && (f > bound || (f == bound && ~(uint32_t)v >= tie)) &&
                      key > (((uint64_t)last.w[0] << 32) | last.w[1]);
      const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
      if (mask == 0) return;
      if (in) held[count + below_me(mask)] = key;
      count += __builtin_popcountll(mask);
      if (count >= 64) {
        sort_in(0, 64);
        const uint64_t rest = held[64 + lane];
        held[lane] = rest;
        count -= 64;
      }
    });
    if (count > 0) sort_in(0, count);
  }
  if (lane < K) list[lane] = ((uint64_t)best.w[0] << 32) | best.w[1];
}

template <typename E, int ITEMS>
__global__ __launch_bounds__(64 * kPartWaves) void beam_parts(const E* __restrict__ scores, int64_t sn, int64_t sw,
                                                              uint32_t W, int V, int K, uint32_t parts,
                                                              uint32_t waves, PartSum* __restrict__ sums,
                                                              uint64_t* __restrict__ lists) {
  __shared__ uint64_t gathered[kPartWaves][kGathered];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wave = blockIdx.x * kPartWaves + w;
  if (wave >= waves) return;
  const uint32_t row = wave / parts, part = wave % parts;
  part_list<E, ITEMS>(scores + (int64_t)(row / W) * sn + (int64_t)(row % W) * sw, V, (int)part, K, gathered[w],
                      sums + wave, lists + (int64_t)wave * K);
}

// ---- the text's next beams -----------------------------------------------------------

__device__ __forceinline__ double wave_sum_f64(double x) {
  auto add = [&](auto m) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint64_t o = ((uint64_t)lane_xor<m>((uint32_t)(u >> 32)) << 32) | lane_xor<m>((uint32_t)u);
    x += __longlong_as_double((long long)o);
  };
  add(std::integral_constant<int, 1>());
  add(std::integral_constant<int, 2>());
  add(std::integral_constant<int, 4>());
  add(std::integral_constant<int, 8>());
  add(std::integral_constant<int, 16>());
  add(std::integral_constant<int, 32>());
  return x;
}

// A sum and what its roundings lost, so that it does not depend on the order of its terms.
struct Sum64 {
  double sum, lost;
  __device__ __forceinline__ void add(double x) {
    const double next = sum + x, part = next - sum;
    lost += (sum - (next - part)) + (x - part);
    sum = next;
  }
};

// L of each beam that goes on, in 64 bits: the scores again, by the whole workgroup.
template <int WAVES, typename E>
__device__ __forceinline__ void exact_levels(const E* scores, int64_t sw, int W, int V, const double* from,
                                             const bool* over, const float* tops, double* level) {
  __shared__ Sum64 partial[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int w = 0; w < W; ++w) {
    if (!(from[w] > (double)kNegInf) || over[w]) continue;  // uniform
    const E* x = scores + w * sw;
    const double top = (double)tops[w];
    Sum64 sum{0., 0.};
#pragma unroll 4
    for (int v = threadIdx.x; v < V; v += 64 * WAVES) sum.add(exp((double)load_f32(x + v) - top));
    for (int m = 1; m < 64; m *= 2) {
      const double other = __shfl_xor(sum.sum, m, 64), lost = __shfl_xor(sum.lost, m, 64);
      sum.add(other);
      sum.lost += lost;
    }
    if (lane == 0) partial[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < WAVES; ++i) {
        sum.add(partial[i].sum);
        sum.lost += partial[i].lost;
      }
      level[w] = top + log(sum.sum + sum.lost);
    }
    __syncthreads();
  }
}

// A text's W parts lists hold W parts K candidates.  The K-th largest of 64 of them,
// the lists' heads and what follows them (of the lanes' best heads where there are
// more lists), as FP32, bounds the next beams from below: each wavefront finds it for
// itself, and the few candidates that reach it are gathered in LDS and sorted by the
// first one.  Values formed with the FP32 sums' L are off by at most `slack`; where a
// candidate of another beam comes that close to one that is taken, which of them is
// larger (and which is the K-th) is decided with L in 64 bits.  Within a beam L is the
// same and the order right as it is, but for scores whose values 64 bits hold as one
// (scores below 1e-7, totals of 1e9): where all of a list may be taken and its last
// value is also that of the next lower score, every candidate is ranked by its value.
// Of texts of 5 to 16 beams fewer than one in a thousand is decided in 64 bits; a batch
// of 64 of 5 beams over 50257 scores with one of them takes 188 us in place of 23 (one
// workgroup's exponentials in 64 bits).
//   sums, lists  the text's, [W, parts] and [W, parts, K]
//   scores, sw   its first beam's scores, and the beams' stride
//   totals, ended and the outputs  the text's rows
template <int WAVES, typename E>
__device__ __forceinline__ void next_beams(const PartSum* sums, const uint64_t* lists, int parts, const E* scores,
                                           int64_t sw, float slack, const float* totals, const unsigned char* ended,
                                           const Stops& stops, int W, int V, int K, float* new_totals,
                                           int64_t* parents, int64_t* tokens, unsigned char* new_ended) {
  __shared__ double level[kMaxBeams];  // L
  __shared__ double from[kMaxBeams];   // the beam's total; -inf where it cannot go on
  __shared__ float tops[kMaxBeams];    // its largest score
  __shared__ bool over[kMaxBeams];     // ended, and goes on
  constexpr int kCandidates = 64 * WAVES;  // that a text gathers
  __shared__ Key<3> gathered[kCandidates];
  __shared__ int count, again, crowded;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x == 0) count = crowded = 0;
  float highest = lane < W ? totals[lane] : 0.f;  // the largest total above 0
  highest = highest > 0.f && highest < __builtin_inff() ? highest : 0.f;
  for (int w = wave; w < W; w += WAVES) {
    const PartSum* part = sums + w * parts;
    const PartSum mine = lane < parts ? part[lane] : PartSum{kNegInf, 0.f};
    const double total = (double)totals[w];
    const bool end = ended && ended[w];
    float top = mine.top;
    for (int i = lane + 64; i < parts; i += 64) top = fmaxf(top, part[i].top);
    top = wave_max_dpp(top);
    const double at = top == kNegInf ? 0. : (double)top;
    // a part with nothing above -inf summed exp x itself: to 0, or NaN with a NaN
    auto scaled = [&](PartSum s) { return s.top == kNegInf ? (double)s.sum : (double)s.sum * exp((double)s.top - at); };
    double sum = scaled(mine);
    for (int i = lane + 64; i < parts; i += 64) sum += scaled(part[i]);
    sum = wave_sum_f64(sum);
    const double l = at + log(sum);  // NaN with a NaN or +inf among the scores
    if (lane == 0) {
      const bool alive = isfinite(total) && (end || (isfinite(l) && top != kNegInf));
      level[w] = l;
      from[w] = alive ? total : (double)kNegInf;
      tops[w] = top;
      over[w] = alive && end;
    }
  }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(highest > 0.f) != 0, 0)) highest = wave_max_dpp(highest);
  __syncthreads();
  const int stop = stops.n ? stops.token[0] : 0;
  // The head'th candidate of a list: its value, its token (V: none) and its score's
  // order key (0: not by a score).  A beam
  // that has ended or cannot go on has one list: the stop token at the beam's
  // total, the others at -inf.
  auto candidate = [&](int list, int head, int& v, uint32_t& order) {
    const int w = list / parts, part = list % parts;
    const double total = from[w];
    v = V;
    order = 0;
    if (total > (double)kNegInf && !over[w]) {
      const uint64_t key = lists[(w * parts + part) * K + head];
      if (key == 0) return 0.;
      v = (int)~(uint32_t)key;
      order = (uint32_t)(key >> 32);
      return total + ((double)key_value(order) - level[w]);
    }
    if (part != 0) return 0.;
    if (!over[w]) {
      v = head;
    } else if (head == 0) {
      v = stop;
      return total;
    } else {
      v = head - 1 + (head - 1 >= stop ? 1 : 0);
    }
    v = min(v, V);
    return (double)kNegInf;
  };
  auto key_of = [&](uint32_t flat, double value) {
    const uint64_t order = order_key64(value);
    return Key<3>{{(uint32_t)(order >> 32), (uint32_t)order, ~flat}};
  };
  auto flat_of = [&](int list, int v) { return (uint32_t)((list / parts) * V + v); };
  auto value_of = [](Key<3> k) { return key64_value(((uint64_t)k.w[0] << 32) | k.w[1]); };
  auto beam_of = [&](const Key<3>& k) { return (int)(~k.w[2] / (uint32_t)V); };
  const int many = W * parts, all = many * K;
  // wave 0: writes the text's rows
  auto write = [&](const Key<3>& best, int parent, float total) {
    if (lane >= K) return;
    const int v = (int)(~best.w[2] % (uint32_t)V);
    bool stopped = ended && ended[parent];
    for (int i = 0; i < stops.n; ++i) stopped = stopped || stops.token[i] == v;
    new_totals[lane] = total;
    parents[lane] = parent;
    tokens[lane] = v;
    new_ended[lane] = stopped ? 1 : 0;
  };
  // The largest of the keys key_at(c), c < end, by wave 0: the K first lanes' (all of
  // them in order where there are at most 64), and the K-th.
  auto largest = [&](int end, Key<3>& best, Key<3>& last, auto&& key_at) {
    best = last = Key<3>{{0, 0, 0}};
    for (int c0 = 0; c0 < end; c0 += 64) {
      Key<3> k = key_at(c0 + lane);
      if (__builtin_amdgcn_ballot_w64(above(k, last)) == 0) continue;
      wave_sort_first(k, end - c0);
      if (c0 == 0)
        best = k;
      else
        merge_lists(best, backwards(k));
      last = key_of_lane(best, K - 1);
    }
  };
  // Selects the next beams with L as it stands (exact: in 64 bits) from the lists and
  // writes them; with nothing written returns kLevels where L does not decide them,
  // kScan where the lists may not hold them.
  constexpr int kLevels = 1, kScan = 2;
  auto select = [&](auto exact_) {
    constexpr bool exact = decltype(exact_)::value;
    // How far apart the values of two beams' candidates are told apart: the errors of
    // both L, and some steps in 64 bits of the largest number in their sums (a value
    // itself where the totals are none above 0).  In FP32 the values' rounding beside.
    const float apart = exact ? 0.f : 2.f * slack + 0x1p-47f * highest;
    auto margin = [&](double value) { return fma(0x1p-48, fabs(value), (double)apart); };
    auto margin32 = [&](float value) { return fmaf(0x1p-22f, fabsf(value), apart); };
    Key<1> heads{{0}};
    for (int c = lane; c < max(many, min(all, 64)); c += 64) {
      int v;
      uint32_t order;
      const double value = candidate(c % many, c / many, v, order);
      if (v < V) heads.w[0] = max(heads.w[0], order_key((float)value + 0.f));
    }
    wave_sort(heads);
    const uint32_t kth = key_of_lane(heads, K - 1).w[0];
    // the K-th value is not below kth but for its rounding; what is close to it counts too
    const float bound = kth ? key_value(kth) : kNegInf, low = bound - margin32(bound);
    for (int c0 = wave * 64; c0 < all; c0 += 64 * WAVES) {
      const int list = (c0 + lane) % many, head = (c0 + lane) / many;
      int v = V;
      uint32_t order = 0;
      double value = 0.;
      if (c0 + lane < all) value = candidate(list, head, v, order);
      const bool in = v < V && (float)value >= low;
      const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
      if (mask == 0) continue;
      int first = 0;
      if (lane == 0) first = atomicAdd(&count, __builtin_popcountll(mask));
      first = __builtin_amdgcn_readfirstlane(first) + below_me(mask);
      if (in && first < kCandidates) gathered[first] = key_of(flat_of(list, v), value);
      if (__builtin_expect(in && head == K - 1 && order != 0, 0)) {
        // A whole list may be taken.  What it leaves out has no larger value, but an
        // equal one, and a lower token, where 64 bits hold a lower score's as the same.
        const double total = from[list / parts], below = total + ((double)key_value(order - 1) - level[list / parts]);
        if (value - below <= 0x1p-49 * (fabs(value) + fabs(total))) crowded = 1;
      }
    }
    __syncthreads();
    if (wave == 0) {
      const int found = count;
      const bool held = found <= kCandidates;  // else every candidate again, against the best so far
      const int end = held ? found : all;
      auto key_at = [&](int c) {
        if (c >= end) return Key<3>{{0, 0, 0}};
        if (held) return gathered[c];
        int v;
        uint32_t order;
        const int list = c % many;
        const double value = candidate(list, c / many, v, order);
        return v < V ? key_of(flat_of(list, v), value) : Key<3>{{0, 0, 0}};
      };
      Key<3> best, last;
      largest(end, best, last, key_at);
      // Neighbours of two beams that are close, among the K and beyond (all of them
      // where at most 64 were gathered): hardly ever any.
      const int parent = beam_of(best), next_parent = (int)next_lane((uint32_t)parent);
      const double value = value_of(best);
      const float total = (float)value;
      const float drop = total - __uint_as_float(next_lane(__float_as_uint(total)));
      bool close = lane + 1 < min(end, 64) && parent != next_parent && drop <= margin32(total);
      bool repeat = false;
      if (__builtin_expect(!exact && (__builtin_amdgcn_ballot_w64(close) != 0 || end > 64), 0)) {
        // In 64 bits: both among the K, or one at the K-th value?  Values of ended beams
        // are exact, and those at -inf equal.
        const double next = value_of({{next_lane(best.w[0]), next_lane(best.w[1]), 0}});
        close = close && lane < K - 1 && value - next <= margin(value) && !(over[parent] && over[next_parent]);
        const double least = value_of(last);
        const int owner = beam_of(last);
        if (least > (double)kNegInf)
          for (int c0 = 0; c0 < end; c0 += 64) {
            const Key<3> k = key_at(c0 + lane);
            if ((k.w[0] | k.w[1] | k.w[2]) != 0 && above(last, k) && least - value_of(k) <= margin(least)) {
              const int beam = beam_of(k);
              close = close || (beam != owner && !(over[beam] && over[owner]));
            }
          }
        repeat = __builtin_amdgcn_ballot_w64(close) != 0;
      }
      const int next = __builtin_expect(crowded, 0) ? kScan : repeat ? kLevels : 0;
      if (__builtin_expect(next == 0, 1)) write(best, parent, total);
      if (lane == 0) again = next;
    }
    __syncthreads();
    return __builtin_expect(again, 0);
  };
  const int next = select(std::false_type());
  if (next == 0) return;
  exact_levels<WAVES>(scores, sw, W, V, from, over, tops, level);
  if (next == kLevels) {
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    if (select(std::true_type()) == 0) return;
  }
  // Every candidate, by its value: each wavefront's K largest, then the largest of these.
  const uint32_t flats = (uint32_t)W * V;
  Key<3> best{{0, 0, 0}}, last{{0, 0, 0}};
  for (uint32_t f0 = wave * 64; f0 < flats; f0 += 64 * WAVES) {
    Key<3> k{{0, 0, 0}};
    if (f0 + lane < flats) {
      const int w = (int)((f0 + lane) / (uint32_t)V), v = (int)((f0 + lane) % (uint32_t)V);
      double value = (double)kNegInf;
      if (over[w])
        value = v == stop ? from[w] : value;
      else if (from[w] > (double)kNegInf)
        value = from[w] + ((double)load_f32(scores + w * sw + v) - level[w]);
      k = key_of(f0 + lane, value);
    }
    if (__builtin_amdgcn_ballot_w64(above(k, last)) == 0) continue;
    wave_sort(k);
    merge_lists(best, backwards(k));
    last = key_of_lane(best, K - 1);
  }
  gathered[threadIdx.x] = best;
  __syncthreads();
  if (wave != 0) return;
  largest(kCandidates, best, last, [&](int c) { return gathered[c]; });
  write(best, beam_of(best), (float)value_of(best));
}

// The arguments of text i: its rows of each array.
struct Beams {
  const float* totals;
  const unsigned char* ended;
  float* new_totals;
  int64_t *parents, *tokens;
  unsigned char* new_ended;
};

template <int WAVES, typename E>
__device__ __forceinline__ void next_beams_of(int64_t i, const PartSum* sums, const uint64_t* lists, int parts,
                                              const E* scores, int64_t sn, int64_t sw, float slack, const Beams& a,
                                              const Stops& stops, int W, int V, int K) {
  next_beams<WAVES>(sums, lists, parts, scores + i * sn, sw, slack, a.totals + i * W,
                    a.ended ? a.ended + i * W : nullptr, stops, W, V, K, a.new_totals + i * K, a.parents + i * K,
                    a.tokens + i * K, a.new_ended + i * K);
}

template <int WAVES, typename E>
__global__ __launch_bounds__(64 * WAVES) void beam_merge(const PartSum* __restrict__ sums,
                                                         const uint64_t* __restrict__ lists, int W, int V, int K,
                                                         int parts, const E* __restrict__ scores, int64_t sn,
                                                         int64_t sw, float slack, Beams a, Stops stops) {
  const int64_t i = blockIdx.x, first = i * W * parts;
  next_beams_of<WAVES>(i, sums + first, lists + first * K, parts, scores, sn, sw, slack, a, stops, W, V, K);
}

// A text of few scores in one launch: a wavefront a part, the lists in LDS.
constexpr int kTextWaves = 16, kTextItems = 32;

template <typename E>
__global__ __launch_bounds__(64 * kTextWaves) void beam_text(const E* __restrict__ scores, int64_t sn, int64_t sw,
                                                             int W, int V, int K, int parts, float slack, Beams a,
                                                             Stops stops) {
  __shared__ uint64_t gathered[kTextWaves][kGathered];
  __shared__ uint64_t lists[kTextWaves * kMaxBeams];
  __shared__ PartSum sums[kTextWaves];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (w < W * parts)
    part_list<E, kTextItems>(scores + (int64_t)blockIdx.x * sn + (int64_t)(w / parts) * sw, V, w % parts, K,
                             gathered[w], sums + w, lists + w * K);
  __syncthreads();
  next_beams_of<kTextWaves>(blockIdx.x, sums, lists, parts, scores, sn, sw, slack, a, stops, W, V, K);
}

// The parts of a beam in beam_text, or 0 where the text takes two launches: where a
// workgroup's wavefronts do not hold its parts, or the texts outnumber the compute
// units.  Measured, us, in a graph and from a program, one launch and two: one text of
// 4 beams over 8192 scores 9.0, 8.3 and 13.9, 17.7; 200 texts 9.8, 11.5 and 13.5, 17.4;
// 8 beams over 4000 11.0, 9.8 and 13.8, 18.1; 16 over 2000 13.8, 12.3 and 13.7, 17.6.
// The rule goes by a program's calls, whose host time it saves; in a graph a few texts
// are 0.7 to 1.5 us slower by it.
int text_parts(int n, int W, int V) {
  const int64_t parts = ((int64_t)V + 64 * kTextItems - 1) / (64 * kTextItems);
  return W * parts <= kTextWaves && n <= compute_units() ? (int)parts : 0;
}

// What the FP32 sums may put a beam's L = log S off by.  A term exp(x - top): the
// argument's rounding, log2 e's and their product's, at most 2.3 2^-24 |x - top|, whose
// mean over the terms is at most log V (their entropy less log S); the exponential, one
// step, 2 2^-24; and a part's 24 additions in turn (at most 18 of a lane's, 6 across
// the lanes), 2^-24 each of terms of one sign.  The parts are joined in 64 bits.
float level_slack(int V) { return (float)((3. * std::log((double)V) + 33.) * 0x1p-24); }

// Scores a lane of a part: 64 where the parts of 4096 fill the GPU, 16 where
// they do not, so that few rows are spread over it.
int part_items(int64_t rows, int V) {
  return rows * (((int64_t)V + 4095) / 4096) >= 4 * (int64_t)compute_units() ? 64 : 16;
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
  if ((int64_t)W * V > (1 << 28) || (int64_t)n * W > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "beam_workspace: n=%d W=%d V=%d is too large", n, W, V);
  if (text_parts(n, W, V)) {
    *bytes = 0;
    return WPTV_OK;
  }
  const int part = 64 * part_items((int64_t)n * W, V);
  if ((int64_t)n * W * (((int64_t)V + part - 1) / part) > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "beam_workspace: n=%d W=%d V=%d is too large", n, W, V);
  *bytes = (size_t)n * W * (((int64_t)V + part - 1) / part) * (sizeof(PartSum) + (size_t)K * sizeof(uint64_t));
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
  if (!scores || !totals || !new_totals || !parents || !tokens || !new_ended || (need && !workspace))
    return fail(WPTV_E_INVALID, "beam_step: a required pointer is NULL");
  if (workspace_bytes < need)
    return fail(WPTV_E_INVALID, "beam_step: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const Beams beams{totals, ended, new_totals, parents, tokens, new_ended};
  const float slack = level_slack(V);
  if (const int parts = text_parts(n, W, V)) {
    if (scores_dtype == WPTV_F32)
      beam_text<<<n, 64 * kTextWaves, 0, stream>>>(static_cast<const float*>(scores), scores_stride_n, scores_stride_w,
                                                   W, V, K, parts, slack, beams, s);
    else
      beam_text<<<n, 64 * kTextWaves, 0, stream>>>(static_cast<const unsigned short*>(scores), scores_stride_n,
                                                   scores_stride_w, W, V, K, parts, slack, beams, s);
    return launched("beam_text");
  }
  const int items = part_items((int64_t)n * W, V), parts = (int)(((int64_t)V + 64 * items - 1) / (64 * items));
  const int64_t waves = (int64_t)n * W * parts, blocks = (waves + kPartWaves - 1) / kPartWaves;
  PartSum* sums = static_cast<PartSum*>(workspace);
  uint64_t* lists = reinterpret_cast<uint64_t*>(sums + waves);
#define WPTV_PARTS(E, ITEMS)                                                                                      \
  beam_parts<E, ITEMS><<<(unsigned)blocks, 64 * kPartWaves, 0, stream>>>(                                         \
      static_cast<const E*>(scores), scores_stride_n, scores_stride_w, W, V, K, parts, waves, sums, lists)
  if (scores_dtype == WPTV_F32) {
    if (items == 64) WPTV_PARTS(float, 64); else WPTV_PARTS(float, 16);
  } else {
    if (items == 64) WPTV_PARTS(unsigned short, 64); else WPTV_PARTS(unsigned short, 16);
  }
#undef WPTV_PARTS
  const int launch = launched("beam_parts");
  if (launch != WPTV_OK) return launch;
#define WPTV_MERGE(WAVES, E)                                                                                       \
  beam_merge<WAVES, E><<<n, 64 * WAVES, 0, stream>>>(sums, lists, W, V, K, parts, static_cast<const E*>(scores),   \
                                                     scores_stride_n, scores_stride_w, slack, beams, s)
  const bool few = (int64_t)W * parts * K <= 4096;
  if (scores_dtype == WPTV_F32) {
    if (few) WPTV_MERGE(8, float); else WPTV_MERGE(16, float);
  } else {
    if (few) WPTV_MERGE(8, unsigned short); else WPTV_MERGE(16, unsigned short);
  }
#undef WPTV_MERGE
  return launched("beam_merge");
}
