// A mixture of experts for the few tokens of a verify step, for gfx950: the
// router's choice (wptv_route) and the experts' products (wptv_experts).
//
//   l[m, e]  = x[m] . router[e]                              in 64 bits
//   chosen   = the k experts of the largest l + bias, gates = softmax of their l
//   y[m]     = sum_j gates[m, j] down_e (silu(gate_e x[m]) * (up_e x[m])),  e = chosen[m, j]
//
// Every (token, choice) is a "pair" p = m k + j.  What bounds the products is
// the stream of the experts' weights, read once each: a pair adds a column to a
// matrix instruction that its expert's weights feed anyway.
//
// Each product is one launch over all experts, in a form by the counts:
//   expert_columns  few tokens, or few row blocks: a workgroup a pair of 16-row
//                   blocks, its wavefronts sharing out the width
//   expert_tiles    more: a pair of blocks a wavefront, the tokens through LDS
//   expert_rows     the down product of a few tokens, joined in the same launch
// then join_experts, or the residual norm, adds a token's terms.  Kernels, us: 160
// rows (120 of them read), 8 of 64 experts of 704 features, width 2048 (0.55 GB):
// products 70 and 36 (5.2 and 5.1 TB/s), router 5 and 5, join 5; one row 12 and 7;
// 512 rows (384 read) over 128 experts (1.1 GB) 141 and 85.
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// ---- the packed weights ------------------------------------------------------
//
// An expert's matrix [N, K] as 1 KiB blocks of 16 rows by KU columns (32 in bf16,
// 16 in FP32), block (rb, ks) at rb KS + ks: lane l = 16 g + j holds row 16 rb + j,
// columns KU ks + EPL g .. + EPL - 1, its operand of one matrix instruction (four
// in FP32, a column of each lane's four at a time: the order of a sum's columns is
// free as long as both operands share it).  A wavefront's weights are then one
// contiguous stream, loaded straight into registers.  Rows and columns are padded
// with zeros.
template <typename T>
struct Operand;

template <>
struct Operand<unsigned short> {
  static constexpr int KU = 32, EPL = 8;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};

template <>
struct Operand<float> {
  static constexpr int KU = 16, EPL = 4;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
};

__host__ __device__ __forceinline__ int padded(int x, int unit) { return (x + unit - 1) / unit * unit; }

// The sizes of the packed matrices: the features padded to the down product's
// column unit, its outputs to two row blocks.
struct ExpertShape {
  int D, F, unit, Fp, KSx, KSf, FB, DB;  // KSx, KSf: k-steps of the two products; FB, DB: their row-block pairs
};

__host__ __device__ __forceinline__ ExpertShape expert_shape(int D, int F, int dtype) {
  const int unit = dtype == WPTV_BF16 ? 32 : 16;
  ExpertShape s;
  s.D = D;
  s.F = F;
  s.unit = unit;
  s.Fp = padded(F, unit);
  s.KSx = padded(D, unit) / unit;
  s.KSf = s.Fp / unit;
  s.FB = s.Fp / 16;
  s.DB = padded(D, 32) / 32;
  return s;
}

// One thread a lane's 16 bytes of one expert's matrix.  PAIRED: row blocks 2 f and
// 2 f + 1 hold the gate and the up rows of features 16 f .. 16 f + 15 (w holds the
// N gate rows, then the N up rows).
template <typename T, bool PAIRED>
__global__ __launch_bounds__(256) void pack_experts(const T* __restrict__ w, int N, int K, int blocks, int KS,
                                                    bool whole, u32x4* __restrict__ out) {
  using O = Operand<T>;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= (int64_t)blocks * KS * 64) return;
  const int lane = (int)(item & 63), ks = (int)((item >> 6) % KS), rb = (int)((item >> 6) / KS);
  const int row = 16 * (PAIRED ? rb >> 1 : rb) + (lane & 15), col = O::KU * ks + O::EPL * (lane >> 4);
  union {
    T element[O::EPL];
    u32x4 all;
  } v;
  v.all = u32x4{0u, 0u, 0u, 0u};
  if (row < N && col < K) {
    const int64_t rows = PAIRED ? 2 * (int64_t)N : N;
    const T* from = w + ((int64_t)blockIdx.y * rows + row + (PAIRED && (rb & 1) ? N : 0)) * K + col;
    if (whole) {  // rows of whole, aligned 16 bytes
      v.all = *reinterpret_cast<const u32x4*>(from);
    } else {
#pragma unroll
      for (int i = 0; i < O::EPL; ++i)
        if (col + i < K) v.element[i] = from[i];
    }
  }
  out[(int64_t)blockIdx.y * blocks * KS * 64 + item] = v.all;
}

// ---- the router --------------------------------------------------------------

// An order-preserving key of a value in 64 bits: a NaN the largest, -0 as 0.
__device__ __forceinline__ uint64_t order_key64(double f) {
  if (f != f) return ~0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(f + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// The key an expert is ranked by; 0, below every key, where its bias takes it out,
// whatever its logit (NaN - inf and inf - inf would be the largest).
__device__ __forceinline__ uint64_t expert_key(double logit, const float* __restrict__ bias, int e) {
  if (!bias) return order_key64(logit);
  const float b = bias[e];
  return b == -__builtin_inff() ? 0 : order_key64(logit + (double)b);
}

constexpr int kMaxExperts = 512, kMaxChosen = 16;

// A token's choices and gates by one wavefront (every lane calls): lane l holds the
// logits of experts l, l + 64, ... and their keys (0, below every key, past the
// last).  k times the largest key left, the lowest expert of equal ones; the softmax
// of the chosen logits in 64 bits.
template <int SLOTS>
__device__ __forceinline__ void choose_experts(const double (&logit)[SLOTS], uint64_t (&key)[SLOTS], int k,
                                               int* __restrict__ chosen, float* __restrict__ gates) {
  const int lane = threadIdx.x & 63;
  const uint64_t none = order_key64(-__builtin_inf());
  int mine = -1;  // lane i keeps choice i
  double l = -__builtin_inf();
  for (int i = 0; i < k; ++i) {
    uint64_t best = key[0];
#pragma unroll
    for (int s = 1; s < SLOTS; ++s) best = key[s] > best ? key[s] : best;
    const int flip = INT_MIN;  // signed maxima of unsigned halves
    const int high = wave_max_i32((int)(best >> 32) ^ flip);
    const int low = wave_max_i32((int)(best >> 32 ^ (unsigned)flip) == high ? (int)(uint32_t)best ^ flip : INT_MIN);
    const uint64_t top = (uint64_t)(unsigned)(high ^ flip) << 32 | (unsigned)(low ^ flip);
    if (top <= none) break;
    int e = -1;
    double its = 0.;
#pragma unroll
    for (int s = SLOTS - 1; s >= 0; --s) {
      const uint64_t same = __builtin_amdgcn_ballot_w64(key[s] == top);
      if (same) {
        const int at = __builtin_ctzll(same);
        e = 64 * s + at;
        its = __shfl(logit[s], at, 64);
      }
    }
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (e == 64 * s + lane) key[s] = 0;
    if (lane == i) {
      mine = e;
      l = its;
    }
  }
  double most = l;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) most = fmax(most, __shfl_xor(most, o, 64));
  const double share = mine < 0 ? 0. : exp(l - most);  // a NaN among them, or +inf, makes the total one
  double total = share;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
  if (lane < k) {
    chosen[lane] = mine;
    gates[lane] = mine < 0 ? 0.f : (float)(share / total);
  }
}

constexpr int kAhead = 4;  // steps whose loads a wavefront waits for together

template <typename T>
__device__ __forceinline__ void load_four(const T* p, float* to) {
  typedef T four __attribute__((ext_vector_type(4)));
  const four v = *reinterpret_cast<const four*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T x = v[i];
    to[i] = load_f32<T>(&x);
  }
}

// A small router in one launch: a workgroup a token, `lanes` of its threads (a power
// of two up to 64, as many as kTokenThreads gives each expert) an expert.  Few lanes an
// expert keep the sums between them short: by whole wavefronts, one CU's LDS moves
// every expert's six 64-bit exchanges (in a graph, us: 16 tokens, 72 experts of 104
// 14.9 -> 5.8; 160 tokens, 64 of 256 8.2 -> 6.2; 512 of 32 30.7 -> 8.3; 256 threads and
// 1024 4.8, 5.3 at 8 of 256, 512 4.9).
constexpr int kTokenThreads = 512;

template <typename T, int SLOTS>
__global__ __launch_bounds__(kTokenThreads) void route_token(const T* __restrict__ x,
                                                             const float* __restrict__ router,
                                                             const float* __restrict__ bias,
                                                             const int64_t* __restrict__ counts, int per_row, int D,
                                                             int E, int lanes, int k, int* __restrict__ chosen,
                                                             float* __restrict__ gates) {
  __shared__ double logit[64 * SLOTS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t m = blockIdx.x;
  const T* row = x + m * D;
  const int e = tid / lanes, piece = tid % lanes;
  const float* w = router + (int64_t)min(e, E - 1) * D;
  double sum = 0.;
  for (int first = 4 * piece; first - 4 * piece < D; first += kAhead * 4 * lanes) {
    float a[kAhead][4], b[kAhead][4];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {  // all asked for at once; past the width nothing is added
      const int d = first + 4 * lanes * u < D ? first + 4 * lanes * u : 0;
      load_four<float>(w + d, a[u]);
      load_four<T>(row + d, b[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (first + 4 * lanes * u < D)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fma((double)a[u][i], (double)b[u][i], sum);
  }
  for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (piece == 0 && e < E) logit[e] = sum;
  __syncthreads();
  if (tid >= 64) return;
  const bool read = !counts || m % per_row < counts[m / per_row];
  double own[SLOTS];
  uint64_t key[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 64 * s;
    own[s] = e < E ? logit[e] : 0.;
    key[s] = read && e < E ? expert_key(own[s], bias, e) : 0;
  }
  choose_experts<SLOTS>(own, key, k, chosen + m * k, gates + m * k);
}

typedef double f64x4 __attribute__((ext_vector_type(4)));

// The logits of a wider one on the 64-bit matrix instruction (16 experts by 16
// tokens by 4 columns; the product of two FP32 values is exact): grid (E / 16,
// rows / 16, splits), workgroup z's four wavefronts taking the 32-column steps
// 4 z + wv, 4 z + wv + 4 splits, ...; sums[z] [rows, E] in 64 bits.  A lane's eight
// neighbouring columns are the step's eight instructions.  The loads bound it, rows of
// 64 bytes and more at a time (512 tokens, 128 experts of 2048, both launches: four
// columns a lane and four steps ahead 18.5 us, eight columns and four steps 18.2, two
// 16.9, one 16.7; 160 tokens, 64 experts 9.8 to 10.3, 11.4, 9.9, 9.3 to 9.8).
template <typename T>
__global__ __launch_bounds__(256) void route_logits(const T* __restrict__ x, const float* __restrict__ router, int rows,
                                                    int D, int E, double* __restrict__ sums) {
  __shared__ double red[4][256];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, j = lane & 15, g = lane >> 4;
  const int e0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const float* w = router + (int64_t)min(e0 + j, E - 1) * D;
  const T* row = x + (int64_t)min(m0 + j, rows - 1) * D;
  f64x4 acc = {0., 0., 0., 0.};
  const int steps = (D + 31) / 32;
  for (int step = 4 * (int)blockIdx.z + __builtin_amdgcn_readfirstlane(wv); step < steps; step += 4 * (int)gridDim.z) {
    const int d = 32 * step + 8 * g;
    const bool inside = d < D;  // past the width zeros
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      load_four<float>(w + (inside ? d + i : 0), a + i);
      load_four<T>(row + (inside ? d + i : 0), b + i);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64(inside ? (double)a[i] : 0., inside ? (double)b[i] : 0., acc, 0, 0, 0);
  }
  // register i of lane (j, g): expert 4 i + g, token j
#pragma unroll
  for (int i = 0; i < 4; ++i) red[wv][j * 16 + 4 * i + g] = acc[i];
  __syncthreads();
  const int m = m0 + (tid >> 4), e = e0 + (tid & 15);
  if (m < rows && e < E)
    sums[((int64_t)blockIdx.z * rows + m) * E + e] = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
}

// A wavefront a token.
template <int SLOTS>
__global__ __launch_bounds__(256) void route_choose(const double* __restrict__ sums, const float* __restrict__ bias,
                                                    const int64_t* __restrict__ counts, int rows, int per_row, int E,
                                                    int splits, int k, int* __restrict__ chosen,
                                                    float* __restrict__ gates) {
  const int lane = threadIdx.x & 63, m = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (m >= rows) return;
  const bool read = !counts || m % per_row < counts[m / per_row];
  double own[SLOTS];
  uint64_t key[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) own[s] = 0.;
  for (int z = 0; z < splits; z += 4) {
    double part[4][SLOTS];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s)
        part[u][s] = sums[((int64_t)min(z + u, splits - 1) * rows + m) * E + min(lane + 64 * s, E - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) own[s] += z + u < splits ? part[u][s] : 0.;
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = lane + 64 * s;
    key[s] = read && e < E ? expert_key(own[s], bias, e) : 0;
  }
  choose_experts<SLOTS>(own, key, k, chosen + (int64_t)m * k, gates + (int64_t)m * k);
}

// The most parts the width is cut into: two steps a wavefront each.
int64_t route_parts(int D) { return D > 32 * 256 ? 32 : (D + 255) / 256; }

// The router's form: 0, one launch, where a token's workgroup and all of them together
// read little, else the parts the width is cut into (the tiles of 16 by 16 cover the
// compute units twice).  One launch and two, us: 160 tokens, 128 experts of 256 7.6, 9.4,
// 16 of 2048 6.4, 8.0; 256 of 256 12.7, 11.1; 1 token, 500 of 64 9.4, 7.9; 512 tokens, 64
// of 256 6.9, 7.9, 128 of 256 10.6, 9.6; 2000 tokens, 8 of 256 8.6, 7.7, 8 of 2048 13.5,
// 10.9.
int route_splits(int64_t rows, int D, int E) {
  const int64_t size = (int64_t)E * D;
  if (rows <= 1024 && size <= (E <= 128 ? 32768 : 16384) && rows * size <= (1 << 23)) return 0;
  const int64_t tiles = (rows + 15) / 16 * ((E + 15) / 16);
  const int64_t want = 512 / tiles, most = route_parts(D);
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

// ---- the experts' products ---------------------------------------------------

// A buffer of up to 2 GiB, read 16 bytes a lane at a lane's offset and a uniform
// one, both unsigned bytes; past the end a load gives zeros, and kOutside is past
// every end.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr unsigned kOutside = 0x80000000u;
constexpr int64_t kBufferBytes = 0x7fffff00;

__device__ __forceinline__ Buffer buffer(const void* base, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ u32x4 load16(Buffer from, unsigned lane_offset, unsigned offset) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, lane_offset, offset, 0));
}

// Weights that one workgroup reads (ONCE): no cache line is kept for them.
template <bool ONCE>
__device__ __forceinline__ u32x4 load16_weights(Buffer from, unsigned lane_offset, unsigned offset) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, lane_offset, offset, ONCE ? 2 : 0));
}

enum Product { kGateUp = 0, kDown = 1 };

// The pairs of a range [r0, r0 + RANGE) that one expert takes, in their order,
// listed by a workgroup of WAVES wavefronts, a stretch of the range each.
template <int WAVES, int RANGE>
struct PairList {
  static constexpr int kTurns = RANGE / WAVES / 64;
  uint16_t list[RANGE];
  int listed[WAVES];

  // A thread's choices of a range (loaded ahead of other loads, whose arrival the
  // list then does not wait for).
  struct Choices {
    int c[kTurns];
  };

  static __device__ __forceinline__ int turns(int here) { return (here + 64 * WAVES - 1) / (64 * WAVES); }

  static __device__ __forceinline__ void load(Choices& choices, const int* __restrict__ chosen, int r0, int pairs) {
    // the stretches follow the pairs' count, in whole wavefronts, so that a few pairs are listed by all at once
    const int here = min(pairs - r0, RANGE), many = turns(here);
    const int at = (threadIdx.x >> 6) * many * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      if (i < many) choices.c[i] = chosen[r0 + min(at + 64 * i, here - 1)];
  }

  // Lists expert e's pairs, counted from r0 (e == E: those of no expert), and
  // returns their count.  Ends with a barrier.
  __device__ __forceinline__ int fill(const Choices& choices, int r0, int pairs, int e, int E) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const uint64_t below = (1ull << lane) - 1ull;
    const int here = min(pairs - r0, RANGE), many = turns(here), begin = wv * many * 64;
    auto mine = [&](int i) {
      const int c = choices.c[i];
      return begin + 64 * i + lane < here && (c == e || (e == E && (unsigned)c >= (unsigned)E));
    };
    int n = 0;
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      if (i < many) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine(i)));
    if (lane == 0) listed[wv] = n;
    __syncthreads();
    int total = 0, at = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      at += w < wv ? listed[w] : 0;
      total += listed[w];
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      if (i < many) {
        const uint64_t found = __builtin_amdgcn_ballot_w64(mine(i));
        if (mine(i)) list[at + __builtin_popcountll(found & below)] = (uint16_t)(begin + 64 * i + lane);
        at += __builtin_popcountll(found);
      }
    __syncthreads();
    return total;
  }
};

// A workgroup's column of row blocks, list of pairs and tile of that list's tokens,
// of a grid in one dimension (product_grid): the tiles of one expert's rows follow
// each other on one XCD (workgroup i runs on XCD i mod 8), whose cache then gives
// the weights to all of them.
struct Place {
  int column, list, tile;
};

__device__ __forceinline__ Place product_place(int columns, int tiles) {
  const int id = blockIdx.x, t = id >> 3, at = t / tiles * 8 + (id & 7);
  return Place{at % columns, at / columns, t % tiles};
}

inline unsigned product_grid(int columns, int lists, int tiles) {
  return (unsigned)(((int64_t)columns * lists + 7) / 8 * 8 * tiles);
}

// The k-steps of one of the `cuts` that the down product's columns are cut into
// (product_cuts), whose sums the join adds in order; the gate/up product's are whole.
struct Cut {
  int first, steps;
};

template <int PRODUCT>
__device__ __forceinline__ Cut product_cut(int KS, int cut, int cuts) {
  if constexpr (PRODUCT == kGateUp) return Cut{0, KS};
  const int most = (KS + cuts - 1) / cuts;
  return Cut{cut * most, min(most, KS - cut * most)};
}

// The parts' rows that no expert of the range writes, cleared by `waves` (at least
// one) wavefronts of their own, one after the other a row each.
__device__ __forceinline__ void clear_rows(const uint16_t* pairs, int n, int r0, int wave, int waves, int first,
                                           int last, int D, int64_t total, int k, float* __restrict__ parts) {
  for (int i = wave; i < n; i += waves) {
    const int p = r0 + pairs[i];
    float* to = parts + ((p % k) * total + p / k) * D;
    for (int d = first + 4 * (threadIdx.x & 63); d < min(D, last); d += 256)
      *reinterpret_cast<f32x4*>(to + d) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// What the two products store.  The gate scales silu(g) u before its one rounding,
// which is a relative one: the down product's sums are then the gated terms.  bf16
// operands are what the caller's dtype asks for (a layer is 0.0023 of its size from 64
// bits, 0.0016 with this product in FP32).
template <typename T, int PRODUCT>
__device__ __forceinline__ void store_block(f32x4 a, f32x4 b, int p, int block, int g, const ExpertShape& shape,
                                            int64_t total, int k, const float* __restrict__ gates,
                                            void* __restrict__ out) {
  if constexpr (PRODUCT == kGateUp) {
    const float gate = gates[p];
    T* to = static_cast<T*>(out) + (int64_t)p * shape.Fp + 16 * block + 4 * g;
    union {
      T element[4];
      unsigned int word[sizeof(T)];
    } v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.element[i] = from_f32<T>(a[i] / (1.f + expf(-a[i])) * b[i] * gate);
    typedef unsigned int words __attribute__((ext_vector_type(sizeof(T))));
    *reinterpret_cast<words*>(to) = *reinterpret_cast<const words*>(v.word);
  } else {
    float* to = static_cast<float*>(out) + ((p % k) * total + p / k) * shape.D + 32 * block + 4 * g;
    const int left = shape.D - 32 * block - 4 * g;
    if (left > 0) *reinterpret_cast<f32x4*>(to) = a;
    if (left > 16) *reinterpret_cast<f32x4*>(to + 16) = b;
  }
}

// A workgroup's four wavefronts share out the k-steps of one row-block pair of one
// expert's matrix (their sums joined in LDS, in order), over tiles of 16 NT of the
// expert's tokens.  The weights are the A operand, the tokens the B operand, both
// straight from memory into registers, kDepth k-steps ahead: three keep the stream
// going and leave room for four workgroups a compute unit (6 tokens, 8 of 64 experts
// of 704, whole layers: 8 ahead 81 us, 6 73, 4 71, 3 69).
//   kGateUp   x [rows, D] -> act [pairs, Fp]: gates[p] silu(g) u of the FP32 sums,
//             rounded once to T, which the down product takes
//   kDown     act -> parts [k, rows, D] FP32
// BY_PAIR (fewer pairs than experts): a workgroup serves the expert of one pair, if
// that is the expert's first.
template <typename T, int PRODUCT, int NT, int WAVES, bool BY_PAIR, bool ONCE>
__global__ __launch_bounds__(64 * WAVES) void expert_columns(const T* __restrict__ in,
                                                             const u32x4* __restrict__ weights,
                                                             const int* __restrict__ chosen,
                                                             const float* __restrict__ gates, ExpertShape shape,
                                                             int rows, int64_t total, int E, int k, int clears,
                                                             int lists, int tiles, int cuts, void* __restrict__ out) {
  using O = Operand<T>;
  // a list of its own a wavefront, for fewer than kMaxExperts pairs; 16 tokens have up to 256 pairs
  constexpr int kDepth = 3, kRange = BY_PAIR ? WAVES * kMaxExperts : NT == 1 ? 1024 : 4096;
  typedef PairList<WAVES, kRange> List;
  __shared__ List list;
  __shared__ float red[WAVES * NT * 2 * 4 * 64];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pairs = rows * k;
  const Place place = product_place((PRODUCT == kGateUp ? shape.FB : shape.DB) * cuts, tiles);
  if (place.list >= lists) return;
  int e = BY_PAIR ? chosen[place.list] : place.list < clears ? E : place.list - clears;
  e = __builtin_amdgcn_readfirstlane(e);
  if ((unsigned)e >= (unsigned)E) e = E;  // no expert
  const int KS = PRODUCT == kGateUp ? shape.KSx : shape.KSf;
  const unsigned width = (PRODUCT == kGateUp ? shape.D : shape.Fp) * sizeof(T);
  const int block = place.column / cuts, blocks = PRODUCT == kGateUp ? shape.FB : shape.DB;
  const Cut cut = product_cut<PRODUCT>(KS, place.column % cuts, cuts);
  const unsigned limit = width - 64 * cut.first;
  const int steps = (cut.steps - wv + WAVES - 1) / WAVES;
  const Buffer w = buffer(weights + ((int64_t)min(e, E - 1) * blocks + block) * 2 * KS * 64 + cut.first * 64,
                          (2u * KS - cut.first) * 1024);
  const Buffer x = buffer(reinterpret_cast<const char*>(in) + 64 * cut.first,
                          (unsigned)((PRODUCT == kGateUp ? rows : pairs) * width - 64 * cut.first));
  if constexpr (PRODUCT == kDown) out = static_cast<float*>(out) + (place.column % cuts) * k * total * shape.D;
  u32x4 wb[kDepth][2], xb[kDepth][NT];
  auto load_weights = [&](int d, int s) {
    const unsigned ks = wv + WAVES * s;
    wb[d][0] = load16_weights<ONCE>(w, 16 * lane, 1024 * ks);
    wb[d][1] = load16_weights<ONCE>(w, 16 * lane, 1024 * (KS + ks));
  };
  // a few pairs: the first weights are asked for before the expert's tokens are known (one token's layer 32.0 -> 30.1
  // us; with more of them the registers cost more than it gives, 16 tokens over wide experts 101 -> 103)
  if constexpr (BY_PAIR) {
    if (e < E && steps > 0) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) load_weights(d, min(d, steps - 1));
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  for (int r0 = 0; r0 < pairs; r0 += kRange) {
    const uint16_t* mine = list.list;
    int n = 0;
    if constexpr (BY_PAIR) {  // fewer pairs than 512: every wavefront lists them for itself
      uint16_t* own = list.list + wv * kMaxExperts;
      for (int p = lane; p - lane < pairs; p += 64) {
        const int c = chosen[min(p, pairs - 1)];
        const bool same = p < pairs && (c == e || (e == E && (unsigned)c >= (unsigned)E));
        const uint64_t found = __builtin_amdgcn_ballot_w64(same);
        if (__builtin_amdgcn_ballot_w64(same && p < place.list)) return;  // an earlier pair's workgroup serves it
        if (same) own[n + __builtin_popcountll(found & ((1ull << lane) - 1ull))] = (uint16_t)p;
        n += __builtin_popcountll(found);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      mine = own;
    } else {
      typename List::Choices choices;
      list.load(choices, chosen, r0, pairs);
      n = list.fill(choices, r0, pairs, e, E);
    }
    if (e == E) {
      if (PRODUCT == kDown && clears > 0 && place.tile == 0)
        clear_rows(mine, n, r0, BY_PAIR ? wv : place.list * WAVES + wv, BY_PAIR ? WAVES : clears * WAVES, 32 * block,
                   32 * block + 32, shape.D, total, k, static_cast<float*>(out));
      __syncthreads();
      continue;
    }
    for (int first = 16 * NT * place.tile; first < n; first += 16 * NT * tiles) {
      int pair[NT];
      unsigned row[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        // columns past the last token repeat it; nothing of them is stored
        pair[t] = r0 + mine[min(first + 16 * t + j, n - 1)];
        row[t] = (PRODUCT == kGateUp ? pair[t] / k : pair[t]) * width + 16 * g;
      }
      f32x4 acc[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      auto load_tokens = [&](int d, int s) {
        const unsigned ks = wv + WAVES * s;
#pragma unroll
        for (int t = 0; t < NT; ++t)  // columns past the width are zero, as the weights' padding
          xb[d][t] = load16(x, 64 * ks + 16 * g < limit ? row[t] : kOutside, 64 * ks);
      };
      auto multiply = [&](int d) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[t][0] = O::mfma(wb[d][0], xb[d][t], acc[t][0]);
          acc[t][1] = O::mfma(wb[d][1], xb[d][t], acc[t][1]);
        }
      };
      if (steps > 0) {
        if (!BY_PAIR || first > 0) {
#pragma unroll
          for (int d = 0; d < kDepth; ++d) load_weights(d, min(d, steps - 1));
        }
#pragma unroll
        for (int d = 0; d < kDepth; ++d) load_tokens(d, min(d, steps - 1));
        int s = 0;
        for (; s + kDepth <= steps; s += kDepth) {
#pragma unroll
          for (int d = 0; d < kDepth; ++d) {
            multiply(d);
            __builtin_amdgcn_sched_barrier(0);
            load_weights(d, min(s + kDepth + d, steps - 1));
            load_tokens(d, min(s + kDepth + d, steps - 1));
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int d = 0; d < kDepth; ++d)
          if (s + d < steps) multiply(d);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) red[((wv * NT + t) * 8 + i) * 64 + lane] = acc[t][i >> 2][i & 3];
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (t % WAVES == wv && first + 16 * t + j < n) {
          float sum[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sum[i] = red[(t * 8 + i) * 64 + lane];
#pragma unroll
            for (int u = 1; u < WAVES; ++u) sum[i] += red[((u * NT + t) * 8 + i) * 64 + lane];
          }
          store_block<T, PRODUCT>(f32x4{sum[0], sum[1], sum[2], sum[3]}, f32x4{sum[4], sum[5], sum[6], sum[7]}, pair[t],
                                  block, g, shape, total, k, gates, out);
        }
      __syncthreads();
    }
    __syncthreads();  // the lists are written again
  }
}

// A workgroup's four wavefronts take a row-block pair of one expert's matrix each,
// over tiles of up to 64 of the expert's tokens.  The tokens' columns go through LDS,
// kChunk k-steps at a time in two buffers, in the order the matrix instructions take
// them; the weights go straight from memory into registers, DEPTH k-steps ahead,
// across the chunks' barriers, which wait for LDS alone.  Whole layers, us, of 160
// and of 512 rows (above): eight wavefronts a workgroup 135, 291, four 125, 254; tiles
// of 32 tokens 138, 314, of 48 132, 270, of 64 125, 255; weights kept in the caches
// 131, 263.  Up to 2048 pairs, shorter lists and two k-steps ahead let four workgroups
// share a compute unit in place of three: 160 rows 124 -> 119.  With hundreds of tokens
// an expert LDS and the cache bound it: 8 matrix instructions take 4 KiB of tokens and
// 2 KiB of weights (4096 tokens of 2048, 8 of 64 experts of 704 278 TFLOP/s).  A sum runs
// along the whole width in one chain.
constexpr int kTileWaves = 4, kTileTokens = 4, kChunk = 4;

// A tile of NT times 16 tokens, `first` the list's place of the first.
template <typename T, int PRODUCT, int NT, int DEPTH, bool ONCE>
__device__ __forceinline__ void tile_pass(Buffer in, Buffer w, int KS, int steps, unsigned width, unsigned limit,
                                          const uint16_t* list,
                                          u32x4 (*xs)[kTileTokens * kChunk * 64], int r0, int first, int n, int block,
                                          bool live, const ExpertShape& shape, int64_t total, int k,
                                          const float* __restrict__ gates, void* __restrict__ out) {
  using O = Operand<T>;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  u32x4 wb[DEPTH][2], xr[NT];
  const unsigned at = live ? 16 * lane : kOutside;  // wavefronts past the last row blocks load nothing
  auto load = [&](int d, int s) {
    const unsigned ks = min(s, steps - 1);
    wb[d][0] = load16_weights<ONCE>(w, at, 1024 * ks);
    wb[d][1] = load16_weights<ONCE>(w, at, 1024 * (KS + ks));
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(d, d);
  // a thread stages one 16-byte piece of a chunk's columns of every 16th token
  static_assert(kTileWaves == kChunk, "16 tokens a turn");
  const int piece = tid % (4 * kChunk), token = tid / (4 * kChunk);
  unsigned row[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int p = r0 + list[min(first + 16 * i + token, n - 1)];
    row[i] = (PRODUCT == kGateUp ? p / k : p) * width + 16 * piece;
  }
  auto fetch = [&](int c) {
    const unsigned column = 64 * kChunk * c;
#pragma unroll
    for (int i = 0; i < NT; ++i)  // columns past the width are zero, as the weights' padding
      xr[i] = load16(in, column + 16 * piece < limit ? row[i] : kOutside, column);
  };
  u32x4* to = xs[0] + (piece >> 2) * 64 + (piece & 3) * 16 + token;
  auto stage = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < NT; ++i) to[buffer * (kTileTokens * kChunk * 64) + i * kChunk * 64] = xr[i];
  };
  f32x4 acc[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](const u32x4* x, int q, int s) {
    const int d = q % DEPTH;
    u32x4 xb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xb[t] = x[(t * kChunk + q) * 64];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      acc[t][0] = O::mfma(wb[d][0], xb[t], acc[t][0]);
      acc[t][1] = O::mfma(wb[d][1], xb[t], acc[t][1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    load(d, s + DEPTH);
    __builtin_amdgcn_sched_barrier(0);
  };
  // LDS alone: this chunk's reads and the next one's writes; the loads from memory go on
  auto barrier = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  const int whole = steps / kChunk, left = steps % kChunk;
  fetch(0);
  stage(0);
  barrier();
  for (int c = 0; c < whole; ++c) {
    const bool more = c + 1 < whole || left;
    if (more) fetch(c + 1);
    __builtin_amdgcn_sched_barrier(0);
    const u32x4* x = xs[c & 1] + lane;
#pragma unroll
    for (int q = 0; q < kChunk; ++q) step(x, q, c * kChunk + q);
    if (more) stage((c + 1) & 1);
    barrier();
  }
  const u32x4* x = xs[whole & 1] + lane;
#pragma unroll
  for (int q = 0; q < kChunk - 1; ++q)
    if (q < left) step(x, q, whole * kChunk + q);
  if (left) barrier();
  if (live)
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (first + 16 * t + j < n)
        store_block<T, PRODUCT>(acc[t][0], acc[t][1], r0 + list[first + 16 * t + j], block, g, shape, total, k, gates,
                                out);
}

template <typename T, int PRODUCT, int RANGE, int DEPTH, bool ONCE>
__global__ __launch_bounds__(64 * kTileWaves, DEPTH == 2 ? 4 : 3) void expert_tiles(
    const T* __restrict__ in, const u32x4* __restrict__ weights, const int* __restrict__ chosen,
    const float* __restrict__ gates, ExpertShape shape, int rows, int64_t total, int E, int k, int clears, int lists,
    int tiles, int cuts, void* __restrict__ out) {
  typedef PairList<kTileWaves, RANGE> List;
  __shared__ List list;
  __shared__ u32x4 xs[2][kTileTokens * kChunk * 64];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pairs = rows * k;
  const Place place =
      product_place(((PRODUCT == kGateUp ? shape.FB : shape.DB) + kTileWaves - 1) / kTileWaves * cuts, tiles);
  if (place.list >= lists) return;
  const int e = place.list < clears ? E : place.list - clears;
  const int KS = PRODUCT == kGateUp ? shape.KSx : shape.KSf;
  const unsigned width = (PRODUCT == kGateUp ? shape.D : shape.Fp) * sizeof(T);
  const int blocks = PRODUCT == kGateUp ? shape.FB : shape.DB;
  const int column = place.column / cuts, block = column * kTileWaves + wv;
  const bool live = block < blocks;
  const Cut cut = product_cut<PRODUCT>(KS, place.column % cuts, cuts);
  const unsigned limit = width - 64 * cut.first;
  const Buffer w = buffer(weights + ((int64_t)min(e, E - 1) * blocks + min(block, blocks - 1)) * 2 * KS * 64 +
                              cut.first * 64,
                          (2u * KS - cut.first) * 1024);
  const Buffer x = buffer(reinterpret_cast<const char*>(in) + 64 * cut.first,
                          (unsigned)((PRODUCT == kGateUp ? rows : pairs) * width - 64 * cut.first));
  if constexpr (PRODUCT == kDown) out = static_cast<float*>(out) + (place.column % cuts) * k * total * shape.D;

  for (int r0 = 0; r0 < pairs; r0 += RANGE) {
    typename List::Choices choices;
    list.load(choices, chosen, r0, pairs);
    const int n = list.fill(choices, r0, pairs, e, E);
    if (e == E) {
      if (PRODUCT == kDown && clears > 0 && place.tile == 0)
        clear_rows(list.list, n, r0, place.list * kTileWaves + wv, clears * kTileWaves, 32 * column * kTileWaves,
                   32 * (column + 1) * kTileWaves, shape.D, total, k, static_cast<float*>(out));
    } else {
      for (int first = 16 * kTileTokens * place.tile; first < n; first += 16 * kTileTokens * tiles) {
#define WPTV_TILE(NT)                                                                                                 \
  tile_pass<T, PRODUCT, NT, DEPTH, ONCE>(x, w, KS, cut.steps, width, limit, list.list, xs, r0, first, n, block, live, \
                                         shape, total, k, gates, out)
        switch ((n - first + 15) / 16) {
          case 1: WPTV_TILE(1); break;
          case 2: WPTV_TILE(2); break;
          case 3: WPTV_TILE(3); break;
          default: WPTV_TILE(4); break;
        }
#undef WPTV_TILE
      }
    }
    __syncthreads();  // the lists are written again
  }
}

// y of at most 16 tokens in one launch after the gate/up product: grid (D / 16), a
// workgroup's eight wavefronts share out the k-steps of 16 output rows over every
// expert that some token takes, one after the other, the tokens' columns in their
// own places, so that the matrix instructions add up the experts' terms as well.
// Pairs of one expert make a group, and one that a token names twice makes another;
// prow[group][token] is the pair, or kNone.
constexpr int kFewTokens = 16, kFewPairs = 128, kFewWaves = 8, kNone = 0xffff;

template <typename T>
__global__ __launch_bounds__(64 * kFewWaves) void expert_rows(const T* __restrict__ act,
                                                              const u32x4* __restrict__ weights,
                                                              const int* __restrict__ chosen, ExpertShape shape,
                                                              int rows, int E, int k, T* __restrict__ y) {
  using O = Operand<T>;
  constexpr int kDepth = 8;
  __shared__ int key[kFewPairs], expert[kFewPairs];
  __shared__ uint64_t leaders[kFewPairs / 64];
  static_assert(kFewPairs == 128, "two wavefronts of pairs");
  __shared__ uint16_t prow[kFewPairs][kFewTokens];
  __shared__ float red[kFewWaves][4 * 64];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pairs = rows * k;  // at most kFewPairs
  int e = -1, times = 0;
  if (tid < pairs) {
    e = chosen[tid];
    for (int i = tid / k * k; i < tid; ++i) times += chosen[i] == e ? 1 : 0;
    if ((unsigned)e >= (unsigned)E) e = -1;
    key[tid] = e < 0 ? -1 - tid : e * kMaxChosen + times;
  }
  for (int i = tid; i < kFewPairs * kFewTokens / 2; i += 64 * kFewWaves) reinterpret_cast<uint32_t*>(prow)[i] = ~0u;
  __syncthreads();
  // the first pair of a group is its leader; the groups in their leaders' order
  int leader = tid;
  if (e >= 0)
    for (int i = tid - 1; i >= 0; --i) leader = key[i] == key[tid] ? i : leader;
  const uint64_t first = __builtin_amdgcn_ballot_w64(e >= 0 && leader == tid);
  if (lane == 0 && wv < kFewPairs / 64) leaders[wv] = first;
  __syncthreads();
  if (e >= 0) {
    int group = __builtin_popcountll(leaders[leader >> 6] & ((1ull << (leader & 63)) - 1ull));
    if (leader >= 64) group += __builtin_popcountll(leaders[0]);
    prow[group][tid / k] = (uint16_t)tid;
    if (leader == tid) expert[group] = e;
  }
  const int groups = __builtin_popcountll(leaders[0]) + __builtin_popcountll(leaders[1]);
  __syncthreads();
  const int KS = shape.KSf, total = groups * KS;
  const unsigned width = shape.Fp * sizeof(T);
  const Buffer x = buffer(act, pairs * width);
  const int64_t matrix = (int64_t)shape.DB * 2 * KS * 64;
  const u32x4* w0 = weights + (int64_t)blockIdx.x * KS * 64;
  const int steps = (total - wv + kFewWaves - 1) / kFewWaves;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  u32x4 wb[kDepth], xb[kDepth];
  bool taken[kDepth];  // by the lane's token
  auto load = [&](int d, int s) {
    const int step = wv + kFewWaves * s, which = step / KS, ks = step - which * KS;
    const u32x4* w = w0 + __builtin_amdgcn_readfirstlane(expert[which]) * matrix;
    wb[d] = load16_weights<true>(buffer(w, 1024u * KS), 16 * lane, 1024 * ks);
    const unsigned p = prow[which][j];
    taken[d] = p != kNone;
    xb[d] = load16(x, taken[d] ? p * width + 16 * g : kOutside, 64 * ks);
  };
  auto multiply = [&](int d) {  // the other tokens' sums stay: 0 times a weight that is not finite is a NaN
    const f32x4 sum = O::mfma(wb[d], xb[d], acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = taken[d] ? sum[i] : acc[i];
  };
  if (steps > 0) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(d, min(d, steps - 1));
    int s = 0;
    for (; s + kDepth <= steps; s += kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        multiply(d);
        __builtin_amdgcn_sched_barrier(0);
        load(d, min(s + kDepth + d, steps - 1));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (s + d < steps) multiply(d);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[wv][i * 64 + lane] = acc[i];
  __syncthreads();
  if (tid < 256) {  // output row 4 g + i of token j
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kFewWaves; ++u) sum += red[u][tid];
    const int n = 16 * blockIdx.x + 4 * g + wv;
    if (j < rows && n < shape.D) y[(int64_t)j * shape.D + n] = from_f32<T>(sum);
  }
}

// y[m] = the sum of a token's parts in the order of its choices, rounded once; the
// parts of no expert hold nothing and are passed over.
template <typename T, bool CUT>
__global__ __launch_bounds__(256) void join_experts(const float* __restrict__ parts, const int* __restrict__ chosen,
                                                    int64_t rows, int D, int E, int k, int cuts,
                                                    T* __restrict__ y) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= rows * D) return;
  const int* choice = chosen + at / D * k;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const int all = CUT ? k * cuts : k;
  for (int first = 0; first < all; first += 8) {
    bool some[8];
    f32x4 part[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int part = min(first + i, all - 1);
      some[i] = first + i < all && (unsigned)choice[CUT ? part % k : part] < (unsigned)E;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)  // all asked for at once
      part[i] = *reinterpret_cast<const f32x4*>(parts + (some[i] ? (first + i) * rows * D : 0) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += some[i] ? part[i] : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  union {
    T element[4];
    unsigned int word[sizeof(T)];
  } v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.element[i] = from_f32<T>(sum[i]);
  typedef unsigned int words __attribute__((ext_vector_type(sizeof(T))));
  *reinterpret_cast<words*>(y + at) = *reinterpret_cast<const words*>(v.word);
}

// ---- host side ---------------------------------------------------------------

int check_dtype(const char* what, int dtype) {
  if (dtype == WPTV_BF16 || dtype == WPTV_F32) return WPTV_OK;
  return fail(WPTV_E_UNSUPPORTED, "%s: dtype %d is neither fp32 nor bf16", what, dtype);
}

int check_shape(const char* what, int64_t rows, int D, int E, int k, int dtype) {
  if (rows < 0 || D <= 0 || E <= 0 || k <= 0) {
    return fail(WPTV_E_INVALID, "%s: bad shape rows=%lld D=%d E=%d k=%d", what, (long long)rows, D, E, k);
  }
  if (k > E) return fail(WPTV_E_INVALID, "%s: k=%d of %d experts", what, k, E);
  if (D % 8 != 0 || D > (1 << 20))
    return fail(WPTV_E_UNSUPPORTED, "%s: width %d is not a multiple of 8 up to 2^20", what, D);
  if (E > kMaxExperts || k > kMaxChosen)
    return fail(WPTV_E_UNSUPPORTED, "%s: k=%d of E=%d experts is above %d of %d", what, k, E, kMaxChosen, kMaxExperts);
  if (rows > (1 << 24)) return fail(WPTV_E_UNSUPPORTED, "%s: %lld rows above 2^24", what, (long long)rows);
  return check_dtype(what, dtype);
}

int check_features(const char* what, int F) {
  if (F <= 0) return fail(WPTV_E_INVALID, "%s: bad width F=%d", what, F);
  if (F > (1 << 20)) return fail(WPTV_E_UNSUPPORTED, "%s: expert width %d above 2^20", what, F);
  return WPTV_OK;
}

// The bytes of the parts' logits, no less for more rows: with more than one part they
// have 512 tiles at most.
size_t route_bytes(int64_t rows, int D, int E) {
  if (rows == 0 || route_splits(rows, D, E) == 0) return 0;
  const int64_t most = route_parts(D) * rows, tiles = 512 / ((E + 15) / 16) * 16, some = most < tiles ? most : tiles;
  return (size_t)(rows > some ? rows : some) * E * sizeof(double);
}

// The experts a lane of a token's wavefront holds.
#define WPTV_SLOTS(FORM) \
  if (E <= 64)           \
    FORM(1);             \
  else if (E <= 128)     \
    FORM(2);             \
  else if (E <= 256)     \
    FORM(4);             \
  else                   \
    FORM(8)

template <typename T>
int run_route(const void* x, const float* router, const float* bias, const int64_t* counts, int rows, int per_row,
              int D, int E, int k, int* chosen, float* gates, void* workspace, hipStream_t stream) {
  const T* xt = static_cast<const T*>(x);
  const int splits = route_splits(rows, D, E);
  if (splits == 0) {
    int lanes = 64;
    while (lanes * E > kTokenThreads) lanes /= 2;
#define WPTV_TOKEN(SLOTS)                                                                                          \
  route_token<T, SLOTS><<<rows, kTokenThreads, 0, stream>>>(xt, router, bias, counts, per_row, D, E, lanes, k, \
                                                            chosen, gates)
    WPTV_SLOTS(WPTV_TOKEN);
#undef WPTV_TOKEN
    return launched("route");
  }
  double* sums = static_cast<double*>(workspace);
  // 2^19 tokens a launch: the grid's second dimension ends at 65535 (more tokens than that have one part)
  for (int m = 0; m < rows; m += 1 << 19) {
    const int here = rows - m < (1 << 19) ? rows - m : 1 << 19;
    route_logits<T><<<dim3((E + 15) / 16, (here + 15) / 16, splits), 256, 0, stream>>>(
        xt + (int64_t)m * D, router, here, D, E, sums + (int64_t)m * E);
  }
  const int status = launched("route (logits)");
  if (status != WPTV_OK) return status;
#define WPTV_CHOOSE(SLOTS) \
  route_choose<SLOTS>      \
      <<<(rows + 3) / 4, 256, 0, stream>>>(sums, bias, counts, rows, per_row, E, splits, k, chosen, gates)
  WPTV_SLOTS(WPTV_CHOOSE);
#undef WPTV_CHOOSE
  return launched("route (choice)");
}

// The down product's columns are cut where the row blocks and the experts leave compute
// units idle: into as many cuts as make 512 workgroups, of at least 16 k-steps each.
// Whole layers in a graph, us, whole and cut: 496 tokens of 448, 4 of 37 experts of 2395
// 132, 100; 160 of 1024, 2 of 16 of 4096 108, 89; 512 of 1024, 2 of 8 of 2816 86, 69; one
// of 2048, 2 of 8 of 5632 38.8, 34.6; FP32, one of 280, 2 of 2 of 4715 39.0, 23.9.  More
// do not give more: towards 768 tiles' workgroups 100, 92, 72 of the first three; towards
// 1024 160 tokens of 512, 4 of 16 of 1408 38.8 -> 41.4, cuts of 8 k-steps among those
// 238 of 1704, 6 of 16 of 509 56.8 -> 63.7.
constexpr int kCutGroups = 512, kCutSteps = 16, kMostCuts = 16;
constexpr int64_t kCutBytes = 32 << 20;  // the most that the terms of all cuts may take

int product_cuts(int KS, int64_t want) {
  int64_t cuts = want < kMostCuts ? want : kMostCuts;
  if (cuts > KS / kCutSteps) cuts = KS / kCutSteps;
  if (cuts <= 1) return 1;
  const int steps = (int)((KS + cuts - 1) / cuts);
  return (KS + steps - 1) / steps;  // none is empty
}

int64_t term_bytes(int64_t rows, int k, const ExpertShape& shape) { return rows * k * shape.D * 4; }

// The bytes of a round's terms, no less for more rows: of as many cuts as k experts'
// row blocks, the fewest there are, could be cut into.
size_t terms_bytes(int round, int k, const ExpertShape& shape) {
  const int64_t one = term_bytes(round, k, shape);
  const int64_t all = one * product_cuts(shape.KSf, kTileWaves * kCutGroups / ((int64_t)k * shape.DB));
  const int64_t some = all < kCutBytes ? all : kCutBytes;
  return (size_t)(one > some ? one : some);
}

template <typename T, int PRODUCT>
int run_product(const void* in, const void* weights, const int* chosen, const float* gates, const ExpertShape& shape,
                int rows, int64_t total, int E, int k, bool clear, int* cut, void* out,
                hipStream_t stream) {
  const int64_t pairs = (int64_t)rows * k;
  const int blocks = PRODUCT == kGateUp ? shape.FB : shape.DB;
  const bool by_pair = pairs < E;
  const int clears = !clear ? 0 : by_pair || pairs < 1024 ? 1 : 16;
  const int lists = by_pair ? (int)pairs : E + clears;
  const T* from = static_cast<const T*>(in);
  const u32x4* w = static_cast<const u32x4*>(weights);
  // tiles of one expert's tokens side by side, as many as its mean count in a range of pairs fills
  const int64_t mean = (pairs < 8192 ? pairs : 8192) / E;
  const int tiles = mean > 1024 ? 16 : (int)((mean + 63) / 64), few = mean > 512 ? 16 : (int)((mean + 31) / 32);
#define WPTV_COLUMNS(NT, TILES, BY, ONCE)                                                                   \
  expert_columns<T, PRODUCT, NT, 4, BY, ONCE><<<product_grid(blocks * cuts, lists, TILES), 256, 0, stream>>>( \
      from, w, chosen, gates, shape, rows, total, E, k, clears, lists, TILES, cuts, out)
#define WPTV_TILES(RANGE, DEPTH, ONCE)                                                                      \
  expert_tiles<T, PRODUCT, RANGE, DEPTH, ONCE>                                                              \
      <<<product_grid((blocks + kTileWaves - 1) / kTileWaves * cuts, lists, tiles), 64 * kTileWaves, 0, stream>>>( \
          from, w, chosen, gates, shape, rows, total, E, k, clears, lists, tiles, cuts, out)
  // The k-steps of a block pair over a workgroup, or tiles of 64 tokens a wavefront.  Whole layers, us, columns and
  // tiles: bf16, E blocks 352 (8 experts of 704, 300 tokens of 1000) 40.8, 39.1; 528 (6 of 1408, 100 tokens of 4096)
  // 99, 83; 1408 (16 of 1408, 256 tokens) 130, 115; FP32, whose instructions take four times as long, 512 (16 of 512,
  // 200 tokens of 1024) 61, 103.
  const int64_t least = sizeof(T) == 2 ? 512 : 1024;
  const bool columns = by_pair || rows <= 16 || (int64_t)E * blocks * tiles < least;
  const int spread = by_pair || rows <= 16 ? 1 : columns ? few : tiles;
  const int64_t groups =
      (int64_t)(by_pair ? pairs : E) * (columns ? blocks : (blocks + kTileWaves - 1) / kTileWaves) * spread;
  const int64_t fit = cut ? kCutBytes / term_bytes(rows, k, shape) : 1, want = kCutGroups / groups;
  const int cuts = PRODUCT == kGateUp ? 1 : product_cuts(shape.KSf, want < fit ? want : fit);
  if (cut) *cut = cuts;
  if (by_pair)
    WPTV_COLUMNS(1, 1, true, true);
  else if (rows <= 16)
    WPTV_COLUMNS(1, 1, false, true);
  else if (columns && few == 1)
    WPTV_COLUMNS(2, 1, false, true);
  else if (columns)
    WPTV_COLUMNS(2, few, false, false);
  else if (tiles > 1 || pairs > 4096)
    WPTV_TILES(8192, 4, false);
  else if (pairs <= 2048)
    WPTV_TILES(2048, 2, true);
  else
    WPTV_TILES(4096, 4, true);
#undef WPTV_TILES
#undef WPTV_COLUMNS
  return launched(PRODUCT == kGateUp ? "experts (gate, up)" : "experts (down)");
}

// The rows of one round of the two products: their operands stay within a buffer,
// and the terms that a join reads within kRoundBytes (a row's are 64 MiB at most).
constexpr int64_t kRoundBytes = 1 << 29;

int round_rows(int64_t rows, int k, const ExpertShape& shape, int dtype, bool join) {
  const int64_t act = (int64_t)k * shape.Fp;
  const int64_t widest = (dtype == WPTV_BF16 ? 2 : 4) * (shape.D > act ? shape.D : act);
  int64_t fit = kBufferBytes / widest;
  const int64_t most = kRoundBytes / term_bytes(1, k, shape);
  if (join && most < fit) fit = most;
  return (int)(rows < fit ? rows : fit);
}

size_t act_bytes(int round, int k, const ExpertShape& shape, int dtype) {
  return align_up((size_t)round * k * shape.Fp * (dtype == WPTV_BF16 ? 2 : 4), 256);
}

// Whether 16 output rows a workgroup, over all experts, are the faster down product
// of a few tokens (of at most kFewPairs pairs, whose rows are one round): where a
// workgroup reads little, which saves the join, or where they cover the compute units.
// Whole layers in a graph, us, this and the other form: one token, D 256, 2 of 8 experts
// of 704 12.6, 13.8; D 4096, 4 of 64 of 1408 42.0, 45.3, 4 tokens 105, 112; D 2048, 8 of
// 64 of 704 30.7, 29.9, 4 tokens, 2 of 8 of 5632 89, 80; FP32, 3 tokens, D 1024, 4 of 64
// of 300 29.9, 25.8.
bool few_rows(int rows, int k, const ExpertShape& shape) {
  if (rows > kFewTokens || rows * k > kFewPairs) return false;
  return (int64_t)rows * k * shape.KSf <= 64 || shape.D >= 4096;
}

template <typename T>
int run_experts(const void* x, const void* gate_up, const void* down, const int* chosen, const float* gates,
                const ExpertShape& shape, int rows, int E, int k, int dtype, float* parts, void* y, void* workspace,
                hipStream_t stream) {
  const int round = round_rows(rows, k, shape, dtype, y != nullptr);
  char* act = static_cast<char*>(workspace);
  float* terms = reinterpret_cast<float*>(act + act_bytes(round, k, shape, dtype));
  for (int64_t m = 0; m < rows; m += round) {
    const int here = rows - m < round ? (int)(rows - m) : round;
    const int* choice = chosen + m * k;
    int status = run_product<T, kGateUp>(static_cast<const T*>(x) + m * shape.D, gate_up, choice, gates + m * k, shape,
                                         here, here, E, k, false, nullptr, act, stream);
    if (status == WPTV_OK && y && few_rows(rows, k, shape)) {
      expert_rows<T><<<(shape.D + 15) / 16, 64 * kFewWaves, 0, stream>>>(
          reinterpret_cast<const T*>(act), static_cast<const u32x4*>(down), chosen, shape, rows, E, k,
          static_cast<T*>(y));
      return launched("experts (rows)");
    }
    int cuts = 1;
    if (status == WPTV_OK)
      status = y ? run_product<T, kDown>(act, down, choice, nullptr, shape, here, here, E, k, false, &cuts,
                                         terms, stream)
                 : run_product<T, kDown>(act, down, choice, nullptr, shape, here, rows, E, k, true, nullptr,
                                         parts + m * shape.D, stream);
    if (status != WPTV_OK) return status;
    if (y) {
      const int64_t threads = (int64_t)here * shape.D / 4;
#define WPTV_JOIN(CUT)                                                                                         \
  join_experts<T, CUT><<<(unsigned)((threads + 255) / 256), 256, 0, stream>>>(terms, choice, here, shape.D, E, \
                                                                              k, cuts, static_cast<T*>(y) + m * shape.D)
      if (cuts > 1)
        WPTV_JOIN(true);
      else
        WPTV_JOIN(false);
#undef WPTV_JOIN
      status = launched("experts (join)");
      if (status != WPTV_OK) return status;
    }
  }
  return WPTV_OK;
}

int check_experts(const char* what, const void* x, const void* gate_up, const void* down, const int* chosen,
                  const float* gates, int64_t rows, int D, int E, int k, int F, int dtype, const float* parts,
                  const void* y, const void* workspace, size_t workspace_bytes) {
  int status = check_shape(what, rows, D, E, k, dtype);
  if (status == WPTV_OK) status = check_features(what, F);
  if (status != WPTV_OK) return status;
  if (rows == 0) return WPTV_OK;
  if ((parts == nullptr) == (y == nullptr))
    return fail(WPTV_E_INVALID, "%s: one of parts and y must be given", what);
  if (!x || !chosen || !gates || !gate_up || !down) return fail(WPTV_E_INVALID, "%s: a required pointer is NULL", what);
  if (!aligned(x, 16) || !aligned(gate_up, 16) || !aligned(down, 16) || !aligned(parts, 16) || !aligned(y, 16) ||
      !aligned(workspace, 16))
    return fail(WPTV_E_INVALID, "%s: rows must be 16-byte aligned", what);
  size_t need = 0;
  status = wptv_experts_workspace((int)rows, D, F, k, dtype, parts ? 1 : 0, &need);
  if (status != WPTV_OK) return status;
  if (!workspace || workspace_bytes < need)
    return fail(WPTV_E_INVALID, "%s: the workspace holds %zu bytes; %zu are needed", what,
                workspace ? workspace_bytes : 0, need);
  return WPTV_OK;
}

int check_route(const char* what, const void* x, const float* router, int B, int T, int D, int E, int k, int dtype,
                const int* chosen, const float* gates, const void* workspace, size_t workspace_bytes) {
  if (B < 0 || T < 0) return fail(WPTV_E_INVALID, "%s: bad shape B=%d T=%d", what, B, T);
  const int status = check_shape(what, (int64_t)B * T, D, E, k, dtype);
  if (status != WPTV_OK) return status;
  if ((int64_t)B * T == 0) return WPTV_OK;
  if (!x || !router || !chosen || !gates) return fail(WPTV_E_INVALID, "%s: a required pointer is NULL", what);
  if (!aligned(x, 16) || !aligned(router, 16) || !aligned(workspace, 16))
    return fail(WPTV_E_INVALID, "%s: rows must be 16-byte aligned", what);
  const size_t need = route_bytes((int64_t)B * T, D, E);
  if (need && (!workspace || workspace_bytes < need))
    return fail(WPTV_E_INVALID, "%s: the workspace holds %zu bytes; %zu are needed", what,
                workspace ? workspace_bytes : 0, need);
  return WPTV_OK;
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_experts_packed(int D, int F, int dtype, size_t* gate_up_bytes, size_t* down_bytes) {
  int status = check_shape("experts_packed", 0, D, 1, 1, dtype);
  if (status == WPTV_OK) status = check_features("experts_packed", F);
  if (status != WPTV_OK) return status;
  if (!gate_up_bytes || !down_bytes) return fail(WPTV_E_INVALID, "experts_packed: a required pointer is NULL");
  const ExpertShape s = expert_shape(D, F, dtype);
  *gate_up_bytes = (size_t)s.FB * 2 * s.KSx * 1024;
  *down_bytes = (size_t)s.DB * 2 * s.KSf * 1024;
  return WPTV_OK;
}

extern "C" int wptv_pack_experts(const void* gate_up, const void* down, int E, int D, int F, int dtype,
                                 void* gate_up_packed, void* down_packed, hipStream_t stream) {
  int status = check_shape("pack_experts", 0, D, E, 1, dtype);
  if (status == WPTV_OK) status = check_features("pack_experts", F);
  if (status != WPTV_OK) return status;
  if (!gate_up || !down || !gate_up_packed || !down_packed)
    return fail(WPTV_E_INVALID, "pack_experts: every pointer must be given");
  if (!aligned(gate_up_packed, 16) || !aligned(down_packed, 16))
    return fail(WPTV_E_INVALID, "pack_experts: the packed weights must be 16-byte aligned");
  const ExpertShape s = expert_shape(D, F, dtype);
  const int64_t gu = (int64_t)s.FB * 2 * s.KSx * 64, dn = (int64_t)s.DB * 2 * s.KSf * 64;
  const dim3 gu_grid((unsigned)((gu + 255) / 256), E), dn_grid((unsigned)((dn + 255) / 256), E);
#define WPTV_PACK(TT)                                                                                             \
  pack_experts<TT, true><<<gu_grid, 256, 0, stream>>>(static_cast<const TT*>(gate_up), F, D, s.FB * 2, s.KSx,     \
                                                      aligned(gate_up, 16), static_cast<u32x4*>(gate_up_packed)); \
  pack_experts<TT, false><<<dn_grid, 256, 0, stream>>>(static_cast<const TT*>(down), D, F, s.DB * 2, s.KSf,       \
                                                       aligned(down, 16) && F % Operand<TT>::EPL == 0,            \
                                                       static_cast<u32x4*>(down_packed))
  if (dtype == WPTV_BF16) {
    WPTV_PACK(unsigned short);
  } else {
    WPTV_PACK(float);
  }
#undef WPTV_PACK
  return launched("pack_experts");
}

extern "C" int wptv_route_workspace(int rows, int D, int E, size_t* bytes) {
  const int status = check_shape("route_workspace", rows, D, E, 1, WPTV_F32);
  if (status != WPTV_OK) return status;
  if (!bytes) return fail(WPTV_E_INVALID, "route_workspace: a required pointer is NULL");
  *bytes = route_bytes(rows, D, E);
  return WPTV_OK;
}

extern "C" int wptv_route(const void* x, int dtype, const float* router, const float* bias, const int64_t* counts,
                          int B, int T, int D, int E, int k, int32_t* chosen, float* gates, void* workspace,
                          size_t workspace_bytes, hipStream_t stream) {
  const int status =
      check_route("route", x, router, B, T, D, E, k, dtype, chosen, gates, workspace, workspace_bytes);
  if (status != WPTV_OK || (int64_t)B * T == 0) return status;
  return dtype == WPTV_BF16
             ? run_route<unsigned short>(x, router, bias, counts, B * T, T, D, E, k, chosen, gates, workspace, stream)
             : run_route<float>(x, router, bias, counts, B * T, T, D, E, k, chosen, gates, workspace, stream);
}

extern "C" int wptv_experts_workspace(int rows, int D, int F, int k, int dtype, int parts_out, size_t* bytes) {
  int status = check_shape("experts_workspace", rows, D, kMaxExperts, k, dtype);
  if (status == WPTV_OK) status = check_features("experts_workspace", F);
  if (status != WPTV_OK) return status;
  if (!bytes) return fail(WPTV_E_INVALID, "experts_workspace: a required pointer is NULL");
  const ExpertShape s = expert_shape(D, F, dtype);
  const int round = round_rows(rows, k, s, dtype, !parts_out);
  *bytes = act_bytes(round, k, s, dtype) + (parts_out || rows == 0 ? 0 : terms_bytes(round, k, s));
  return WPTV_OK;
}

extern "C" int wptv_experts(const void* x, int dtype, const void* gate_up_packed, const void* down_packed,
                            const int32_t* chosen, const float* gates, int rows, int D, int E, int k, int F,
                            float* parts, void* y, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const int status = check_experts("experts", x, gate_up_packed, down_packed, chosen, gates, rows, D, E, k, F, dtype,
                                   parts, y, workspace, workspace_bytes);
  if (status != WPTV_OK || rows == 0) return status;
  const ExpertShape s = expert_shape(D, F, dtype);
  return dtype == WPTV_BF16 ? run_experts<unsigned short>(x, gate_up_packed, down_packed, chosen, gates, s, rows, E, k,
                                                          dtype, parts, y, workspace, stream)
                            : run_experts<float>(x, gate_up_packed, down_packed, chosen, gates, s, rows, E, k, dtype,
                                                 parts, y, workspace, stream);
}

extern "C" int wptv_mixture_workspace(int rows, int D, int E, int F, int k, int dtype, int parts_out, size_t* bytes) {
  size_t products = 0, sums = 0;
  int status = wptv_experts_workspace(rows, D, F, k, dtype, parts_out, &products);
  if (status == WPTV_OK) status = wptv_route_workspace(rows, D, E, &sums);
  if (status != WPTV_OK) return status;
  if (!bytes) return fail(WPTV_E_INVALID, "mixture_workspace: a required pointer is NULL");
  *bytes = products > sums ? products : sums;  // one after the other
  return WPTV_OK;
}

extern "C" int wptv_mixture(const void* x, int dtype, const float* router, const float* bias, const int64_t* counts,
                            int B, int T, int D, int E, int k, int F, const void* gate_up_packed,
                            const void* down_packed, int32_t* chosen, float* gates, float* parts, void* y,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int status = check_route("mixture", x, router, B, T, D, E, k, dtype, chosen, gates, workspace, workspace_bytes);
  if (status == WPTV_OK)
    status = check_experts("mixture", x, gate_up_packed, down_packed, chosen, gates, (int64_t)B * T, D, E, k, F, dtype,
                           parts, y, workspace, workspace_bytes);
  if (status != WPTV_OK) return status;
  // the router's sums are read before the products write
  status = wptv_route(x, dtype, router, bias, counts, B, T, D, E, k, chosen, gates, workspace, workspace_bytes, stream);
  if (status != WPTV_OK) return status;
  return wptv_experts(x, dtype, gate_up_packed, down_packed, chosen, gates, B * T, D, E, k, F, parts, y, workspace,
                      workspace_bytes, stream);
}
