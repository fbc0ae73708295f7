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
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
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
                                                    u32x4* __restrict__ out) {
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
  if (row < N) {
    const int64_t rows = PAIRED ? 2 * (int64_t)N : N;
    const T* from = w + ((int64_t)blockIdx.y * rows + row + (PAIRED && (rb & 1) ? N : 0)) * K;
#pragma unroll
    for (int i = 0; i < O::EPL; ++i)
      if (col + i < K) v.element[i] = from[col + i];
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

constexpr int kRouteThreads = 512, kMaxExperts = 512, kMaxChosen = 16;

// A workgroup TM tokens: its wavefronts share out the experts, the lanes the width;
// the products of two FP32 values are exact in 64 bits, and so is the order of the
// logits but for the sums' own rounding.  An expert's place is the count of those
// before it.
template <typename T, int TM>
__global__ __launch_bounds__(kRouteThreads) void route(const T* __restrict__ x, const float* __restrict__ router,
                                                       const float* __restrict__ bias,
                                                       const int64_t* __restrict__ counts, int rows, int per_row, int D,
                                                       int E, int k, int* __restrict__ chosen,
                                                       float* __restrict__ gates) {
  constexpr int kWaves = kRouteThreads / 64, kTokenThreads = kRouteThreads / TM;
  __shared__ double logit[TM][kMaxExperts];
  __shared__ uint64_t key[TM][kMaxExperts];
  __shared__ int place[TM][kMaxChosen];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int m0 = blockIdx.x * TM;
  const T* xr[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) xr[t] = x + (int64_t)min(m0 + t, rows - 1) * D;
  for (int e = wv; e < E; e += kWaves) {
    const float* w = router + (int64_t)e * D;
    double sum[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) sum[t] = 0.;
    for (int d = 4 * lane; d < D; d += 256) {
      const float4 a = *reinterpret_cast<const float4*>(w + d);
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        float b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = load_f32<T>(xr[t] + d + i);
        sum[t] = fma((double)a.x, (double)b[0], sum[t]);
        sum[t] = fma((double)a.y, (double)b[1], sum[t]);
        sum[t] = fma((double)a.z, (double)b[2], sum[t]);
        sum[t] = fma((double)a.w, (double)b[3], sum[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum[t] += __shfl_xor(sum[t], o, 64);
      if (lane == 0) {
        logit[t][e] = sum[t];
        key[t][e] = order_key64(bias ? sum[t] + (double)bias[e] : sum[t]);
      }
    }
  }
  const int t = threadIdx.x / kTokenThreads, tt = threadIdx.x % kTokenThreads, m = m0 + t;
  if (tt < k) place[t][tt] = -1;
  __syncthreads();
  const bool read = m < rows && (!counts || m % per_row < counts[m / per_row]);
  const uint64_t none = order_key64(-__builtin_inf());
  if (read)
    for (int e = tt; e < E; e += kTokenThreads) {
      const uint64_t mine = key[t][e];
      int before = 0;
      for (int i = 0; i < E; ++i) {
        const uint64_t other = key[t][i];
        before += other > mine || (other == mine && i < e) ? 1 : 0;
      }
      if (before < k && mine != none) place[t][before] = e;
    }
  __syncthreads();
  if (m < rows && tt < k) {
    double high = -__builtin_inf(), total = 0.;
    bool nan = false;
    for (int i = 0; i < k; ++i)
      if (place[t][i] >= 0) {
        const double l = logit[t][place[t][i]];
        nan |= l != l;
        high = fmax(high, l);
      }
    for (int i = 0; i < k; ++i)
      if (place[t][i] >= 0) total += exp(logit[t][place[t][i]] - high);
    const int e = place[t][tt];
    chosen[(int64_t)m * k + tt] = e;
    gates[(int64_t)m * k + tt] =
        e < 0 ? 0.f : nan ? __builtin_nanf("") : (float)(exp(logit[t][e] - high) / total);
  }
}

// ---- the experts' products ---------------------------------------------------

constexpr int kRange = 4096;  // pairs whose expert is looked up at a time

enum Product { kGateUp = 0, kDown = 1 };

// The pairs of the range [r0, r0 + kRange) that expert e takes, in their order:
// wavefront w lists those of its quarter in list[w].  Returns their count.
// e == E: the pairs of no expert.
__device__ __forceinline__ int list_pairs(const int* __restrict__ chosen, int64_t r0, int64_t pairs, int e, int E,
                                          int (*list)[kRange / 4], int* listed) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int n = 0;
  const uint64_t below = (1ull << lane) - 1ull;
  for (int i = 0; i < kRange / 4; i += 64) {
    const int64_t p = r0 + wv * (kRange / 4) + i + lane;
    if (r0 + wv * (kRange / 4) + i >= pairs) break;
    bool mine = false;
    if (p < pairs) {
      const int c = chosen[p];
      mine = c == e || (e == E && (unsigned)c >= (unsigned)E);
    }
    const uint64_t found = __builtin_amdgcn_ballot_w64(mine);
    if (mine) list[wv][n + __builtin_popcountll(found & below)] = (int)(p - r0);
    n += __builtin_popcountll(found);
  }
  if (lane == 0) listed[wv] = n;
  __syncthreads();
  return listed[0] + listed[1] + listed[2] + listed[3];
}

// The i-th listed pair of the range.
__device__ __forceinline__ int listed_pair(int i, const int (*list)[kRange / 4], const int* listed) {
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    if (i < listed[w]) return list[w][i];
    i -= listed[w];
  }
  return list[3][i];
}

// grid (row-block pairs / (4 / KW), experts or pairs): a workgroup's four
// wavefronts take 4 / KW row-block pairs of one expert's matrix, KW of them the
// k-steps of one pair in turn (their sums joined in LDS, in order), over tiles of
// 16 NT of the expert's tokens.  The weights are the A operand, the tokens the B
// operand, both straight from memory into registers, kDepth k-steps ahead.
//   kGateUp   x [rows, D] -> act [pairs, Fp]: silu(g) u of the FP32 sums, rounded
//             once to T, which the down product takes
//   kDown     act -> parts [k, rows, D]: gates[p] times the product, FP32
// BY_PAIR (fewer pairs than experts): workgroup y serves the expert of pair y,
// if that is the expert's first.
template <typename T, int PRODUCT, int NT, int KW, bool BY_PAIR>
__global__ __launch_bounds__(256) void expert_product(const T* __restrict__ in, const u32x4* __restrict__ weights,
                                                      const int* __restrict__ chosen, const float* __restrict__ gates,
                                                      ExpertShape shape, int64_t rows, int E, int k,
                                                      void* __restrict__ out) {
  using O = Operand<T>;
  constexpr int kDepth = NT == 1 ? 8 : 4;
  __shared__ int list[4][kRange / 4];
  __shared__ int listed[4];
  __shared__ float red[KW == 1 ? 1 : 4 * NT * 2 * 4 * 64];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t pairs = rows * k;
  int e = blockIdx.y;
  if constexpr (BY_PAIR) {
    const int at = e;
    e = chosen[at];
    for (int p = lane; p - lane < at; p += 64)
      if (__builtin_amdgcn_ballot_w64(p < at && chosen[p] == e)) return;
    if ((unsigned)e >= (unsigned)E) e = E;  // no expert: several of them clear the same rows
  }
  const int pairs_of_blocks = PRODUCT == kGateUp ? shape.FB : shape.DB;
  const int KS = PRODUCT == kGateUp ? shape.KSx : shape.KSf;
  const int K = PRODUCT == kGateUp ? shape.D : shape.Fp;
  const int block = blockIdx.x * (4 / KW) + wv / KW, part = wv % KW;
  const bool live = block < pairs_of_blocks;
  const int steps = live ? (KS - part + KW - 1) / KW : 0;
  const u32x4* w0 = weights + (((int64_t)e * pairs_of_blocks + block) * 2 * KS + part) * 64 + lane;
  const u32x4* w1 = w0 + (int64_t)KS * 64;

  for (int64_t r0 = 0; r0 < pairs; r0 += kRange) {
    const int n = list_pairs(chosen, r0, pairs, e, E, list, listed);
    if (e == E) {  // rows that no expert takes
      if constexpr (PRODUCT == kDown)
        for (int i = 0; i < n; ++i) {
          const int64_t p = r0 + listed_pair(i, list, listed);
          float* to = static_cast<float*>(out) + ((p % k) * rows + p / k) * shape.D;
          for (int d = blockIdx.x * (4 / KW) * 32 + threadIdx.x; d < min(shape.D, (int)(blockIdx.x + 1) * (4 / KW) * 32);
               d += 256)
            to[d] = 0.f;
        }
      __syncthreads();
      continue;
    }
    for (int first = 0; first < n; first += 16 * NT) {
      int64_t pair[NT];
      const T* row[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        // columns past the last token repeat it; nothing of them is stored
        pair[t] = r0 + listed_pair(min(first + 16 * t + j, n - 1), list, listed);
        row[t] = PRODUCT == kGateUp ? in + pair[t] / k * shape.D : in + pair[t] * shape.Fp;
      }
      f32x4 acc[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      u32x4 wb[kDepth][2], xb[kDepth][NT];
      auto load = [&](int d, int s) {
        wb[d][0] = w0[(int64_t)s * KW * 64];
        wb[d][1] = w1[(int64_t)s * KW * 64];
        const int col = O::KU * (part + KW * s) + O::EPL * g;
        const bool inside = col < K;  // the last k-step's columns past the width are zero
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(row[t] + (inside ? col : 0));
          xb[d][t] = inside ? v : u32x4{0u, 0u, 0u, 0u};
        }
      };
      auto multiply = [&](int d) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[t][0] = O::mfma(wb[d][0], xb[d][t], acc[t][0]);
          acc[t][1] = O::mfma(wb[d][1], xb[d][t], acc[t][1]);
        }
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
      auto store = [&](int t, f32x4 a, f32x4 b) {
        if (!live || first + 16 * t + j >= n) return;
        if constexpr (PRODUCT == kGateUp) {
          T* to = static_cast<T*>(out) + pair[t] * shape.Fp + 16 * block + 4 * g;
#pragma unroll
          for (int i = 0; i < 4; ++i) to[i] = from_f32<T>(a[i] / (1.f + expf(-a[i])) * b[i]);
        } else {
          const int64_t p = pair[t];
          const float gate = gates[p];
          float* to = static_cast<float*>(out) + ((p % k) * rows + p / k) * shape.D + 32 * block + 4 * g;
          const int left = shape.D - 32 * block - 4 * g;
          if (left > 0) *reinterpret_cast<f32x4*>(to) = gate * a;
          if (left > 16) *reinterpret_cast<f32x4*>(to + 16) = gate * b;
        }
      };
      if constexpr (KW == 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t) store(t, acc[t][0], acc[t][1]);
      } else {
        static_assert(KW == 1 || KW == 4, "a block pair's k-steps over the whole workgroup, or one wavefront");
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 8; ++i) red[((wv * NT + t) * 8 + i) * 64 + lane] = acc[t][i >> 2][i & 3];
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (t % 4 == wv) {
            float sum[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              sum[i] = red[(t * 8 + i) * 64 + lane];
#pragma unroll
              for (int u = 1; u < 4; ++u) sum[i] += red[((u * NT + t) * 8 + i) * 64 + lane];
            }
            store(t, f32x4{sum[0], sum[1], sum[2], sum[3]}, f32x4{sum[4], sum[5], sum[6], sum[7]});
          }
        __syncthreads();
      }
    }
    __syncthreads();  // the lists are written again
  }
}

// y[m] = the sum of a token's parts in the order of its choices, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void join_experts(const float* __restrict__ parts, int64_t rows, int D, int k,
                                                    T* __restrict__ y) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= rows * D) return;
  f32x4 sum = *reinterpret_cast<const f32x4*>(parts + at);
  for (int i = 1; i < k; ++i) sum += *reinterpret_cast<const f32x4*>(parts + i * rows * D + at);
#pragma unroll
  for (int i = 0; i < 4; ++i) y[at + i] = from_f32<T>(sum[i]);
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
  if (D % 8 != 0 || D > (1 << 20)) return fail(WPTV_E_UNSUPPORTED, "%s: width %d is not a multiple of 8 up to 2^20", what, D);
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

template <typename T>
int run_route(const void* x, const float* router, const float* bias, const int64_t* counts, int rows, int per_row, int D,
              int E, int k, int* chosen, float* gates, hipStream_t stream) {
  const T* xt = static_cast<const T*>(x);
  if (rows <= 256)
    route<T, 1><<<rows, kRouteThreads, 0, stream>>>(xt, router, bias, counts, rows, per_row, D, E, k, chosen, gates);
  else
    route<T, 4><<<(rows + 3) / 4, kRouteThreads, 0, stream>>>(xt, router, bias, counts, rows, per_row, D, E, k, chosen,
                                                             gates);
  return launched("route");
}

template <typename T, int PRODUCT>
int run_product(const void* in, const void* weights, const int* chosen, const float* gates, const ExpertShape& shape,
                int64_t rows, int E, int k, void* out, hipStream_t stream) {
  const int64_t pairs = rows * k;
  const int blocks = PRODUCT == kGateUp ? shape.FB : shape.DB;
  const bool by_pair = pairs < E;
  // one workgroup more clears the rows of no expert
  const int lists = by_pair ? (int)pairs : E + (PRODUCT == kDown ? 1 : 0);
#define WPTV_PRODUCT(NT, KW, BY)                                                                               \
  expert_product<T, PRODUCT, NT, KW, BY><<<dim3((blocks * KW + 3) / 4, lists), 256, 0, stream>>>(              \
      static_cast<const T*>(in), static_cast<const u32x4*>(weights), chosen, gates, shape, rows, E, k, out)
  if (by_pair)
    WPTV_PRODUCT(1, 4, true);
  else if (rows <= 16)
    WPTV_PRODUCT(1, 4, false);
  else if (pairs <= 16 * (int64_t)E)
    WPTV_PRODUCT(2, 1, false);
  else
    WPTV_PRODUCT(4, 1, false);
#undef WPTV_PRODUCT
  return launched(PRODUCT == kGateUp ? "experts (gate, up)" : "experts (down)");
}

size_t act_bytes(int64_t rows, int k, const ExpertShape& shape, int dtype) {
  return align_up((size_t)rows * k * shape.Fp * (dtype == WPTV_BF16 ? 2 : 4), 256);
}

template <typename T>
int run_experts(const void* x, const void* gate_up, const void* down, const int* chosen, const float* gates,
                const ExpertShape& shape, int64_t rows, int E, int k, int dtype, float* parts, void* y, void* workspace,
                hipStream_t stream) {
  char* act = static_cast<char*>(workspace);
  float* sums = parts ? parts : reinterpret_cast<float*>(act + act_bytes(rows, k, shape, dtype));
  int status = run_product<T, kGateUp>(x, gate_up, chosen, gates, shape, rows, E, k, act, stream);
  if (status != WPTV_OK) return status;
  status = run_product<T, kDown>(act, down, chosen, gates, shape, rows, E, k, sums, stream);
  if (status != WPTV_OK || parts) return status;
  const int64_t threads = rows * shape.D / 4;
  join_experts<T><<<(unsigned)((threads + 255) / 256), 256, 0, stream>>>(sums, rows, shape.D, k, static_cast<T*>(y));
  return launched("experts (join)");
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
    return fail(WPTV_E_INVALID, "%s: the workspace holds %zu bytes; %zu are needed", what, workspace ? workspace_bytes : 0,
                need);
  return WPTV_OK;
}

int check_route(const char* what, const void* x, const float* router, int B, int T, int D, int E, int k, int dtype,
                const int* chosen, const float* gates) {
  if (B < 0 || T < 0) return fail(WPTV_E_INVALID, "%s: bad shape B=%d T=%d", what, B, T);
  const int status = check_shape(what, (int64_t)B * T, D, E, k, dtype);
  if (status != WPTV_OK) return status;
  if ((int64_t)B * T == 0) return WPTV_OK;
  if (!x || !router || !chosen || !gates) return fail(WPTV_E_INVALID, "%s: a required pointer is NULL", what);
  if (!aligned(x, 16) || !aligned(router, 16)) return fail(WPTV_E_INVALID, "%s: rows must be 16-byte aligned", what);
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
                                                      static_cast<u32x4*>(gate_up_packed));                       \
  pack_experts<TT, false><<<dn_grid, 256, 0, stream>>>(static_cast<const TT*>(down), D, F, s.DB * 2, s.KSf,       \
                                                       static_cast<u32x4*>(down_packed))
  if (dtype == WPTV_BF16) {
    WPTV_PACK(unsigned short);
  } else {
    WPTV_PACK(float);
  }
#undef WPTV_PACK
  return launched("pack_experts");
}

extern "C" int wptv_route(const void* x, int dtype, const float* router, const float* bias, const int64_t* counts, int B,
                          int T, int D, int E, int k, int32_t* chosen, float* gates, hipStream_t stream) {
  const int status = check_route("route", x, router, B, T, D, E, k, dtype, chosen, gates);
  if (status != WPTV_OK || (int64_t)B * T == 0) return status;
  return dtype == WPTV_BF16
             ? run_route<unsigned short>(x, router, bias, counts, B * T, T, D, E, k, chosen, gates, stream)
             : run_route<float>(x, router, bias, counts, B * T, T, D, E, k, chosen, gates, stream);
}

extern "C" int wptv_experts_workspace(int rows, int D, int F, int k, int dtype, int parts_out, size_t* bytes) {
  int status = check_shape("experts_workspace", rows, D, kMaxExperts, k, dtype);
  if (status == WPTV_OK) status = check_features("experts_workspace", F);
  if (status != WPTV_OK) return status;
  if (!bytes) return fail(WPTV_E_INVALID, "experts_workspace: a required pointer is NULL");
  const ExpertShape s = expert_shape(D, F, dtype);
  *bytes = act_bytes(rows, k, s, dtype) + (parts_out ? 0 : (size_t)k * rows * D * 4);
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

extern "C" int wptv_mixture(const void* x, int dtype, const float* router, const float* bias, const int64_t* counts,
                            int B, int T, int D, int E, int k, int F, const void* gate_up_packed,
                            const void* down_packed, int32_t* chosen, float* gates, float* parts, void* y,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
  int status = check_route("mixture", x, router, B, T, D, E, k, dtype, chosen, gates);
  if (status == WPTV_OK)
    status = check_experts("mixture", x, gate_up_packed, down_packed, chosen, gates, (int64_t)B * T, D, E, k, F, dtype,
                           parts, y, workspace, workspace_bytes);
  if (status != WPTV_OK) return status;
  status = wptv_route(x, dtype, router, bias, counts, B, T, D, E, k, chosen, gates, stream);
  if (status != WPTV_OK) return status;
  return wptv_experts(x, dtype, gate_up_packed, down_packed, chosen, gates, B * T, D, E, k, F, parts, y, workspace,
                      workspace_bytes, stream);
}
