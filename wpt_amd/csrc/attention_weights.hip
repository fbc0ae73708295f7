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
// No atomics: a wavefront owns its rows and takes the queries in order, and the
// parts that many queries are cut into are joined in order, so the sums do not
// depend on the launch.
//   attention_weights_mfma     head widths 64 and 128: the products on the
//                              matrix cores
//   attention_weights_join     the parts' sums
//   attention_weights_generic  any other width up to 256, or unaligned rows
//
// A term's exponent is formed in FP32 from lse log2 e and scale log2 e, each rounded: a
// weight is off by a few steps of 2^-24 times |lse| + |scale q . k|.
//
// Per 16 query heads x 16 rows at head width 128, a SIMD's matrix cores take 64
// cycles and its vector unit about 110 (16.6 instructions, of them four exponentials at
// a quarter of the rate).  Two prompts of 4096 tokens, 16 heads: 62 us and 4 for the
// join, 1.1 PFLOP/s of the products alone; by the counters the matrix cores are busy 25 %
// of that time and the vector units 40 %, with two wavefronts a SIMD on average: neither
// is full, a wavefront's products and exponentials follow each other, and the parts of a
// causal prompt end at different times.  Few queries are bound
// by the keys: 32 texts of 4100 rows, 5 queries, 11.4 us for 27 MB, of which the chain
// positions, keys, products, write takes 4 whatever is read.
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

constexpr int kKeys = 64;   // table rows of a workgroup of the generic kernel
constexpr int kGT = 256;
constexpr int kMaxWidth = 256;

// The counted queries of batch row b.
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

// ---- the matrix-core form ------------------------------------------------------

constexpr int kBlockKeys = 256;  // table rows of a workgroup of four wavefronts of 64
constexpr int kStage = 512;      // query heads whose lse and position are staged in LDS at once
constexpr float kUnseen = -1.f;  // a part's sum for a row that none of its queries sees (sums are not negative)

// 16 rows of C values as an operand of the 16-row matrix instructions, in 16-byte
// pieces: piece f of lane 16 g + j holds bytes 64 f + 16 g of row j.  The products
// only need both operands to agree on the order of the C values.
template <typename E, int C>
struct Rows16;

template <int C>
struct Rows16<unsigned short, C> {
  static constexpr int kPieces = C / 32, kSteps = C / 32;
  bf16x8 v[kPieces];
  static __device__ __forceinline__ f32x4 step(const Rows16& a, const Rows16& b, int s, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[s], b.v[s], acc, 0, 0, 0);
  }
};

template <int C>
struct Rows16<float, C> {
  static constexpr int kPieces = C / 16, kSteps = C / 4;
  f32x4 v[kPieces];
  static __device__ __forceinline__ f32x4 step(const Rows16& a, const Rows16& b, int s, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[s / 4][s % 4], b.v[s / 4][s % 4], acc, 0, 0, 0);
  }
};

// A wavefront holds 64 table rows as the second operand of four products and
// streams the query heads, 16 at a time, through the first: a lane ends with
// four query heads of one row in each, whose exponentials it adds to that row's
// sum in a register.  Nothing but the sums is written.  The query heads come into
// LDS by DMA in the order of the operand's registers (1 KiB a piece, read back
// without a bank conflict), 64 at a time for the four wavefronts, the next ones
// while these are multiplied.
// At least two wavefronts a SIMD: the compiler then keeps the products out of the
// accumulation registers, which the exponentials cannot read.
template <typename E, int C, int U>
__global__ __launch_bounds__(256, 2) void attention_weights_mfma(
    const E* __restrict__ q, const E* __restrict__ k, int64_t ksb, int64_t ksn, const int64_t* __restrict__ positions,
    const float* __restrict__ lse, const int64_t* __restrict__ counts, const int64_t* __restrict__ start, int B, int T,
    int H, int N, float scale_log2, int nkb, int parts, int part_rows, int by_xcd, float* __restrict__ weights,
    int64_t wsb, float* __restrict__ sums, int64_t sums_stride) {
  typedef Rows16<E, C> Op;
  static_assert(U == 2 || U == 4, "blocks of 16 rows a wavefront holds");
  constexpr int kP = Op::kPieces, kWaveKeys = 16 * U;
  __shared__ __attribute__((aligned(16))) unsigned char queries[2][4 * kP * 1024];  // blocks of 16, then pieces
  __shared__ __attribute__((aligned(16))) float l2s[kStage];
  __shared__ __attribute__((aligned(16))) int seen[kStage];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, g = lane >> 4;
  int kb = blockIdx.x % nkb, chunk = blockIdx.x / nkb;
  if (by_xcd) {  // workgroups go to the 8 XCDs in turn: the queries of a part are read through one XCD's L2
    kb = blockIdx.x / 8 % nkb;
    chunk = blockIdx.x / 8 / nkb * 8 + blockIdx.x % 8;
    if (chunk >= parts * B) return;
  }
  const int b = chunk / parts, part = chunk % parts;
  const int64_t rows_b = (int64_t)b * T * H;
  const int first = part * part_rows;
  // The rows that the part's queries see end at hi, and each sees those up to lo.
  const int64_t* pos = positions + (int64_t)b * T;
  auto reach = [&](int64_t p) { return p < 0 ? -1 : p < N ? (int)p : N - 1; };
  int lo = N - 1, hi = -1, end;
  {
    const int t0 = first / H;
    const int64_t p0 = pos[min(t0 + lane, T - 1)];  // read with the count, not after it
    end = min(counted(counts, b, T) * H, first + part_rows);
    const int t1 = (end - 1) / H;
    if (first < end && t0 + lane <= t1) lo = hi = reach(p0);
    if (first < end)
      for (int t = t0 + 64 + lane; t <= t1; t += 64) {
        const int c = reach(pos[t]);
        lo = min(lo, c);
        hi = max(hi, c);
      }
    lo = __builtin_amdgcn_readfirstlane(wave_min_i32(lo));
    hi = __builtin_amdgcn_readfirstlane(wave_max_i32(hi));
  }
  const int n0 = kb * 4 * kWaveKeys, wn0 = n0 + kWaveKeys * w, n = wn0 + lane;
  const bool mine = lane < kWaveKeys;  // lane l ends with row wn0 + l's sum
  float total = 0.f, before = 0.f;
  if (n0 <= hi) {
    const int heads = end - first;
    // the lse and reach of query heads r0 .. r0 + kStage - 1, from memory and into
    // LDS; padding query heads have no weight
    float l2[kStage / 256];
    int see[kStage / 256];
    auto read_stage = [&](int r0) {
#pragma unroll
      for (int i = 0; i < kStage / 256; ++i) {
        const int r = min(r0 + tid + 256 * i, heads - 1);
        l2[i] = lse[rows_b + first + r];
        see[i] = reach(pos[(first + r) / H]);
      }
    };
    auto write_stage = [&](int r0) {
#pragma unroll
      for (int i = 0; i < kStage / 256; ++i) {
        const bool padding = r0 + tid + 256 * i >= heads;
        l2s[tid + 256 * i] = padding ? __builtin_inff() : l2[i] * kLog2e;
        seen[tid + 256 * i] = padding ? -1 : see[i];
      }
    };
    // everything is asked for at once: what is waited for first, first
    read_stage(0);
    if (parts == 1 && mine && n <= hi && !(start && n >= start[b])) before = weights[(int64_t)b * wsb + n];
    // query heads first + r0 .. first + r0 + 63 into a buffer, block w by wavefront w
    // (past the end: the last one again)
    auto fetch = [&](int r0, int buffer) {
      const i32x4 rsrc = buffer_resource(q + (rows_b + first + r0) * C);
      const int row = min(16 * w + j, heads - r0 - 1);
      const uint32_t at = lds_address(&queries[buffer][w * kP * 1024]);
#pragma unroll
      for (int f = 0; f < kP; ++f)
        dma_16B(rsrc, (uint32_t)row * (C * sizeof(E)) + 64 * f + 16 * g, __builtin_amdgcn_readfirstlane(at + 1024 * f));
    };
    fetch(0, 0);
    Op keys[U];
    float sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sum[u] = 0.f;
      const E* row = k + (int64_t)b * ksb + (int64_t)min(wn0 + 16 * u + j, N - 1) * ksn;
#pragma unroll
      for (int f = 0; f < kP; ++f)
        keys[u].v[f] = *reinterpret_cast<const decltype(keys[u].v[f] + 0)*>(reinterpret_cast<const unsigned char*>(row) +
                                                                            64 * f + 16 * g);
    }
    write_stage(0);
    // the keys are waited for here: in the loop, the wait would be for the DMA too
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < kP; ++f) asm volatile("" : "+v"(keys[u].v[f]));
    const bool whole = wn0 + kWaveKeys - 1 <= lo, idle = wn0 > hi;
    for (int r0 = 0; r0 < heads; r0 += 64) {
      const int buffer = (r0 / 64) & 1;
      if (r0 > 0 && r0 % kStage == 0) {  // the last barrier is behind the reads of the stage before
        read_stage(r0);
        write_stage(r0);
      }
      if (r0 + 64 < heads) {
        fetch(r0 + 64, buffer ^ 1);
        wait_vmcnt<kP>();  // these 64 have come
      } else {
        wait_vmcnt<0>();
      }
      __syncthreads();
      const int blocks = idle ? 0 : min(4, (heads - r0 + 15) / 16);
      for (int m = 0; m < blocks; ++m) {
        Op query;
#pragma unroll
        for (int f = 0; f < kP; ++f)
          query.v[f] = *reinterpret_cast<const decltype(query.v[f] + 0)*>(&queries[buffer][(m * kP + f) * 1024 + lane * 16]);
        const f32x4 l2 = *reinterpret_cast<const f32x4*>(&l2s[r0 % kStage + 16 * m + 4 * g]);
        f32x4 acc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < Op::kSteps; ++s)
#pragma unroll
          for (int u = 0; u < U; ++u) acc[u] = Op::step(query, keys[u], s, acc[u]);
        // acc[u][i]: query head 16 m + 4 g + i, row wn0 + 16 u + j
        if (whole) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(acc[u][i], scale_log2, -l2[i]));
            sum[u] += (e[0] + e[1]) + (e[2] + e[3]);
          }
        } else {
          const i32x4 p = *reinterpret_cast<const i32x4*>(&seen[r0 % kStage + 16 * m + 4 * g]);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = __builtin_amdgcn_exp2f(fmaf(acc[u][i], scale_log2, -l2[i]));
              e[i] = wn0 + 16 * u + j <= p[i] ? x : 0.f;  // an unseen row may hold anything
            }
            sum[u] += (e[0] + e[1]) + (e[2] + e[3]);
          }
        }
      }
      __syncthreads();  // the buffer is read
    }
    // the four lane groups' sums of each block, block u into lane group u (two blocks:
    // into the first two groups)
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[0]), __float_as_uint(sum[1]), false, false);
    const float z01 = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    float z23 = z01;
    if constexpr (U == 4) {
      const auto c = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[2]), __float_as_uint(sum[3]), false, false);
      z23 = __uint_as_float(c[0]) + __uint_as_float(c[1]);
    }
    const auto d = __builtin_amdgcn_permlane32_swap(__float_as_uint(z01), __float_as_uint(z23), false, false);
    total = __uint_as_float(d[0]) + __uint_as_float(d[1]);
  }
  if (!mine) return;
  if (parts > 1) {
    sums[((int64_t)part * B + b) * sums_stride + n] = n <= hi ? total : kUnseen;
  } else if (n <= hi) {
    float* out = weights + (int64_t)b * wsb + n;
    *out = before + total;
  }
}

// weights += the parts' sums in order, a fourth of them by each wavefront of a
// workgroup of 64 rows; rows that no part sees are left alone.
__global__ __launch_bounds__(256) void attention_weights_join(const float* __restrict__ sums, int parts, int64_t sums_stride,
                                                              int B, int N, const int64_t* __restrict__ start,
                                                              float* __restrict__ weights, int64_t wsb) {
  __shared__ float shared[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int b = blockIdx.y, n = blockIdx.x * 64 + lane;
  const int64_t stride = B * sums_stride;
  const int some = (parts + 3) / 4, end = min(parts, (w + 1) * some);
  const float* s = sums + b * sums_stride + n;
  float total = kUnseen;
#pragma unroll 8
  for (int p = w * some; p < end; ++p) {
    const float x = s[p * stride];
    total = x == kUnseen ? total : total == kUnseen ? x : total + x;
  }
  shared[w][lane] = total;
  __syncthreads();
  if (w != 0 || n >= N) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const float x = shared[i][lane];
    total = x == kUnseen ? total : total == kUnseen ? x : total + x;
  }
  if (total == kUnseen) return;
  float* out = weights + (int64_t)b * wsb + n;
  *out = (start && n >= start[b] ? 0.f : *out) + total;
}

// The parts the T H query heads are cut into.  A workgroup a compute unit where
// parts of 32 query heads give them; above that, parts of about 512 query heads
// balance what a causal prompt leaves of them, up to 16 workgroups a compute unit
// (the parts' sums have to be joined).  Measured, us, by parts: two prompts of 4096
// tokens 121 [32], 73 [64], 67 [128], 71 [192]; a chunk of 1024 tokens over 4096 rows
// 38 [16], 26 [32], 32 [96], 39 [192]; one of 64 over 8192 34 [1], 14 [4], 11 [8],
// 14 [32]; a prompt of 512 36 [8], 11.2 [64], 10.4 [128], 12.9 [192]; 9 queries of 32
// heads over 1000 rows 9.1 [1], 9.0 [4], 8.1 [12].
int weight_parts(int B, int T, int H, int N) {
  const int64_t rows = (int64_t)T * H, units = (int64_t)B * ((N + kBlockKeys - 1) / kBlockKeys);
  const int64_t cus = compute_units();
  const int64_t parts = max(min(cus / units, rows / 32), min(rows / 512, 16 * cus / units));
  // few query heads in few parts: the join costs more than it gives (80 over 2000 rows
  // of 16 texts 5.9 [1], 8.6 [2]; 256 over 16000 of two 8.9 [1], 10.6 [2])
  if (rows < 256 || (rows <= 512 && parts < 4)) return 1;
  return (int)max((int64_t)1, parts);
}

bool matrix_width(int c) { return c == 64 || c == 128; }

// Blocks of 16 rows a wavefront holds: four, so that a query head read from LDS meets
// 64 rows; two where the queries are few and the workgroups of four do not fill the
// compute units four times, so that twice as many share the chain's latency.
// Measured, us, two and four: 32 texts of 4100 rows, 5 queries of 16 heads, 11.4, 12.6;
// 8 texts 5.9, 7.4; one token over 4096 rows 4.2, 5.1; 6 texts of 3001 FP32 rows, 7
// queries of 4 heads, 5.6, 7.3; 64 texts of 4100, one query, 14.3, 13.4.
int wave_blocks(int B, int64_t heads, int N, int parts) {
  const int64_t units = (int64_t)B * ((N + kBlockKeys - 1) / kBlockKeys);
  return parts == 1 && heads <= 320 && units <= 4 * (int64_t)compute_units() ? 2 : 4;
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
  if (N > (1 << 30) || (int64_t)T * H > (1 << 29) || (int64_t)B * ((N + kKeys - 1) / kKeys) > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "attention_weights: B=%d T=%d H=%d N=%d is too large", B, T, H, N);
  if (*splits < 0) return fail(WPTV_E_INVALID, "attention_weights: splits = %d", *splits);
  const int64_t rows = (int64_t)T * H;
  if (!matrix_width(c) || B == 0 || rows == 0 || B > 65535) {  // (the join's grid has B rows)
    *splits = 1;
  } else if (*splits == 0) {
    *splits = weight_parts(B, T, H, N);
  } else {
    *splits = (int)min((int64_t)*splits, (rows + 15) / 16);  // a part holds at least one block of query heads
  }
  const int64_t nkb = (N + kBlockKeys - 1) / kBlockKeys;
  if ((int64_t)B * nkb * *splits + nkb * 8 > INT32_MAX)
    return fail(WPTV_E_UNSUPPORTED, "attention_weights: B=%d N=%d in %d parts is too large", B, N, *splits);
  *bytes = *splits == 1 ? 0 : (size_t)*splits * B * nkb * kBlockKeys * sizeof(float);
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
  const int elem = dtype == WPTV_BF16 ? 2 : 4;
  if (matrix_width(c) && aligned(q, 16) && aligned(k, 16) && k_stride_n * elem % 16 == 0 && k_stride_b * elem % 16 == 0) {
    const int held = wave_blocks(B, (int64_t)T * H, N, splits);
    const int blocks = (N + 64 * held - 1) / (64 * held);
    const int64_t sums_stride = (int64_t)((N + kBlockKeys - 1) / kBlockKeys) * kBlockKeys;
    const int part_rows = (int)(((int64_t)T * H + splits - 1) / splits + 15) / 16 * 16;
    const int chunks = splits * B;
    const int by_xcd = splits > 1 && (chunks % 8 == 0 || chunks >= 64);  // as many chunks an XCD, nearly
    const int groups = by_xcd ? (chunks + 7) / 8 * 8 : chunks;
    float* sums = static_cast<float*>(workspace);
#define WPTV_WEIGHTS(E, C, U)                                                                                         \
  attention_weights_mfma<E, C, U><<<blocks * groups, 256, 0, stream>>>(                                              \
      static_cast<const E*>(q), static_cast<const E*>(k), k_stride_b, k_stride_n, positions, lse, counts, start, B, T, \
      H, N, scale * kLog2e, blocks, splits, part_rows, by_xcd, weights, weights_stride_b, sums, sums_stride)
#define WPTV_WEIGHTS_U(E, C) (held == 2 ? WPTV_WEIGHTS(E, C, 2) : WPTV_WEIGHTS(E, C, 4))
    if (dtype == WPTV_BF16) {
      if (c == 64) WPTV_WEIGHTS_U(unsigned short, 64); else WPTV_WEIGHTS_U(unsigned short, 128);
    } else {
      if (c == 64) WPTV_WEIGHTS_U(float, 64); else WPTV_WEIGHTS_U(float, 128);
    }
#undef WPTV_WEIGHTS_U
#undef WPTV_WEIGHTS
    const int launch = launched("attention_weights_mfma");
    if (launch != WPTV_OK || splits == 1) return launch;
    attention_weights_join<<<dim3((N + 63) / 64, B), 256, 0, stream>>>(sums, splits, sums_stride, B, N, start, weights,
                                                                       weights_stride_b);
    return launched("attention_weights_join");
  }
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
