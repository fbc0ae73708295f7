// The K-th largest of a workgroup's 32-bit keys, held in its threads' registers or read
// again for each pass (long texts): what the choice of rows (choice.hip) and the eviction
// (eviction.hip) select by.
#pragma once

#include "wptv_common.h"

namespace wptv {
namespace {

// The sum over the lanes up to and including this one; every lane must be
// active (DPP: shifts within the rows of 16, then the rows' totals carried on).
__device__ __forceinline__ int wave_scan_i32(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

constexpr int kSelectBins = 1024, kSelectCand = 256;

template <int THREADS>
struct SelectShared {
  __attribute__((aligned(16))) int hist[kSelectBins];
  __attribute__((aligned(16))) uint32_t cand[kSelectCand];
  int range[2][THREADS / 64], sel[3], ncand;
  uint32_t found;
};

// The `remaining`-th largest key, the same in every thread, of those that
// each(f) calls f(item, key) with in each thread (at least `remaining` in all).
// Histograms of 1024 equal bins over the range of keys still open (first smallest
// to largest): the bin that holds it, then, when that holds at most kSelectCand
// keys, the one among them, else a histogram of the bin's own range.  A range
// shrinks 2^9 times a pass at the least, so four passes end it whatever the keys
// are (equal ones end in a bin of width one); scores take one pass.
//
// Among the bin's keys: BY_BITS, a search of its bits by ballots, else their ranks
// by counting, a loop as long as the bin is full.  Weights fill it (384 selections
// of 3964 weights 16 us by counting, 13.6 by bits), scores do not (160 selections
// among 3972 half a microsecond longer by bits).
template <int THREADS, bool BY_BITS, typename Each>
__device__ __forceinline__ uint32_t kth_largest(Each&& each, int remaining, SelectShared<THREADS>& shared) {
  constexpr int kWaves = THREADS / 64, kBins = kSelectBins, kCand = kSelectCand;
  constexpr int kPerLane = kBins / 64;
  static_assert(kBins % THREADS == 0 && kCand <= THREADS, "bins and candidates a thread");
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  auto& hist = shared.hist;
  auto& cand = shared.cand;
  auto& range = shared.range;
  auto& sel = shared.sel;
  auto& ncand = shared.ncand;
  uint32_t tau;
#pragma unroll
  for (int i = 0; i < kBins / THREADS; ++i) hist[tid + i * THREADS] = 0;
  if (tid == 0) ncand = 0;
  int kmin = INT32_MAX, kmax = INT32_MIN;  // as signed, order kept
  each([&](int, uint32_t x) {
    const int y = (int)(x ^ 0x80000000u);
    kmin = min(kmin, y);
    kmax = max(kmax, y);
  });
  kmin = wave_min_i32(kmin);
  kmax = wave_max_i32(kmax);
  if (lane == 0) {
    range[0][w] = kmin;
    range[1][w] = kmax;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    kmin = min(kmin, range[0][i]);
    kmax = max(kmax, range[1][i]);
  }
  uint32_t lo = (uint32_t)kmin ^ 0x80000000u, hi = (uint32_t)kmax ^ 0x80000000u;
  // the key sought is the remaining-th largest of those in lo .. hi
  for (;;) {
    const uint32_t span = hi - lo;
    const int shift = span < kBins ? 0 : 22 - __builtin_clz(span);  // span >> shift < kBins
    each([&](int, uint32_t x) {
      if (x >= lo && x <= hi) atomicAdd(&hist[(x - lo) >> shift], 1);
    });
    __syncthreads();
    if (w == 0) {
      // lane l holds bins top - 15 .. top, top = kBins - 1 - 16 l
      int cnt[kPerLane], total = 0;
      const int first = kBins - kPerLane * (lane + 1);
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) total += (cnt[e] = hist[first + e]);
      const int upto = wave_scan_i32(total);
      if (upto >= remaining && upto - total < remaining) {  // one lane
        int above = upto - total, bin = first, c = 0;
#pragma unroll
        for (int e = kPerLane - 1; e >= 0; --e) {
          if (c == 0 && above + cnt[e] >= remaining) {
            bin = first + e;
            c = cnt[e];
          }
          if (c == 0) above += cnt[e];
        }
        sel[0] = bin;
        sel[1] = above;
        sel[2] = c;
      }
    }
    __syncthreads();
    const int count = sel[2];
    remaining -= sel[1];
    lo += (uint32_t)sel[0] << shift;
    if (shift == 0) {  // the bin's keys are equal
      tau = lo;
      break;
    }
    const uint32_t width = (1u << shift) - 1u;
    if (hi - lo > width) hi = lo + width;
    if (count <= kCand) {
      each([&](int, uint32_t x) {
        if (x >= lo && x <= hi) cand[atomicAdd(&ncand, 1)] = x;
      });
      __syncthreads();
      if constexpr (BY_BITS) {
        // every wavefront for itself: the largest offset into the bin that
        // `remaining` of its keys reach, a bit at a time
        uint32_t offset[kCand / 64], reached = 0;
#pragma unroll
        for (int i = 0; i < kCand / 64; ++i) offset[i] = lane + 64 * i < count ? cand[lane + 64 * i] - lo : 0u;
        for (int bit = shift - 1; bit >= 0; --bit) {
          const uint32_t trial = reached | (1u << bit);
          int many = 0;
#pragma unroll
          for (int i = 0; i < kCand / 64; ++i)
            many += __builtin_popcountll(__builtin_amdgcn_ballot_w64(offset[i] >= trial));
          if (many >= remaining) reached = trial;
        }
        tau = lo + reached;
      } else {
        if (tid < count) {
          const uint32_t mine = cand[tid];
          int gt = 0, ge = 0;
          for (int i = 0; i < count; ++i) {
            const uint32_t x = cand[i];
            gt += x > mine ? 1 : 0;
            ge += x >= mine ? 1 : 0;
          }
          if (gt < remaining && ge >= remaining) shared.found = mine;  // the same key from each that writes
        }
        __syncthreads();
        tau = shared.found;
      }
      break;
    }
#pragma unroll
    for (int i = 0; i < kBins / THREADS; ++i) hist[tid + i * THREADS] = 0;
    __syncthreads();
  }
  return tau;
}

}  // namespace
}  // namespace wptv
