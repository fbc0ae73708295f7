// The generation cache's rows under beam search and eviction, moved in place
// for gfx950: a text's beams take over each other's states
// (wptv_reorder_rows), and the rows that a bounded cache keeps move together
// (wptv_keep_rows).
//
// Both read and write every moved row once, which is all they have to do, and
// need neither a second table nor a wait between workgroups: each workgroup
// owns every place that its own moves read and write.
//   reorder_rows  a thread owns one column piece of one token row of ALL the
//                 beams of a text: it reads the sources of the beams that
//                 change, then writes them, whatever cycles they form
//   keep_rows     a workgroup owns one column slice of ALL the rows of a batch
//                 row.  The kept list ascends, so a row's source is never
//                 below it: step by step, the sources of a step are read
//                 before the barrier and its rows written after it, and no
//                 later step reads what this one writes
#include "wptv_common.h"

#include <climits>

namespace wptv {
namespace {

constexpr int kMaxBeams = 64;
constexpr int kTables = 32;  // tables of one launch

struct Table {
  unsigned char* base;
  int64_t stride_b, stride_n;  // bytes
  int capacity;
  int pieces;  // a row's pieces of the launch's unit
};

struct Tables {
  Table t[kTables];
};

template <int BYTES>
struct Unit;
template <>
struct Unit<16> {
  typedef unsigned int type __attribute__((ext_vector_type(4)));
};
template <>
struct Unit<8> {
  typedef unsigned int type __attribute__((ext_vector_type(2)));
};
template <>
struct Unit<4> {
  typedef unsigned int type;
};
template <>
struct Unit<2> {
  typedef unsigned short type;
};
template <>
struct Unit<1> {
  typedef unsigned char type;
};

constexpr int kThreads = 256;

// The source beam of beam w of a text: itself where the given one is none of
// the text's.
__device__ __forceinline__ int source_beam(const int64_t* parents, int w, int W) {
  const int64_t p = parents[w];
  return p >= 0 && p < W ? (int)p : w;
}

// W <= WMAX: the beams' pieces of one place in registers.
template <int BYTES, int WMAX>
__global__ __launch_bounds__(kThreads) void reorder_rows(Tables tables, const int64_t* __restrict__ parents,
                                                         const int64_t* __restrict__ lengths, int W) {
  typedef typename Unit<BYTES>::type U;
  const Table& t = tables.t[blockIdx.z];
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t n = at / t.pieces;
  const int piece = (int)(at % t.pieces);
  if (n >= t.capacity) return;
  const int64_t text = blockIdx.y;
  const int64_t* p = parents + text * W;
  unsigned char* place = t.base + text * W * t.stride_b + n * t.stride_n + (int64_t)piece * BYTES;
  U held[WMAX];
  bool moves[WMAX];
#pragma unroll
  for (int w = 0; w < WMAX; ++w) {
    moves[w] = false;
    if (w < W) {
      const int from = source_beam(p, w, W);
      moves[w] = from != w && (!lengths || n < lengths[text * W + from]);
      if (moves[w]) held[w] = *reinterpret_cast<const U*>(place + from * t.stride_b);
    }
  }
#pragma unroll
  for (int w = 0; w < WMAX; ++w)
    if (w < W && moves[w]) *reinterpret_cast<U*>(place + w * t.stride_b) = held[w];
}

template <int BYTES>
__global__ __launch_bounds__(kThreads) void keep_rows(Tables tables, const int64_t* __restrict__ kept, int first_list,
                                                      int lists, int B, int keep, const int64_t* __restrict__ counts,
                                                      int slice_pieces) {
  typedef typename Unit<BYTES>::type U;
  const Table& t = tables.t[blockIdx.z];
  const int b = blockIdx.y;
  const int piece = blockIdx.x * slice_pieces + threadIdx.x % slice_pieces;
  const int rows = kThreads / slice_pieces;  // rows a step
  const int r = threadIdx.x / slice_pieces;
  int64_t live = counts[b];
  live = live < keep ? live : keep;
  const int64_t* list = kept + ((int64_t)((first_list + blockIdx.z) % lists) * B + b) * keep;
  unsigned char* column = t.base + b * t.stride_b + (int64_t)piece * BYTES;
  for (int64_t j0 = 0; j0 < live; j0 += rows) {
    const int64_t j = j0 + r;
    U held;
    bool moves = false;
    if (r < rows && piece < t.pieces && j < live && j < t.capacity) {
      const int64_t from = list[j];
      moves = from > j && from < t.capacity;
      if (moves) held = *reinterpret_cast<const U*>(column + from * t.stride_n);
    }
    __syncthreads();  // every source of the step is read
    if (moves) *reinterpret_cast<U*>(column + j * t.stride_n) = held;
  }
}

// The widest unit that divides a table's addresses, strides and row.
int unit_of(const void* base, int64_t sb, int64_t sn, int64_t row_bytes) {
  const uint64_t bits = reinterpret_cast<uint64_t>(base) | (uint64_t)sb | (uint64_t)sn | (uint64_t)row_bytes | 16;
  return (int)(bits & ~(bits - 1));
}

// Host checks of one table of `rows_b` batch rows.
int check_table(const char* what, int i, const void* base, int64_t sb, int64_t sn, int64_t capacity, int64_t row_bytes,
                int64_t rows_b) {
  if (capacity < 0 || capacity > INT32_MAX || row_bytes <= 0 || row_bytes > INT32_MAX)
    return fail(WPTV_E_INVALID, "%s: table %d has capacity %lld and rows of %lld bytes", what, i, (long long)capacity,
                (long long)row_bytes);
  if (capacity > 0 && rows_b > 0 && !base) return fail(WPTV_E_INVALID, "%s: table %d is NULL", what, i);
  // rows apart within a batch row and batch rows apart, in either nesting: a place written twice would race
  const bool apart_n = capacity <= 1 || sn >= row_bytes;
  const bool apart_b = rows_b <= 1 || sb >= row_bytes;
  const bool nested = capacity <= 1 || rows_b <= 1 || sb >= (capacity - 1) * sn + row_bytes ||
                      sn >= (rows_b - 1) * sb + row_bytes;
  if (!apart_n || !apart_b || !nested)
    return fail(WPTV_E_INVALID, "%s: the rows of table %d overlap (strides %lld and %lld bytes, rows of %lld)", what, i,
                (long long)sb, (long long)sn, (long long)row_bytes);
  return WPTV_OK;
}

template <int BYTES>
int launch_reorder(const Tables& tables, int count, int64_t blocks, int n, const int64_t* parents,
                   const int64_t* lengths, int W, hipStream_t stream) {
  const dim3 grid((unsigned)blocks, n, count);
  if (W <= 4)
    reorder_rows<BYTES, 4><<<grid, kThreads, 0, stream>>>(tables, parents, lengths, W);
  else if (W <= 8)
    reorder_rows<BYTES, 8><<<grid, kThreads, 0, stream>>>(tables, parents, lengths, W);
  else if (W <= 16)
    reorder_rows<BYTES, 16><<<grid, kThreads, 0, stream>>>(tables, parents, lengths, W);
  else
    reorder_rows<(BYTES < 4 ? BYTES : 4), 64><<<grid, kThreads, 0, stream>>>(tables, parents, lengths, W);
  return launched("reorder_rows");
}

template <int BYTES>
int launch_keep(const Tables& tables, int count, int slices, int slice_pieces, const int64_t* kept, int first_list,
                int lists, int B, int keep, const int64_t* counts, hipStream_t stream) {
  keep_rows<BYTES><<<dim3(slices, B, count), kThreads, 0, stream>>>(tables, kept, first_list, lists, B, keep, counts,
                                                                    slice_pieces);
  return launched("keep_rows");
}

}  // namespace
}  // namespace wptv

using namespace wptv;

extern "C" int wptv_reorder_rows(void* const* tables, const int64_t* strides_b, const int64_t* strides_n,
                                 const int64_t* capacities, const int64_t* row_bytes, int count,
                                 const int64_t* parents, const int64_t* lengths, int64_t rows, int n, int W,
                                 hipStream_t stream) {
  if (count < 0 || n < 0 || W <= 0 || rows < 0)
    return fail(WPTV_E_INVALID, "reorder_rows: bad shape count=%d n=%d W=%d rows=%lld", count, n, W, (long long)rows);
  if (W > kMaxBeams) return fail(WPTV_E_UNSUPPORTED, "reorder_rows: at most %d beams a text (got %d)", kMaxBeams, W);
  if (n > 65535) return fail(WPTV_E_UNSUPPORTED, "reorder_rows: at most 65535 texts (got %d)", n);
  if (count && (!tables || !strides_b || !strides_n || !capacities || !row_bytes))
    return fail(WPTV_E_INVALID, "reorder_rows: the tables' addresses and shapes must be given");
  for (int i = 0; i < count; ++i) {
    const int status = check_table("reorder_rows", i, tables[i], strides_b[i], strides_n[i], capacities[i],
                                   row_bytes[i], (int64_t)n * W);
    if (status != WPTV_OK) return status;
  }
  if (count == 0 || n == 0 || W == 1) return WPTV_OK;
  if (!parents) return fail(WPTV_E_INVALID, "reorder_rows: parents is NULL");
  // a launch for up to kTables tables of one unit
  for (int unit = 16; unit >= 1; unit /= 2) {
    Tables held;
    int many = 0;
    int64_t blocks = 0;
    for (int i = 0; i <= count; ++i) {
      if (i < count && capacities[i] > 0) {
        int u = unit_of(tables[i], strides_b[i], strides_n[i], row_bytes[i]);
        if (W > 16 && u > 4) u = 4;  // 64 beams' pieces in registers
        if (u == unit) {
          const int64_t reach = lengths && rows < capacities[i] ? rows : capacities[i];
          const int64_t pieces = row_bytes[i] / unit;
          held.t[many++] = Table{static_cast<unsigned char*>(tables[i]), strides_b[i], strides_n[i], (int)reach,
                                 (int)pieces};
          const int64_t need = (reach * pieces + kThreads - 1) / kThreads;
          if (need > INT32_MAX) return fail(WPTV_E_UNSUPPORTED, "reorder_rows: table %d is too large", i);
          blocks = blocks > need ? blocks : need;
        }
      }
      if (many == kTables || (i == count && many)) {
        int status = WPTV_OK;
        if (blocks) {
          switch (unit) {
            case 16: status = launch_reorder<16>(held, many, blocks, n, parents, lengths, W, stream); break;
            case 8: status = launch_reorder<8>(held, many, blocks, n, parents, lengths, W, stream); break;
            case 4: status = launch_reorder<4>(held, many, blocks, n, parents, lengths, W, stream); break;
            case 2: status = launch_reorder<2>(held, many, blocks, n, parents, lengths, W, stream); break;
            default: status = launch_reorder<1>(held, many, blocks, n, parents, lengths, W, stream); break;
          }
        }
        if (status != WPTV_OK) return status;
        many = 0;
        blocks = 0;
      }
    }
  }
  return WPTV_OK;
}

extern "C" int wptv_keep_rows(void* const* tables, const int64_t* strides_b, const int64_t* strides_n,
                              const int64_t* capacities, const int64_t* row_bytes, int count, const int64_t* kept,
                              int lists, int keep, const int64_t* counts, int B, hipStream_t stream) {
  if (count < 0 || lists < 0 || keep < 0 || B < 0 || (count && (lists == 0 || count % lists)))
    return fail(WPTV_E_INVALID, "keep_rows: %d tables for %d lists of %d rows, B=%d", count, lists, keep, B);
  if (B > 65535) return fail(WPTV_E_UNSUPPORTED, "keep_rows: at most 65535 batch rows (got %d)", B);
  if (count && (!tables || !strides_b || !strides_n || !capacities || !row_bytes))
    return fail(WPTV_E_INVALID, "keep_rows: the tables' addresses and shapes must be given");
  for (int i = 0; i < count; ++i) {
    const int status =
        check_table("keep_rows", i, tables[i], strides_b[i], strides_n[i], capacities[i], row_bytes[i], B);
    if (status != WPTV_OK) return status;
  }
  if (count == 0 || B == 0 || keep == 0) return WPTV_OK;
  if (!kept || !counts) return fail(WPTV_E_INVALID, "keep_rows: kept and counts must be given");
  for (int i = 0; i < count; ++i) {
    if (capacities[i] == 0) continue;
    Tables held;
    const int unit = unit_of(tables[i], strides_b[i], strides_n[i], row_bytes[i]);
    const int pieces = (int)(row_bytes[i] / unit);
    const int slice = pieces < 8 ? pieces : 8;
    const int slices = (pieces + slice - 1) / slice;
    held.t[0] = Table{static_cast<unsigned char*>(tables[i]), strides_b[i], strides_n[i], (int)capacities[i], pieces};
    int status;
    switch (unit) {
      case 16: status = launch_keep<16>(held, 1, slices, slice, kept, i, lists, B, keep, counts, stream); break;
      case 8: status = launch_keep<8>(held, 1, slices, slice, kept, i, lists, B, keep, counts, stream); break;
      case 4: status = launch_keep<4>(held, 1, slices, slice, kept, i, lists, B, keep, counts, stream); break;
      case 2: status = launch_keep<2>(held, 1, slices, slice, kept, i, lists, B, keep, counts, stream); break;
      default: status = launch_keep<1>(held, 1, slices, slice, kept, i, lists, B, keep, counts, stream); break;
    }
    if (status != WPTV_OK) return status;
  }
  return WPTV_OK;
}
