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
// Bound by HBM: a copy of 1 GiB runs at 5.15 TB/s, read and written.  24 tables of 8
// texts of 4 beams, three of them moved, 1125 rows of 512 bytes on average: 117 us, 4.7
// TB/s (8 and 16 beams 5.4 and 5.2); 24 tables of 16 texts, 2048 rows kept: 115 us, 4.4
// TB/s, the rows left out breaking its reads up.
#include "wptv_common.h"

#include <climits>
#include <initializer_list>

namespace wptv {
namespace {

constexpr int kMaxBeams = 64;
constexpr int kTables = 32;  // tables of one launch

struct Table {
  unsigned char* base;
  int64_t stride_b, stride_n;  // bytes
  int capacity;
  int pieces;  // a row's pieces of the launch's unit
  int list;    // keep_rows: which layer's list of rows
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

// p[i] of an input that no kernel of the launch writes: a scalar load where i
// is uniform.
__device__ __forceinline__ int64_t const_load(const int64_t* p, int64_t i) {
  return ((const __attribute__((address_space(4))) int64_t*)(uintptr_t)p)[i];
}

// The pieces of beams w .. WMAX - 1, each in a register of its own: of an array of
// eight 16-byte pieces the compiler made one 32-register value that it copied at
// each of them (2.5 TB/s in place of 5).  All are read before the first is written,
// and written in the order they were asked for, so that the first write waits for
// one read and not for all (5.7 TB/s against 4.4 the other way round).
template <int BYTES, int WMAX, int w = 0>
struct Pieces {
  typename Unit<BYTES>::type held;
  Pieces<BYTES, WMAX, w + 1> rest;
  __device__ __forceinline__ void read(const unsigned char* place, int64_t stride_b, int n, int source, int taken) {
    const int from = __builtin_amdgcn_readlane(source, w);
    if (n < __builtin_amdgcn_readlane(taken, w))
      held = *reinterpret_cast<const typename Unit<BYTES>::type*>(place + from * stride_b);
    rest.read(place, stride_b, n, source, taken);
  }
  __device__ __forceinline__ void write(unsigned char* place, int64_t stride_b, int n, int taken) {
    if (n < __builtin_amdgcn_readlane(taken, w))
      *reinterpret_cast<typename Unit<BYTES>::type*>(place + w * stride_b) = held;
    rest.write(place, stride_b, n, taken);
  }
};

template <int BYTES, int WMAX>
struct Pieces<BYTES, WMAX, WMAX> {
  __device__ __forceinline__ void read(const unsigned char*, int64_t, int, int, int) {}
  __device__ __forceinline__ void write(unsigned char*, int64_t, int, int) {}
};

// W <= WMAX: the beams' pieces of one place in registers.
template <int BYTES, int WMAX>
__global__ __launch_bounds__(kThreads) void reorder_rows(Tables tables, const int64_t* __restrict__ parents,
                                                         const int64_t* __restrict__ lengths, int W) {
  const Table& t = tables.t[blockIdx.z];
  const int text = blockIdx.y;
  // lane w: beam w's source, and how many of its rows beam w takes (none where
  // it stays as it is, or the source is no beam of the text)
  const int lane = threadIdx.x & 63;
  int source = 0, taken = 0;
  if (lane < W) {
    const int64_t p = parents[(int64_t)text * W + lane];
    if (p >= 0 && p < W && p != lane) {
      source = (int)p;
      taken = t.capacity;
      if (lengths) taken = (int)min(max(lengths[(int64_t)text * W + p], (int64_t)0), (int64_t)t.capacity);
    }
  }
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;  // below 2^31: checked on the host
  const int n = (int)(at / (uint32_t)t.pieces);
  const int piece = (int)(at % (uint32_t)t.pieces);
  unsigned char* place = t.base + (int64_t)text * W * t.stride_b + n * t.stride_n + (int64_t)piece * BYTES;
  Pieces<BYTES, WMAX> pieces;
  pieces.read(place, t.stride_b, n, source, taken);
  pieces.write(place, t.stride_b, n, taken);
}

constexpr int kKeepThreads = 512;
constexpr int kKeepLoads = 8;  // rows a thread holds at once

// A step holds kKeepLoads rows a thread of the slice, 64 KB a workgroup at the
// widest unit: its sources' loads are all in flight together, and the step costs
// one memory round trip however the rows lie.  24 tables, us, with 4, 8 and 16 rows a
// thread: 16 texts from 4096 to 2048 rows 122, 115, 115; 32 texts, a quarter of them
// over 1024 rows, 39, 38, 50.
template <int BYTES>
__global__ __launch_bounds__(kKeepThreads) void keep_rows(Tables tables, const int64_t* __restrict__ kept, int B,
                                                          int keep, const int64_t* __restrict__ counts,
                                                          int slice_shift) {
  typedef typename Unit<BYTES>::type U;
  const Table& t = tables.t[blockIdx.z];
  const int b = blockIdx.y;
  const int piece = (blockIdx.x << slice_shift) + (threadIdx.x & ((1 << slice_shift) - 1));
  const int rows = kKeepThreads >> slice_shift;  // rows of one load of the workgroup
  const int r = threadIdx.x >> slice_shift;
  const int64_t count = const_load(counts, b);
  const int live = (int)min(count, (int64_t)min(keep, t.capacity));
  const int64_t* list = kept + ((int64_t)t.list * B + b) * keep;
  unsigned char* column = t.base + b * t.stride_b + (int64_t)piece * BYTES;
  const bool inside = piece < t.pieces;
  for (int j0 = 0; j0 < live; j0 += rows * kKeepLoads) {
    int64_t from[kKeepLoads];
    U held[kKeepLoads];
#pragma unroll
    for (int i = 0; i < kKeepLoads; ++i) {
      const int j = j0 + i * rows + r;
      from[i] = inside && j < live ? list[j] : -1;
      if (from[i] <= j || from[i] >= t.capacity) from[i] = -1;  // in its place already, or no row
    }
#pragma unroll
    for (int i = 0; i < kKeepLoads; ++i)
      if (from[i] >= 0) held[i] = *reinterpret_cast<const U*>(column + from[i] * t.stride_n);
    __syncthreads();  // every source of the step is read
#pragma unroll
    for (int i = 0; i < kKeepLoads; ++i)
      if (from[i] >= 0) *reinterpret_cast<U*>(column + (j0 + i * rows + r) * t.stride_n) = held[i];
  }
}

// The widest unit that divides a table's addresses, strides and row.
int unit_of(const void* base, int64_t sb, int64_t sn, int64_t row_bytes) {
  const uint64_t bits = reinterpret_cast<uint64_t>(base) | (uint64_t)sb | (uint64_t)sn | (uint64_t)row_bytes | 16;
  return (int)(bits & ~(bits - 1));
}

// A table's bytes: `count` blocks `stride` apart, of blocks, of `bytes` bytes; batch rows
// outermost ([0]), or token rows where those are.
struct Extent {
  uint64_t base;
  int64_t stride[2], count[2], bytes;

  __int128 size(int level) const {
    __int128 n = bytes;
    for (int i = level; i < 2; ++i) n += (__int128)(count[i] - 1) * stride[i];
    return n;
  }
};

// Whether a byte is both in a and in b, whose base lies d bytes behind a's: blocks m
// strides apart meet where what is in them does.  Tables of other strides whose ranges
// meet are not told apart, and taken to.
bool meet(const Extent& a, const Extent& b, __int128 d, int level = 0) {
  if (d >= a.size(level) || d + b.size(level) <= 0) return false;
  if (level == 2) return true;
  const bool one = a.count[level] == 1, other = b.count[level] == 1;
  if (!one && !other && a.stride[level] != b.stride[level]) return true;
  if (one && other) return meet(a, b, d, level + 1);
  const __int128 s = one ? b.stride[level] : a.stride[level];
  const __int128 in_a = a.size(level + 1), in_b = b.size(level + 1);
  const __int128 least = -(a.count[level] - 1), most = b.count[level] - 1;
  // -in_b < d + m s < in_a
  __int128 m = (-in_b - d) / s - 1, end = (in_a - d) / s + 1;
  m = m > least ? m : least;
  end = end < most ? end : most;
  if (end - m > 256) return true;
  for (; m <= end; ++m)
    if (meet(a, b, d + m * s, level + 1)) return true;
  return false;
}

// rows_first: token rows outermost.
Extent extent(const void* base, int64_t sb, int64_t sn, int64_t capacity, int64_t row_bytes, int64_t rows_b,
              bool rows_first) {
  Extent e{reinterpret_cast<uint64_t>(base), {sb, sn}, {rows_b, capacity}, row_bytes};
  if (rows_first) {
    e.stride[0] = sn, e.stride[1] = sb;
    e.count[0] = capacity, e.count[1] = rows_b;
  }
  return e;
}

// What a launch reads while it moves the rows.
struct List {
  const void* base;
  int64_t bytes;
};

constexpr int kRanges = 256;  // tables whose range of addresses is kept for the tables after them

// Host checks of `count` tables of `rows_b` batch rows: a place written twice, or read
// as a list, would race.
int check_tables(const char* what, void* const* bases, const int64_t* strides_b, const int64_t* strides_n,
                 const int64_t* capacities, const int64_t* row_bytes, int count, int64_t rows_b,
                 std::initializer_list<List> lists) {
  uint64_t from[kRanges], to[kRanges];
  auto extent_of = [&](int i, bool rows_first) {
    return extent(bases[i], strides_b[i], strides_n[i], capacities[i], row_bytes[i], rows_b, rows_first);
  };
  // batch rows (or token rows) may stand outermost: their blocks hold those of the others
  auto nests = [&](int i, bool rows_first) {
    return capacities[i] <= 1 || rows_b <= 1 ||
           (rows_first ? strides_n[i] >= strides_b[i] : strides_b[i] >= strides_n[i]);
  };
  auto range = [&](int i, uint64_t& begin, uint64_t& end) {
    begin = reinterpret_cast<uint64_t>(bases[i]);
    end = begin;
    if (capacities[i] > 0 && rows_b > 0) end += (uint64_t)extent_of(i, false).size(0);
  };
  for (int i = 0; i < count; ++i) {
    const void* base = bases[i];
    const int64_t sb = strides_b[i], sn = strides_n[i], capacity = capacities[i], bytes = row_bytes[i];
    if (capacity < 0 || capacity > INT32_MAX || bytes <= 0 || bytes > INT32_MAX)
      return fail(WPTV_E_INVALID, "%s: table %d has capacity %lld and rows of %lld bytes", what, i, (long long)capacity,
                  (long long)bytes);
    if (capacity > 0 && rows_b > 0 && !base) return fail(WPTV_E_INVALID, "%s: table %d is NULL", what, i);
    if (capacity == 0 || rows_b == 0) {  // no bytes
      if (i < kRanges) from[i] = to[i] = 0;
      continue;
    }
    // rows apart within a batch row and batch rows apart, in either nesting
    const bool apart_n = capacity <= 1 || sn >= bytes;
    const bool apart_b = rows_b <= 1 || sb >= bytes;
    const bool nested = capacity <= 1 || rows_b <= 1 || sb >= (__int128)(capacity - 1) * sn + bytes ||
                        sn >= (__int128)(rows_b - 1) * sb + bytes;
    if (!apart_n || !apart_b || !nested)
      return fail(WPTV_E_INVALID, "%s: the rows of table %d overlap (strides %lld and %lld bytes, rows of %lld)", what, i,
                  (long long)sb, (long long)sn, (long long)bytes);
    uint64_t begin, end;
    range(i, begin, end);
    if (i < kRanges) from[i] = begin, to[i] = end;
    for (int other = 0; other < i; ++other) {
      uint64_t first, last;
      if (other < kRanges)
        first = from[other], last = to[other];
      else
        range(other, first, last);
      if (begin >= last || first >= end || first == last) continue;
      const bool rows_first = !(nests(i, false) && nests(other, false));
      const Extent a = extent_of(other, rows_first), b = extent_of(i, rows_first);
      if ((rows_first && !(nests(i, true) && nests(other, true))) || meet(a, b, (__int128)b.base - a.base))
        return fail(WPTV_E_INVALID, "%s: tables %d and %d are the same, or overlap", what, other, i);
    }
    for (const List& list : lists) {
      const uint64_t at = reinterpret_cast<uint64_t>(list.base);
      if (!list.base || list.bytes <= 0 || begin >= at + (uint64_t)list.bytes || at >= end) continue;
      const Extent a = extent_of(i, !nests(i, false)), b = extent(list.base, 0, 0, 1, list.bytes, 1, false);
      if (meet(a, b, (__int128)b.base - a.base))
        return fail(WPTV_E_INVALID, "%s: table %d is also read as a list of rows", what, i);
    }
  }
  return WPTV_OK;
}

// W <= 16, or a unit of at most 4 bytes.
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
int launch_keep(const Tables& tables, int count, int widest, const int64_t* kept, int B, int keep,
                const int64_t* counts, hipStream_t stream) {
  // Slices of a row, one a workgroup: whole 128-byte lines, thinner where there
  // would be hardly any workgroup.  Measured, us, 24 layers, rows of 512 bytes, slices
  // of 32, 64, 128 and 256 bytes: 16 texts from 4096 to 2048 rows 231, 151, 115, 111; one
  // text 25, 16, 14, 23; 32 texts, a quarter of them over 1024 rows, 90, 51, 38, 43; one
  // layer of one text of 16000 rows 29, 35, 51, 100.
  int shift = 0;
  while ((BYTES << (shift + 1)) <= 128 && (1 << shift) < widest) ++shift;
  while (shift > 0 && (int64_t)count * B * ((widest + (1 << shift) - 1) >> shift) < 16) --shift;
  const int slices = (widest + (1 << shift) - 1) >> shift;
  keep_rows<BYTES><<<dim3(slices, B, count), kKeepThreads, 0, stream>>>(tables, kept, B, keep, counts, shift);
  return launched("keep_rows");
}

// Calls launch(unit, tables, how many, the largest `size` of them) for up to
// kTables tables of one unit at a time, wider units first.
template <typename Size, typename Launch>
int each_launch(void* const* tables, const int64_t* strides_b, const int64_t* strides_n, const int64_t* capacities,
                const int64_t* row_bytes, int count, int lists, int widest_unit, Size size, Launch launch) {
  for (int unit = widest_unit; unit >= 1; unit /= 2) {
    Tables held;
    int many = 0;
    int64_t most = 0;
    for (int i = 0; i <= count; ++i) {
      if (i < count && capacities[i] > 0 &&
          min(unit_of(tables[i], strides_b[i], strides_n[i], row_bytes[i]), widest_unit) == unit) {
        Table& t = held.t[many++];
        t = Table{static_cast<unsigned char*>(tables[i]), strides_b[i], strides_n[i], (int)capacities[i],
                  (int)(row_bytes[i] / unit), i % lists};
        most = max(most, (int64_t)size(t));
      }
      if (many == kTables || (i == count && many)) {
        const int status = launch(unit, held, many, most);
        if (status != WPTV_OK) return status;
        many = 0;
        most = 0;
      }
    }
  }
  return WPTV_OK;
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
  const int64_t listed = (int64_t)n * W * sizeof(int64_t);
  const int status = check_tables("reorder_rows", tables, strides_b, strides_n, capacities, row_bytes, count,
                                  (int64_t)n * W, {{parents, listed}, {lengths, listed}});
  if (status != WPTV_OK) return status;
  if (count == 0 || n == 0 || W == 1) return WPTV_OK;
  if (!parents) return fail(WPTV_E_INVALID, "reorder_rows: parents is NULL");
  const int widest = W > 16 ? 4 : 16;  // 64 beams' pieces are held in registers
  auto size = [&](Table& t) {
    if (lengths) t.capacity = (int)min((int64_t)t.capacity, rows);
    return (int64_t)t.capacity * t.pieces;
  };
  auto launch = [&](int unit, const Tables& held, int many, int64_t most) {
    if (most > INT32_MAX - kThreads) return fail(WPTV_E_UNSUPPORTED, "reorder_rows: a batch row of 2^31 pieces");
    const int64_t blocks = (most + kThreads - 1) / kThreads;
    if (blocks == 0) return (int)WPTV_OK;
    switch (unit) {
      case 16: return launch_reorder<16>(held, many, blocks, n, parents, lengths, W, stream);
      case 8: return launch_reorder<8>(held, many, blocks, n, parents, lengths, W, stream);
      case 4: return launch_reorder<4>(held, many, blocks, n, parents, lengths, W, stream);
      case 2: return launch_reorder<2>(held, many, blocks, n, parents, lengths, W, stream);
      default: return launch_reorder<1>(held, many, blocks, n, parents, lengths, W, stream);
    }
  };
  return each_launch(tables, strides_b, strides_n, capacities, row_bytes, count, 1, widest, size, launch);
}

extern "C" int wptv_keep_rows(void* const* tables, const int64_t* strides_b, const int64_t* strides_n,
                              const int64_t* capacities, const int64_t* row_bytes, int count, const int64_t* kept,
                              int lists, int keep, const int64_t* counts, int B, hipStream_t stream) {
  if (count < 0 || lists < 0 || keep < 0 || B < 0 || (count && (lists == 0 || count % lists)))
    return fail(WPTV_E_INVALID, "keep_rows: %d tables for %d lists of %d rows, B=%d", count, lists, keep, B);
  if (B > 65535) return fail(WPTV_E_UNSUPPORTED, "keep_rows: at most 65535 batch rows (got %d)", B);
  if (count && (!tables || !strides_b || !strides_n || !capacities || !row_bytes))
    return fail(WPTV_E_INVALID, "keep_rows: the tables' addresses and shapes must be given");
  if ((__int128)lists * B * keep > INT64_MAX / 8) return fail(WPTV_E_INVALID, "keep_rows: lists of 2^60 rows");
  const int status = check_tables("keep_rows", tables, strides_b, strides_n, capacities, row_bytes, count, B,
                                  {{kept, (int64_t)lists * B * keep * (int64_t)sizeof(int64_t)},
                                   {counts, B * (int64_t)sizeof(int64_t)}});
  if (status != WPTV_OK) return status;
  if (count == 0 || B == 0 || keep == 0) return WPTV_OK;
  if (!kept || !counts) return fail(WPTV_E_INVALID, "keep_rows: kept and counts must be given");
  auto size = [](Table& t) { return t.pieces; };
  auto launch = [&](int unit, const Tables& held, int many, int64_t most) {
    switch (unit) {
      case 16: return launch_keep<16>(held, many, (int)most, kept, B, keep, counts, stream);
      case 8: return launch_keep<8>(held, many, (int)most, kept, B, keep, counts, stream);
      case 4: return launch_keep<4>(held, many, (int)most, kept, B, keep, counts, stream);
      case 2: return launch_keep<2>(held, many, (int)most, kept, B, keep, counts, stream);
      default: return launch_keep<1>(held, many, (int)most, kept, B, keep, counts, stream);
    }
  };
  return each_launch(tables, strides_b, strides_n, capacities, row_bytes, count, lists, 16, size, launch);
}
