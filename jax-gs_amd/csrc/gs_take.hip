// Rows of many tensors by one index, on gfx950: taken into new tensors, or moved in place.
//
//   take   out_k[i] = index[i] in [0, n) ? t_k[index[i]] : fill_k           i < r
//   move   t_k[i]   = t_k[index[i]]  where index[i] != i and index[index[i]] = index[i],
//                     fill_k         where index[i] < 0
//
// Rows are bytes, so that any type moves, and every value arrives as it was.  In a move no row that is
// read is written (a source is a row that stays), so the order of the writes does not matter; a row whose
// index asks for anything else stays and is counted.
//
// Both are bound by memory: what is taken is read and written once.  A row is dealt out in units, the
// largest power of two up to 16 bytes that divides its length, its stride and its addresses.
#include "gs_common.h"
#include "gs_pieces.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kRowTensors = 56;       // per launch: the argument block stays below 4 KiB
constexpr int kTakeBytes = 16384;     // of one output, per workgroup: 4 vectors of 16 bytes a lane
constexpr int64_t kMaxRowBytes = (int64_t)1 << 31;

struct RowRecord {
  const char* src;
  char* dst;
  const char* fill;
  int64_t stride;      // bytes from row to row of src (of both in a move)
  int64_t bytes;       // of all rows of dst, and zeros behind them
  uint32_t units;      // units per row
  uint32_t magic;      // floor(2^32 / units) + 1, 0 for rows of one unit
  uint8_t unit_log2;   // of a unit's bytes
};

struct RowArgs {
  RowRecord t[kRowTensors];
  uint32_t begin[kRowTensors];  // first workgroup of each tensor
  const void* index;
  int64_t count;                // entries of the index
  uint32_t rows;                // of the tensors that are read
  int32_t n;
  uint32_t groups;
  int32_t wide;                 // the index is int64
};
static_assert(sizeof(RowArgs) <= 4096, "kernel arguments");

// Entry i of the index, -1 for one that is no row.
__device__ inline int32_t row_at(const RowArgs& A, int64_t i) {
  if (A.wide) {
    const int64_t x = ((const int64_t*)A.index)[i];
    return x >= 0 && x < (int64_t)A.rows ? (int32_t)x : -1;
  }
  const int32_t x = ((const int32_t*)A.index)[i];
  return x >= 0 && (uint32_t)x < A.rows ? x : -1;
}

template <int kBytes> struct Unit;
template <> struct Unit<1> { typedef uint8_t type; };
template <> struct Unit<2> { typedef uint16_t type; };
template <> struct Unit<4> { typedef uint32_t type; };
template <> struct Unit<8> { typedef uint64_t type; };
template <> struct Unit<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };

typedef uint32_t vec16 __attribute__((ext_vector_type(4)));

// One workgroup's part of one output, 16 bytes a lane and store.
template <int kBytes>
__device__ inline void take_part(const RowArgs& A, const RowRecord& t, int64_t base) {
  typedef typename Unit<kBytes>::type unit;
  constexpr int kUnits = 16 / kBytes;  // in a vector
  constexpr int kVecs = kTakeBytes / 16 / 256;
  const uint32_t units = t.units;
  // the row of the workgroup's first unit: once, in scalar registers
  const uint64_t first = (uint64_t)base / kBytes, row0 = first / units;
  const uint32_t at = (uint32_t)(first - row0 * units);
  unit got[kVecs][kUnits];
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const uint32_t e0 = at + (v * 256 + threadIdx.x) * kUnits;
#pragma unroll
    for (int j = 0; j < kUnits; ++j) {
      const uint32_t e = e0 + j;
      uint32_t q;
      if (units > kTakeBytes / kBytes) q = e >= units ? 1u : 0u;
      else q = t.magic ? __umulhi(e, t.magic) : e;
      const uint32_t off = e - q * units;
      const int64_t row = (int64_t)(row0 + q);
      unit x{};
      if (row < A.count) {
        const int32_t s = row_at(A, row);
        if (s >= 0) x = *reinterpret_cast<const unit*>(t.src + s * t.stride + (int64_t)off * kBytes);
        else if (t.fill) x = *reinterpret_cast<const unit*>(t.fill + (int64_t)off * kBytes);
      }
      got[v][j] = x;
    }
  }
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int64_t to = base + (int64_t)(v * 256 + threadIdx.x) * 16;
    if (to + 16 <= t.bytes) {
      vec16 w;
      __builtin_memcpy(&w, got[v], 16);
      *reinterpret_cast<vec16*>(t.dst + to) = w;
    } else {
#pragma unroll
      for (int j = 0; j < kUnits; ++j)
        if (to + (j + 1) * kBytes <= t.bytes) *reinterpret_cast<unit*>(t.dst + to + j * kBytes) = got[v][j];
    }
  }
}

// The tensor of this workgroup: the last that begins at or before it.
__device__ inline int tensor_of(const RowArgs& A, uint32_t b) {
  const int lane = threadIdx.x & 63;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < A.n && b >= A.begin[min(lane, A.n - 1)])) - 1);
}

__global__ __launch_bounds__(256) void take_rows_kernel(RowArgs A) {
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const RowRecord& t = A.t[k];
  const int64_t base = (int64_t)(b - A.begin[k]) * kTakeBytes;
  switch (t.unit_log2) {
    case 4: take_part<16>(A, t, base); break;
    case 3: take_part<8>(A, t, base); break;
    case 2: take_part<4>(A, t, base); break;
    case 1: take_part<2>(A, t, base); break;
    default: take_part<1>(A, t, base);
  }
}

constexpr int kMoveRows = 1024;  // per workgroup

// One tensor's units of the `moved` rows listed: consecutive lanes, consecutive units.
template <int kBytes>
__device__ inline void move_part(const RowRecord& t, const int32_t* __restrict__ to, const int32_t* __restrict__ of,
                                 int moved, int64_t base) {
  typedef typename Unit<kBytes>::type unit;
  const uint64_t all = (uint64_t)moved * t.units;
  for (uint64_t e = threadIdx.x; e < all; e += 256) {
    // kMoveRows * units * units below 2^32: the reciprocal is exact
    const uint32_t q = t.units <= 1024 ? (t.magic ? __umulhi((uint32_t)e, t.magic) : (uint32_t)e) : (uint32_t)(e / t.units);
    const int64_t off = (int64_t)(e - (uint64_t)q * t.units) * kBytes;
    const int32_t s = of[q];
    unit x{};
    if (s >= 0) x = *reinterpret_cast<const unit*>(t.src + s * t.stride + off);
    else if (t.fill) x = *reinterpret_cast<const unit*>(t.fill + off);
    *reinterpret_cast<unit*>(t.dst + (base + to[q]) * t.stride + off) = x;
  }
}

__global__ __launch_bounds__(256) void move_rows_kernel(RowArgs A, int32_t* left) {
  __shared__ int32_t to[kMoveRows], of[kMoveRows];
  __shared__ int32_t moved;
  if (threadIdx.x == 0) moved = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kMoveRows;
  int bad = 0;
  for (int j = threadIdx.x; j < kMoveRows; j += 256) {
    const int64_t i = base + j;
    if (i >= A.count) continue;
    const int64_t x = A.wide ? ((const int64_t*)A.index)[i] : ((const int32_t*)A.index)[i];
    if (x == i) continue;
    if (x >= 0) {
      const int32_t s = row_at(A, i);
      if (s < 0 || row_at(A, s) != s) {
        ++bad;
        continue;
      }
    }
    const int p = atomicAdd(&moved, 1);
    to[p] = j;
    of[p] = x < 0 ? -1 : (int32_t)x;
  }
  if (left && bad) atomicAdd(left, bad);
  __syncthreads();
  const int m = moved;
  if (m == 0) return;
  for (int k = 0; k < A.n; ++k) {
    const RowRecord& t = A.t[k];
    switch (t.unit_log2) {
      case 4: move_part<16>(t, to, of, m, base); break;
      case 3: move_part<8>(t, to, of, m, base); break;
      case 2: move_part<4>(t, to, of, m, base); break;
      case 1: move_part<2>(t, to, of, m, base); break;
      default: move_part<1>(t, to, of, m, base);
    }
  }
}

// A record's unit: the largest that divides everything.
int unit_log2(int64_t row_bytes, int64_t stride, const void* a, const void* b, const void* c) {
  const uint64_t all = (uint64_t)row_bytes | (uint64_t)stride | (uint64_t)(uintptr_t)a | (uint64_t)(uintptr_t)b |
                       (uint64_t)(uintptr_t)c | 16u;
  return __builtin_ctzll(all);
}

void fill_record(RowRecord& t, const void* src, void* dst, const void* fill, int64_t row_bytes, int64_t stride) {
  t.src = (const char*)src;
  t.dst = (char*)dst;
  t.fill = (const char*)fill;
  t.stride = stride;
  t.unit_log2 = (uint8_t)unit_log2(row_bytes, stride, src, dst, fill);
  t.units = (uint32_t)(row_bytes >> t.unit_log2);
  t.magic = t.units > 1 ? (uint32_t)((((uint64_t)1 << 32) / t.units) + 1) : 0;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_take_rows(void* stream, int num, const void* const* tensors, const int64_t* row_bytes,
                            const int64_t* strides, int64_t rows, void* const* out, const int64_t* out_bytes,
                            const void* const* fills, const void* index, int index_bits, int64_t count) {
  GS_REQUIRE(num >= 0, "gs_take_rows: %d tensors", num);
  GS_REQUIRE(num == 0 || (tensors && row_bytes && strides && out), "gs_take_rows: NULL argument");
  GS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && count >= 0 && count < ((int64_t)1 << 31),
             "gs_take_rows: %lld rows by %lld indices", (long long)rows, (long long)count);
  GS_REQUIRE(index_bits == 32 || index_bits == 64, "gs_take_rows: indices of 32 or 64 bits, not %d", index_bits);
  GS_REQUIRE(count == 0 || index, "gs_take_rows: NULL index");
  GS_REQUIRE((reinterpret_cast<uintptr_t>(index) & (index_bits / 8 - 1)) == 0, "gs_take_rows: the index is not aligned");
  for (int i = 0; i < num; ++i) {
    GS_REQUIRE(row_bytes[i] >= 0 && row_bytes[i] < kMaxRowBytes, "gs_take_rows: rows of %lld bytes", (long long)row_bytes[i]);
    const int64_t need = row_bytes[i] * count, all = out_bytes ? out_bytes[i] : need;
    GS_REQUIRE(all >= need && all <= kMaxGroups * kTakeBytes && (all == 0 || row_bytes[i] > 0), "gs_take_rows: output %d of %lld bytes for %lld", i,
               (long long)all, (long long)need);
    GS_REQUIRE(all == 0 || out[i], "gs_take_rows: NULL output %d", i);
    GS_REQUIRE(need == 0 || rows == 0 || tensors[i], "gs_take_rows: NULL tensor %d", i);
    GS_REQUIRE((reinterpret_cast<uintptr_t>(out[i]) & 15) == 0, "gs_take_rows: output %d must be 16-byte aligned", i);
  }
  RowArgs A{};
  A.index = index;
  A.count = count;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  for (int i = 0; i < num;) {
    int k = 0;
    int64_t groups = 0;
    for (; i < num && k < kRowTensors; ++i) {
      const int64_t all = out_bytes ? out_bytes[i] : row_bytes[i] * count;
      if (all == 0) continue;
      const int64_t more = (all + kTakeBytes - 1) / kTakeBytes;
      if (groups + more > kMaxGroups) break;
      RowRecord& t = A.t[k];
      fill_record(t, tensors[i], out[i], fills ? fills[i] : nullptr, row_bytes[i], strides[i]);
      t.bytes = all;
      A.begin[k++] = (uint32_t)groups;
      groups += more;
    }
    if (k == 0) continue;
    A.n = k;
    A.groups = (uint32_t)groups;
    hipLaunchKernelGGL(take_rows_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, A);
    GS_LAUNCH_CHECK("take_rows_kernel");
  }
  return GS_OK;
}

extern "C" int gs_move_rows(void* stream, int num, void* const* tensors, const int64_t* row_bytes,
                            const int64_t* strides, int64_t rows, const void* const* fills, const void* index,
                            int index_bits, int32_t* left) {
  GS_REQUIRE(num >= 0, "gs_move_rows: %d tensors", num);
  GS_REQUIRE(num == 0 || (tensors && row_bytes && strides), "gs_move_rows: NULL argument");
  GS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31), "gs_move_rows: %lld rows", (long long)rows);
  GS_REQUIRE(index_bits == 32 || index_bits == 64, "gs_move_rows: indices of 32 or 64 bits, not %d", index_bits);
  GS_REQUIRE(rows == 0 || index, "gs_move_rows: NULL index");
  GS_REQUIRE((reinterpret_cast<uintptr_t>(index) & (index_bits / 8 - 1)) == 0, "gs_move_rows: the index is not aligned");
  for (int i = 0; i < num; ++i) {
    GS_REQUIRE(row_bytes[i] >= 0 && row_bytes[i] < kMaxRowBytes, "gs_move_rows: rows of %lld bytes", (long long)row_bytes[i]);
    GS_REQUIRE(rows <= 1 || strides[i] >= row_bytes[i], "gs_move_rows: the rows of tensor %d overlap", i);
    GS_REQUIRE(row_bytes[i] == 0 || rows == 0 || tensors[i], "gs_move_rows: NULL tensor %d", i);
  }
  if (rows == 0) return GS_OK;
  RowArgs A{};
  A.index = index;
  A.count = rows;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  const dim3 grid((unsigned)div_up(rows, kMoveRows));
  int i = 0;
  do {  // one launch at least: it counts the rows that are left
    A.n = 0;
    for (; i < num && A.n < kRowTensors; ++i)
      if (row_bytes[i]) fill_record(A.t[A.n++], tensors[i], tensors[i], fills ? fills[i] : nullptr, row_bytes[i], strides[i]);
    hipLaunchKernelGGL(move_rows_kernel, grid, dim3(256), 0, (hipStream_t)stream, A, left);
    GS_LAUNCH_CHECK("move_rows_kernel");
    left = nullptr;
  } while (i < num);
  return GS_OK;
}
