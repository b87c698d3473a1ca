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
// Both are bound by memory: what is taken is read and written once.  Rows lie at any byte, so loads of up to
// 16 bytes go to any address; outputs are written 16 bytes a lane, a vector that two rows share joined from both,
// rows shorter than a vector by way of LDS (2M rows: 90 bytes 64 us, 279 in units of two bytes; 12 bytes at random 40
// us, 57 in units of four).  192 bytes 133 us (6.1 TB/s; a copy of the same size 155), pages of 16 KiB 343 (6.3).
#include "gs_common.h"
#include "gs_pieces.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kRowTensors = 56;  // per launch: the argument block stays below 4 KiB
constexpr int kTakeVecs = 2;     // vectors of 16 bytes a lane (192-byte rows 133 us; one 149, four 134)
constexpr int kTakeBytes = kTakeVecs * 256 * 16;  // of one output, per workgroup
constexpr int kTakeRows = 512;   // per workgroup where rows are shorter than 16 bytes
// Outputs go past the caches from here on: 128 MB 49 us and 41 past them, but with a sweep that reads them
// next 92 and 97; 192 MB 82 and 69, with the sweep 150 and 145.
constexpr int64_t kStreamBytes = (int64_t)160 << 20;
constexpr int64_t kMaxRowBytes = (int64_t)1 << 31;

struct RowRecord {
  const char* src;
  char* dst;
  const char* fill;
  int64_t stride;      // bytes from row to row of src (of both in a move)
  int64_t bytes;       // of all rows of dst, and zeros behind them
  uint64_t magic64;    // floor(2^64 / row) + 1, 0 where a division is needed
  uint32_t row;        // bytes
  uint32_t magic;      // floor(2^32 / row) + 1; in a move of the 16-byte pieces of a row, 0 for one
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

// Loads and stores at any address.
typedef uint16_t any2 __attribute__((aligned(1)));
typedef uint32_t any4 __attribute__((aligned(1)));
typedef uint32_t any8 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t vec16 __attribute__((ext_vector_type(4)));

// Row s of t, the fill for s < 0, or null (zeros).
__device__ inline const char* row_ptr(const RowRecord& t, int32_t s) { return s >= 0 ? t.src + s * t.stride : t.fill; }

// The 16 bytes that begin `k` bytes before the end of a (1 <= k <= 15) and go on with b.
__device__ inline vec16 join(vec16 a, vec16 b, uint32_t k) {
  const uint32_t w[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  const uint32_t word = (16 - k) >> 2, byte = (16 - k) & 3;  // where they begin
  uint32_t x[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) x[j] = word == 0 ? w[j] : word == 1 ? w[j + 1] : word == 2 ? w[j + 2] : w[j + 3];
  vec16 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_alignbyte(x[j + 1], x[j], byte);
  return r;
}

template <bool kStream>
__device__ inline void put(char* to, vec16 x) {
  if (kStream) __builtin_nontemporal_store(x, reinterpret_cast<vec16*>(to));
  else *reinterpret_cast<vec16*>(to) = x;
}

// A workgroup's part of an output with rows of 16 bytes and more: a lane's vectors lie in one row or, where
// kSplit, in two.
template <bool kSplit, bool kStream>
__device__ inline void take_long(const RowArgs& A, const RowRecord& t, uint32_t group) {
  const int64_t base = (int64_t)group * kTakeBytes;
  const uint32_t row = t.row;
  // the row of the workgroup's first byte: once, in scalar registers
  const uint64_t row0 = t.magic64 ? __umul64hi((uint64_t)base, t.magic64) : (uint64_t)base / row;
  const uint32_t at = (uint32_t)((uint64_t)base - row0 * row);
  vec16 got[kTakeVecs];
#pragma unroll
  for (int v = 0; v < kTakeVecs; ++v) {
    const uint32_t e = at + (v * 256 + threadIdx.x) * 16;
    // e < row + kTakeBytes; with row <= kTakeBytes the reciprocal is exact
    const uint32_t q = row > kTakeBytes ? (e >= row ? 1u : 0u) : __umulhi(e, t.magic);
    const uint32_t off = e - q * row;
    const int64_t i = (int64_t)(row0 + q);
    vec16 x{};
    if (i < A.count) {
      const char* p = row_ptr(t, row_at(A, i));
      if (!kSplit || off + 16 <= row) {
        if (p) x = *reinterpret_cast<const any16*>(p + off);
      } else {
        vec16 a{}, b{};
        if (p) a = *reinterpret_cast<const any16*>(p + row - 16);
        if (i + 1 < A.count) {
          const char* next = row_ptr(t, row_at(A, i + 1));
          if (next) b = *reinterpret_cast<const any16*>(next);
        }
        x = join(a, b, row - off);
      }
    }
    got[v] = x;
  }
#pragma unroll
  for (int v = 0; v < kTakeVecs; ++v) {
    const int64_t to = base + (int64_t)(v * 256 + threadIdx.x) * 16;
    if (to + 16 <= t.bytes) {
      put<kStream>(t.dst + to, got[v]);
    } else if (to < t.bytes) {
      uint8_t b[16];
      __builtin_memcpy(b, &got[v], 16);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (to + j < t.bytes) t.dst[to + j] = (char)b[j];
    }
  }
}

// Copies a row of fewer than 16 bytes, or zeros.
__device__ inline void copy_short(char* to, const char* from, uint32_t row) {
  any8 a = {};
  any4 b = 0;
  any2 c = 0;
  uint8_t d = 0;
  if (from) {
    if (row & 8) a = *reinterpret_cast<const any8*>(from);
    if (row & 4) b = *reinterpret_cast<const any4*>(from + (row & 8));
    if (row & 2) c = *reinterpret_cast<const any2*>(from + (row & 12));
    if (row & 1) d = *reinterpret_cast<const uint8_t*>(from + (row & 14));
  }
  if (row & 8) *reinterpret_cast<any8*>(to) = a;
  if (row & 4) *reinterpret_cast<any4*>(to + (row & 8)) = b;
  if (row & 2) *reinterpret_cast<any2*>(to + (row & 12)) = c;
  if (row & 1) *reinterpret_cast<uint8_t*>(to + (row & 14)) = d;
}

// A workgroup's part of an output with shorter rows: a lane fetches rows, which go out by way of LDS.
template <bool kStream>
__device__ inline void take_short(const RowArgs& A, const RowRecord& t, uint32_t group, char* lds) {
  const int64_t i0 = (int64_t)group * kTakeRows;
  const uint32_t row = t.row;
#pragma unroll
  for (int v = 0; v < kTakeRows / 256; ++v) {
    const uint32_t r = v * 256 + threadIdx.x;
    const int64_t i = i0 + r;
    copy_short(lds + r * row, i < A.count ? row_ptr(t, row_at(A, i)) : nullptr, row);
  }
  __syncthreads();
  const int64_t base = i0 * row;  // a multiple of 16
  for (uint32_t e = threadIdx.x * 16; e < kTakeRows * row; e += 256 * 16) {
    const vec16 x = *reinterpret_cast<const vec16*>(lds + e);
    if (base + e + 16 <= t.bytes) {
      put<kStream>(t.dst + base + e, x);
    } else {
      for (int j = 0; j < 16 && base + e + j < t.bytes; ++j) t.dst[base + e + j] = lds[e + j];
    }
  }
}

// The tensor of this workgroup: the last that begins at or before it.
__device__ inline int tensor_of(const RowArgs& A, uint32_t b) {
  const int lane = threadIdx.x & 63;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(lane < A.n && b >= A.begin[min(lane, A.n - 1)])) - 1);
}

template <bool kStream>
__global__ __launch_bounds__(256) void take_rows_kernel(RowArgs A) {
  __shared__ __attribute__((aligned(16))) char lds[kTakeRows * 15];
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const RowRecord& t = A.t[k];
  const uint32_t group = b - A.begin[k];
  if (t.row < 16) take_short<kStream>(A, t, group, lds);
  else if (t.row % 16) take_long<true, kStream>(A, t, group);
  else take_long<false, kStream>(A, t, group);
}

// A move: a workgroup looks at up to 256 rows and copies those that change, in pieces of 16 bytes -- the last of a row up
// to its end (it writes what the piece before it writes too) -- or whole shorter rows.
constexpr int kMoveRows = 256;     // per workgroup at most
constexpr int kMovePieces = 512;   // of a row's in all tensors, up to which they are dealt out together
constexpr int kWidePieces = 4096;  // of wide rows, per workgroup
constexpr int kMoveAhead = 4;      // pieces in flight a lane

// A piece on its way: a vector, or a short row's parts of 8, 4, 2 and 1 bytes.
__device__ inline vec16 load_piece(const char* from, uint32_t row) {
  vec16 x{};
  if (row >= 16) {
    if (from) x = *reinterpret_cast<const any16*>(from);
    return x;
  }
  if (from) {
    if (row & 8) {
      const any8 a = *reinterpret_cast<const any8*>(from);
      x[0] = a[0];
      x[1] = a[1];
    }
    if (row & 4) x[2] = *reinterpret_cast<const any4*>(from + (row & 8));
    if (row & 2) x[3] = *reinterpret_cast<const any2*>(from + (row & 12));
    if (row & 1) x[3] |= (uint32_t)*reinterpret_cast<const uint8_t*>(from + (row & 14)) << 16;
  }
  return x;
}
__device__ inline void store_piece(char* to, uint32_t row, vec16 x) {
  if (row >= 16) {
    *reinterpret_cast<any16*>(to) = x;
    return;
  }
  if (row & 8) *reinterpret_cast<any8*>(to) = any8{x[0], x[1]};
  if (row & 4) *reinterpret_cast<any4*>(to + (row & 8)) = x[2];
  if (row & 2) *reinterpret_cast<any2*>(to + (row & 12)) = (uint16_t)x[3];
  if (row & 1) *reinterpret_cast<uint8_t*>(to + (row & 14)) = (uint8_t)(x[3] >> 16);
}

struct MoveArgs {
  RowArgs rows;      // records: bytes holds the first piece of the tensor, magic is of its pieces
  int32_t tile;      // rows per workgroup
  uint32_t pieces;   // of one row in all tensors, 0 where they are too many to be dealt out together
};
static_assert(sizeof(MoveArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(256) void move_rows_kernel(MoveArgs M, int32_t* left) {
  const RowArgs& A = M.rows;
  __shared__ int32_t to[kMoveRows], of[kMoveRows];
  __shared__ int32_t moved;
  __shared__ uint8_t tensor[kMovePieces];
  __shared__ RowRecord rec[kRowTensors];
  if (threadIdx.x == 0) moved = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * M.tile, i = base + threadIdx.x;
  bool some = false, bad = false;
  int64_t x = i;
  if ((int)threadIdx.x < M.tile && i < A.count) {
    x = A.wide ? ((const int64_t*)A.index)[i] : ((const int32_t*)A.index)[i];
    some = x != i;
    if (some && x >= 0) bad = x >= (int64_t)A.rows || row_at(A, x) != x;
  }
  const uint64_t move = __ballot(some && !bad), stay = __ballot(bad);
  const int lane = threadIdx.x & 63;
  if (lane == 0 && stay && left && blockIdx.y == 0 && blockIdx.z == 0) atomicAdd(left, __popcll(stay));
  int32_t at = 0;
  if (lane == 0 && move) at = atomicAdd(&moved, __popcll(move));
  at = __builtin_amdgcn_readfirstlane(at);
  if (some && !bad) {
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(move >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)move, 0));
    to[at + below] = threadIdx.x;
    of[at + below] = x < 0 ? -1 : (int32_t)x;
  }
  __syncthreads();
  const uint32_t m = moved;
  if (m == 0) return;
  if (M.pieces == 0) {  // wide rows: kWidePieces of one tensor's
    const RowRecord& t = A.t[blockIdx.y];
    const uint32_t row = t.row, first = blockIdx.z * kWidePieces, all_pieces = (row + 15) / 16;
    if (first >= all_pieces) return;
    const uint32_t pieces = min(all_pieces - first, (uint32_t)kWidePieces), all = m * pieces;
    const uint32_t by = pieces > 1 ? 0xffffffffu / pieces + 1 : 0;
    for (uint32_t e0 = threadIdx.x; e0 < all; e0 += 256 * kMoveAhead) {
      vec16 got[kMoveAhead];
      char* at[kMoveAhead];
#pragma unroll
      for (int u = 0; u < kMoveAhead; ++u) {
        const uint32_t e = e0 + 256 * u;
        at[u] = nullptr;
        if (e < all) {
          const uint32_t q = by ? __umulhi(e, by) : e, c = (first + e - q * pieces) * 16;
          const uint32_t off = row < 16 ? 0 : min(c, row - 16);
          const char* from = row_ptr(t, of[q]);
          got[u] = load_piece(from ? from + off : from, row);
          at[u] = t.dst + (base + to[q]) * t.stride + off;
        }
      }
#pragma unroll
      for (int u = 0; u < kMoveAhead; ++u)
        if (at[u]) store_piece(at[u], row, got[u]);
    }
    return;
  }
  // the records and every piece's tensor at hand
  for (int j = threadIdx.x; j < A.n * (int)(sizeof(RowRecord) / 8); j += 256)
    reinterpret_cast<uint64_t*>(rec)[j] = reinterpret_cast<const uint64_t*>(A.t)[j];
  for (int k = threadIdx.x >> 6; k < A.n; k += 4) {
    const uint32_t first = (uint32_t)A.t[k].bytes, pieces = (A.t[k].row + 15) / 16;
    for (uint32_t c = lane; c < pieces; c += 64) tensor[first + c] = (uint8_t)k;
  }
  __syncthreads();
  const uint32_t all = m * M.pieces;
  const uint32_t by_m = m > 1 ? 0xffffffffu / m + 1 : 0;
  for (uint32_t e0 = threadIdx.x; e0 < all; e0 += 256 * kMoveAhead) {
    vec16 got[kMoveAhead];
    char* at[kMoveAhead];
    uint32_t row[kMoveAhead];
#pragma unroll
    for (int u = 0; u < kMoveAhead; ++u) {
      const uint32_t e = e0 + 256 * u;
      row[u] = 0;
      if (e < all) {
        // tensor after tensor, row after row: neighbours write side by side
        const RowRecord& t = rec[tensor[by_m ? __umulhi(e, by_m) : e]];
        row[u] = t.row;
        const uint32_t pieces = (row[u] + 15) / 16, r = e - m * (uint32_t)t.bytes;
        const uint32_t q = t.magic ? __umulhi(r, t.magic) : r;
        const uint32_t off = row[u] < 16 ? 0 : min((r - q * pieces) * 16, row[u] - 16);
        const char* from = row_ptr(t, of[q]);
        got[u] = load_piece(from ? from + off : from, row[u]);
        at[u] = t.dst + (base + to[q]) * t.stride + off;
      }
    }
#pragma unroll
    for (int u = 0; u < kMoveAhead; ++u)
      if (row[u]) store_piece(at[u], row[u], got[u]);
  }
}

// Bytes of an output that a workgroup writes.
int64_t take_bytes(int64_t row) { return row < 16 ? kTakeRows * row : kTakeBytes; }

uint32_t reciprocal(uint32_t d) { return d > 1 ? (uint32_t)((((uint64_t)1 << 32) / d) + 1) : 0; }

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
    GS_REQUIRE(all >= need && all <= kMaxGroups * take_bytes(row_bytes[i]) && (all == 0 || row_bytes[i] > 0),
               "gs_take_rows: output %d of %lld bytes for %lld", i, (long long)all, (long long)need);
    GS_REQUIRE(all == 0 || out[i], "gs_take_rows: NULL output %d", i);
    GS_REQUIRE(need == 0 || rows == 0 || tensors[i], "gs_take_rows: NULL tensor %d", i);
    GS_REQUIRE((reinterpret_cast<uintptr_t>(out[i]) & 15) == 0, "gs_take_rows: output %d must be 16-byte aligned", i);
  }
  RowArgs A{};
  A.index = index;
  A.count = count;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  int64_t written = 0;
  for (int i = 0; i < num; ++i) written += out_bytes ? out_bytes[i] : row_bytes[i] * count;
  auto* kernel = written >= kStreamBytes ? take_rows_kernel<true> : take_rows_kernel<false>;
  for (int i = 0; i < num;) {
    int k = 0;
    int64_t groups = 0;
    for (; i < num && k < kRowTensors; ++i) {
      const int64_t all = out_bytes ? out_bytes[i] : row_bytes[i] * count;
      if (all == 0) continue;
      const int64_t per = take_bytes(row_bytes[i]), more = (all + per - 1) / per;
      if (groups + more > kMaxGroups) break;
      RowRecord& t = A.t[k];
      t.src = (const char*)tensors[i];
      t.dst = (char*)out[i];
      t.fill = fills ? (const char*)fills[i] : nullptr;
      t.stride = strides[i];
      t.bytes = all;
      t.row = (uint32_t)row_bytes[i];
      t.magic = reciprocal(t.row);
      // exact for offsets times rows below 2^64; outputs stay below 2^37 bytes
      t.magic64 = row_bytes[i] < ((int64_t)1 << 26) ? ~(uint64_t)0 / t.row + 1 : 0;
      A.begin[k++] = (uint32_t)groups;
      groups += more;
    }
    if (k == 0) continue;
    A.n = k;
    A.groups = (uint32_t)groups;
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, A);
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
  MoveArgs M{};
  RowArgs& A = M.rows;
  A.index = index;
  A.count = rows;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  int i = 0;
  do {  // one launch at least: it counts the rows that are left
    A.n = 0;
    int64_t pieces = 0, most = 0;
    for (; i < num && A.n < kRowTensors; ++i)
      if (row_bytes[i]) {
        RowRecord& t = A.t[A.n++];
        t.src = t.dst = (char*)tensors[i];
        t.fill = fills ? (const char*)fills[i] : nullptr;
        t.stride = strides[i];
        t.row = (uint32_t)row_bytes[i];
        t.bytes = pieces;
        t.magic = reciprocal((t.row + 15) / 16);
        pieces += (t.row + 15) / 16;
        most = std::max<int64_t>(most, (t.row + 15) / 16);
      }
    M.pieces = pieces <= kMovePieces ? (uint32_t)pieces : 0;
    dim3 grid;
    if (M.pieces || A.n == 0) {
      // few rows a workgroup where there are few workgroups, as the rows that change may lie together: 200k rows of 15
      // arrays, the last 5 % change, 12.7 us by 64, 17.8 by 128, 29.9 by 256; but 3M rows of four tensors, one in six
      // changes, 109, 82 and 69
      M.tile = rows <= ((int64_t)1 << 18) ? 64 : rows <= ((int64_t)1 << 19) ? 128 : kMoveRows;
      while (M.tile > 32 && M.tile * pieces > 16384 && div_up(rows, M.tile / 2) <= kMaxGroups) M.tile /= 2;
    } else {
      const int64_t fit = kWidePieces / std::min<int64_t>(most, kWidePieces);
      M.tile = (int)std::min<int64_t>(fit, 64);
      while (div_up(rows, M.tile) > kMaxGroups) M.tile *= 2;
      grid.y = (unsigned)A.n;
      grid.z = (unsigned)div_up(most, kWidePieces);
    }
    grid.x = (unsigned)div_up(rows, M.tile);
    hipLaunchKernelGGL(move_rows_kernel, grid, dim3(256), 0, (hipStream_t)stream, M, left);
    GS_LAUNCH_CHECK("move_rows_kernel");
    left = nullptr;
  } while (i < num);
  return GS_OK;
}
