// Rows of moments in 8 bits by one index, on gfx950: taken into a new state, or moved in place.
//
// A tensor's moments are rows of row_len elements one after another, in blocks of 256 that share an
// exponent (gs_moments.h); a row's new neighbours are others than its old ones, so a block is decoded element by element from where
// its rows come from and encoded again, to nearest even.  Values come back as they were but where a
// larger neighbour raises the exponent of their block.
//
// A wave makes four blocks, four elements of each a lane, the loads of all four under way before the first is
// encoded.  In a move, blocks without a changed row are left out; the others go to a copy first, for a block is
// read by others while it changes.
#include "gs_moments.h"
#include "gs_pieces.h"
#include "gs_rows.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kMomentTensors = 80;  // per launch: the argument block stays below 4 KiB
constexpr int kMomentAhead = 4;     // blocks per wave
constexpr int kMomentGroup = 4 * kMomentAhead;  // per workgroup

struct MomentRecord {
  int64_t count;     // elements behind which there is nothing
  uint64_t magic;    // row_magic
  uint32_t src_at, dst_at;  // blocks
  uint32_t row_len;
  uint32_t blocks;
};

struct MomentArgs {
  MomentRecord t[kMomentTensors];
  uint32_t begin[kMomentTensors];
  const uint8_t *m8, *r8, *fields;
  uint8_t *to_m8, *to_r8, *to_fields;
  uint8_t* changed;  // per block of a move
  const void* index;
  uint32_t rows;     // of the tensors that are read
  int32_t n;
  uint32_t groups;
  int32_t wide;
};
static_assert(sizeof(MomentArgs) <= 4096, "kernel arguments");

// Entry i of the index, -1 for one that is no row.
__device__ inline int32_t entry(const MomentArgs& A, int64_t i) {
  if (A.wide) {
    const int64_t x = ((const int64_t*)A.index)[i];
    return x >= 0 && x < (int64_t)A.rows ? (int32_t)x : -1;
  }
  const int32_t x = ((const int32_t*)A.index)[i];
  return x >= 0 && (uint32_t)x < A.rows ? x : -1;
}

// Where row i comes from, -1 for nowhere.
template <bool kMove>
__device__ inline int32_t source(const MomentArgs& A, int32_t i) {
  const int32_t s = entry(A, i);
  if (!kMove || s == i) return s;
  if (s >= 0) return entry(A, s) == s ? s : i;
  // a negative index frees the row, one beyond the rows leaves it
  const int64_t x = A.wide ? ((const int64_t*)A.index)[i] : ((const int32_t*)A.index)[i];
  return x < 0 ? -1 : i;
}

// The tensor of this workgroup: the last that begins at or before it.
__device__ inline int tensor_of(const MomentArgs& A, uint32_t b) {
  const int lane = threadIdx.x & 63;
  int k = -1;
  for (int at = 0; at < A.n; at += 64) k += __popcll(__ballot(at + lane < A.n && b >= A.begin[min(at + lane, A.n - 1)]));
  return __builtin_amdgcn_readfirstlane(k);
}

// The blocks from `first` on of one tensor (the whole wave).  kQuad: rows of a multiple of four elements, of
// which a lane's four are of one row and of one block.
template <bool kMove, bool kQuad>
__device__ inline void make_blocks(const MomentArgs& A, const MomentRecord& t, uint32_t first) {
  constexpr int kOf = kQuad ? 1 : 4;  // sources of a lane's elements
  const int lane = threadIdx.x & 63;
  const uint32_t len = t.row_len;
  const int64_t base0 = (int64_t)first * kMomBlock;
  const uint64_t row0 = t.magic ? __umul64hi((uint64_t)base0, t.magic) : (uint64_t)base0;
  const uint32_t at0 = (uint32_t)((uint64_t)base0 - row0 * len);
  int32_t s[kMomentAhead][kOf];
  uint32_t off[kMomentAhead][kOf];
  uint32_t some = 0;  // blocks to make
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) {
    bool moved = false;
#pragma unroll
    for (int j = 0; j < kOf; ++j) {
      const uint32_t d = g * kMomBlock + lane * 4 + j, e = at0 + d;
      // less than row_len + 1024 elements from the first row
      const uint32_t q = len > 4096u ? (e >= len ? 1u : 0u) : t.magic ? __umulhi(e, (uint32_t)(t.magic >> 32) + 1u) : e;
      const int32_t row = (int32_t)(row0 + q);
      const bool in = base0 + d < t.count;
      off[g][j] = e - q * len;
      s[g][j] = in ? source<kMove>(A, row) : -1;
      if (kMove) moved |= in && s[g][j] != row;
    }
    if (first + g < t.blocks && (!kMove || __ballot(moved))) some |= 1u << g;
  }
  if (kMove) {
    if (lane < kMomentAhead && first + lane < t.blocks) A.changed[t.dst_at + first + lane] = some >> lane & 1u;
    if (some == 0) return;
  }
  const uint64_t from = (uint64_t)t.src_at * kMomBlock;
  uint32_t wm[kMomentAhead], wr[kMomentAhead], f[kMomentAhead][kOf];
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) {
    wm[g] = wr[g] = 0;
    if (!(some >> g & 1u)) continue;
#pragma unroll
    for (int j = 0; j < kOf; ++j) {
      f[g][j] = 0;
      if (s[g][j] < 0) continue;
      const uint64_t at = from + (uint64_t)s[g][j] * len + off[g][j];
      if (kQuad) {
        wm[g] = *reinterpret_cast<const uint32_t*>(A.m8 + at);
        wr[g] = *reinterpret_cast<const uint32_t*>(A.r8 + at);
      } else {
        wm[g] |= (uint32_t)A.m8[at] << (8 * j);
        wr[g] |= (uint32_t)A.r8[at] << (8 * j);
      }
      f[g][j] = *(const uint16_t*)(A.fields + 2 * (at >> 8));
    }
  }
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) {
    if (!(some >> g & 1u)) continue;
    int fm[4], fr[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      fm[j] = (int)(f[g][j % kOf] & 255u);
      fr[j] = (int)(f[g][j % kOf] >> 8);
    }
    float m[4], r[4];
    decode_m4(wm[g], fm, m);
    decode_r4(wr[g], fr, r);
    const uint32_t none[4] = {0, 0, 0, 0};
    uint32_t cm, cr, fields;
    encode_block<false>(m, r, none, cm, cr, fields);
    const uint64_t to = ((uint64_t)t.dst_at + first + g) * kMomBlock + lane * 4;
    *reinterpret_cast<uint32_t*>(A.to_m8 + to) = cm;
    *reinterpret_cast<uint32_t*>(A.to_r8 + to) = cr;
    if (lane == 0) *(uint16_t*)(A.to_fields + 2 * (to >> 8)) = (uint16_t)fields;
  }
}

template <bool kMove>
__global__ __launch_bounds__(256) void moment_rows_kernel(MomentArgs A) {
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const MomentRecord& t = A.t[k];
  const uint32_t first =
      __builtin_amdgcn_readfirstlane((b - A.begin[k]) * kMomentGroup + (threadIdx.x >> 6) * kMomentAhead);
  if (first >= t.blocks) return;
  if (t.row_len % 4 == 0) make_blocks<kMove, true>(A, t, first);
  else make_blocks<kMove, false>(A, t, first);
}

// The changed blocks from the copy into their places, 16 bytes a lane and array.
__global__ __launch_bounds__(256) void moment_back_kernel(MomentArgs A) {
  typedef uint32_t vec __attribute__((ext_vector_type(4)));
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const uint32_t block = (b - A.begin[k]) * kMomentGroup + (threadIdx.x >> 4);
  if (block >= A.t[k].blocks) return;
  const uint64_t i = (uint64_t)A.t[k].dst_at + block;
  if (!A.changed[i]) return;
  const uint64_t at = i * kMomBlock + (threadIdx.x & 15) * 16;
  *reinterpret_cast<vec*>(const_cast<uint8_t*>(A.m8) + at) = *reinterpret_cast<const vec*>(A.to_m8 + at);
  *reinterpret_cast<vec*>(const_cast<uint8_t*>(A.r8) + at) = *reinterpret_cast<const vec*>(A.to_r8 + at);
  if ((threadIdx.x & 15) == 0) *(uint16_t*)(const_cast<uint8_t*>(A.fields) + 2 * i) = *(const uint16_t*)(A.to_fields + 2 * i);
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Layout checks of one side: the moments of each tensor behind those before, inside the state.
int check_side(const char* what, int num, const int64_t* row_lens, int64_t rows, const int64_t* offsets, int64_t size) {
  int64_t used = 0;
  for (int i = 0; i < num; ++i) {
    GS_REQUIRE(row_lens[i] >= 0 && row_lens[i] < kMaxRowLen, "%s: rows of %lld elements", what, (long long)row_lens[i]);
    if (row_lens[i] == 0 || rows == 0) continue;
    GS_REQUIRE(rows < ((int64_t)1 << 40) / row_lens[i], "%s: tensor %d is too large", what, i);
    GS_REQUIRE(offsets[i] >= used && offsets[i] % kMomBlock == 0 && offsets[i] <= size &&
                   rows * row_lens[i] <= size - offsets[i],
               "%s: the moments of tensor %d lie outside the state, or on those before", what, i);
    used = offsets[i] + rows * row_lens[i];
  }
  return GS_OK;
}

enum { kTake, kMove, kBack };

int launch(int what, hipStream_t stream, int num, const int64_t* row_lens, const int64_t* offsets, const int64_t* out_offsets,
           int64_t count, MomentArgs& A) {
  for (int i = 0; i < num;) {
    int k = 0;
    int64_t groups = 0;
    for (; i < num && k < kMomentTensors; ++i) {
      const int64_t elements = row_lens[i] * count, blocks = (elements + kMomBlock - 1) / kMomBlock;
      if (blocks == 0) continue;
      const int64_t more = (blocks + kMomentGroup - 1) / kMomentGroup;
      GS_REQUIRE(more <= kMaxGroups, "gs_moments: tensor %d is too large", i);
      if (groups + more > kMaxGroups) break;
      MomentRecord& t = A.t[k];
      t.count = elements;
      t.row_len = (uint32_t)row_lens[i];
      t.magic = row_magic(row_lens[i]);
      t.src_at = (uint32_t)(offsets[i] / kMomBlock);
      t.dst_at = (uint32_t)(out_offsets[i] / kMomBlock);
      t.blocks = (uint32_t)blocks;
      A.begin[k++] = (uint32_t)groups;
      groups += more;
    }
    if (k == 0) continue;
    A.n = k;
    A.groups = (uint32_t)groups;
    auto* kernel = what == kTake ? moment_rows_kernel<false> : what == kMove ? moment_rows_kernel<true> : moment_back_kernel;
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, stream, A);
    GS_LAUNCH_CHECK("moment_rows_kernel");
  }
  return GS_OK;
}

size_t padded(int64_t bytes) { return ((size_t)bytes + 255) & ~(size_t)255; }

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_moments_take(void* stream, int num, const int64_t* row_lens, int64_t rows, const int64_t* offsets,
                               int64_t state_size, const uint8_t* mu8, const uint8_t* nu8, const uint8_t* fields,
                               const void* index, int index_bits, int64_t count, const int64_t* out_offsets,
                               int64_t out_size, uint8_t* out_mu8, uint8_t* out_nu8, uint8_t* out_fields) {
  const char* what = "gs_moments_take";
  GS_REQUIRE(num >= 0 && (num == 0 || (row_lens && offsets && out_offsets)), "%s: NULL argument", what);
  GS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && count >= 0 && count < ((int64_t)1 << 31),
             "%s: %lld rows by %lld indices", what, (long long)rows, (long long)count);
  GS_REQUIRE(index_bits == 32 || index_bits == 64, "%s: indices of 32 or 64 bits, not %d", what, index_bits);
  GS_REQUIRE(count == 0 || index, "%s: NULL index", what);
  GS_REQUIRE(aligned(index, index_bits / 8), "%s: the index is not aligned", what);
  GS_REQUIRE(state_size >= 0 && state_size % kMomBlock == 0 && state_size < ((int64_t)1 << 40) && out_size >= 0 &&
                 out_size % kMomBlock == 0 && out_size < ((int64_t)1 << 40),
             "%s: states of %lld and %lld elements", what, (long long)state_size, (long long)out_size);
  GS_REQUIRE(state_size == 0 || (mu8 && nu8 && fields), "%s: NULL state", what);
  GS_REQUIRE(out_size == 0 || (out_mu8 && out_nu8 && out_fields), "%s: NULL state", what);
  GS_REQUIRE(aligned(mu8, 16) && aligned(nu8, 16) && aligned(fields, 2) && aligned(out_mu8, 16) && aligned(out_nu8, 16) &&
                 aligned(out_fields, 2),
             "%s: the states' arrays must be 16-byte aligned", what);
  int rc = check_side(what, num, row_lens, rows, offsets, state_size);
  if (rc == GS_OK) rc = check_side(what, num, row_lens, count, out_offsets, out_size);
  if (rc != GS_OK) return rc;
  MomentArgs A{};
  A.m8 = mu8;
  A.r8 = nu8;
  A.fields = fields;
  A.to_m8 = out_mu8;
  A.to_r8 = out_nu8;
  A.to_fields = out_fields;
  A.index = index;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  return launch(kTake, (hipStream_t)stream, num, row_lens, offsets, out_offsets, count, A);
}

extern "C" size_t gs_moments_move_workspace_size(int64_t state_size) {
  if (state_size < 0 || state_size % kMomBlock) return 0;
  const int64_t blocks = state_size / kMomBlock;
  return (size_t)state_size * 2 + padded(blocks * 2) + padded(blocks);
}

extern "C" int gs_moments_move(void* stream, int num, const int64_t* row_lens, int64_t rows, const int64_t* offsets,
                               int64_t state_size, uint8_t* mu8, uint8_t* nu8, uint8_t* fields, const void* index,
                               int index_bits, void* workspace, size_t workspace_bytes) {
  const char* what = "gs_moments_move";
  GS_REQUIRE(num >= 0 && (num == 0 || (row_lens && offsets)), "%s: NULL argument", what);
  GS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31), "%s: %lld rows", what, (long long)rows);
  GS_REQUIRE(index_bits == 32 || index_bits == 64, "%s: indices of 32 or 64 bits, not %d", what, index_bits);
  GS_REQUIRE(rows == 0 || index, "%s: NULL index", what);
  GS_REQUIRE(aligned(index, index_bits / 8), "%s: the index is not aligned", what);
  GS_REQUIRE(state_size >= 0 && state_size % kMomBlock == 0 && state_size < ((int64_t)1 << 40),
             "%s: state of %lld elements", what, (long long)state_size);
  GS_REQUIRE(state_size == 0 || (mu8 && nu8 && fields && workspace), "%s: NULL state", what);
  GS_REQUIRE(aligned(mu8, 16) && aligned(nu8, 16) && aligned(fields, 2) && aligned(workspace, 16),
             "%s: the state's arrays and the workspace must be 16-byte aligned", what);
  const size_t need = gs_moments_move_workspace_size(state_size);
  GS_REQUIRE(workspace_bytes >= need, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  const int rc = check_side(what, num, row_lens, rows, offsets, state_size);
  if (rc != GS_OK) return rc;
  const int64_t blocks = state_size / kMomBlock;
  uint8_t* ws = (uint8_t*)workspace;
  MomentArgs A{};
  A.m8 = mu8;
  A.r8 = nu8;
  A.fields = fields;
  A.to_m8 = ws;
  A.to_r8 = ws + state_size;
  A.to_fields = ws + 2 * state_size;
  A.changed = ws + 2 * state_size + padded(blocks * 2);
  A.index = index;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  const int done = launch(kMove, (hipStream_t)stream, num, row_lens, offsets, offsets, rows, A);
  if (done != GS_OK) return done;
  return launch(kBack, (hipStream_t)stream, num, row_lens, offsets, offsets, rows, A);
}
