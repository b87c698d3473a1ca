// Rows of moments in 8 bits by one index, on gfx950: taken into a new state, or moved in place.
//
// A tensor's moments are rows of row_len elements one after another, in blocks of 256 that share an
// exponent (gs_moments.h); a row's new neighbours are others than its old ones, so a block is decoded element by element from where
// its rows come from and encoded again, to nearest even.  Values come back as they were but where a
// larger neighbour raises the exponent of their block.
//
// A wave makes a block, four elements a lane.  In a move, blocks without a changed row are left out; the
// others go to a copy first, for a block is read by others while it changes.
#include "gs_moments.h"
#include "gs_pieces.h"
#include "gs_rows.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kMomentTensors = 80;  // per launch: the argument block stays below 4 KiB
constexpr int kMomentGroup = 4;     // blocks per workgroup

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

template <bool kMove>
__global__ __launch_bounds__(256) void moment_rows_kernel(MomentArgs A) {
  const uint32_t b = blockIdx.x;
  const int lane = threadIdx.x & 63;
  if (b >= A.groups) return;
  int k = -1;
  for (int at = 0; at < A.n; at += 64) k += __popcll(__ballot(at + lane < A.n && b >= A.begin[min(at + lane, A.n - 1)]));
  k = __builtin_amdgcn_readfirstlane(k);
  const MomentRecord& t = A.t[k];
  const uint32_t block = __builtin_amdgcn_readfirstlane((b - A.begin[k]) * kMomentGroup + (threadIdx.x >> 6));
  if (block >= t.blocks) return;
  const int64_t base = (int64_t)block * kMomBlock;
  const uint64_t row0 = t.magic ? __umul64hi((uint64_t)base, t.magic) : (uint64_t)base;
  const uint32_t len = t.row_len;
  const uint32_t e0 = (uint32_t)((uint64_t)base - row0 * len) + lane * 4;
  const uint64_t from = (uint64_t)t.src_at * kMomBlock;
  uint32_t wm = 0, wr = 0;
  int fm[4], fr[4];
  bool moved = false;
  int32_t row[4], s[4];
  uint32_t off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t e = e0 + j;
    // a lane is less than row_len + 256 from its block's first row
    const uint32_t q = len > 4096u ? (e >= len ? 1u : 0u) : t.magic ? __umulhi(e, (uint32_t)(t.magic >> 32) + 1u) : e;
    row[j] = (int32_t)(row0 + q);
    off[j] = e - q * len;
    s[j] = base + lane * 4 + j < t.count ? source<kMove>(A, row[j]) : -1;
    if (kMove) moved |= base + lane * 4 + j < t.count && s[j] != row[j];
  }
  if (kMove) {
    const bool any = __ballot(moved) != 0;
    if (lane == 0) A.changed[t.dst_at + block] = any;
    if (!any) return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t cm = 0, cr = 0, f = 0;
    if (s[j] >= 0) {
      const uint64_t at = from + (uint64_t)s[j] * len + off[j];
      cm = A.m8[at];
      cr = A.r8[at];
      f = *(const uint16_t*)(A.fields + 2 * (at >> 8));
    }
    wm |= cm << (8 * j);
    wr |= cr << (8 * j);
    fm[j] = (int)(f & 255u);
    fr[j] = (int)(f >> 8);
  }
  float m[4], r[4];
  decode_m4(wm, fm, m);
  decode_r4(wr, fr, r);
  const uint32_t none[4] = {0, 0, 0, 0};
  uint32_t cm, cr, f;
  encode_block<false>(m, r, none, cm, cr, f);
  const uint64_t to = (uint64_t)t.dst_at * kMomBlock + base + lane * 4;
  *reinterpret_cast<uint32_t*>(A.to_m8 + to) = cm;
  *reinterpret_cast<uint32_t*>(A.to_r8 + to) = cr;
  if (lane == 0) *(uint16_t*)(A.to_fields + 2 * ((uint64_t)t.dst_at + block)) = (uint16_t)f;
}

// The changed blocks from the copy into their places.
__global__ __launch_bounds__(256) void moment_back_kernel(int64_t blocks, const uint8_t* __restrict__ changed,
                                                          const uint8_t* __restrict__ from_m8,
                                                          const uint8_t* __restrict__ from_r8,
                                                          const uint8_t* __restrict__ from_fields,
                                                          uint8_t* __restrict__ m8, uint8_t* __restrict__ r8,
                                                          uint8_t* __restrict__ fields) {
  const int64_t block = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (block >= blocks || !changed[block]) return;
  const int64_t at = block * kMomBlock + lane * 4;
  *reinterpret_cast<uint32_t*>(m8 + at) = *reinterpret_cast<const uint32_t*>(from_m8 + at);
  *reinterpret_cast<uint32_t*>(r8 + at) = *reinterpret_cast<const uint32_t*>(from_r8 + at);
  if (lane == 0) *(uint16_t*)(fields + 2 * block) = *(const uint16_t*)(from_fields + 2 * block);
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

template <bool kMove>
int launch(hipStream_t stream, int num, const int64_t* row_lens, const int64_t* offsets, const int64_t* out_offsets,
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
    hipLaunchKernelGGL(moment_rows_kernel<kMove>, dim3((unsigned)groups), dim3(256), 0, stream, A);
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
  return launch<false>((hipStream_t)stream, num, row_lens, offsets, out_offsets, count, A);
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
  const int done = launch<true>((hipStream_t)stream, num, row_lens, offsets, offsets, rows, A);
  if (done != GS_OK) return done;
  // tensor by tensor: blocks between them belong to nobody
  for (int i = 0; i < num; ++i) {
    const int64_t first = offsets[i] / kMomBlock, here = (row_lens[i] * rows + kMomBlock - 1) / kMomBlock;
    if (here == 0) continue;
    const int64_t at = first * kMomBlock;
    hipLaunchKernelGGL(moment_back_kernel, dim3((unsigned)div_up(here, 4)), dim3(256), 0, (hipStream_t)stream, here,
                       A.changed + first, A.to_m8 + at, A.to_r8 + at, A.to_fields + 2 * first, mu8 + at, nu8 + at,
                       fields + 2 * first);
    GS_LAUNCH_CHECK("moment_back_kernel");
  }
  return GS_OK;
}
