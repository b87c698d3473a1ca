// The k rows with the best scores, in index order, on gfx950.
//
// A score's key is a 32-bit number in the order of the scores: 0 for NaN (below everything), -0 as +0.
// The k-th largest key T is found digit by digit from the top (11, 11 and 10 bits; half types have 16
// bits, in the upper digits): a histogram of the digit among the rows that agree with T so far, and the
// bin in which the k-th falls.  Rows with a key above T are taken, and of those with T the first.  Counts are integers, so
// the result does not depend on the order of the atomics.
#include "gs_common.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kBestBlock = 1024;
constexpr int kBestGroups = 512;   // at most, for the passes over the scores
constexpr int kBins = 2048;

struct BestControl {
  uint32_t hist[3][kBins];
  uint32_t prefix[4];   // T's digits before digit d, in place
  uint32_t want[4];     // how many rows are still wanted among those that agree
};

struct BestArgs {
  const void* scores;      // NULL: all alike
  const uint8_t* active;
  int64_t n;
  int64_t chunk;           // rows per workgroup, a multiple of kBestBlock
  int type;
  int digits;
  BestControl* ctl;
  uint32_t* above;         // per workgroup: rows above T, rows with T (then: those before)
  uint32_t* equal;
  int32_t* out;
  uint32_t k;
};

__device__ inline uint32_t key_of(float x) {
  const uint32_t b = float_to_bits(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0;
  return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}

__device__ inline uint32_t key_at(const BestArgs& A, int64_t i) {
  if (!A.scores) return 1u;
  if (A.type == GS_TYPE_F32) return key_of(((const float*)A.scores)[i]);
  const uint32_t b = ((const uint16_t*)A.scores)[i];
  if (A.type == GS_TYPE_BF16) return key_of(bits_to_float(b << 16)) & 0xffff0000u;
  // float16: its 16 bits in their own order, in the upper half
  const uint32_t c = b == 0x8000u ? 0u : b;
  if ((c & 0x7fffu) > 0x7c00u) return 0;
  return ((c & 0x8000u) ? ~c & 0xffffu : c | 0x8000u) << 16;
}

// digit d of a key: 11, 11, 10 bits
__device__ inline int shift_of(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }

__global__ __launch_bounds__(kBestBlock) void best_clear_kernel(BestControl* ctl, uint32_t k) {
  for (int i = threadIdx.x; i < 3 * kBins; i += kBestBlock) (&ctl->hist[0][0])[i] = 0;
  if (threadIdx.x == 0) {
    ctl->prefix[0] = 0;
    ctl->want[0] = k;
  }
}

__global__ __launch_bounds__(kBestBlock) void best_hist_kernel(BestArgs A, int d) {
  __shared__ uint32_t h[kBins];
  for (int i = threadIdx.x; i < kBins; i += kBestBlock) h[i] = 0;
  __syncthreads();
  const uint32_t prefix = A.ctl->prefix[d];
  const int sh = shift_of(d), above = sh + (d == 2 ? 10 : 11);
  const int64_t begin = blockIdx.x * A.chunk, end = min(begin + A.chunk, A.n);
  for (int64_t i = begin + threadIdx.x; i < end; i += kBestBlock) {
    if (A.active && !A.active[i]) continue;
    const uint32_t key = key_at(A, i);
    if (d > 0 && (key >> above) != (prefix >> above)) continue;
    atomicAdd(&h[(key >> sh) & (d == 2 ? 1023u : 2047u)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kBestBlock)
    if (h[i]) atomicAdd(&A.ctl->hist[d][i], h[i]);
}

// Inclusive sum over the workgroup's threads of x, in thread order.
__device__ inline uint32_t block_scan(uint32_t x, uint32_t* w) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) w[wave] = x;
  __syncthreads();
  for (int q = 0; q < wave; ++q) x += w[q];
  return x;
}

// The bin of digit d in which the wanted row falls, counted from the largest.
__global__ __launch_bounds__(kBestBlock) void best_pick_kernel(BestArgs A, int d) {
  __shared__ uint32_t w[kBestBlock / 64];
  const uint32_t want = A.ctl->want[d];
  const uint32_t* h = A.ctl->hist[d];
  const int hi = kBins - 1 - 2 * (int)threadIdx.x;
  const uint32_t a = h[hi], b = h[hi - 1];
  const uint32_t all = block_scan(a + b, w), before = all - a - b;
  const int sh = shift_of(d);
  if (before < want && want <= all) {
    const bool second = before + a < want;
    A.ctl->prefix[d + 1] = A.ctl->prefix[d] | ((uint32_t)(second ? hi - 1 : hi) << sh);
    A.ctl->want[d + 1] = want - before - (second ? a : 0);
  }
  // fewer rows than wanted: everything is above T = 0 or, with key 0, among the first
  if (threadIdx.x == kBestBlock - 1 && all < want) {
    A.ctl->prefix[d + 1] = 0;
    A.ctl->want[d + 1] = want;
  }
}

__global__ __launch_bounds__(kBestBlock) void best_count_kernel(BestArgs A) {
  __shared__ uint32_t w[kBestBlock / 64];
  const uint32_t T = A.ctl->prefix[A.digits];
  const int64_t begin = blockIdx.x * A.chunk, end = min(begin + A.chunk, A.n);
  uint32_t above = 0, equal = 0;
  for (int64_t i = begin + threadIdx.x; i < end; i += kBestBlock) {
    if (A.active && !A.active[i]) continue;
    const uint32_t key = key_at(A, i);
    above += key > T;
    equal += key == T;
  }
  const uint32_t a = block_scan(above, w), e = block_scan(equal, w);
  if (threadIdx.x == kBestBlock - 1) {
    A.above[blockIdx.x] = a;
    A.equal[blockIdx.x] = e;
  }
}

__global__ __launch_bounds__(kBestBlock) void best_write_kernel(BestArgs A) {
  __shared__ uint32_t w[kBestBlock / 64];
  __shared__ uint32_t sum[2];
  const uint32_t T = A.ctl->prefix[A.digits], want = A.ctl->want[A.digits];
  const int b = blockIdx.x, groups = gridDim.x;
  // what the workgroups before this one have
  uint32_t a = 0, e = 0, all_a = 0, all_e = 0;
  if ((int)threadIdx.x < groups) {
    all_a = A.above[threadIdx.x];
    all_e = A.equal[threadIdx.x];
    a = (int)threadIdx.x < b ? all_a : 0;
    e = (int)threadIdx.x < b ? all_e : 0;
  }
  a = block_scan(a, w);
  e = block_scan(e, w);
  if (threadIdx.x == kBestBlock - 1) {
    sum[0] = a;
    sum[1] = e;
  }
  all_a = block_scan(all_a, w);
  all_e = block_scan(all_e, w);
  __shared__ uint32_t total;
  if (threadIdx.x == kBestBlock - 1) total = all_a + min(all_e, want);
  __syncthreads();
  uint32_t base_a = sum[0], base_e = sum[1];
  const int64_t begin = b * A.chunk, end = min(begin + A.chunk, A.n);
  for (int64_t at = begin; at < end; at += kBestBlock) {
    const int64_t i = at + threadIdx.x;
    uint32_t up = 0, eq = 0;
    if (i < end && !(A.active && !A.active[i])) {
      const uint32_t key = key_at(A, i);
      up = key > T;
      eq = key == T;
    }
    const uint32_t both = block_scan(up | (eq << 16), w);  // at most 1024 of each
    const uint32_t ia = base_a + (both & 0xffffu), ie = base_e + (both >> 16);
    // rows above T before this one, and those of T that are taken
    if (up || (eq && ie <= want)) {
      const uint32_t p = (ia - up) + min(ie - eq, want);
      if (p < A.k) A.out[p] = (int32_t)i;
    }
    __shared__ uint32_t last;
    if (threadIdx.x == kBestBlock - 1) last = both;
    __syncthreads();
    base_a += last & 0xffffu;
    base_e += last >> 16;
  }
  // nothing behind the last
  for (int64_t p = total + (int64_t)b * kBestBlock + threadIdx.x; p < A.k; p += (int64_t)groups * kBestBlock) A.out[p] = -1;
}

int64_t best_chunk(int64_t n) {
  const int64_t steps = (n + kBestBlock - 1) / kBestBlock;
  return (steps + kBestGroups - 1) / kBestGroups * kBestBlock;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_best_rows_workspace_size(int64_t rows) {
  return rows >= 0 ? sizeof(BestControl) + 2 * kBestGroups * sizeof(uint32_t) : 0;
}

extern "C" int gs_best_rows(void* stream, int64_t rows, const void* scores, int type, const uint8_t* active, int64_t k,
                            void* workspace, size_t workspace_bytes, int32_t* out) {
  GS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31), "gs_best_rows: %lld rows", (long long)rows);
  GS_REQUIRE(k >= 0 && k < ((int64_t)1 << 31), "gs_best_rows: the best %lld", (long long)k);
  GS_REQUIRE(!scores || (type >= GS_TYPE_F32 && type <= GS_TYPE_F16), "gs_best_rows: type %d", type);
  GS_REQUIRE((reinterpret_cast<uintptr_t>(scores) & (type == GS_TYPE_F32 ? 3 : 1)) == 0,
             "gs_best_rows: the scores are not aligned to their type");
  if (k == 0) return GS_OK;
  GS_REQUIRE(out && workspace, "gs_best_rows: NULL argument");
  const size_t need = gs_best_rows_workspace_size(rows);
  GS_REQUIRE(workspace_bytes >= need, "gs_best_rows: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  GS_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 3) == 0, "gs_best_rows: the workspace must be 4-byte aligned");
  BestArgs A{};
  A.scores = scores;
  A.active = active;
  A.n = rows;
  A.chunk = std::max<int64_t>(best_chunk(rows), kBestBlock);
  A.type = type;
  A.digits = !scores ? 0 : type == GS_TYPE_F32 ? 3 : 2;
  A.ctl = (BestControl*)workspace;
  A.above = (uint32_t*)(A.ctl + 1);
  A.equal = A.above + kBestGroups;
  A.out = out;
  A.k = (uint32_t)k;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)std::max<int64_t>(1, (rows + A.chunk - 1) / A.chunk));
  hipLaunchKernelGGL(best_clear_kernel, dim3(1), dim3(kBestBlock), 0, s, A.ctl, A.k);
  GS_LAUNCH_CHECK("best_clear_kernel");
  for (int d = 0; d < A.digits; ++d) {
    hipLaunchKernelGGL(best_hist_kernel, grid, dim3(kBestBlock), 0, s, A, d);
    GS_LAUNCH_CHECK("best_hist_kernel");
    hipLaunchKernelGGL(best_pick_kernel, dim3(1), dim3(kBestBlock), 0, s, A, d);
    GS_LAUNCH_CHECK("best_pick_kernel");
  }
  hipLaunchKernelGGL(best_count_kernel, grid, dim3(kBestBlock), 0, s, A);
  GS_LAUNCH_CHECK("best_count_kernel");
  hipLaunchKernelGGL(best_write_kernel, grid, dim3(kBestBlock), 0, s, A);
  GS_LAUNCH_CHECK("best_write_kernel");
  return GS_OK;
}
