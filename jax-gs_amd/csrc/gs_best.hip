// The k rows with the best scores, in index order, on gfx950.
//
// A score's key is a 32-bit number in the order of the scores: 0 for NaN (below everything), -0 as +0.
// The k-th largest key T is found digit by digit from the top (11, 11 and 10 bits; half types have 16
// bits, in the upper two digits): a histogram of the digit among the rows that agree with T so far, and the
// bin in which the k-th falls.  Rows with a key above T are taken, and of those with T the first.  Counts are
// integers, so the result does not depend on the order of the atomics.
//
// Few bytes move (3M half scores and their mask 9 MB, 1.3 us), so launches and their latency bound it, and for many rows
// the atomics in LDS.  Up to 16384 rows one workgroup does everything with its keys in registers (2000 rows 10 us, 16000 16).
// Beyond, a launch for each digit, one that counts what each workgroup takes and one that writes; the bin of a digit is
// found by every workgroup of the next launch for itself, which reads 16 KiB but saves a launch.  500k rows 23 us in float32
// and 20 in half types, 3M 37 and 32, 20M 113 and 95.
#include "gs_common.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kBestBlock = 512;
constexpr int kBestRun = 8;        // consecutive rows a thread
constexpr int kBestTile = kBestBlock * kBestRun;
constexpr int kOneBlock = 1024;    // of the workgroup that does everything
constexpr int kOneTile = kOneBlock * kBestRun;
constexpr int kBestGroups = 512;   // at most
constexpr int kBestOne = 2;        // tiles that one workgroup holds in registers
constexpr int kBins = 2048;
// Histograms in memory, by turns of the workgroups, whose atomics wait for each other (3M float32 36.5 us, one 40.8, four 37.2).
constexpr int kSplit = 2;
constexpr int kAlike = 3;          // in place of a type: no scores

struct Pick {
  uint32_t prefix;  // T's digits so far, in place
  uint32_t want;    // how many rows are still wanted among those that agree with them
};

struct BestControl {
  uint32_t hist[3][kSplit][kBins];
  uint32_t above[kBestGroups], equal[kBestGroups];  // rows above T and with T of each workgroup
  Pick picks[4];                                    // before digit d
};

struct BestArgs {
  const void* scores;
  const uint8_t* active;
  int64_t n;
  int64_t tiles;  // per workgroup
  BestControl* ctl;
  int32_t* out;
  uint32_t k;
};

__device__ inline uint32_t key_of(float x) {
  const uint32_t b = float_to_bits(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0;
  return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}

// The key in the 16 bits of a half type (of either: sign, exponent, mantissa).
template <int kType>
__device__ inline uint32_t half_key(uint32_t b) {
  constexpr uint32_t kInf = kType == GS_TYPE_BF16 ? 0x7f80u : 0x7c00u;
  if ((b & 0x7fffu) > kInf) return 0;
  if (b == 0x8000u) b = 0;
  return ((b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u) << 16;
}

template <int kType>
__device__ inline uint32_t key_at(const BestArgs& A, int64_t i) {
  if constexpr (kType == kAlike) return 1u;
  else if constexpr (kType == GS_TYPE_F32) return key_of(((const float*)A.scores)[i]);
  else return half_key<kType>(((const uint16_t*)A.scores)[i]);
}

// The keys of the rows from i on and which of them count (bit by bit).
template <int kType>
__device__ inline uint32_t keys_at(const BestArgs& A, int64_t i, uint32_t (&key)[kBestRun]) {
  typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));
  typedef uint8_t u8x8 __attribute__((ext_vector_type(8), aligned(1)));
  uint32_t on = 0;
  if (i + kBestRun <= A.n) {
    on = 255u;
    if (A.active) {
      const u8x8 a = *reinterpret_cast<const u8x8*>(A.active + i);
      on = 0;
#pragma unroll
      for (int j = 0; j < kBestRun; ++j) on |= (uint32_t)(a[j] != 0) << j;
    }
    if constexpr (kType == GS_TYPE_F32) {
      const f32x4 a = *reinterpret_cast<const f32x4*>((const float*)A.scores + i);
      const f32x4 b = *reinterpret_cast<const f32x4*>((const float*)A.scores + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        key[j] = key_of(a[j]);
        key[j + 4] = key_of(b[j]);
      }
    } else if constexpr (kType == kAlike) {
#pragma unroll
      for (int j = 0; j < kBestRun; ++j) key[j] = 1u;
    } else {
      const u16x8 a = *reinterpret_cast<const u16x8*>((const uint16_t*)A.scores + i);
#pragma unroll
      for (int j = 0; j < kBestRun; ++j) key[j] = half_key<kType>(a[j]);
    }
    return on;
  }
#pragma unroll
  for (int j = 0; j < kBestRun; ++j) {
    key[j] = 0;
    if (i + j < A.n && !(A.active && !A.active[i + j])) {
      key[j] = key_at<kType>(A, i + j);
      on |= 1u << j;
    }
  }
  return on;
}

// digit d of a key: 11, 11, 10 bits
__device__ inline int shift_of(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__device__ inline uint32_t bin_of(uint32_t key, int d) { return (key >> shift_of(d)) & (d == 2 ? 1023u : 2047u); }
// whether the digits above digit d agree
__device__ inline bool agrees(uint32_t key, uint32_t prefix, int d) {
  return d == 0 || (key ^ prefix) >> (d == 1 ? 21 : 10) == 0;
}

struct Sums {
  uint32_t w[kOneBlock / 64];
};

// Inclusive sum over the workgroup's threads of x, in thread order, and the sum of all.
template <int kBlock>
__device__ inline uint32_t block_scan(uint32_t x, Sums& s, uint32_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) s.w[wave] = x;
  __syncthreads();
  all = 0;
  uint32_t before = 0;
#pragma unroll
  for (int q = 0; q < kBlock / 64; ++q) {
    before += q < wave ? s.w[q] : 0;
    all += s.w[q];
  }
  return x + before;
}

// Digit d of T, from the histogram of the rows that agree so far: the bin in which the wanted row falls,
// counted from the largest.  Where there are fewer rows than wanted, all are: T is 0 then, and of
// the rows with key 0 all are among the first.
template <int kBlock, int kHists>
__device__ inline Pick pick(const uint32_t* h, Pick p, int d, Sums& s, Pick& shared) {
  constexpr int kEach = kBins / kBlock;  // bins a thread
  uint32_t x[kEach], own = 0, all;
  const int hi = kBins - 1 - kEach * (int)threadIdx.x;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    x[j] = h[hi - j];
#pragma unroll
    for (int q = 1; q < kHists; ++q) x[j] += h[q * kBins + hi - j];
    own += x[j];
  }
  uint32_t before = block_scan<kBlock>(own, s, all) - own;
  if (threadIdx.x == 0 && all < p.want) shared = Pick{0, p.want};
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (before < p.want && p.want <= before + x[j])
      shared = Pick{p.prefix | (uint32_t)(hi - j) << shift_of(d), p.want - before};
    before += x[j];
  }
  __syncthreads();
  return shared;
}

// Rows above and with T among a run's, `equal` in the upper half.
__device__ inline uint32_t count_run(const uint32_t (&key)[kBestRun], uint32_t on, uint32_t T) {
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < kBestRun; ++j)
    if (on >> j & 1u) c += key[j] > T ? 1u : key[j] == T ? 0x10000u : 0u;
  return c;
}

// The rows of a tile that are taken, which follow one another in the result: `a` rows above T and `e` with T come before
// the tile, `own` are this run's and `to` those of the tile before it.  By way of LDS, so that neighbours write
// side by side.
template <int kBlock>
__device__ inline void write_tile(const BestArgs& A, int64_t i, const uint32_t (&key)[kBestRun], uint32_t on, Pick p,
                                  uint32_t a, uint32_t e, uint32_t to, uint32_t all, int32_t* lds) {
  const uint32_t base = a + min(e, p.want), end = a + (all & 0xffffu) + min(e + (all >> 16), p.want);
  uint32_t ra = a + (to & 0xffffu), re = e + (to >> 16);
#pragma unroll
  for (int j = 0; j < kBestRun; ++j) {
    if (!(on >> j & 1u)) continue;
    const bool up = key[j] > p.prefix, eq = key[j] == p.prefix;
    if (up || (eq && re < p.want)) lds[ra + min(re, p.want) - base] = (int32_t)(i + j);
    ra += up;
    re += eq;
  }
  __syncthreads();
  for (uint32_t at = base + threadIdx.x; at < min(end, A.k); at += kBlock) A.out[at] = lds[at - base];
}

template <int kType>
__global__ __launch_bounds__(kOneBlock) void best_one_kernel(BestArgs A) {
  __shared__ uint32_t h[kBins];
  __shared__ int32_t lds[kOneTile];
  __shared__ Sums s;
  __shared__ Pick shared;
  constexpr int kDigits = kType == kAlike ? 0 : kType == GS_TYPE_F32 ? 3 : 2;
  uint32_t key[kBestOne][kBestRun], on[kBestOne];
#pragma unroll
  for (int v = 0; v < kBestOne; ++v) on[v] = keys_at<kType>(A, v * kOneTile + threadIdx.x * kBestRun, key[v]);
  Pick p{0, A.k};
#pragma unroll
  for (int d = 0; d < kDigits; ++d) {
#pragma unroll
    for (int j = 0; j < kBins / kOneBlock; ++j) h[threadIdx.x + j * kOneBlock] = 0;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kBestOne; ++v)
#pragma unroll
      for (int j = 0; j < kBestRun; ++j)
        if ((on[v] >> j & 1u) && agrees(key[v][j], p.prefix, d)) atomicAdd(&h[bin_of(key[v][j], d)], 1u);
    __syncthreads();
    p = pick<kOneBlock, 1>(h, p, d, s, shared);
  }
  uint32_t a = 0, e = 0;
#pragma unroll
  for (int v = 0; v < kBestOne; ++v) {
    uint32_t all;
    const uint32_t own = count_run(key[v], on[v], p.prefix), to = block_scan<kOneBlock>(own, s, all) - own;
    write_tile<kOneBlock>(A, v * kOneTile + threadIdx.x * kBestRun, key[v], on[v], p, a, e, to, all, lds);
    a += all & 0xffffu;
    e += all >> 16;
  }
  for (uint32_t at = a + min(e, p.want) + threadIdx.x; at < A.k; at += kOneBlock) A.out[at] = -1;
}

__global__ __launch_bounds__(kBestBlock) void best_clear_kernel(BestControl* ctl) {
  for (int i = threadIdx.x; i < 3 * kSplit * kBins; i += kBestBlock) (&ctl->hist[0][0][0])[i] = 0;
}

// T's digits before digit d: those before d - 1 are there from the launch before, the last is found by every workgroup.
__device__ inline Pick picks(const BestArgs& A, int d, Sums& s, Pick& shared) {
  if (d == 0) return Pick{0, A.k};
  const Pick p = pick<kBestBlock, kSplit>(A.ctl->hist[d - 1][0], d == 1 ? Pick{0, A.k} : A.ctl->picks[d - 1], d - 1, s, shared);
  if (blockIdx.x == 0 && threadIdx.x == 0) A.ctl->picks[d] = p;
  return p;
}

// Four histograms in LDS, one word beside another: lanes with one bin (scores that are zero, or all alike) then wait for
// a quarter of the others (20M equal scores 266 -> 115 us, eight 98; 3M different ones are as fast with one).
constexpr int kCopies = 4;
template <int kType>
__global__ __launch_bounds__(kBestBlock) void best_hist_kernel(BestArgs A, int d) {
  __shared__ uint32_t h[kBins * kCopies];
  __shared__ Sums s;
  __shared__ Pick shared;
  // the first keys come while the last digit is found
  int64_t i = blockIdx.x * A.tiles * kBestTile + threadIdx.x * kBestRun;
  uint32_t key[kBestRun], on = keys_at<kType>(A, i, key);
#pragma unroll
  for (int j = 0; j < kBins / kBestBlock * kCopies; ++j) h[threadIdx.x + j * kBestBlock] = 0;
  const Pick p = picks(A, d, s, shared);
  __syncthreads();
  for (int64_t v = 0;;) {
#pragma unroll
    for (int j = 0; j < kBestRun; ++j) {
      if (!((on >> j & 1u) && agrees(key[j], p.prefix, d))) continue;
      atomicAdd(&h[bin_of(key[j], d) * kCopies + threadIdx.x % kCopies], 1u);
    }
    if (++v == A.tiles) break;
    i += kBestTile;
    on = keys_at<kType>(A, i, key);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kBins / kBestBlock; ++j) {
    const uint32_t bin = threadIdx.x + j * kBestBlock;
    uint32_t c = 0;
#pragma unroll
    for (int q = 0; q < kCopies; ++q) c += h[bin * kCopies + q];
    if (c) atomicAdd(&A.ctl->hist[d][blockIdx.x % kSplit][bin], c);
  }
}

template <int kType>
__global__ __launch_bounds__(kBestBlock) void best_count_kernel(BestArgs A) {
  __shared__ Sums s;
  __shared__ Pick shared;
  constexpr int kDigits = kType == kAlike ? 0 : kType == GS_TYPE_F32 ? 3 : 2;
  int64_t i = blockIdx.x * A.tiles * kBestTile + threadIdx.x * kBestRun;
  uint32_t key[kBestRun], on = keys_at<kType>(A, i, key);
  const Pick p = picks(A, kDigits, s, shared);
  uint32_t above = 0, equal = 0;
  for (int64_t v = 0;;) {
    const uint32_t c = count_run(key, on, p.prefix);
    above += c & 0xffffu;
    equal += c >> 16;
    if (++v == A.tiles) break;
    i += kBestTile;
    on = keys_at<kType>(A, i, key);
  }
  uint32_t a, e;
  block_scan<kBestBlock>(above, s, a);
  block_scan<kBestBlock>(equal, s, e);
  if (threadIdx.x == 0) {
    A.ctl->above[blockIdx.x] = a;
    A.ctl->equal[blockIdx.x] = e;
  }
}

template <int kType>
__global__ __launch_bounds__(kBestBlock) void best_write_kernel(BestArgs A) {
  __shared__ int32_t lds[kBestTile];
  __shared__ Sums s;
  constexpr int kDigits = kType == kAlike ? 0 : kType == GS_TYPE_F32 ? 3 : 2;
  int64_t i = blockIdx.x * A.tiles * kBestTile + threadIdx.x * kBestRun;
  uint32_t key[kBestRun], on = keys_at<kType>(A, i, key);
  const Pick p = kDigits ? A.ctl->picks[kDigits] : Pick{0, A.k};
  // what the workgroups have, and those before this one
  const uint32_t b = blockIdx.x, groups = gridDim.x;
  uint32_t a = 0, e = 0, all_a = 0, all_e = 0;
#pragma unroll
  for (int j = 0; j < kBestGroups / kBestBlock; ++j) {
    const uint32_t g = threadIdx.x + j * kBestBlock;
    const uint32_t xa = g < groups ? A.ctl->above[g] : 0, xe = g < groups ? A.ctl->equal[g] : 0;
    all_a += xa;
    all_e += xe;
    a += g < b ? xa : 0;
    e += g < b ? xe : 0;
  }
  block_scan<kBestBlock>(a, s, a);
  block_scan<kBestBlock>(e, s, e);
  block_scan<kBestBlock>(all_a, s, all_a);
  block_scan<kBestBlock>(all_e, s, all_e);
  for (int64_t v = 0;;) {
    uint32_t all;
    const uint32_t own = count_run(key, on, p.prefix), to = block_scan<kBestBlock>(own, s, all) - own;
    write_tile<kBestBlock>(A, i, key, on, p, a, e, to, all, lds);
    a += all & 0xffffu;
    e += all >> 16;
    if (++v == A.tiles) break;
    i += kBestTile;
    on = keys_at<kType>(A, i, key);
  }
  // nothing behind the last
  const int64_t total = (int64_t)all_a + min(all_e, p.want);
  for (int64_t at = total + (int64_t)b * kBestBlock + threadIdx.x; at < A.k; at += (int64_t)groups * kBestBlock) A.out[at] = -1;
}

template <int kType>
int best_rows(hipStream_t s, BestArgs& A) {
  // (what it writes behind the last row takes one workgroup long, where that is much more)
  if (A.n <= kBestOne * kOneTile && A.k <= 16 * kBestOne * kOneTile) {
    hipLaunchKernelGGL(best_one_kernel<kType>, dim3(1), dim3(kOneBlock), 0, s, A);
    GS_LAUNCH_CHECK("best_one_kernel");
    return GS_OK;
  }
  const int64_t tiles = (A.n + kBestTile - 1) / kBestTile;
  A.tiles = std::max<int64_t>((tiles + kBestGroups - 1) / kBestGroups, 1);
  const int64_t groups = (tiles + A.tiles - 1) / A.tiles;
  const dim3 grid((unsigned)std::max(groups, std::min<int64_t>(A.k >> 16, kBestGroups)));
  constexpr int kDigits = kType == kAlike ? 0 : kType == GS_TYPE_F32 ? 3 : 2;
  if (kDigits) {
    hipLaunchKernelGGL(best_clear_kernel, dim3(1), dim3(kBestBlock), 0, s, A.ctl);
    GS_LAUNCH_CHECK("best_clear_kernel");
  }
  for (int d = 0; d < kDigits; ++d) {
    hipLaunchKernelGGL(best_hist_kernel<kType>, grid, dim3(kBestBlock), 0, s, A, d);
    GS_LAUNCH_CHECK("best_hist_kernel");
  }
  hipLaunchKernelGGL(best_count_kernel<kType>, grid, dim3(kBestBlock), 0, s, A);
  GS_LAUNCH_CHECK("best_count_kernel");
  hipLaunchKernelGGL(best_write_kernel<kType>, grid, dim3(kBestBlock), 0, s, A);
  GS_LAUNCH_CHECK("best_write_kernel");
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_best_rows_workspace_size(int64_t rows) { return rows >= 0 ? sizeof(BestControl) : 0; }

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
  A.ctl = (BestControl*)workspace;
  A.out = out;
  A.k = (uint32_t)k;
  hipStream_t s = (hipStream_t)stream;
  if (!scores) return best_rows<kAlike>(s, A);
  if (type == GS_TYPE_F32) return best_rows<GS_TYPE_F32>(s, A);
  if (type == GS_TYPE_BF16) return best_rows<GS_TYPE_BF16>(s, A);
  return best_rows<GS_TYPE_F16>(s, A);
}
