// Norms of many gradients at once, and the factor that clips them, on gfx950.
//
//   n_k = |s| sqrt(sum_i g_ki^2),   n = sqrt(sum_k n_k^2),
//   scale = s min(1, c / (n + 1e-6))   (s without c; NaN unless the float64 n is finite, that is
//                                       unless s and every gradient are),
// s a device scalar (a loss scale's inverse) or 1.  Rows whose mask is 0 are left out, whatever
// they hold.  Squares and sums are float64: no square of a float32 overflows or vanishes there,
// and the order of the sums, which is fixed, does not show in the float32 results.
//
// Every workgroup sums one run of consecutive elements of one tensor into one partial sum (runs are
// the multiple of 8192 elements with which at most 2048 whole ones cover all tensors: for large lists
// 1025 to 2048 of them); a second launch of one
// workgroup adds the partial sums of each tensor and the tensors' sums.  Reading bounds the first:
// 59M float32 44 us (5.3 TB/s), 148 bfloat16 tensors of 22M elements 13 us, 124M float32 under a
// mask 110 us (150 us behind a step, whose dirty lines are written back meanwhile); the second
// takes 3 to 5 us, a chain of two reads and two reductions.
#include "gs_rows.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kNormTensors = 152;  // per launch: the argument block stays below 4 KiB
constexpr int kNormRuns = 2048;    // 8 workgroups of 4 waves on each of 256 CUs

struct NormArgs {
  const void* grad[kNormTensors];
  int64_t count[kNormTensors];
  uint32_t begin[kNormTensors];  // first workgroup of each tensor
  int32_t row_len[kNormTensors];
  uint8_t type[kNormTensors];
  const uint8_t* active;
  double* partial;  // of this launch's first workgroup
  int32_t* first;   // this launch's tensors: their first partial sums
  int32_t first_partial;
  int32_t n;
  uint32_t groups;
  int64_t run;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

struct NormLayout {
  int64_t run, partials;
  size_t sums, first, total;
};

NormLayout norm_layout(int num, const int64_t* counts) {
  NormLayout L;
  int64_t total = 0;
  for (int i = 0; i < num; ++i) total += counts[i];
  L.run = std::max<int64_t>(8192, ((total + kNormRuns - 1) / kNormRuns + 8191) / 8192 * 8192);
  L.partials = 0;
  for (int i = 0; i < num; ++i) L.partials += (counts[i] + L.run - 1) / L.run;
  L.sums = (size_t)L.partials * sizeof(double);
  L.first = L.sums + (size_t)num * sizeof(double);
  L.total = L.first + ((size_t)num + 2) * sizeof(int32_t);
  return L;
}

// Deals the tensors out to launches, in order.
struct NormList {
  int num;
  const void* const* grads;
  const int* types;
  const int64_t* counts;
  const int64_t* row_lens;
  const uint8_t* active;
  int64_t run;
  int tensor = 0;
  int64_t done = 0;  // workgroups of the launches before

  NormList(int num_, const void* const* grads_, const int* types_, const int64_t* counts_, const int64_t* row_lens_,
           const uint8_t* active_, const NormLayout& L)
      : num(num_), grads(grads_), types(types_), counts(counts_), row_lens(row_lens_), active(active_), run(L.run) {}

  bool next(NormArgs& A) {
    if (tensor >= num) return false;
    int k = 0;
    int64_t groups = 0;
    for (; tensor < num && k < kNormTensors; ++tensor) {
      A.grad[k] = grads[tensor];
      A.count[k] = counts[tensor];
      A.row_len[k] = active && counts[tensor] ? (int32_t)row_lens[tensor] : 1;
      A.type[k] = (uint8_t)types[tensor];
      A.begin[k++] = (uint32_t)groups;
      groups += (counts[tensor] + run - 1) / run;
    }
    A.active = active;
    A.run = run;
    A.n = k;
    A.groups = (uint32_t)groups;
    A.first_partial = (int32_t)done;
    done += groups;
    return true;
  }
};

__device__ inline double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

template <class G>
__device__ inline double run_sum(const G* __restrict__ g, const uint8_t* __restrict__ active, int32_t row_len,
                                 int64_t begin, int64_t end) {
  constexpr int kVec = 16 / sizeof(G);  // 16 bytes a lane
  constexpr int kStep = 256 * kVec;
  constexpr int kAhead = 4;  // vectors in flight
  typedef G vec __attribute__((ext_vector_type(kVec), aligned(sizeof(G))));
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  const uint32_t l = threadIdx.x * kVec;
  // the reciprocal of the row length: a division, but one per workgroup
  const uint64_t magic = active && row_len > 1 ? ~(uint64_t)0 / (uint32_t)row_len + 1 : 0;
  int64_t base = begin;
  uint32_t on[kAhead];
  if (active && base + kAhead * kStep <= end)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) on[u] = rows_on<kVec>(active, magic, row_len, base + u * kStep, l, kVec);
  for (; base + kAhead * kStep <= end; base += kAhead * kStep) {
    vec v[kAhead];
    if (active == nullptr) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) v[u] = *reinterpret_cast<const vec*>(g + base + u * kStep + l);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const double x = (double)(float)v[u][j];
          acc[u] = fma(x, x, acc[u]);
        }
    } else {
      // masked rows are not read; the next masks come while these elements do
      uint32_t now[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        now[u] = on[u];
        v[u] = (vec)(G)0.0f;
        if (now[u]) v[u] = *reinterpret_cast<const vec*>(g + base + u * kStep + l);
      }
      if (base + 2 * kAhead * kStep <= end)
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          on[u] = rows_on<kVec>(active, magic, row_len, base + (kAhead + u) * kStep, l, kVec);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const double x = now[u] >> j & 1u ? (double)(float)v[u][j] : 0.0;
          acc[u] = fma(x, x, acc[u]);
        }
    }
  }
  for (; base < end; base += kStep) {
    const int64_t left = end - base - l;
    const int n = left >= kVec ? kVec : left > 0 ? (int)left : 0;
    const uint32_t some = active ? rows_on<kVec>(active, magic, row_len, base, l, n) : (1u << n) - 1u;
    if (some == 0) continue;
    vec v = (vec)(G)0.0f;
    if (n == kVec) {
      v = *reinterpret_cast<const vec*>(g + base + l);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (j < n) v[j] = g[base + l + j];
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const double x = some >> j & 1u ? (double)(float)v[j] : 0.0;
      acc[j & 3] = fma(x, x, acc[j & 3]);
    }
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

__global__ __launch_bounds__(256) void grad_norms_kernel(NormArgs A) {
  const uint32_t b = blockIdx.x;
  const int lane = threadIdx.x & 63;
  if (b == 0)
    for (int k = threadIdx.x; k < A.n; k += 256) A.first[k] = A.first_partial + (int32_t)A.begin[k];
  if (b >= A.groups) return;  // every tensor is empty
  int k = -1;  // the last tensor that begins at or before this workgroup
  for (int at = 0; at < A.n; at += 64) k += __popcll(__ballot(at + lane < A.n && b >= A.begin[min(at + lane, A.n - 1)]));
  k = __builtin_amdgcn_readfirstlane(k);
  const int64_t begin = (int64_t)(b - A.begin[k]) * A.run, count = A.count[k];
  const int64_t end = begin + A.run < count ? begin + A.run : count;
  const int type = A.type[k], row_len = A.row_len[k];
  const void* g = A.grad[k];
  double x;
  if (type == GS_TYPE_F32) x = run_sum((const float*)g, A.active, row_len, begin, end);
  else if (type == GS_TYPE_BF16) x = run_sum((const __bf16*)g, A.active, row_len, begin, end);
  else x = run_sum((const _Float16*)g, A.active, row_len, begin, end);
  x = wave_sum(x);
  __shared__ double w[4];
  if (lane == 0) w[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x == 0) A.partial[b] = (w[0] + w[1]) + (w[2] + w[3]);
}

// One workgroup: 2^group_log2 threads sum a tensor's partial sums, the first wave the tensors'.
__global__ __launch_bounds__(1024) void grad_norms_total_kernel(int num, int partials, int group_log2,
                                                                const double* __restrict__ partial,
                                                                const int32_t* __restrict__ first, double* sums,
                                                                const float* __restrict__ grad_scale, double max_norm,
                                                                float* __restrict__ norms, float* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = 1 << group_log2, within = threadIdx.x & (group - 1);
  const double s = grad_scale ? fabs((double)*grad_scale) : 1.0;
  __shared__ double w[16];
  for (int k0 = 0; k0 < num; k0 += 1024 >> group_log2) {
    const int k = k0 + (threadIdx.x >> group_log2);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    if (k < num) {
      const int e = k + 1 < num ? first[k + 1] : partials;
      for (int i = first[k] + within; i < e; i += 8 * group) {
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = partial[min(i + u * group, e - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u) acc[u & 3] += i + u * group < e ? v[u] : 0.0;
      }
    }
    double x = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    for (int o = min(group, 64) >> 1; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if (group > 64) {
      if (lane == 0) w[wave] = x;
      __syncthreads();
      x = 0.0;
      for (int q = 0; q < group >> 6; ++q) x += w[(wave & ~((group >> 6) - 1)) + q];
      __syncthreads();
    }
    if (within == 0 && k < num) {
      sums[k] = x;
      if (norms) norms[k] = (float)(sqrt(x) * s);
    }
  }
  __syncthreads();
  if (wave != 0) return;
  double x = 0.0;
  for (int k = lane; k < num; k += 64) x += sums[k];
  x = wave_sum(x);
  if (lane == 0) {
    const double n = sqrt(x) * s;
    double f = grad_scale ? (double)*grad_scale : 1.0;
    if (max_norm > 0.0) f *= fmin(1.0, max_norm / (n + 1e-6));
    out[0] = (float)n;
    out[1] = n < __builtin_huge_val() ? (float)f : bits_to_float(0x7fc00000u);
  }
}

// Gradients times the factor, in place: the norms' runs, 16 bytes a lane, each product rounded once.
// Masked rows keep what they hold.  Past the caches from kStreamBytes on: 472 MB with their norms 294 us
// and 234 past them, 236 MB 121 and 115 (under a mask 102 and 106: there not), 118 MB 58 either way, 88 MB 48 and 51.
constexpr int64_t kStreamBytes = (int64_t)160 << 20;

template <bool kStream, class G>
__device__ inline void run_scale(G* __restrict__ g, const uint8_t* __restrict__ active, int32_t row_len, int64_t begin,
                                 int64_t end, float f) {
  constexpr int kVec = 16 / sizeof(G);
  constexpr int kStep = 256 * kVec;
  constexpr int kAhead = 4;
  constexpr uint32_t kAll = (1u << kVec) - 1u;
  typedef G vec __attribute__((ext_vector_type(kVec), aligned(sizeof(G))));
  const uint32_t l = threadIdx.x * kVec;
  const uint64_t magic = active && row_len > 1 ? ~(uint64_t)0 / (uint32_t)row_len + 1 : 0;
  int64_t base = begin;
  for (; base + kAhead * kStep <= end; base += kAhead * kStep) {
    vec v[kAhead];
    uint32_t on[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      on[u] = active ? rows_on<kVec>(active, magic, row_len, base + u * kStep, l, kVec) : kAll;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (on[u]) {
        const vec* from = reinterpret_cast<const vec*>(g + base + u * kStep + l);
        v[u] = kStream ? __builtin_nontemporal_load(from) : *from;
      }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (!on[u]) continue;
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (on[u] >> j & 1u) v[u][j] = (G)((float)v[u][j] * f);
      vec* to = reinterpret_cast<vec*>(g + base + u * kStep + l);
      if (kStream) __builtin_nontemporal_store(v[u], to);
      else *to = v[u];
    }
  }
  for (; base < end; base += kStep) {
    const int64_t left = end - base - l;
    const int n = left >= kVec ? kVec : left > 0 ? (int)left : 0;
    const uint32_t some = active ? rows_on<kVec>(active, magic, row_len, base, l, n) : (1u << n) - 1u;
    if (some == 0) continue;
    G* p = g + base + l;
    if (n == kVec) {
      vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (some >> j & 1u) v[j] = (G)((float)v[j] * f);
      *reinterpret_cast<vec*>(p) = v;
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (some >> j & 1u) p[j] = (G)((float)p[j] * f);
    }
  }
}

struct ScaleArgs {
  NormArgs a;              // its partial and first are not used
  const double* partial;   // of all launches; NULL: the factor is there already
  int32_t partials;
  int32_t writes;          // this launch's first workgroup writes the results
  double max_norm;
  const float* grad_scale;
  float* norms;            // of this launch's first tensor, or NULL
  float* out;
};
static_assert(sizeof(ScaleArgs) <= 4096, "kernel arguments");

// The sum of n partial sums, in a fixed order, in every thread.
__device__ inline double sum_of(const double* __restrict__ partial, int n, double (&w)[4]) {
  double acc[2] = {0.0, 0.0};
  for (int i = threadIdx.x; i < n; i += 2 * 256 * 4) {
    double v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = partial[min(i + u * 256, n - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[u & 1] += i + u * 256 < n ? v[u] : 0.0;
  }
  const double x = wave_sum(acc[0] + acc[1]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = x;
  __syncthreads();
  return (w[0] + w[1]) + (w[2] + w[3]);
}

// Every workgroup adds all partial sums for itself, up to 2 * kNormRuns of them (32 KiB out of L2), which takes less than a
// launch that does it once for all: one tensor of 16M elements (2048 sums) 17.6 us, 19.8 with the launch; beside it 1000
// tensors of 1000 elements 75 and 81, 3000 of them (4024 sums) 203 and 205.  Beyond, the launch is faster: 6000 such
// tensors alone 394 and 379.
template <bool kStream>
__global__ __launch_bounds__(256) void grad_scale_kernel(ScaleArgs S) {
  const NormArgs& A = S.a;
  const uint32_t b = blockIdx.x;
  const int lane = threadIdx.x & 63;
  __shared__ double w[4];
  float f;
  if (S.partial) {
    const double s = S.grad_scale ? (double)*S.grad_scale : 1.0;
    const double n = sqrt(sum_of(S.partial, S.partials, w)) * fabs(s);
    f = (float)(s * fmin(1.0, S.max_norm / (n + 1e-6)));
    if (!(n < __builtin_huge_val())) f = bits_to_float(0x7fc00000u);
    if (b == 0 && S.writes && threadIdx.x == 0) {
      S.out[0] = (float)n;
      S.out[1] = f;
    }
    if (b == 0 && S.norms)
      for (int k = threadIdx.x; k < A.n; k += 256)
        if (A.count[k] == 0) S.norms[k] = (float)fabs(0.0 * s);
  } else {
    f = S.out[1];
  }
  if (b >= A.groups) return;
  int k = -1;
  for (int at = 0; at < A.n; at += 64) k += __popcll(__ballot(at + lane < A.n && b >= A.begin[min(at + lane, A.n - 1)]));
  k = __builtin_amdgcn_readfirstlane(k);
  const int64_t begin = (int64_t)(b - A.begin[k]) * A.run, count = A.count[k];
  const int64_t end = begin + A.run < count ? begin + A.run : count;
  if (S.partial && S.norms && begin == 0) {  // a tensor's first workgroup: its own norm
    const double x = sum_of(S.partial + A.first_partial + b, (int)((count + A.run - 1) / A.run), w);
    if (threadIdx.x == 0) S.norms[k] = (float)(sqrt(x) * (S.grad_scale ? fabs((double)*S.grad_scale) : 1.0));
  }
  if (f == 1.0f || !(fabsf(f) < __builtin_huge_valf())) return;
  const int type = A.type[k], row_len = A.row_len[k];
  void* g = const_cast<void*>(A.grad[k]);
  if (type == GS_TYPE_F32) run_scale<kStream>((float*)g, A.active, row_len, begin, end, f);
  else if (type == GS_TYPE_BF16) run_scale<kStream>((__bf16*)g, A.active, row_len, begin, end, f);
  else run_scale<kStream>((_Float16*)g, A.active, row_len, begin, end, f);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_grad_norms_workspace_size(int num, const int64_t* counts) {
  if (num < 0 || (num > 0 && !counts)) return 0;
  for (int i = 0; i < num; ++i)
    if (counts[i] < 0 || counts[i] >= ((int64_t)1 << 40)) return 0;
  return norm_layout(num, counts).total;
}

namespace {

// Both norms and clipping: checks, and the launches of the partial sums.
int norm_launches(const char* what, hipStream_t s, int num, const void* const* grads, const int* grad_types,
                  const int64_t* counts, const int64_t* row_lens, const uint8_t* active, int64_t rows, double max_norm,
                  void* workspace, size_t workspace_bytes, const float* out, NormLayout& L) {
  GS_REQUIRE(num >= 0, "%s: %d tensors", what, num);
  GS_REQUIRE(num == 0 || (grads && grad_types && counts), "%s: NULL argument", what);
  GS_REQUIRE(out && workspace, "%s: NULL argument", what);
  GS_REQUIRE(!active || row_lens, "%s: a mask needs row lengths", what);
  GS_REQUIRE(max_norm == max_norm, "%s: the norm to clip to is not a number", what);
  for (int i = 0; i < num; ++i) {
    GS_REQUIRE(counts[i] >= 0 && counts[i] < ((int64_t)1 << 40), "%s: tensor %d has %lld elements", what, i,
               (long long)counts[i]);
    GS_REQUIRE(counts[i] == 0 || grads[i], "%s: NULL tensor %d", what, i);
    GS_REQUIRE(grad_types[i] >= GS_TYPE_F32 && grad_types[i] <= GS_TYPE_F16, "%s: type of tensor %d", what, i);
    GS_REQUIRE((reinterpret_cast<uintptr_t>(grads[i]) & (grad_types[i] == GS_TYPE_F32 ? 3 : 1)) == 0,
               "%s: tensor %d is not aligned to its type", what, i);
    if (active && counts[i])
      GS_REQUIRE(row_lens[i] >= 1 && row_lens[i] < kMaxRowLen && rows >= 0 &&
                     counts[i] % row_lens[i] == 0 && counts[i] / row_lens[i] == rows,
                 "%s: tensor %d has %lld elements, not rows x row length", what, i, (long long)counts[i]);
  }
  L = norm_layout(num, counts);
  GS_REQUIRE(workspace_bytes >= L.total, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, L.total);
  GS_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "%s: the workspace must be 8-byte aligned", what);
  GS_REQUIRE(L.partials < 0x7fffffff, "%s: too many elements", what);
  char* ws = (char*)workspace;
  NormArgs A{};
  NormList list(num, grads, grad_types, counts, active ? row_lens : nullptr, active, L);
  while (list.next(A)) {
    A.first = (int32_t*)(ws + L.first) + list.tensor - A.n;
    A.partial = (double*)ws + A.first_partial;
    hipLaunchKernelGGL(grad_norms_kernel, dim3(A.groups ? A.groups : 1), dim3(256), 0, s, A);
    GS_LAUNCH_CHECK("grad_norms_kernel");
  }
  return GS_OK;
}

int total_launch(hipStream_t s, int num, const NormLayout& L, double max_norm, const float* grad_scale, void* workspace,
                 float* norms, float* out) {
  const char* ws = (const char*)workspace;
  // all threads at once for few tensors; at least eight a tensor, whose loads then wait together
  int group_log2 = 10;
  while (group_log2 > 3 && (1024 >> group_log2) < num) --group_log2;
  hipLaunchKernelGGL(grad_norms_total_kernel, dim3(1), dim3(1024), 0, s, num, (int)L.partials, group_log2, (const double*)ws,
                     (const int32_t*)(ws + L.first), (double*)(ws + L.sums), grad_scale, max_norm, norms, out);
  GS_LAUNCH_CHECK("grad_norms_total_kernel");
  return GS_OK;
}

}  // namespace

extern "C" int gs_grad_norms(void* stream, int num, const void* const* grads, const int* grad_types,
                             const int64_t* counts, const int64_t* row_lens, const uint8_t* active, int64_t rows,
                             double max_norm, const float* grad_scale, void* workspace, size_t workspace_bytes,
                             float* norms, float* out) {
  NormLayout L;
  const int rc = norm_launches("gs_grad_norms", (hipStream_t)stream, num, grads, grad_types, counts, row_lens, active, rows,
                               max_norm, workspace, workspace_bytes, out, L);
  if (rc != GS_OK) return rc;
  return total_launch((hipStream_t)stream, num, L, max_norm, grad_scale, workspace, norms, out);
}

extern "C" int gs_clip_grads(void* stream, int num, void* const* grads, const int* grad_types, const int64_t* counts,
                             const int64_t* row_lens, const uint8_t* active, int64_t rows, double max_norm,
                             const float* grad_scale, void* workspace, size_t workspace_bytes, float* norms, float* out) {
  GS_REQUIRE(max_norm > 0.0, "gs_clip_grads: the norm to clip to must be positive");
  hipStream_t s = (hipStream_t)stream;
  NormLayout L;
  int rc = norm_launches("gs_clip_grads", s, num, grads, grad_types, counts, row_lens, active, rows, max_norm, workspace,
                         workspace_bytes, out, L);
  if (rc != GS_OK) return rc;
  ScaleArgs S{};
  // more partial sums (of very many tensors) are added up once
  const bool apart = L.partials > 2 * kNormRuns;
  if (apart || num == 0) {
    rc = total_launch(s, num, L, max_norm, grad_scale, workspace, norms, out);
    if (rc != GS_OK) return rc;
  }
  S.partial = apart ? nullptr : (const double*)workspace;
  S.partials = (int32_t)L.partials;
  S.writes = 1;
  S.max_norm = max_norm;
  S.grad_scale = grad_scale;
  S.out = out;
  int64_t bytes = 0;
  for (int i = 0; i < num; ++i) bytes += counts[i] * (grad_types[i] == GS_TYPE_F32 ? 4 : 2);
  NormList list(num, grads, grad_types, counts, active ? row_lens : nullptr, active, L);
  while (list.next(S.a)) {
    S.norms = norms ? norms + list.tensor - S.a.n : nullptr;
    hipLaunchKernelGGL(bytes >= kStreamBytes && !active ? grad_scale_kernel<true> : grad_scale_kernel<false>, dim3(S.a.groups ? S.a.groups : 1), dim3(256), 0, s, S);
    GS_LAUNCH_CHECK("grad_scale_kernel");
    S.writes = 0;
  }
  return GS_OK;
}
