// Norms of many gradients at once, and the factor that clips them, on gfx950.
//
//   n_k = |s| sqrt(sum_i g_ki^2),   n = sqrt(sum_k n_k^2),
//   scale = s min(1, c / (n + 1e-6))   (s without c; NaN unless n is finite),
// s a device scalar (a loss scale's inverse) or 1.  Rows whose mask is 0 are left out, whatever
// they hold.  Squares and sums are float64: no square of a float32 overflows or vanishes there,
// and the order of the sums, which is fixed, does not show in the float32 results.
//
// Every workgroup sums one run of consecutive elements of one tensor (the runs' length is chosen
// so that about 2048 of them cover all tensors) into one partial sum; a second launch of one
// workgroup adds the partial sums of each tensor and the tensors' sums.
#include "gs_common.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kNormTensors = 64;  // per launch
constexpr int kNormRuns = 2048;   // 8 workgroups of 4 waves on each of 256 CUs

struct NormTensor {
  const void* grad;
  int64_t count;
  uint64_t row_magic;  // floor(2^64 / row_len) + 1 (0: row_len 1)
  int32_t row_len;
  int32_t type;
};

struct NormArgs {
  NormTensor t[kNormTensors];
  uint32_t begin[64];  // first workgroup of each tensor, ~0 after the last
  const uint8_t* active;
  double* partial;     // of this launch's first workgroup
  int32_t* first;      // this launch's tensors: their first partial sums
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
  L.run = std::max<int64_t>(4096, ((total + kNormRuns - 1) / kNormRuns + 2047) / 2048 * 2048);
  L.partials = 0;
  for (int i = 0; i < num; ++i) L.partials += (counts[i] + L.run - 1) / L.run;
  L.sums = (size_t)L.partials * sizeof(double);
  L.first = L.sums + (size_t)num * sizeof(double);
  L.total = L.first + ((size_t)num + 2) * sizeof(int32_t);
  return L;
}

__device__ inline double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

template <class G>
__device__ inline double run_sum(const NormArgs& A, const NormTensor& t, int64_t begin, int64_t end) {
  constexpr int kVec = 16 / sizeof(G);  // 16 bytes a lane
  typedef G vec __attribute__((ext_vector_type(kVec), aligned(sizeof(G))));
  const G* g = (const G*)t.grad;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  if (A.active == nullptr) {
    const int64_t step = 256 * kVec;
    int64_t e = begin + threadIdx.x * kVec;
    for (; e + 3 * step + kVec <= end; e += 4 * step) {
      vec v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const vec*>(g + e + u * step);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const double x = (double)(float)v[u][j];
          acc[u] = fma(x, x, acc[u]);
        }
    }
    for (; e < end; e += step)
      for (int j = 0; j < kVec; ++j)
        if (e + j < end) {
          const double x = (double)(float)g[e + j];
          acc[0] = fma(x, x, acc[0]);
        }
  } else {
    for (int64_t e = begin + threadIdx.x; e < end; e += 256) {
      const uint64_t row = t.row_magic ? __umul64hi((uint64_t)e, t.row_magic) : (uint64_t)e;
      const float gx = (float)g[e];
      const double x = A.active[row] ? (double)gx : 0.0;
      acc[0] = fma(x, x, acc[0]);
    }
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

__global__ __launch_bounds__(256) void grad_norms_kernel(NormArgs A) {
  const uint32_t b = blockIdx.x;
  if (b == 0 && threadIdx.x < (uint32_t)A.n)
    A.first[threadIdx.x] = A.first_partial + (int32_t)A.begin[threadIdx.x];
  if (b >= A.groups) return;  // every tensor is empty
  const int k = __popcll(__ballot(b >= A.begin[threadIdx.x & 63u])) - 1;
  const NormTensor t = A.t[k];
  const uint32_t within = b - A.begin[k];
  const int64_t begin = (int64_t)within * A.run;
  const int64_t end = begin + A.run < t.count ? begin + A.run : t.count;
  double x;
  if (t.type == GS_TYPE_F32) x = run_sum<float>(A, t, begin, end);
  else if (t.type == GS_TYPE_BF16) x = run_sum<__bf16>(A, t, begin, end);
  else x = run_sum<_Float16>(A, t, begin, end);
  x = wave_sum(x);
  __shared__ double w[4];
  if ((threadIdx.x & 63u) == 0) w[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x == 0) A.partial[b] = (w[0] + w[1]) + (w[2] + w[3]);
}

// One workgroup: a wave sums a tensor's partial sums, the first wave the tensors'.
__global__ __launch_bounds__(1024) void grad_norms_total_kernel(int num, int partials, const double* __restrict__ partial,
                                                                const int32_t* __restrict__ first, double* sums,
                                                                const float* __restrict__ grad_scale, double max_norm,
                                                                float* __restrict__ norms, float* __restrict__ out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double s = grad_scale ? fabs((double)*grad_scale) : 1.0;
  for (int k = wave; k < num; k += 16) {
    const int b = first[k], e = k + 1 < num ? first[k + 1] : partials;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    int i = b + lane;
    for (; i + 192 < e; i += 256)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] += partial[i + 64 * u];
    for (; i < e; i += 64) acc[0] += partial[i];
    const double x = wave_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (lane == 0) {
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

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_grad_norms_workspace_size(int num, const int64_t* counts) {
  if (num < 0 || (num > 0 && !counts)) return 0;
  for (int i = 0; i < num; ++i)
    if (counts[i] < 0 || counts[i] >= ((int64_t)1 << 40)) return 0;
  return norm_layout(num, counts).total;
}

extern "C" int gs_grad_norms(void* stream, int num, const void* const* grads, const int* grad_types,
                             const int64_t* counts, const int64_t* row_lens, const uint8_t* active, int64_t rows,
                             double max_norm, const float* grad_scale, void* workspace, size_t workspace_bytes,
                             float* norms, float* out) {
  GS_REQUIRE(num >= 0, "gs_grad_norms: %d tensors", num);
  GS_REQUIRE(num == 0 || (grads && grad_types && counts), "gs_grad_norms: NULL argument");
  GS_REQUIRE(out && workspace, "gs_grad_norms: NULL argument");
  GS_REQUIRE(!active || row_lens, "gs_grad_norms: a mask needs row lengths");
  GS_REQUIRE(max_norm == max_norm, "gs_grad_norms: the norm to clip to is not a number");
  for (int i = 0; i < num; ++i) {
    GS_REQUIRE(counts[i] >= 0 && counts[i] < ((int64_t)1 << 40), "gs_grad_norms: tensor %d has %lld elements", i,
               (long long)counts[i]);
    GS_REQUIRE(counts[i] == 0 || grads[i], "gs_grad_norms: NULL tensor %d", i);
    GS_REQUIRE(grad_types[i] >= GS_TYPE_F32 && grad_types[i] <= GS_TYPE_F16, "gs_grad_norms: type of tensor %d", i);
    GS_REQUIRE((reinterpret_cast<uintptr_t>(grads[i]) & (grad_types[i] == GS_TYPE_F32 ? 3 : 1)) == 0,
               "gs_grad_norms: tensor %d is not aligned to its type", i);
    if (active && counts[i])
      GS_REQUIRE(row_lens[i] >= 1 && row_lens[i] < ((int64_t)1 << 24) && rows >= 0 &&
                     counts[i] % row_lens[i] == 0 && counts[i] / row_lens[i] == rows,
                 "gs_grad_norms: tensor %d has %lld elements, not rows x row length", i, (long long)counts[i]);
  }
  const NormLayout L = norm_layout(num, counts);
  GS_REQUIRE(workspace_bytes >= L.total, "gs_grad_norms: workspace of %zu bytes, %zu needed", workspace_bytes,
             L.total);
  GS_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "gs_grad_norms: the workspace must be 8-byte aligned");
  GS_REQUIRE(L.partials < 0x7fffffff, "gs_grad_norms: too many elements");
  char* ws = (char*)workspace;
  NormArgs A{};
  A.active = active;
  A.run = L.run;
  hipStream_t s = (hipStream_t)stream;
  int64_t done = 0;
  for (int i = 0; i < num;) {
    int k = 0;
    int64_t groups = 0;
    for (; i < num && k < kNormTensors; ++i) {
      NormTensor& t = A.t[k];
      t.grad = grads[i];
      t.count = counts[i];
      t.row_len = active && counts[i] ? (int32_t)row_lens[i] : 1;
      t.row_magic = t.row_len > 1 ? ~(uint64_t)0 / (uint64_t)t.row_len + 1 : 0;
      t.type = grad_types[i];
      A.begin[k++] = (uint32_t)groups;
      groups += (counts[i] + L.run - 1) / L.run;
    }
    A.n = k;
    A.groups = (uint32_t)groups;
    A.first = (int32_t*)(ws + L.first) + (i - k);
    for (; k < 64; ++k) A.begin[k] = 0xffffffffu;
    A.partial = (double*)ws + done;
    A.first_partial = (int32_t)done;
    done += groups;
    hipLaunchKernelGGL(grad_norms_kernel, dim3((unsigned)(groups > 0 ? groups : 1)), dim3(256), 0, s, A);
    GS_LAUNCH_CHECK("grad_norms_kernel");
  }
  hipLaunchKernelGGL(grad_norms_total_kernel, dim3(1), dim3(1024), 0, s, num, (int)L.partials, (const double*)ws,
                     (const int32_t*)(ws + L.first), (double*)(ws + L.sums), grad_scale, max_norm, norms, out);
  GS_LAUNCH_CHECK("grad_norms_total_kernel");
  return GS_OK;
}
