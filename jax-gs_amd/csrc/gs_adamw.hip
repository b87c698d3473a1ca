// AdamW over many tensors at once on gfx950, with moments in 32 or in 8 bits, and the
// conversion of moments between the two.
//
// Per element, with g = scale * grad (0 in masked rows), t = updates made, this one included:
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//   u = (m / (1 - b1^t)) / (sqrt(v) / sqrt(1 - b2^t) + eps),
//   w = w - lr (u + decay w)                       (masked rows keep w).
// Moments, weights and every operation are float32; half parameters are rounded once to
// nearest even from the float32 result, which a master copy keeps when there is one.  A scale
// that is not finite leaves everything as it is and does not count as an update.
//
// The state is flat: tensor i's moments begin at offsets[i], a multiple of 256, so that blocks
// of the 8-bit form, whole quads and their alignment do not depend on the tensors' sizes.
// A workgroup takes 1024 consecutive elements of one tensor, a wave one block, a lane four
// elements: 16-byte accesses of float32, and a block's two maxima are one reduction over a wave.
// The tensor is found by one comparison per lane and a ballot.
//
// One pass over memory, which bounds it: 28 B an element with float32 everywhere, 16 B with 8-bit
// moments; a large copy reaches 5.1 TB/s.  Measured: 59M float32 elements 260 us in 32 bits (6.3
// TB/s), 152 us in 8 bits (6.2 TB/s; 257 vector instructions a wave, which would take 110 us by
// themselves and are what bounds bfloat16 weights and gradients, 128 us for 10 B an element);
// 2.1M Gaussians (124M elements, 40 % of the rows masked) in 32 bits 487 us; 3M (177M, 20 %
// masked) in 8 bits 462 us; 59M half weights and gradients without masters in 32 bits 203 us (6.4
// TB/s, either type).  The smallest call takes 4.4 us, five dependent reads.
#include "gs_moments.h"
#include "gs_pieces.h"
#include "gs_rows.h"

namespace gs {
namespace {

struct StepTensor {
  void* param;
  const void* grad;
  int64_t at;     // first element in the state
  int64_t count;
  uint64_t magic; // of the row length
  uint32_t row_len;
  float lr, decay;
  int kind;       // parameter type * 6 + gradient type * 2 + master
};

// As it is passed: one record per tensor (per 2^30 elements of one), which a wave reads from one or two cache lines (arrays
// per field, ten lines, cost a tenth of the whole step in 8 bits: 158 -> 172 us).
struct StepRecord {
  void* param;
  const void* grad;
  uint64_t magic;
  uint32_t at;      // first block in the state
  uint32_t blocks;
  uint32_t row_len;
  float lr, decay;
  uint8_t last;     // elements of the last block, less one
  uint8_t kind;
  uint16_t piece;   // the record's workgroups begin at piece * kPieceGroups of the tensor
};

struct StepArgs {
  StepRecord t[kStepTensors];
  uint32_t begin[kStepTensors];  // first workgroup of each record
  int32_t n;
  uint32_t groups;
  void* mu;
  void* nu;
  uint8_t* fields;
  float* master;
  const uint8_t* active;
  double b1d, b2d;
  float b1, b2, omb1, omb2, eps;
  uint32_t key;
  bool stream_params;
};
static_assert(sizeof(StepArgs) + 3 * sizeof(void*) <= 4096, "kernel arguments");

// From this many bytes on (parameters, gradients and moments of a call) the arrays go past the
// caches: nothing of them is left there for the next call, and what is written does not push out
// what is about to be read.  float32, us with caches -> past them: 4M elements 21 -> 24, 8M
// (128 MB) 46 -> 41, 16M 87 -> 73, 59M 296 -> 272, 177M 901 -> 823; in 8 bits 8M (80 MB)
// 25 -> 27, 16M 52 -> 46, 32M 98 -> 89; encoding 12M (120 MB) 20 -> 23, 30M 55 -> 50, decoding
// 30M 55 -> 45.
constexpr int64_t kStreamBytes = (int64_t)128 << 20;
// Parameters are read next by whatever uses the model: they go past the caches only when they
// alone are as large (16M: 79 us past them, 73 not; 59M: 272 and 304).

// Four elements at p, which is only as aligned as its element: a tensor may begin anywhere.
template <bool kStream, class T>
__device__ inline void load4(const T* p, float (&x)[4]) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const vec* q = reinterpret_cast<const vec*>(p);
  const vec v = kStream ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = (float)v[j];
}
template <bool kStream, class T>
__device__ inline void store4(T* p, const float (&x)[4]) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  vec v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (T)x[j];
  vec* q = reinterpret_cast<vec*>(p);
  if (kStream) __builtin_nontemporal_store(v, q);
  else *q = v;
}
// Four 8-bit codes.
template <bool kStream>
__device__ inline uint32_t load_codes(const void* p, int64_t at) {
  const uint32_t* q = (const uint32_t*)((const uint8_t*)p + at);
  return kStream ? __builtin_nontemporal_load(q) : *q;
}
template <bool kStream>
__device__ inline void store_codes(void* p, int64_t at, uint32_t x) {
  uint32_t* q = (uint32_t*)((uint8_t*)p + at);
  if (kStream) __builtin_nontemporal_store(x, q);
  else *q = x;
}

// How a wave reads and writes its 256 elements of gradient and weight, the lane's four from l4 on.
// Whole blocks know their types, so that all loads are on their way before the first wait.
template <bool kStream, class P, class G, bool kMaster>
struct WholeBlock {
  typedef P params __attribute__((ext_vector_type(4), aligned(sizeof(P))));
  const G* grad;
  P* param;
  float* master;
  bool stream_params;
  params old;  // of a lane with masters and some of its four masked
  __device__ WholeBlock(const StepArgs& A, const StepTensor& t, int64_t base)
      : grad((const G*)t.grad + base), param((P*)t.param + base), master(A.master + t.at + base),
        stream_params(A.stream_params) {}
  __device__ int n(uint32_t) const { return 4; }
  // on: which of the four are not masked.
  __device__ void load(uint32_t l4, float (&g)[4], float (&w)[4], uint32_t on) {
    load4<kStream>(grad + l4, g);
    if (kMaster) load4<kStream>(master + l4, w);
    else load4<kStream>((const P*)param + l4, w);
    if (kMaster && on != 15u) old = *reinterpret_cast<const params*>(param + l4);
  }
  // The masked of the four are stored as what was read from there.  With masters that is one more
  // read, which takes less than storing the others one by one (30M bfloat16 with masters, 40 % of the
  // elements masked, 32 and 8 bits: 138 and 98 us, one by one 166 and 118).
  __device__ void store(uint32_t l4, const float (&w)[4], uint32_t on) const {
    if (kMaster && on != 15u) {
      params v = old;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (on >> j & 1u) v[j] = (P)w[j];
      *reinterpret_cast<params*>(param + l4) = v;
    } else if (kStream && stream_params) {
      asm volatile("");  // keeps the compiler from merging the two stores into one of the second kind
      store4<true>(param + l4, w);
      asm volatile("");
    } else {
      store4<false>(param + l4, w);
    }
    if (kMaster) store4<kStream>(master + l4, w);
  }
};

// The last, partial block of a tensor: element by element, of any types.  All loads are on their
// way before the first is looked at: lanes past the end read the last element again.
struct PartBlock {
  const void* grad;
  void* param;
  float* master;
  int64_t base;
  int left, gtype, ptype;
  __device__ PartBlock(const StepArgs& A, const StepTensor& t, int64_t base_)
      : grad(t.grad), param(t.param), master(t.kind & 1 ? A.master + t.at + base_ : nullptr), base(base_),
        left((int)(t.count - base_)), gtype((t.kind >> 1) % 3), ptype(t.kind / 6) {}
  __device__ int n(uint32_t l4) const { return min(max(left - (int)l4, 0), 4); }
  __device__ void raw(const void* p, int64_t from, bool wide, uint32_t l4, uint32_t (&x)[4]) const {
    const int last = left - 1;
    if (wide) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = ((const uint32_t*)p)[from + min((int)l4 + j, last)];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = ((const uint16_t*)p)[from + min((int)l4 + j, last)];
    }
  }
  static __device__ float value(uint32_t x, int type) {
    if (type == GS_TYPE_F32) return bits_to_float(x);
    if (type == GS_TYPE_BF16) return bits_to_float(x << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
  }
  __device__ void load(uint32_t l4, float (&g)[4], float (&w)[4], uint32_t) const {
    uint32_t a[4], b[4];
    raw(grad, base, gtype == GS_TYPE_F32, l4, a);
    raw(master ? (const void*)master : param, master ? 0 : base, master || ptype == GS_TYPE_F32, l4, b);
    const int k = n(l4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] = j < k ? value(a[j], gtype) : 0.0f;
      w[j] = j < k ? value(b[j], master ? GS_TYPE_F32 : ptype) : 0.0f;
    }
  }
  __device__ void store(uint32_t l4, const float (&w)[4], uint32_t on) const {
    const int k = n(l4);
    for (int j = 0; j < 4; ++j) {
      if (j >= k || !(on >> j & 1u)) continue;
      const int64_t i = base + l4 + j;
      if (ptype == GS_TYPE_F32) ((float*)param)[i] = w[j];
      else if (ptype == GS_TYPE_BF16) ((__bf16*)param)[i] = (__bf16)w[j];
      else ((_Float16*)param)[i] = (_Float16)w[j];
      if (master) master[l4 + j] = w[j];
    }
  }
};

__device__ inline bool is_finite(float x) { return fabsf(x) < __builtin_huge_valf(); }

template <bool k8, bool kMask, bool kStream, class Block>
__device__ inline void step_block(const StepArgs& A, const StepTensor& t, int64_t base, float scale, double r1d,
                                  double r2d) {
  const uint32_t l4 = (threadIdx.x & 63u) * 4u;
  const int64_t at = t.at + base;
  Block io(A, t, base);
  float w[4] = {0.0f, 0.0f, 0.0f, 0.0f}, g[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m[4], r[4], v[4];
  uint32_t m8 = 0, r8 = 0, f = 0;
  if (k8) {
    m8 = load_codes<kStream>(A.mu, at + l4);
    r8 = load_codes<kStream>(A.nu, at + l4);
    f = *(const uint16_t*)(A.fields + (at >> 7));
  } else {
    load4<kStream>((const float*)A.mu + at + l4, m);
    load4<kStream>((const float*)A.nu + at + l4, v);
  }
  // masked rows: neither gradient nor parameter is read or written
  const uint32_t on = kMask ? rows_on<4>(A.active, t.magic, t.row_len, base, l4, io.n(l4)) : 15u;
  if (!kMask || on) io.load(l4, g, w, on);
  if (k8 && !is_finite(scale)) return;
  const float r1 = (float)r1d, r2 = (float)r2d;
  if (k8) {
    decode_m4(m8, (int)(f & 255u), m);
    decode_r4(r8, (int)(f >> 8), r);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = r[j] * r[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = !kMask || (on >> j & 1u) ? g[j] * scale : 0.0f;
    m[j] = m[j] * A.b1 + x * A.omb1;
    v[j] = v[j] * A.b2 + (x * x) * A.omb2;
  }
  roots4(v, r);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // the divisor's reciprocal to within one step: 2^-23 of a step of the weight
    const float u = (m[j] * r1) * __builtin_amdgcn_rcpf(r[j] * r2 + A.eps);
    const float y = w[j] - t.lr * (u + t.decay * w[j]);
    w[j] = !kMask || (on >> j & 1u) ? y : w[j];
  }
  if (!kMask || on) io.store(l4, w, on);
  if (k8) {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = place_hash(at, l4 + j, A.key);
    encode_block<true>(m, r, h, m8, r8, f);
    store_codes<kStream>(A.mu, at + l4, m8);
    store_codes<kStream>(A.nu, at + l4, r8);
    if (l4 == 0) *(uint16_t*)(A.fields + (at >> 7)) = (uint16_t)f;
  } else {
    store4<kStream>((float*)A.mu + at + l4, m);
    store4<kStream>((float*)A.nu + at + l4, v);
  }
}

template <bool k8, bool kMask, bool kStream>
__global__ __launch_bounds__(256) void adamw_kernel(
    StepArgs A, const float* __restrict__ grad_scale,
    const double* __restrict__ powers,  // b1^(t-1), b2^(t-1), 1 / (1 - b1^t), 1 / sqrt(1 - b2^t)
    double* __restrict__ powers_next) {  // NULL in all launches of a step but the first
  const float scale = grad_scale ? *grad_scale : 1.0f;
  const double r1 = powers[2], r2 = powers[3];
  if (powers_next != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    const bool ok = is_finite(scale);
    const double p1 = ok ? powers[0] * A.b1d : powers[0], p2 = ok ? powers[1] * A.b2d : powers[1];
    powers_next[0] = p1;
    powers_next[1] = p2;
    powers_next[2] = ok ? 1.0 / (1.0 - p1 * A.b1d) : powers[2];
    powers_next[3] = ok ? 1.0 / sqrt(1.0 - p2 * A.b2d) : powers[3];
  }
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;  // nothing to update
  // A scale that is not finite: nothing changes.  In 8 bits this is asked only after the loads are on
  // their way (3M Gaussians 784 -> 764 us); in 32 bits, where more of them at once crowd the
  // memory (35M bfloat16 weights with masters 164 us asked here, 189 asked there), before.
  if (!k8 && !is_finite(scale)) return;
  int k = -1;  // the last record that begins at or before this workgroup
  for (int i = 0; i < A.n; i += 64) {
    const int q = i + (int)(threadIdx.x & 63u);
    k += __popcll(__ballot(q < A.n && b >= A.begin[min(q, kStepTensors - 1)]));
  }
  k = __builtin_amdgcn_readfirstlane(k);
  const StepRecord q = A.t[k];
  const StepTensor t{q.param,
                     q.grad,
                     (int64_t)q.at * kMomBlock,
                     ((int64_t)q.blocks - 1) * kMomBlock + q.last + 1,
                     q.magic,
                     q.row_len,
                     q.lr,
                     q.decay,
                     q.kind};
  const int64_t base = (q.piece * kPieceGroups + (b - A.begin[k])) * kStepChunk +
                       __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * kMomBlock;
  if (base >= t.count) return;  // the wave's block is past the end
  if (t.count - base < kMomBlock) {
    step_block<k8, kMask, false, PartBlock>(A, t, base, scale, r1, r2);
    return;
  }
  switch (t.kind) {
#define GS_STEP(i, P, G, M)                                                                       \
  case i:                                                                                         \
    step_block<k8, kMask, kStream, WholeBlock<kStream, P, G, M>>(A, t, base, scale, r1, r2);      \
    break;
    GS_STEP(0, float, float, false)
    GS_STEP(2, float, __bf16, false)
    GS_STEP(4, float, _Float16, false)
    GS_STEP(6, __bf16, float, false)
    GS_STEP(7, __bf16, float, true)
    GS_STEP(8, __bf16, __bf16, false)
    GS_STEP(9, __bf16, __bf16, true)
    GS_STEP(10, __bf16, _Float16, false)
    GS_STEP(11, __bf16, _Float16, true)
    GS_STEP(12, _Float16, float, false)
    GS_STEP(13, _Float16, float, true)
    GS_STEP(14, _Float16, __bf16, false)
    GS_STEP(15, _Float16, __bf16, true)
    GS_STEP(16, _Float16, _Float16, false)
    GS_STEP(17, _Float16, _Float16, true)
#undef GS_STEP
  }
}

// Conversion: a wave per block, 10 B an element and little arithmetic, so memory bounds both.
// 12M elements 22 us to 8 bits and 18 us back (5.3 and 6.5 TB/s), 124M 196 and 212 us (6.3, 5.9).
template <bool kStream>
__global__ __launch_bounds__(256) void moments_encode_kernel(int64_t blocks, const float* __restrict__ mu,
                                                             const float* __restrict__ nu, uint8_t* __restrict__ m8,
                                                             uint8_t* __restrict__ r8, uint8_t* __restrict__ fields) {
  const int64_t block = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (block >= blocks) return;
  const int64_t at = block * kMomBlock + (threadIdx.x & 63u) * 4;
  float m[4], r[4], v[4];
  load4<kStream>(mu + at, m);
  load4<kStream>(nu + at, v);
  roots4(v, r);
  const uint32_t none[4] = {0, 0, 0, 0};
  uint32_t cm, cr, f;
  encode_block<false>(m, r, none, cm, cr, f);
  store_codes<kStream>(m8, at, cm);
  store_codes<kStream>(r8, at, cr);
  if ((threadIdx.x & 63u) == 0) *(uint16_t*)(fields + 2 * block) = (uint16_t)f;
}

template <bool kStream>
__global__ __launch_bounds__(256) void moments_decode_kernel(int64_t blocks, const uint8_t* __restrict__ m8,
                                                             const uint8_t* __restrict__ r8,
                                                             const uint8_t* __restrict__ fields,
                                                             float* __restrict__ mu, float* __restrict__ nu) {
  const int64_t block = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (block >= blocks) return;
  const int64_t at = block * kMomBlock + (threadIdx.x & 63u) * 4;
  const uint32_t f = *(const uint16_t*)(fields + 2 * block);
  float m[4], r[4];
  decode_m4(load_codes<kStream>(m8, at), (int)(f & 255u), m);
  decode_r4(load_codes<kStream>(r8, at), (int)(f >> 8), r);
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = r[j] * r[j];
  store4<kStream>(mu + at, m);
  store4<kStream>(nu + at, r);
}

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

size_t size_of(int type) { return type == GS_TYPE_F32 ? 4 : 2; }

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_adamw_step(void* stream, int num, void* const* params, const int* param_types,
                             const void* const* grads, const int* grad_types, const int64_t* offsets,
                             const int64_t* counts, const int64_t* row_lens, const double* lrs,
                             const double* decays, int moment_bits, int64_t state_size, void* mu, void* nu,
                             uint8_t* fields, float* master, const uint8_t* active, int64_t rows,
                             const float* grad_scale, const double* powers, double* powers_next, double b1,
                             double b2, double eps, uint32_t key) {
  GS_REQUIRE(num >= 0, "gs_adamw_step: %d tensors", num);
  GS_REQUIRE(num == 0 || (params && param_types && grads && grad_types && offsets && counts && lrs && decays),
             "gs_adamw_step: NULL argument");
  GS_REQUIRE(moment_bits == 32 || moment_bits == 8, "gs_adamw_step: moments in 32 or 8 bits, not %d", moment_bits);
  GS_REQUIRE(state_size >= 0 && state_size % kMomBlock == 0 && state_size < ((int64_t)1 << 40),
             "gs_adamw_step: state of %lld elements",
             (long long)state_size);
  GS_REQUIRE(state_size == 0 || (mu && nu && (moment_bits == 32 || fields)), "gs_adamw_step: NULL state");
  GS_REQUIRE(aligned(mu, 16) && aligned(nu, 16) && aligned(fields, 2) && aligned(master, 16),
             "gs_adamw_step: the state's arrays must be 16-byte aligned");
  GS_REQUIRE(powers && powers_next && powers != powers_next, "gs_adamw_step: two arrays of powers are needed");
  GS_REQUIRE(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0, "gs_adamw_step: b1 and b2 must be in [0, 1)");
  GS_REQUIRE(eps >= 0.0, "gs_adamw_step: eps must not be negative");
  GS_REQUIRE(!active || row_lens, "gs_adamw_step: a mask needs row lengths");
  int64_t used = 0;  // end of the moments of the tensors before
  for (int i = 0; i < num; ++i) {
    if (!grads[i] || counts[i] == 0) continue;
    const int pt = param_types[i], gt = grad_types[i];
    GS_REQUIRE(pt >= GS_TYPE_F32 && pt <= GS_TYPE_F16 && gt >= GS_TYPE_F32 && gt <= GS_TYPE_F16,
               "gs_adamw_step: type of tensor %d", i);
    GS_REQUIRE(counts[i] > 0 && counts[i] < ((int64_t)1 << 40), "gs_adamw_step: tensor %d has %lld elements", i,
               (long long)counts[i]);
    GS_REQUIRE(params[i], "gs_adamw_step: NULL tensor %d", i);
    GS_REQUIRE(aligned(params[i], size_of(pt)) && aligned(grads[i], size_of(gt)),
               "gs_adamw_step: tensor %d is not aligned to its type", i);
    GS_REQUIRE(offsets[i] >= 0 && offsets[i] % kMomBlock == 0 && offsets[i] <= state_size &&
                   counts[i] <= state_size - offsets[i],
               "gs_adamw_step: tensor %d lies outside the state", i);
    GS_REQUIRE(offsets[i] >= used, "gs_adamw_step: the moments of tensor %d do not lie behind those before", i);
    used = offsets[i] + counts[i];
    if (active)
      GS_REQUIRE(row_lens[i] >= 1 && row_lens[i] < kMaxRowLen && rows >= 0 &&
                     counts[i] % row_lens[i] == 0 && counts[i] / row_lens[i] == rows,
                 "gs_adamw_step: tensor %d has %lld elements, not rows x row length", i, (long long)counts[i]);
  }
  StepArgs A{};
  A.mu = mu;
  A.nu = nu;
  A.fields = fields;
  A.master = master;
  A.active = active;
  A.b1d = b1;
  A.b2d = b2;
  A.b1 = (float)b1;
  A.b2 = (float)b2;
  A.omb1 = (float)(1.0 - b1);
  A.omb2 = (float)(1.0 - b2);
  A.eps = (float)eps;
  A.key = key;
  hipStream_t s = (hipStream_t)stream;
  const int64_t state_bytes = (moment_bits == 8 ? 2 : 8) + (master ? 4 : 0);
  int64_t param_bytes = 0, bytes = 0;
  for (int j = 0; j < num; ++j)
    if (grads[j]) {
      param_bytes += counts[j] * (int64_t)size_of(param_types[j]);
      bytes += counts[j] * ((int64_t)size_of(grad_types[j]) + state_bytes);
    }
  A.stream_params = param_bytes >= kStreamBytes;
  const bool stream_all = param_bytes + bytes >= kStreamBytes;
#define GS_KERNEL(k8, kMask) (stream_all ? adamw_kernel<k8, kMask, true> : adamw_kernel<k8, kMask, false>)
  auto* kernel = moment_bits == 8 ? (active ? GS_KERNEL(true, true) : GS_KERNEL(true, false))
                                  : (active ? GS_KERNEL(false, true) : GS_KERNEL(false, false));
#undef GS_KERNEL
  // Shared memory that nobody uses, so that four workgroups of 32-bit moments fit a CU instead of
  // eight: past the caches, seven streams of more waves than that crowd the memory (59M float32
  // 275 us with eight, 265 with six, 260 with four; 177M 869, 840, 829; 35M bfloat16 with masters
  // 158, 156, 151).  In 8 bits, where the arithmetic counts, eight are best (35M 91 us, 114
  // with four), and under a mask, whose loads come first (124M, 40 % off: 489 us, 502 with four).
  const unsigned lds = stream_all && moment_bits == 32 && !active ? 40960 : 0;
  // always one launch, so that the powers move on; further ones take what does not fit it
  StepPieces pieces(num, grads, counts);
  do {
    StepPiece out[kStepTensors];
    int64_t groups = 0;
    A.n = pieces.next(out, groups);
    A.groups = (uint32_t)groups;
    for (int k = 0; k < A.n; ++k) {
      const int i = out[k].tensor;
      const int64_t blocks = (counts[i] + kMomBlock - 1) / kMomBlock;
      StepRecord& t = A.t[k];
      t.param = params[i];
      t.grad = grads[i];
      t.at = (uint32_t)(offsets[i] / kMomBlock);
      t.blocks = (uint32_t)blocks;
      t.last = (uint8_t)(counts[i] - (blocks - 1) * kMomBlock - 1);
      t.piece = (uint16_t)out[k].piece;
      t.row_len = active ? (uint32_t)row_lens[i] : 1u;
      t.magic = row_magic(t.row_len);
      t.lr = (float)lrs[i];
      t.decay = (float)decays[i];
      t.kind = (uint8_t)(param_types[i] * 6 + grad_types[i] * 2 + (param_types[i] != GS_TYPE_F32 && master ? 1 : 0));
      A.begin[k] = (uint32_t)out[k].begin;
    }
    const dim3 grid((unsigned)(groups > 0 ? groups : 1));
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, A, grad_scale, powers, powers_next);
    GS_LAUNCH_CHECK("adamw_kernel");
    powers_next = nullptr;
  } while (!pieces.done());
  return GS_OK;
}

extern "C" int gs_moments_encode(void* stream, int64_t state_size, const float* mu, const float* nu, uint8_t* mu8,
                                 uint8_t* nu8, uint8_t* fields) {
  GS_REQUIRE(state_size >= 0 && state_size % kMomBlock == 0 && state_size < ((int64_t)1 << 40),
             "gs_moments_encode: state of %lld elements", (long long)state_size);
  if (state_size == 0) return GS_OK;
  GS_REQUIRE(mu && nu && mu8 && nu8 && fields, "gs_moments_encode: NULL argument");
  GS_REQUIRE(aligned(mu, 16) && aligned(nu, 16) && aligned(mu8, 16) && aligned(nu8, 16) && aligned(fields, 2),
             "gs_moments_encode: the state's arrays must be 16-byte aligned");
  const int64_t blocks = state_size / kMomBlock;
  auto* kernel = state_size * 10 >= kStreamBytes ? moments_encode_kernel<true> : moments_encode_kernel<false>;
  for (int64_t first = 0, here; first < blocks; first += here) {
    here = conversion_blocks(first, blocks);
    const int64_t at = first * kMomBlock;
    hipLaunchKernelGGL(kernel, dim3((unsigned)div_up(here, 4)), dim3(256), 0, (hipStream_t)stream, here,
                       mu + at, nu + at, mu8 + at, nu8 + at, fields + 2 * first);
    GS_LAUNCH_CHECK("moments_encode_kernel");
  }
  return GS_OK;
}

extern "C" int gs_moments_decode(void* stream, int64_t state_size, const uint8_t* mu8, const uint8_t* nu8,
                                 const uint8_t* fields, float* mu, float* nu) {
  GS_REQUIRE(state_size >= 0 && state_size % kMomBlock == 0 && state_size < ((int64_t)1 << 40),
             "gs_moments_decode: state of %lld elements", (long long)state_size);
  if (state_size == 0) return GS_OK;
  GS_REQUIRE(mu && nu && mu8 && nu8 && fields, "gs_moments_decode: NULL argument");
  GS_REQUIRE(aligned(mu, 16) && aligned(nu, 16) && aligned(mu8, 16) && aligned(nu8, 16) && aligned(fields, 2),
             "gs_moments_decode: the state's arrays must be 16-byte aligned");
  const int64_t blocks = state_size / kMomBlock;
  auto* kernel = state_size * 10 >= kStreamBytes ? moments_decode_kernel<true> : moments_decode_kernel<false>;
  for (int64_t first = 0, here; first < blocks; first += here) {
    here = conversion_blocks(first, blocks);
    const int64_t at = first * kMomBlock;
    hipLaunchKernelGGL(kernel, dim3((unsigned)div_up(here, 4)), dim3(256), 0, (hipStream_t)stream, here,
                       mu8 + at, nu8 + at, fields + 2 * first, mu + at, nu + at);
    GS_LAUNCH_CHECK("moments_decode_kernel");
  }
  return GS_OK;
}
