// Rows of moments in 8 bits by one index, on gfx950: taken into a new state, or moved in place.
//
// A tensor's moments are rows of row_len elements one after another, in blocks of 256 that share an
// exponent (gs_moments.h); a row's new neighbours are others than its old ones, so a block is decoded element by element from where
// its rows come from and encoded again, to nearest even.  Values come back as they were but where a
// larger neighbour raises the exponent of their block.
//
// Taken: sixteen lanes make two blocks where rows are a multiple of sixteen elements, else a wave four, four elements of each
// a lane, with all loads under way before the first is encoded.  70 % of 2M rows of 48 elements: 63 us, bound by memory (at
// 5.4 TB/s with the lines of rows that are skipped); of the Gaussians' five tensors 92, where the 11 of 59 elements in
// short rows take 30: their fields and codes come element by element.
//
// Moved: a first launch looks the index over, marks the rows that change bit by bit, and copies the codes and exponents
// that they get; a second (one for each kind of rows, as they want registers or waves) makes the blocks that hold such a row
// anew, in place, from their own codes and those.  So no block is read by others while it changes, and blocks without a
// changed row are not touched.  2M Gaussians, 8 % of them at random: 139 us (187 where changed blocks went to a copy and
// back, and each tensor looked the index over), 8 % at the end 62 (60), none 17 (27).
#include "gs_moments.h"
#include "gs_pieces.h"
#include "gs_rows.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kMomentTensors = 72;  // per launch: the argument block stays below 4 KiB
constexpr int kMomentAhead = 4;     // blocks per wave
constexpr int kOddGroup = 4 * kMomentAhead;  // per workgroup
constexpr int kEvenAhead = 2;       // blocks of sixteen lanes (1.5M rows of 48 taken: 63 us, one 70, four 68)
constexpr int kEvenGroup = 16 * kEvenAhead;
constexpr int kRemakeGroup = 64;    // in a move's second launch
constexpr int kOddAhead = 2;        // blocks of a wave there (139 us; four 148)

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
  int64_t state_size;
  const void* index;
  uint32_t rows;     // of the tensors that are read
  int32_t n;
  uint32_t groups;
};
static_assert(sizeof(MomentArgs) <= 4096, "kernel arguments");

// Entry i of the index: a row, -1 for a negative one, -2 for one beyond the rows.
template <bool kWide, class Args>
__device__ inline int32_t entry(const Args& A, int64_t i) {
  if constexpr (kWide) {
    const int64_t x = ((const int64_t*)A.index)[i];
    return x < 0 ? -1 : x < (int64_t)A.rows ? (int32_t)x : -2;
  } else {
    const int32_t x = ((const int32_t*)A.index)[i];
    return x < 0 ? -1 : (uint32_t)x < A.rows ? x : -2;
  }
}

// Where the rows come from, negative for nowhere.
template <bool kWide, int kN>
__device__ inline void sources(const MomentArgs& A, const int32_t (&row)[kN], const bool (&in)[kN], int32_t (&s)[kN]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) s[j] = entry<kWide>(A, in[j] ? row[j] : 0);
#pragma unroll
  for (int j = 0; j < kN; ++j)
    if (!in[j]) s[j] = -1;
}

// The tensor of this workgroup: the last that begins at or before it.
template <class Args>
__device__ inline int tensor_of(const Args& A, uint32_t b) {
  const int lane = threadIdx.x & 63;
  int k = -1;
  for (int at = 0; at < A.n; at += 64) k += __popcll(__ballot(at + lane < A.n && b >= A.begin[min(at + lane, A.n - 1)]));
  return __builtin_amdgcn_readfirstlane(k);
}

// A block's first row, and how far into it the block begins.
template <class Record>
__device__ inline uint64_t first_row(const Record& t, int64_t base, uint32_t& at) {
  const uint64_t row = t.magic ? __umul64hi((uint64_t)base, t.magic) : (uint64_t)base;
  at = (uint32_t)((uint64_t)base - row * t.row_len);
  return row;
}
// The row of element e from a block's first row on, e less than row_len + 256.
template <class Record>
__device__ inline uint32_t row_of(const Record& t, uint32_t e) {
  return t.row_len > 4096u ? (e >= t.row_len ? 1u : 0u) : t.magic ? __umulhi(e, (uint32_t)(t.magic >> 32) + 1u) : e;
}

// Maxima over each sixteen lanes, in every one of them.
__device__ inline void row_max2_u32(uint32_t& x, uint32_t& y) {
#define GS_DPP_MAX(ctrl)                                                                                  \
  {                                                                                                       \
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true));                   \
    y = max(y, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)y, ctrl, 0xf, 0xf, true));                   \
  }
  GS_DPP_MAX(0xB1);   // quad_perm [1, 0, 3, 2]
  GS_DPP_MAX(0x4E);   // quad_perm [2, 3, 0, 1]
  GS_DPP_MAX(0x141);  // row_half_mirror
  GS_DPP_MAX(0x140);  // row_mirror
#undef GS_DPP_MAX
}

typedef uint32_t vec4u __attribute__((ext_vector_type(4)));
typedef uint16_t pair __attribute__((ext_vector_type(2)));

// Codes of roots under another exponent of their block, as integers: a code above gradual underflow that stays there
// changes by 16 for each power of two.  all: the largest (exponent field * 16 + code) * 2 + (code >= 16) of the block;
// false where the general way is needed.
__device__ inline bool shift_roots(vec4u& w, uint32_t field, uint32_t all, uint32_t least, uint32_t& fields) {
  const uint32_t top = all >> 1;
  // a float32's exponent field of the largest root, as moment_field takes it
  const uint32_t to = all ? (top >> 4) - 15u + ((top & 15u) == 15u ? 1u : 0u) : 0u;
  fields |= to << 8;
  const bool fine = all == 0 || ((all & 1u) && (top >> 4) >= 16u && to < 253u);
  const int by = 16 * ((int)field - (int)to);
  const bool kept = least == 0xffffu || by == 0 || (least >= 15u && (int)least + 1 + by >= 16);  // least: smallest code above 0, less 1
  const uint32_t step = (uint32_t)(by < 0 ? -by : by) * 0x01010101u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t y = (((w[j] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[j]) & 0x80808080u;  // bytes that are not zero
    const uint32_t d = step & (y | (y - (y >> 7)));
    w[j] = by < 0 ? w[j] - d : w[j] + d;
  }
  return fine && kept;
}

// The general way, as encode_block_odd: decode, and encode to nearest.  Everything is decoded twice, so that four values
// at a time are in registers.
__device__ inline void remake(vec4u& wm, vec4u& wr, uint32_t f, uint32_t& fields) {
  constexpr uint32_t kInf = 0x7f800000u;
  uint32_t mm = 0, rr = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float x[4], y[4];
    decode_m4(wm[w], (int)(f & 255u), x);
    decode_r4(wr[w], (int)(f >> 8), y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = float_to_bits(x[j]) & 0x7fffffffu, b = float_to_bits(y[j]);
      mm = max(mm, a < kInf ? a : 0u);
      rr = max(rr, b < kInf ? b : 0u);
    }
  }
  row_max2_u32(mm, rr);
  const uint32_t fm = moment_field<3>(mm), fr = moment_field<4>(rr);
  fields = fm | (fr << 8);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float x[4], y[4];
    decode_m4(wm[w], (int)(f & 255u), x);
    decode_r4(wr[w], (int)(f >> 8), y);
    uint32_t cm[4], cr[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = float_to_bits(x[j]) & 0x7fffffffu, b = float_to_bits(y[j]);
      const uint32_t c = a >= kInf ? 127u << 24 : min(moment_top<3, false>(bits_to_float(a), (int)fm, 0), (126u << 24) | 0xffffffu);
      cm[j] = (c & 0x7fffffffu) | (float_to_bits(x[j]) & 0x80000000u);
      cr[j] = b >= kInf ? 255u << 24 : min(moment_top<4, false>(y[j], (int)fr, 0), (254u << 24) | 0xffffffu);
    }
    wm[w] = pack_top(cm);
    wr[w] = pack_top(cr);
  }
}

// Sixteen codes a lane, of a block in sixteen lanes, under the exponents of their new block.  The signed codes go through
// the machine's scaled conversions, two values each, the roots' as integers; waves with values that are not finite, with
// float32's least exponents or with roots under gradual underflow take the general way, with twice the instructions.
__device__ inline void recode(vec4u& wm, vec4u& wr, uint32_t f, uint32_t& fields) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  constexpr uint32_t kLeastField = 18;  // all values are normal float32s from here on
  const uint32_t fm = f & 255u, fr = f >> 8;
  const float scale = bits_to_float((max(fm, kLeastField) - 8u) << 23);
  float m[16];
  uint32_t mm = 0, some = 0;
  pair most = 0, least = (uint16_t)0xffffu;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(wm[w], scale, false);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(wm[w], scale, true);
    m[4 * w] = a[0];
    m[4 * w + 1] = a[1];
    m[4 * w + 2] = b[0];
    m[4 * w + 3] = b[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) mm = max(mm, float_to_bits(m[4 * w + j]) & 0x7fffffffu);
    some |= wm[w];
    const pair even = __builtin_bit_cast(pair, wr[w] & 0x00ff00ffu), odd = __builtin_bit_cast(pair, (wr[w] >> 8) & 0x00ff00ffu);
    most = __builtin_elementwise_max(__builtin_elementwise_max(most, even), odd);
    // zero becomes the largest
    least = __builtin_elementwise_min(__builtin_elementwise_min(least, (pair)(even - (uint16_t)1)), (pair)(odd - (uint16_t)1));
  }
  const uint32_t top = max((uint32_t)most[0], (uint32_t)most[1]), low = min((uint32_t)least[0], (uint32_t)least[1]);
  uint32_t key = top ? (fr * 16 + top) * 2 + (top >= 16 ? 1u : 0u) : 0u;
  bool fine = mm < 0x7e800000u && top != 255u && (fm >= kLeastField || (some & 0x7f7f7f7fu) == 0);
  row_max2_u32(mm, key);
  const uint32_t to = moment_field<3>(mm);
  fields = to;
  vec4u roots = wr;
  fine &= shift_roots(roots, fr, key, low, fields) && (mm == 0 || to >= kLeastField);
  if (__ballot(!fine)) {
    remake(wm, wr, f, fields);
    return;
  }
  wr = roots;
  const float down = bits_to_float((max(to, kLeastField) - 8u) << 23);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    s16x2 c{};
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, m[4 * w], m[4 * w + 1], down, false);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, m[4 * w + 2], m[4 * w + 3], down, true);
    wm[w] = __builtin_bit_cast(uint32_t, c);
  }
}

// kEvenAhead blocks of a tensor with rows of a multiple of sixteen elements by sixteen lanes (those with `make`; the
// others may be none of the tensor's): sixteen elements a lane, which are of one row and of one block.
template <bool kWide>
__device__ inline void make_even(const MomentArgs& A, const MomentRecord& t, const uint32_t (&block)[kEvenAhead],
                                 const bool (&make)[kEvenAhead]) {
  const int lane = threadIdx.x & 15;
  const uint32_t len = t.row_len;
  int32_t row[kEvenAhead], s[kEvenAhead];
  uint32_t off[kEvenAhead];
  bool in[kEvenAhead];
#pragma unroll
  for (int g = 0; g < kEvenAhead; ++g) {
    const int64_t base = (int64_t)block[g] * kMomBlock;
    uint32_t at0;
    const uint64_t row0 = first_row(t, base, at0);
    const uint32_t e = at0 + lane * 16, q = row_of(t, e);
    row[g] = (int32_t)(row0 + q);
    off[g] = e - q * len;
    in[g] = make[g] && base + lane * 16 < t.count;
  }
  sources<kWide>(A, row, in, s);
  vec4u wm[kEvenAhead], wr[kEvenAhead];
  uint32_t f[kEvenAhead];
#pragma unroll
  for (int g = 0; g < kEvenAhead; ++g) {
    wm[g] = wr[g] = vec4u{};
    f[g] = 0;
    if (s[g] < 0) continue;
    const uint64_t at = (uint64_t)t.src_at * kMomBlock + (uint64_t)s[g] * len + off[g];
    wm[g] = *reinterpret_cast<const vec4u*>(A.m8 + at);
    wr[g] = *reinterpret_cast<const vec4u*>(A.r8 + at);
    f[g] = *(const uint16_t*)(A.fields + 2 * (at >> 8));
  }
#pragma unroll
  for (int g = 0; g < kEvenAhead; ++g) {
    uint32_t fields;
    recode(wm[g], wr[g], f[g], fields);
    if (!make[g]) continue;
    const uint64_t to = ((uint64_t)t.dst_at + block[g]) * kMomBlock + lane * 16;
    *reinterpret_cast<vec4u*>(A.to_m8 + to) = wm[g];
    *reinterpret_cast<vec4u*>(A.to_r8 + to) = wr[g];
    if (lane == 0) *(uint16_t*)(A.to_fields + 2 * (to >> 8)) = (uint16_t)fields;
  }
}

// Four bytes from `at` on, of which those that lie in the array are right.
__device__ inline uint32_t four_at(const uint8_t* p, uint64_t at, uint64_t size) {
  typedef uint32_t any4 __attribute__((aligned(1)));
  const uint64_t from = at < size - 4 ? at : size - 4;
  return *reinterpret_cast<const any4*>(p + from) >> (8 * (uint32_t)(at - from));
}

// Four blocks (the same for the wave, none beyond `some`) of a tensor with other rows, four elements of each a lane.
// kOf rows they can be of: 1 with rows of a multiple of four elements, 2 with rows of three and more, 4.
template <bool kWide, int kOf>
__device__ inline void make_odd(const MomentArgs& A, const MomentRecord& t, const uint32_t (&block)[kMomentAhead], int some) {
  constexpr int kN = kMomentAhead * kOf;
  const uint32_t len = t.row_len, l = (threadIdx.x & 63) * 4;
  int32_t row[kN], s[kN];
  uint32_t off[kN];  // of the first element that is of the row
  bool in[kN];
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) {
    const int64_t base = (int64_t)block[g] * kMomBlock;
    uint32_t at0;
    const uint64_t row0 = first_row(t, base, at0);
    if (kOf == 4) {
#pragma unroll
      for (int j = 0; j < kOf; ++j) {
        const uint32_t e = at0 + l + j, q = row_of(t, e);
        row[g * kOf + j] = (int32_t)(row0 + q);
        off[g * kOf + j] = e - q * len;
        in[g * kOf + j] = g < some && base + l + j < t.count;
      }
    } else {
      const uint32_t e = at0 + l, q = row_of(t, e);
      row[g * kOf] = (int32_t)(row0 + q);
      off[g * kOf] = e - q * len;
      in[g * kOf] = g < some && base + l < t.count;
      if (kOf == 2) {
        const uint32_t here = len - off[g * kOf];  // elements of the first row from this lane's on
        row[g * kOf + 1] = row[g * kOf] + 1;
        off[g * kOf + 1] = 0;
        in[g * kOf + 1] = g < some && here < 4 && base + l + here < t.count;
      }
    }
  }
  sources<kWide>(A, row, in, s);
  const uint64_t from = (uint64_t)t.src_at * kMomBlock, size = (uint64_t)A.state_size;
  uint32_t wm[kMomentAhead], wr[kMomentAhead], f[kMomentAhead][4];
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) {
    wm[g] = wr[g] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[g][j] = 0;
    if (g >= some || A.rows == 0) continue;
    if (kOf == 4) {
      uint32_t cm[4], cr[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = g * kOf + j;
        // a row that comes from nowhere reads the first, and is none
        const uint64_t at = from + (s[k] >= 0 ? (uint64_t)s[k] * len + off[k] : 0u);
        cm[j] = A.m8[at];
        cr[j] = A.r8[at];
        f[g][j] = *(const uint16_t*)(A.fields + 2 * (at >> 8));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        wm[g] |= s[g * kOf + j] >= 0 ? cm[j] << (8 * j) : 0u;
        wr[g] |= s[g * kOf + j] >= 0 ? cr[j] << (8 * j) : 0u;
      }
    } else if (kOf == 2) {
      const int k = g * kOf;
      const uint64_t a = from + (s[k] >= 0 ? (uint64_t)s[k] * len + off[k] : 0u);
      const uint64_t b = from + (s[k + 1] >= 0 ? (uint64_t)s[k + 1] * len : 0u);
      const uint32_t here = len - off[k] < 4 ? len - off[k] : 4;
      const uint32_t am = four_at(A.m8, a, size), ar = four_at(A.r8, a, size);
      const uint32_t bm = four_at(A.m8, b, size), br = four_at(A.r8, b, size);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t at = (uint32_t)j < here ? a + j : b + (j - here);
        f[g][j] = *(const uint16_t*)(A.fields + 2 * ((at < size ? at : 0u) >> 8));
      }
      const uint32_t mask = here < 4 ? (1u << (8 * here)) - 1u : ~0u;
      wm[g] = (s[k] >= 0 ? am & mask : 0u) | (s[k + 1] >= 0 && here < 4 ? bm << (8 * (here & 3)) : 0u);
      wr[g] = (s[k] >= 0 ? ar & mask : 0u) | (s[k + 1] >= 0 && here < 4 ? br << (8 * (here & 3)) : 0u);
    } else if (s[g] >= 0) {
      const uint64_t at = from + (uint64_t)s[g] * len + off[g];
      wm[g] = *reinterpret_cast<const uint32_t*>(A.m8 + at);
      wr[g] = *reinterpret_cast<const uint32_t*>(A.r8 + at);
      f[g][0] = f[g][1] = f[g][2] = f[g][3] = *(const uint16_t*)(A.fields + 2 * (at >> 8));
    }
  }
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) {
    if (g >= some) continue;
    int fm[4], fr[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      fm[j] = (int)(f[g][j] & 255u);
      fr[j] = (int)(f[g][j] >> 8);
    }
    float m[4], r[4];
    decode_m4(wm[g], fm, m);
    decode_r4(wr[g], fr, r);
    const uint32_t none[4] = {0, 0, 0, 0};
    uint32_t cm, cr, fields;
    encode_block<false>(m, r, none, cm, cr, fields);
    const uint64_t to = ((uint64_t)t.dst_at + block[g]) * kMomBlock + l;
    *reinterpret_cast<uint32_t*>(A.to_m8 + to) = cm;
    *reinterpret_cast<uint32_t*>(A.to_r8 + to) = cr;
    if (l == 0) *(uint16_t*)(A.to_fields + 2 * (to >> 8)) = (uint16_t)fields;
  }
}

template <bool kWide>
__device__ inline void take_odd(const MomentArgs& A, const MomentRecord& t, uint32_t group) {
  const uint32_t first = __builtin_amdgcn_readfirstlane(group * kOddGroup + (threadIdx.x >> 6) * kMomentAhead);
  if (first >= t.blocks) return;
  uint32_t block[kMomentAhead];
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) block[g] = first + g;
  const int some = (int)min(t.blocks - first, (uint32_t)kMomentAhead);
  if (t.row_len % 4 == 0) make_odd<kWide, 1>(A, t, block, some);
  else if (t.row_len >= 3) make_odd<kWide, 2>(A, t, block, some);
  else make_odd<kWide, 4>(A, t, block, some);
}

// Where there are rows of a multiple of sixteen elements, which want registers (of 48: 65 us at five waves a SIMD, 133 at
// eight), all tensors go together, at five waves; where there are none at seven (1.4M of 2M rows of 45: 106 us by an int32
// index, 107 by an int64 one; the same at eight waves, which keep two or seven registers in scratch; 115 on another card,
// on which rows of 16 beside them take 137 together and 21 alone).
template <bool kWide>
__global__ __launch_bounds__(256) void moment_take_kernel(MomentArgs A) {
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const MomentRecord& t = A.t[k];
  if (t.row_len % 16) {
    take_odd<kWide>(A, t, b - A.begin[k]);
    return;
  }
  uint32_t block[kEvenAhead];
  bool make[kEvenAhead];
#pragma unroll
  for (int g = 0; g < kEvenAhead; ++g) {
    block[g] = (b - A.begin[k]) * kEvenGroup + g * 16 + (threadIdx.x >> 4);
    make[g] = block[g] < t.blocks;
  }
  make_even<kWide>(A, t, block, make);
}

template <bool kWide>
__global__ __launch_bounds__(256, 7) void moment_take_odd_kernel(MomentArgs A) {
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  take_odd<kWide>(A, A.t[k], b - A.begin[k]);
}

// ---- moves --------------------------------------------------------------------------------------------

// What changed rows get is laid out as the tensor: with rows of a multiple of sixteen elements the codes of both arrays and
// two exponents for each sixteen elements, with others a word an element, m | r << 8 | exponents << 16.
struct MoveRecord {
  int64_t count;
  uint64_t magic;    // row_magic
  uint8_t* stage;
  int64_t plane;     // bytes from the one array's codes to the other's, and on to the exponents; 0: a word an element
  uint32_t at;       // blocks
  uint32_t row_len;
  uint32_t blocks;
  uint32_t pieces;   // of a row: sixteen elements, or four
  uint32_t piece;    // the first among those of all tensors
  uint32_t by_pieces;  // floor(2^32 / pieces) + 1, 0 for one
};

constexpr int kMoveTensors = 60;     // per launch: the argument block stays below 4 KiB
constexpr int kMovePieces = 512;     // of a row in all tensors, up to which they are dealt out together
constexpr int kWidePieces = 256;     // of longer rows, per workgroup
constexpr int kMoveRows = 256;       // per workgroup at most

struct MoveArgs {
  MoveRecord t[kMoveTensors];
  uint32_t begin[kMoveTensors];  // first workgroup of each tensor in the second launch
  uint8_t *m8, *r8, *fields;
  uint32_t* bits;     // rows that change
  int64_t state_size;
  const void* index;
  uint32_t rows;
  int32_t n;
  uint32_t groups;
  int32_t tile;       // rows per workgroup of the first launch, a multiple of 64
  uint32_t pieces;    // of a row in all tensors, 0 where they are too many to be dealt out together
};
static_assert(sizeof(MoveArgs) <= 4096, "kernel arguments");

// Piece c of what `row` gets from row s (nothing for s < 0).
__device__ inline void gather_piece(const MoveArgs& A, const MoveRecord& t, int64_t row, int32_t s, uint32_t c) {
  const uint32_t len = t.row_len;
  const uint64_t from = (uint64_t)t.at * kMomBlock;
  if (t.plane) {
    const uint64_t to = (uint64_t)row * len + c * 16;
    vec4u wm{}, wr{};
    uint16_t f = 0;
    if (s >= 0) {
      const uint64_t at = from + (uint64_t)s * len + c * 16;
      wm = *reinterpret_cast<const vec4u*>(A.m8 + at);
      wr = *reinterpret_cast<const vec4u*>(A.r8 + at);
      f = *(const uint16_t*)(A.fields + 2 * (at >> 8));
    }
    *reinterpret_cast<vec4u*>(t.stage + to) = wm;
    *reinterpret_cast<vec4u*>(t.stage + t.plane + to) = wr;
    *(uint16_t*)(t.stage + 2 * t.plane + (to >> 4) * 2) = f;
    return;
  }
  typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(4)));
  const uint32_t here = min(len - c * 4, 4u);
  uint32_t* to = reinterpret_cast<uint32_t*>(t.stage) + (uint64_t)row * len + c * 4;
  uint32_t w[4] = {0, 0, 0, 0};
  if (s >= 0) {
    const uint64_t at = from + (uint64_t)s * len + c * 4, size = (uint64_t)A.state_size;
    const uint32_t wm = four_at(A.m8, at, size), wr = four_at(A.r8, at, size);
    // the elements lie in one block or in two
    const uint32_t f0 = *(const uint16_t*)(A.fields + 2 * (at >> 8)), f1 = *(const uint16_t*)(A.fields + 2 * ((at + here - 1) >> 8));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = ((wm >> (8 * j)) & 255u) | ((wr >> (8 * j)) & 255u) << 8 | (((at + j) >> 8) == (at >> 8) ? f0 : f1) << 16;
  }
  if (here == 4) {
    *reinterpret_cast<any16*>(to) = any16{w[0], w[1], w[2], w[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if ((uint32_t)j < here) to[j] = w[j];
  }
}

// The first launch: a workgroup looks at up to 256 rows, marks those that change and gathers what they get.
template <bool kWide>
__global__ __launch_bounds__(256) void moment_gather_kernel(MoveArgs A) {
  __shared__ int32_t to[kMoveRows], of[kMoveRows];
  __shared__ int32_t moved;
  __shared__ uint8_t tensor[kMovePieces];
  __shared__ MoveRecord rec[kMoveTensors];
  if (threadIdx.x == 0) moved = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int64_t base = (int64_t)blockIdx.x * A.tile, i = base + threadIdx.x;
  const bool in = (int)threadIdx.x < A.tile && i < (int64_t)A.rows;
  bool change = false;
  int32_t s = -1;
  if (in) {
    s = entry<kWide>(A, i);
    // a row stays whose source does not, or is none
    change = s == -1 || (s >= 0 && s != i && entry<kWide>(A, s) == s);
  }
  const uint64_t move = __ballot(change);
  if (lane == 0 && in && blockIdx.y == 0 && blockIdx.z == 0) {
    A.bits[i >> 5] = (uint32_t)move;
    A.bits[(i >> 5) + 1] = (uint32_t)(move >> 32);
  }
  int32_t at = 0;
  if (lane == 0 && move) at = atomicAdd(&moved, __popcll(move));
  at = __builtin_amdgcn_readfirstlane(at);
  if (change) {
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(move >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)move, 0));
    to[at + below] = threadIdx.x;
    of[at + below] = s;
  }
  __syncthreads();
  const uint32_t m = moved;
  if (m == 0) return;
  if (A.pieces == 0) {  // long rows: kWidePieces of one tensor's
    const MoveRecord& t = A.t[blockIdx.y];
    const uint32_t first = blockIdx.z * kWidePieces;
    if (first >= t.pieces) return;
    const uint32_t pieces = min(t.pieces - first, (uint32_t)kWidePieces), by = pieces > 1 ? 0xffffffffu / pieces + 1 : 0;
    for (uint32_t e = threadIdx.x; e < m * pieces; e += 256) {
      const uint32_t q = by ? __umulhi(e, by) : e;
      gather_piece(A, t, base + to[q], of[q], first + e - q * pieces);
    }
    return;
  }
  // the records and every piece's tensor at hand
  for (int j = threadIdx.x; j < A.n * (int)(sizeof(MoveRecord) / 8); j += 256)
    reinterpret_cast<uint64_t*>(rec)[j] = reinterpret_cast<const uint64_t*>(A.t)[j];
  for (int k = threadIdx.x >> 6; k < A.n; k += 4)
    for (uint32_t c = lane; c < A.t[k].pieces; c += 64) tensor[A.t[k].piece + c] = (uint8_t)k;
  __syncthreads();
  const uint32_t by_m = m > 1 ? 0xffffffffu / m + 1 : 0;
  for (uint32_t e = threadIdx.x; e < m * A.pieces; e += 256) {
    // tensor after tensor, row after row
    const MoveRecord& t = rec[tensor[by_m ? __umulhi(e, by_m) : e]];
    const uint32_t r = e - m * t.piece, q = t.by_pieces ? __umulhi(r, t.by_pieces) : r;
    gather_piece(A, t, base + to[q], of[q], r - q * t.pieces);
  }
}

__device__ inline bool changes(const MoveArgs& A, uint32_t row) { return A.bits[row >> 5] >> (row & 31u) & 1u; }

// Whether a row with elements in a block changes, from every kStep-th of their words, this lane's from `from` on.
template <int kStep>
__device__ inline bool block_changes(const MoveArgs& A, const MoveRecord& t, uint32_t block, uint32_t from) {
  const int64_t base = (int64_t)block * kMomBlock;
  if (base >= t.count) return false;
  uint32_t at0, at1;
  const uint32_t row0 = (uint32_t)first_row(t, base, at0);
  const uint32_t row1 = (uint32_t)first_row(t, min(base + kMomBlock, t.count) - 1, at1);
  uint32_t any = 0;
  for (uint32_t w = (row0 >> 5) + from; w <= row1 >> 5; w += kStep) {
    uint32_t x = A.bits[w];
    if (w == row0 >> 5) x &= ~0u << (row0 & 31u);
    if (w == row1 >> 5) x &= ~0u >> (31u - (row1 & 31u));
    any |= x;
  }
  return any != 0;
}

// The second launch: blocks with a changed row, in place; 64 a workgroup are looked over.
__device__ inline void remake_even(const MoveArgs& A, const MoveRecord& t, uint32_t first, uint8_t* list) {
  const int lane = threadIdx.x & 15, block = threadIdx.x & 63;
  const uint64_t bits = __ballot(block_changes<1>(A, t, first + block, 0));  // the same in every wave
  if (bits == 0) return;
  if (threadIdx.x < kRemakeGroup && (bits >> block & 1u))
    list[__popcll(bits & (((uint64_t)1 << block) - 1u))] = (uint8_t)block;
  __syncthreads();
  const int n = __popcll(bits);
  for (int i = threadIdx.x >> 4; (i & ~3) < n; i += 16 * kEvenAhead) {
    vec4u wm[kEvenAhead], wr[kEvenAhead];
    uint32_t f[kEvenAhead];
    uint64_t at[kEvenAhead];
#pragma unroll
    for (int g = 0; g < kEvenAhead; ++g) {
      wm[g] = wr[g] = vec4u{};
      f[g] = 0;
      if (i + 16 * g >= n) continue;
      const int64_t base = (int64_t)(first + list[i + 16 * g]) * kMomBlock;
      uint32_t at0;
      const uint32_t row = (uint32_t)first_row(t, base, at0) + row_of(t, at0 + lane * 16);
      at[g] = (uint64_t)t.at * kMomBlock + base + lane * 16;
      const uint8_t *m = A.m8 + at[g], *r = A.r8 + at[g], *e = A.fields + 2 * (at[g] >> 8);
      if (base + lane * 16 < t.count && changes(A, row)) {
        m = t.stage + base + lane * 16;
        r = m + t.plane;
        e = t.stage + 2 * t.plane + ((base >> 4) + lane) * 2;
      }
      wm[g] = *reinterpret_cast<const vec4u*>(m);
      wr[g] = *reinterpret_cast<const vec4u*>(r);
      f[g] = *(const uint16_t*)e;
    }
#pragma unroll
    for (int g = 0; g < kEvenAhead; ++g) {
      uint32_t fields;
      recode(wm[g], wr[g], f[g], fields);
      if (i + 16 * g >= n) continue;
      *reinterpret_cast<vec4u*>(A.m8 + at[g]) = wm[g];
      *reinterpret_cast<vec4u*>(A.r8 + at[g]) = wr[g];
      if (lane == 0) *(uint16_t*)(A.fields + 2 * (at[g] >> 8)) = (uint16_t)fields;
    }
  }
}

// Four blocks a wave are looked over, sixteen lanes each; those that change are made kOddAhead at a time.
__device__ inline void remake_odd(const MoveArgs& A, const MoveRecord& t, uint32_t first) {
  const uint32_t lane = threadIdx.x & 63, l = lane * 4;
  const uint32_t* stage = reinterpret_cast<const uint32_t*>(t.stage);
  constexpr int kLanes = 16;  // a block
  uint64_t left = __ballot(block_changes<kLanes>(A, t, first + lane / kLanes, lane % kLanes));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) left |= left >> o;
  left &= 0x0001000100010001u;
  while (left) {
    int some = 0;
    uint32_t block[kOddAhead];
#pragma unroll
    for (int g = 0; g < kOddAhead; ++g) {
      block[g] = first;
      if (left == 0) continue;
      block[g] = first + __builtin_ctzll(left) / kLanes;
      left &= left - 1;
      some = g + 1;
    }
    uint32_t wm[kOddAhead], wr[kOddAhead], f[kOddAhead], change[kOddAhead];
    vec4u got[kOddAhead];
#pragma unroll
    for (int g = 0; g < kOddAhead; ++g) {
      change[g] = 0;
      if (g >= some) continue;
      const int64_t base = (int64_t)block[g] * kMomBlock;
      const uint64_t at = (uint64_t)t.at * kMomBlock + base + l;
      wm[g] = *reinterpret_cast<const uint32_t*>(A.m8 + at);
      wr[g] = *reinterpret_cast<const uint32_t*>(A.r8 + at);
      f[g] = *(const uint16_t*)(A.fields + 2 * (at >> 8));
      // the rows of four elements are four at most: their bits lie in two words
      uint32_t at0;
      const uint32_t row0 = (uint32_t)first_row(t, base, at0), q = row_of(t, at0 + l), off = at0 + l - q * t.row_len;
      uint32_t row[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        row[j] = row0 + q + (t.row_len >= 3 ? (off + j >= t.row_len ? 1u : 0u) : (off + j) >> (t.row_len - 1));
      const int64_t here = t.count - base - l;  // elements from the lane's first on
      if (here <= 0) continue;
      const uint32_t last = here >= 4 ? row[3] : here == 3 ? row[2] : here == 2 ? row[1] : row[0];
      const uint32_t w0 = A.bits[row[0] >> 5], w1 = A.bits[last >> 5];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < here && (row[j] >> 5 == row[0] >> 5 ? w0 : w1) >> (row[j] & 31u) & 1u) change[g] |= 1u << j;
      if (change[g]) got[g] = *reinterpret_cast<const vec4u*>(stage + base + l);
    }
#pragma unroll
    for (int g = 0; g < kOddAhead; ++g) {
      if (g >= some) continue;
      const uint64_t at = ((uint64_t)t.at + block[g]) * kMomBlock + l;
      int fm[4], fr[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t e = f[g];
        if (change[g] >> j & 1u) {
          const uint32_t w = got[g][j], keep = ~(255u << (8 * j));
          wm[g] = (wm[g] & keep) | (w & 255u) << (8 * j);
          wr[g] = (wr[g] & keep) | (w >> 8 & 255u) << (8 * j);
          e = w >> 16;
        }
        fm[j] = (int)(e & 255u);
        fr[j] = (int)(e >> 8);
      }
      float m[4], r[4];
      decode_m4(wm[g], fm, m);
      decode_r4(wr[g], fr, r);
      const uint32_t none[4] = {0, 0, 0, 0};
      uint32_t cm, cr, fields;
      encode_block<false>(m, r, none, cm, cr, fields);
      *reinterpret_cast<uint32_t*>(A.m8 + at) = cm;
      *reinterpret_cast<uint32_t*>(A.r8 + at) = cr;
      if (l == 0) *(uint16_t*)(A.fields + 2 * (at >> 8)) = (uint16_t)fields;
    }
  }
}

__global__ __launch_bounds__(256) void moment_remake_even_kernel(MoveArgs A) {
  __shared__ uint8_t list[kRemakeGroup];
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  remake_even(A, A.t[k], (b - A.begin[k]) * kRemakeGroup, list);
}

__global__ __launch_bounds__(256, 8) void moment_remake_odd_kernel(MoveArgs A) {
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  remake_odd(A, A.t[k], __builtin_amdgcn_readfirstlane((b - A.begin[k]) * kOddGroup + (threadIdx.x >> 6) * 4));
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

int64_t padded(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }

// A move's workspace: the bits of the rows, and of each tensor what changed rows get.
int64_t bits_bytes(int64_t rows) { return padded((rows + 63) / 64 * 8); }
int64_t stage_bytes(int64_t row_len, int64_t rows) {
  const int64_t elements = row_len * rows;
  return row_len % 16 ? padded(elements * 4) : 2 * padded(elements) + padded(elements / 8);
}

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
  A.state_size = state_size;
  A.to_m8 = out_mu8;
  A.to_r8 = out_nu8;
  A.to_fields = out_fields;
  A.index = index;
  A.rows = (uint32_t)rows;
  bool even = false;
  for (int i = 0; i < num; ++i) even |= row_lens[i] > 0 && row_lens[i] % 16 == 0;
  auto* kernel = even ? (index_bits == 64 ? moment_take_kernel<true> : moment_take_kernel<false>)
                      : (index_bits == 64 ? moment_take_odd_kernel<true> : moment_take_odd_kernel<false>);
  for (int i = 0; i < num;) {
    int64_t groups = 0;
    A.n = 0;
    for (; i < num && A.n < kMomentTensors; ++i) {
      const int64_t elements = row_lens[i] * count, blocks = (elements + kMomBlock - 1) / kMomBlock;
      if (blocks == 0) continue;
      const int64_t per = row_lens[i] % 16 ? kOddGroup : kEvenGroup, more = (blocks + per - 1) / per;
      GS_REQUIRE(more <= kMaxGroups, "%s: tensor %d is too large", what, i);
      if (groups + more > kMaxGroups) break;
      MomentRecord& t = A.t[A.n];
      t.count = elements;
      t.row_len = (uint32_t)row_lens[i];
      t.magic = row_magic(row_lens[i]);
      t.src_at = (uint32_t)(offsets[i] / kMomBlock);
      t.dst_at = (uint32_t)(out_offsets[i] / kMomBlock);
      t.blocks = (uint32_t)blocks;
      A.begin[A.n++] = (uint32_t)groups;
      groups += more;
    }
    if (A.n == 0) continue;
    A.groups = (uint32_t)groups;
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, A);
    GS_LAUNCH_CHECK("moment_take_kernel");
  }
  return GS_OK;
}

extern "C" size_t gs_moments_move_workspace_size(int num, const int64_t* row_lens, int64_t rows) {
  if (num < 0 || (num > 0 && !row_lens) || rows < 0 || rows >= ((int64_t)1 << 31)) return 0;
  int64_t bytes = bits_bytes(rows);
  for (int i = 0; i < num; ++i) {
    if (row_lens[i] < 0 || row_lens[i] >= kMaxRowLen) return 0;
    bytes += stage_bytes(row_lens[i], rows);
  }
  return (size_t)bytes;
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
  const int rc = check_side(what, num, row_lens, rows, offsets, state_size);
  if (rc != GS_OK) return rc;
  const size_t need = gs_moments_move_workspace_size(num, row_lens, rows);
  GS_REQUIRE(workspace_bytes >= need, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
  if (rows == 0 || state_size == 0) return GS_OK;
  uint8_t* const ws = (uint8_t*)workspace;
  MoveArgs A{};
  A.m8 = mu8;
  A.r8 = nu8;
  A.fields = fields;
  A.bits = (uint32_t*)ws;
  A.state_size = state_size;
  A.index = index;
  A.rows = (uint32_t)rows;
  // everything is gathered before anything is made anew
  enum { kGather, kEven, kOdd };
  for (const int pass : {kGather, kEven, kOdd}) {
    uint8_t* stage = ws + bits_bytes(rows);
    const int64_t per = pass == kEven ? kRemakeGroup : kOddGroup;
    for (int i = 0; i < num;) {
      int64_t groups = 0, pieces = 0, most = 0;
      A.n = 0;
      for (; i < num && A.n < kMoveTensors; ++i) {
        const int64_t elements = row_lens[i] * rows, blocks = (elements + kMomBlock - 1) / kMomBlock;
        const int64_t more = (blocks + per - 1) / per;
        const bool even = row_lens[i] % 16 == 0;
        if (pass == kGather || even == (pass == kEven)) {
          GS_REQUIRE(more <= kMaxGroups, "%s: tensor %d is too large", what, i);
          if (pass != kGather && groups + more > kMaxGroups) break;
          if (blocks) {
            MoveRecord& t = A.t[A.n];
            t.count = elements;
            t.magic = row_magic(row_lens[i]);
            t.stage = stage;
            t.plane = even ? padded(elements) : 0;
            t.at = (uint32_t)(offsets[i] / kMomBlock);
            t.row_len = (uint32_t)row_lens[i];
            t.blocks = (uint32_t)blocks;
            t.pieces = (uint32_t)(even ? row_lens[i] / 16 : (row_lens[i] + 3) / 4);
            t.piece = (uint32_t)pieces;
            t.by_pieces = t.pieces > 1 ? (uint32_t)((((uint64_t)1 << 32) / t.pieces) + 1) : 0;
            pieces += t.pieces;
            most = std::max<int64_t>(most, t.pieces);
            A.begin[A.n++] = (uint32_t)groups;
            groups += more;
          }
        }
        stage += stage_bytes(row_lens[i], rows);
      }
      if (A.n == 0) continue;
      A.groups = (uint32_t)groups;
      dim3 grid((unsigned)groups);
      if (pass == kGather) {
        A.pieces = pieces <= kMovePieces ? (uint32_t)pieces : 0;
        // few rows a workgroup where there are few workgroups, as the rows that change may lie together (2M Gaussians, 8 % of
        // them at random: 188 us by 64, 167 by 128, 158 by 256)
        A.tile = !A.pieces || rows <= ((int64_t)1 << 18) ? 64 : rows <= ((int64_t)1 << 19) ? 128 : kMoveRows;
        while (div_up(rows, A.tile) > kMaxGroups) A.tile *= 2;
        grid = dim3((unsigned)div_up(rows, A.tile), A.pieces ? 1u : (unsigned)A.n,
                    A.pieces ? 1u : (unsigned)div_up(most, kWidePieces));
        GS_REQUIRE(grid.z < 65536, "%s: rows are too long", what);
      }
      auto* kernel = pass == kEven  ? moment_remake_even_kernel
                     : pass == kOdd ? moment_remake_odd_kernel
                     : index_bits == 64 ? moment_gather_kernel<true> : moment_gather_kernel<false>;
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, A);
      GS_LAUNCH_CHECK("moment_move_kernel");
    }
  }
  return GS_OK;
}
