// Rows of moments in 8 bits by one index, on gfx950: taken into a new state, or moved in place.
//
// A tensor's moments are rows of row_len elements one after another, in blocks of 256 that share an
// exponent (gs_moments.h); a row's new neighbours are others than its old ones, so a block is decoded element by element from where
// its rows come from and encoded again, to nearest even.  Values come back as they were but where a
// larger neighbour raises the exponent of their block.
//
// Sixteen lanes make two blocks where rows are a multiple of sixteen elements, else a wave four, four elements of each a
// lane, with all loads under way before the first is encoded.  In a move a workgroup first finds which of its 64 blocks
// hold a changed row, and makes those; they go to a copy first, for a block is read by others while it changes.
//
// 70 % of 2M rows of 48 elements taken: 63 us, bound by memory (at 5.4 TB/s with the lines of rows that are skipped); of the
// Gaussians' five tensors 92, where the 11 of 59 elements in short rows take 30: their fields and codes come element by
// element.  2M Gaussians moved, 8 % at random: 182 us, 8 % at the end 60, none 26.
#include "gs_moments.h"
#include "gs_pieces.h"
#include "gs_rows.h"

#include <algorithm>

namespace gs {
namespace {

constexpr int kMomentTensors = 72;  // per launch: the argument block stays below 4 KiB
constexpr int kMomentAhead = 4;     // blocks per wave
constexpr int kTakeGroup = 4 * kMomentAhead;  // per workgroup
constexpr int kEvenAhead = 2;       // blocks of sixteen lanes (1.5M rows of 48 taken: 63 us, one 70, four 68)
constexpr int kMoveGroup = 64;      // in a move; 16 with rows of fewer elements than 16, of which they hold as many rows

struct MomentRecord {
  int64_t count;     // elements behind which there is nothing
  uint64_t magic;    // row_magic
  uint32_t src_at, dst_at;  // blocks
  uint32_t row_len;
  uint32_t blocks;
  uint32_t group;    // blocks per workgroup
};

struct MomentArgs {
  MomentRecord t[kMomentTensors];
  uint32_t begin[kMomentTensors];
  const uint8_t *m8, *r8, *fields;
  uint8_t *to_m8, *to_r8, *to_fields;
  uint64_t* changed;  // per workgroup of a move: its blocks, bit by bit
  int64_t state_size;
  const void* index;
  uint32_t rows;     // of the tensors that are read
  int32_t n;
  uint32_t groups;
  int32_t wide;
};
static_assert(sizeof(MomentArgs) <= 4096, "kernel arguments");

// Entry i of the index: a row, -1 for a negative one, -2 for one beyond the rows.
template <bool kWide>
__device__ inline int32_t entry(const MomentArgs& A, int64_t i) {
  if constexpr (kWide) {
    const int64_t x = ((const int64_t*)A.index)[i];
    return x < 0 ? -1 : x < (int64_t)A.rows ? (int32_t)x : -2;
  } else {
    const int32_t x = ((const int32_t*)A.index)[i];
    return x < 0 ? -1 : (uint32_t)x < A.rows ? x : -2;
  }
}

// Where the rows come from, negative for nowhere, from their entries, all loads under way at once: in a move a row stays
// whose source does not.
template <bool kMove, bool kWide, int kN>
__device__ inline void sources(const MomentArgs& A, const int32_t (&row)[kN], const bool (&in)[kN], int32_t (&s)[kN]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) s[j] = entry<kWide>(A, in[j] ? row[j] : 0);
  if (kMove) {
    bool check = false;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      if (s[j] == -2) s[j] = row[j];
      check |= in[j] && s[j] >= 0 && s[j] != row[j];
    }
    if (__ballot(check)) {
      int32_t of[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) of[j] = entry<kWide>(A, s[j] >= 0 ? s[j] : 0);
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (s[j] >= 0 && of[j] != s[j]) s[j] = row[j];
    }
  }
#pragma unroll
  for (int j = 0; j < kN; ++j)
    if (!in[j]) s[j] = -1;
}

// The tensor of this workgroup: the last that begins at or before it.
__device__ inline int tensor_of(const MomentArgs& A, uint32_t b) {
  const int lane = threadIdx.x & 63;
  int k = -1;
  for (int at = 0; at < A.n; at += 64) k += __popcll(__ballot(at + lane < A.n && b >= A.begin[min(at + lane, A.n - 1)]));
  return __builtin_amdgcn_readfirstlane(k);
}

// A block's first row, and how far into it the block begins.
__device__ inline uint64_t first_row(const MomentRecord& t, int64_t base, uint32_t& at) {
  const uint64_t row = t.magic ? __umul64hi((uint64_t)base, t.magic) : (uint64_t)base;
  at = (uint32_t)((uint64_t)base - row * t.row_len);
  return row;
}
// The row of element e from a block's first row on, e less than row_len + 256.
__device__ inline uint32_t row_of(const MomentRecord& t, uint32_t e) {
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
// float32's least exponents or with roots under gradual underflow take the general way, with twice the instructions
// (2M rows moved, 8 % at random: 83 us, 98 where all went that way).
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
template <bool kMove, bool kWide>
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
  sources<kMove, kWide>(A, row, in, s);
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
template <bool kMove, bool kWide, int kOf>
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
  sources<kMove, kWide>(A, row, in, s);
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

template <bool kMove, bool kWide>
__device__ inline void make_four(const MomentArgs& A, const MomentRecord& t, const uint32_t (&block)[kMomentAhead], int some) {
  if (t.row_len % 4 == 0) make_odd<kMove, kWide, 1>(A, t, block, some);
  else if (t.row_len >= 3) make_odd<kMove, kWide, 2>(A, t, block, some);
  else make_odd<kMove, kWide, 4>(A, t, block, some);
}

template <bool kWide>
__global__ __launch_bounds__(256) void moment_take_kernel(MomentArgs A) {
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const MomentRecord& t = A.t[k];
  const uint32_t group = (b - A.begin[k]) * t.group;
  if (t.row_len % 16 == 0) {
    uint32_t block[kEvenAhead];
    bool make[kEvenAhead];
#pragma unroll
    for (int g = 0; g < kEvenAhead; ++g) {
      block[g] = group + g * 16 + (threadIdx.x >> 4);
      make[g] = block[g] < t.blocks;
    }
    make_even<false, kWide>(A, t, block, make);
    return;
  }
  const uint32_t first = __builtin_amdgcn_readfirstlane(group + (threadIdx.x >> 6) * kMomentAhead);
  if (first >= t.blocks) return;
  uint32_t block[kMomentAhead];
#pragma unroll
  for (int g = 0; g < kMomentAhead; ++g) block[g] = first + g;
  make_four<false, kWide>(A, t, block, (int)min(t.blocks - first, (uint32_t)kMomentAhead));
}

template <bool kWide>
__global__ __launch_bounds__(256) void moment_move_kernel(MomentArgs A) {
  __shared__ uint32_t changed[2];
  __shared__ uint8_t list[kMoveGroup];
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const int k = tensor_of(A, b);
  const MomentRecord& t = A.t[k];
  const uint32_t group = t.group, first = (b - A.begin[k]) * group, len = t.row_len;
  if (threadIdx.x < 2) changed[threadIdx.x] = 0;
  __syncthreads();
  // the rows with an element in these blocks, four of them under way at once
  const int64_t base = (int64_t)first * kMomBlock, end = min(base + group * kMomBlock, t.count);
  uint32_t at0, at1;
  const int64_t row0 = (int64_t)first_row(t, base, at0), row1 = (int64_t)first_row(t, end - 1, at1);
  uint32_t lo = 0, hi = 0;
  for (int64_t r = row0 + threadIdx.x; r <= row1; r += 256 * 4) {
    int32_t row[4], s[4];
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      row[j] = (int32_t)(r + 256 * j);
      in[j] = r + 256 * j <= row1;
    }
    sources<true, kWide>(A, row, in, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!in[j] || s[j] == row[j]) continue;
      const int64_t e = (int64_t)row[j] * len - base;
      const int from = e > 0 ? (int)(e / kMomBlock) : 0, to = (int)(min(e + len, end - base) - 1) / kMomBlock;
      const uint64_t bits = ((uint64_t)2 << to) - ((uint64_t)1 << from);
      lo |= (uint32_t)bits;
      hi |= (uint32_t)(bits >> 32);
    }
  }
  if (lo | hi) {  // once for each lane's part: lanes beside each other mostly have the same
    const uint32_t first_lo = __builtin_amdgcn_readfirstlane(lo), first_hi = __builtin_amdgcn_readfirstlane(hi);
    const bool other = lo != first_lo || hi != first_hi;
    if (other || (threadIdx.x & 63) == __builtin_ctzll(__ballot(!other))) {
      if (lo) atomicOr(&changed[0], lo);
      if (hi) atomicOr(&changed[1], hi);
    }
  }
  __syncthreads();
  const uint64_t bits = (uint64_t)changed[1] << 32 | changed[0];
  if (threadIdx.x == 0) A.changed[b] = bits;
  if (bits == 0) return;
  if (threadIdx.x < kMoveGroup && (bits >> threadIdx.x & 1u))
    list[__popcll(bits & (((uint64_t)1 << threadIdx.x) - 1u))] = (uint8_t)threadIdx.x;
  __syncthreads();
  const int n = __popcll(bits);
  if (len % 16 == 0) {
    for (int i = threadIdx.x >> 4; (i & ~3) < n; i += 16 * kEvenAhead) {
      uint32_t block[kEvenAhead];
      bool make[kEvenAhead];
#pragma unroll
      for (int g = 0; g < kEvenAhead; ++g) {
        make[g] = i + 16 * g < n;
        block[g] = first + list[min(i + 16 * g, n - 1)];
      }
      make_even<true, kWide>(A, t, block, make);
    }
    return;
  }
  for (int i = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kMomentAhead; i < n; i += 4 * kMomentAhead) {
    uint32_t block[kMomentAhead];
#pragma unroll
    for (int g = 0; g < kMomentAhead; ++g) block[g] = first + __builtin_amdgcn_readfirstlane(list[min(i + g, n - 1)]);
    make_four<true, kWide>(A, t, block, min(n - i, kMomentAhead));
  }
}

// The changed blocks from the copy into their places, 16 bytes a lane and array.
__global__ __launch_bounds__(256) void moment_back_kernel(MomentArgs A) {
  typedef uint32_t vec __attribute__((ext_vector_type(4)));
  const uint32_t b = blockIdx.x;
  if (b >= A.groups) return;
  const uint64_t bits = A.changed[b];
  if (bits == 0) return;
  const int k = tensor_of(A, b), lane = threadIdx.x & 15;
  const uint64_t first = (uint64_t)A.t[k].dst_at + (b - A.begin[k]) * A.t[k].group;
#pragma unroll
  for (int g = 0; g < kMoveGroup / 16; ++g) {
    const uint32_t block = g * 16 + (threadIdx.x >> 4);
    if (!(bits >> block & 1u)) continue;
    const uint64_t i = first + block, at = i * kMomBlock + lane * 16;
    *reinterpret_cast<vec*>(const_cast<uint8_t*>(A.m8) + at) = *reinterpret_cast<const vec*>(A.to_m8 + at);
    *reinterpret_cast<vec*>(const_cast<uint8_t*>(A.r8) + at) = *reinterpret_cast<const vec*>(A.to_r8 + at);
    if (lane == 0) *(uint16_t*)(const_cast<uint8_t*>(A.fields) + 2 * i) = *(const uint16_t*)(A.to_fields + 2 * i);
  }
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
  uint64_t* const changed = A.changed;
  int64_t done = 0;  // workgroups of the launches before
  for (int i = 0; i < num;) {
    int k = 0;
    int64_t groups = 0;
    for (; i < num && k < kMomentTensors; ++i) {
      const int64_t elements = row_lens[i] * count, blocks = (elements + kMomBlock - 1) / kMomBlock;
      if (blocks == 0) continue;
      const int64_t per = what != kTake ? (row_lens[i] < 16 ? 16 : kMoveGroup) : row_lens[i] % 16 ? kTakeGroup : 16 * kEvenAhead, more = (blocks + per - 1) / per;
      GS_REQUIRE(more <= kMaxGroups, "gs_moments: tensor %d is too large", i);
      if (groups + more > kMaxGroups) break;
      MomentRecord& t = A.t[k];
      t.count = elements;
      t.row_len = (uint32_t)row_lens[i];
      t.magic = row_magic(row_lens[i]);
      t.src_at = (uint32_t)(offsets[i] / kMomBlock);
      t.dst_at = (uint32_t)(out_offsets[i] / kMomBlock);
      t.blocks = (uint32_t)blocks;
      t.group = (uint32_t)per;
      A.begin[k++] = (uint32_t)groups;
      groups += more;
    }
    if (k == 0) continue;
    A.n = k;
    A.groups = (uint32_t)groups;
    A.changed = changed + done;
    done += groups;
    auto* kernel = what == kBack   ? moment_back_kernel
                   : what == kMove ? (A.wide ? moment_move_kernel<true> : moment_move_kernel<false>)
                                   : (A.wide ? moment_take_kernel<true> : moment_take_kernel<false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, stream, A);
    GS_LAUNCH_CHECK("moment_rows_kernel");
  }
  A.changed = changed;
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
  A.state_size = state_size;
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
  // codes, exponents, and which blocks changed: eight bytes for each workgroup, at most one a block
  return (size_t)state_size * 2 + padded(blocks * 2) + padded(blocks * 8);
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
  A.changed = (uint64_t*)(ws + 2 * state_size + padded(blocks * 2));
  A.state_size = state_size;
  A.index = index;
  A.rows = (uint32_t)rows;
  A.wide = index_bits == 64;
  const int done = launch(kMove, (hipStream_t)stream, num, row_lens, offsets, offsets, rows, A);
  if (done != GS_OK) return done;
  return launch(kBack, (hipStream_t)stream, num, row_lens, offsets, offsets, rows, A);
}
