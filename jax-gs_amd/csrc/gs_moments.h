// Optimizer moments in 8 bits, per block of 256 consecutive elements of a tensor.
//
//   m:  sign, 4 exponent bits, 3 mantissa bits          value = +-f(code) 2^e_m
//   r = sqrt(v):  4 exponent bits, 4 mantissa bits      value =   f(code) 2^e_r
//   f(E, M) = (1 + M / 2^k) 2^(E - 15) for E > 0 and (M / 2^k) 2^-14 for E = 0  (k = 3, 4)
//
// with e_m and e_r per block, kept as the float32 exponent field e + 127 (0..254) in two
// bytes.  The largest magnitude code stands for "not finite"; such values take no part in
// the choice of e, so that they do not spread to their neighbours.  e is the least
// exponent for which the block's largest finite value is at most the largest code,
// (2 - 2 / 2^k) 2^e.  A float's relative steps (1/16 and 1/32 at worst to nearest) reach
// 2^-14 below the block's largest value and its gradual underflow 2^-17 and 2^-18; the
// root of v is held because the update divides by it, and because it halves the exponent
// range that v needs.  A root that is not zero is never held as zero: the update divides
// by it, and the smallest code errs to the side of a short step.
//
// The arithmetic is exact: scaling by 2^(15 - field) moves a value's exponent field to the
// code's (float32's own gradual underflow lines up with the code's), after which the code
// is the top of the bits; rounding is an integer addition below them.  Decoded values are
// encoded to themselves by rounding to nearest.
#pragma once

#include "gs_common.h"

namespace gs {

constexpr int kMomBlock = GS_MOMENT_BLOCK;  // elements per block: one wave, four elements a lane

// Maxima of x and of y over the wave, in every lane (unsigned order is that of non-negative
// floats).  A lane without a source reads 0, so that each step is one instruction; the two
// chains fill each other's wait states.
__device__ inline void wave_max2_u32(uint32_t& x, uint32_t& y) {
#define GS_DPP_MAX(ctrl)                                                                          \
  {                                                                                               \
    const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true);    \
    const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)y, ctrl, 0xf, 0xf, true);    \
    x = x > a ? x : a;                                                                            \
    y = y > b ? y : b;                                                                            \
  }
  GS_DPP_MAX(0xB1);   // quad_perm [1, 0, 3, 2]
  GS_DPP_MAX(0x4E);   // quad_perm [2, 3, 0, 1]
  GS_DPP_MAX(0x141);  // row_half_mirror: eight lanes
  GS_DPP_MAX(0x140);  // row_mirror: sixteen lanes
  GS_DPP_MAX(0x142);  // row_bcast15: rows 1 and 3 hold pairs of rows
  GS_DPP_MAX(0x143);  // row_bcast31: row 3 holds all
#undef GS_DPP_MAX
  x = (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
  y = (uint32_t)__builtin_amdgcn_readlane((int)y, 63);
}

// Exponent field of a block whose largest finite magnitude has the given bits.
template <int kMant>
__device__ inline uint32_t moment_field(uint32_t most) {
  const uint32_t f = (most + (1u << (24 - kMant)) - 1u) >> 23;
  return f < 254u ? f : 254u;
}

// The code of a finite value x >= 0 in the top bits of the result (kMant 4: in the upper eight,
// 3: in the seven below the sign's): x scaled so that its code is the top of its bits, with what
// rounds it added: 16 random bits in bits 8..23 (kStochastic), or what rounds to nearest even.
// A root (kMant 4) above zero gets at least code 1, which lies in bit 24; the root of a float32
// that is not zero has larger bits than that.
template <int kMant, bool kStochastic>
__device__ inline uint32_t moment_top(float x, int field, uint32_t noise) {
  constexpr int drop = 23 - kMant, up = 24 - drop;  // the code's lowest bit goes to bit 24
  const uint32_t b = float_to_bits(ldexpf(x, 15 - field));
  uint32_t c;
  if (kStochastic) c = (b << up) + noise;
  else c = (b + (1u << (drop - 1)) - 1u + ((b >> drop) & 1u)) << up;
  if (kMant == 4) {
    const uint32_t least = min(float_to_bits(x), 1u << 24);
    c = max(c, least);
  }
  return c;
}
// Upper and lower half of 32 random bits, where moment_top takes them.
__device__ inline uint32_t noise_hi(uint32_t h) { return __builtin_amdgcn_perm(0, h, 0x0c03020cu); }
__device__ inline uint32_t noise_lo(uint32_t h) { return __builtin_amdgcn_perm(0, h, 0x0c01000cu); }

// Four decoded values of the packed codes w of one lane; fields as stored, one for each value.  The
// signed code is the machine's own 8-bit float (bias 7, the same "not finite" code).
__device__ inline void decode_m4(uint32_t w, const int (&field)[4], float (&m)[4]) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  m[0] = ldexpf(a[0], field[0] - 135);
  m[1] = ldexpf(a[1], field[1] - 135);
  m[2] = ldexpf(b[0], field[2] - 135);
  m[3] = ldexpf(b[1], field[3] - 135);
}
__device__ inline void decode_r4(uint32_t w, const int (&field)[4], float (&r)[4]) {
  constexpr uint32_t mask = 255u << 19;
  r[0] = ldexpf(bits_to_float((w << 19) & mask), field[0] - 15);
  r[1] = ldexpf(bits_to_float((w << 11) & mask), field[1] - 15);
  r[2] = ldexpf(bits_to_float((w << 3) & mask), field[2] - 15);
  r[3] = ldexpf(bits_to_float((w >> 5) & mask), field[3] - 15);
  if ((~w - 0x01010101u) & w & 0x80808080u) {  // some code is 255
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((w >> (8 * j)) & 255u) == 255u) r[j] = bits_to_float(0x7fc00000u);
  }
}
__device__ inline void decode_m4(uint32_t w, int field, float (&m)[4]) {
  const int f[4] = {field, field, field, field};
  decode_m4(w, f, m);
}
__device__ inline void decode_r4(uint32_t w, int field, float (&r)[4]) {
  const int f[4] = {field, field, field, field};
  decode_r4(w, f, r);
}

// The top bytes of four words.
__device__ inline uint32_t pack_top(const uint32_t (&x)[4]) {
  const uint32_t lo = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0703u), hi = __builtin_amdgcn_perm(x[3], x[2], 0x0c0c0703u);
  return (hi << 16) | lo;
}

// encode_block where the block holds values that are not finite or the largest exponents.
template <bool kStochastic>
__device__ inline void encode_block_odd(const float (&m)[4], const float (&r)[4], const uint32_t (&h)[4],
                                        uint32_t& m8, uint32_t& r8, uint32_t& fields) {
  constexpr uint32_t kInf = 0x7f800000u;
  uint32_t mb[4], rb[4], mm = 0, rr = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mb[j] = float_to_bits(m[j]) & 0x7fffffffu;
    rb[j] = float_to_bits(r[j]) & 0x7fffffffu;
    if (mb[j] < kInf && mb[j] > mm) mm = mb[j];
    if (rb[j] < kInf && rb[j] > rr) rr = rb[j];
  }
  wave_max2_u32(mm, rr);
  const uint32_t fm = moment_field<3>(mm), fr = moment_field<4>(rr);
  fields = fm | (fr << 8);
  m8 = r8 = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t cm = moment_top<3, kStochastic>(bits_to_float(mb[j]), (int)fm, noise_hi(h[j])) >> 24;
    uint32_t cr = moment_top<4, kStochastic>(bits_to_float(rb[j]), (int)fr, noise_lo(h[j])) >> 24;
    cm = mb[j] >= kInf ? 127u : cm < 126u ? cm : 126u;
    cr = rb[j] >= kInf ? 255u : cr < 254u ? cr : 254u;
    cm |= (float_to_bits(m[j]) >> 24) & 128u;
    m8 |= cm << (8 * j);
    r8 |= cr << (8 * j);
  }
}

// Codes and exponent fields of one block, four values a lane (the whole wave calls).
// h: 32 random bits per value (the upper half rounds m, the lower half r), unused for round to
// nearest even.
template <bool kStochastic>
__device__ inline void encode_block(const float (&m)[4], const float (&r)[4], const uint32_t (&h)[4], uint32_t& m8,
                                    uint32_t& r8, uint32_t& fields) {
  uint32_t mb[4], rb[4], mm = 0, rr = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mb[j] = float_to_bits(m[j]) & 0x7fffffffu;
    rb[j] = float_to_bits(r[j]);
    mm = mm > mb[j] ? mm : mb[j];
    rr = rr > rb[j] ? rr : rb[j];
  }
  wave_max2_u32(mm, rr);
  // from 2^126 on (not finite, or a field that would pass 254): rare, and the same for the wave
  if (mm >= 0x7e800000u || rr >= 0x7e800000u) {
    encode_block_odd<kStochastic>(m, r, h, m8, r8, fields);
    return;
  }
  const uint32_t fm = moment_field<3>(mm), fr = moment_field<4>(rr);
  fields = fm | (fr << 8);
  uint32_t cm[4], cr[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t c = moment_top<3, kStochastic>(fabsf(m[j]), (int)fm, noise_hi(h[j]));
    cm[j] = (c & 0x7fffffffu) | (float_to_bits(m[j]) & 0x80000000u);
    cr[j] = moment_top<4, kStochastic>(r[j], (int)fr, noise_lo(h[j]));
  }
  m8 = pack_top(cm);
  r8 = pack_top(cr);
}

// Correctly rounded roots of four values v >= 0.  The hardware's reciprocal root and one
// Newton step from the exact residual (s + (v - s^2) / (2 s), s = v times that) give the rounded root of every float from 2^-100 on (all
// 1.9e9 of them compared with the compiler's sequence); a lane with smaller ones, whose residual
// would underflow, or with one that is not finite takes that sequence.
__device__ inline void roots4(const float (&v)[4], float (&r)[4]) {
  constexpr float kLeast = 7.888609052210118e-31f;  // 2^-100: bits 0x0d800000
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float up = fmaxf(v[j], kLeast);
    const float y = __builtin_amdgcn_rsqf(up);
    const float s = v[j] * y;
    r[j] = fmaf(fmaf(-s, s, v[j]), 0.5f * y, s);
    lo = min(lo, float_to_bits(v[j]) - 1u);
    hi = max(hi, float_to_bits(v[j]));
  }
  if (lo < 0x0d7fffffu || hi >= 0x7f800000u) {  // above 0 and below 2^-100, or not finite
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = sqrtf(v[j]);
  }
}

// 32 hashed bits of an element's place in the state: a Weyl step by a prime near 2^32 over the
// golden ratio, then one multiplication by an odd constant between two shifts, the usual finish of
// integer hashes; the multipliers are known ones of such hashes.  key holds the seed and the step.
// The element is block + j with block a multiple of 256 that is the same for the wave and j < 256.
__device__ inline uint32_t place_hash(int64_t block, uint32_t j, uint32_t key) {
  const uint32_t x = (uint32_t)block + (uint32_t)((uint64_t)block >> 32) * 0x632be5abu;
  uint32_t h = j * 0x9e3779b1u + (x * 0x9e3779b1u + key);
  h ^= h >> 15;
  h *= 0xd1b54a35u;
  return h ^ (h >> 13);
}

}  // namespace gs
