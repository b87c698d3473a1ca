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

constexpr int kMomBlock = 256;  // elements per block: one wave, four elements a lane

typedef float floatx4 __attribute__((ext_vector_type(4)));

// Maximum over the wave, in every lane (unsigned order is that of non-negative floats).
__device__ inline uint32_t wave_max_u32(uint32_t x) {
#define GS_DPP_MAX(ctrl)                                                                            \
  {                                                                                                 \
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, ctrl, 0xf, 0xf, false); \
    x = x > y ? x : y;                                                                              \
  }
  GS_DPP_MAX(0xB1);   // quad_perm [1, 0, 3, 2]
  GS_DPP_MAX(0x4E);   // quad_perm [2, 3, 0, 1]
  GS_DPP_MAX(0x141);  // row_half_mirror: eight lanes
  GS_DPP_MAX(0x140);  // row_mirror: sixteen lanes
  GS_DPP_MAX(0x142);  // row_bcast15: rows 1 and 3 hold pairs of rows
  GS_DPP_MAX(0x143);  // row_bcast31: row 3 holds all
#undef GS_DPP_MAX
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// Exponent field of a block whose largest finite magnitude has the given bits.
template <int kMant>
__device__ inline uint32_t moment_field(uint32_t most) {
  const uint32_t f = (most + (1u << (24 - kMant)) - 1u) >> 23;
  return f < 254u ? f : 254u;
}

// The code's magnitude of a finite value x >= 0; `low` is what is added below the code's
// bits: a random number of 23 - kMant bits, or kNearest for round to nearest even.
constexpr uint32_t kNearest = 0xffffffffu;
template <int kMant>
__device__ inline uint32_t moment_code(float x, int field, uint32_t low) {
  constexpr int drop = 23 - kMant;
  constexpr uint32_t top = (16u << kMant) - 2u;
  const uint32_t b = float_to_bits(ldexpf(x, 15 - field));
  if (low == kNearest) low = (1u << (drop - 1)) - 1u + ((b >> drop) & 1u);
  uint32_t c = (b + low) >> drop;
  if (kMant == 4) c = c > 0 || x == 0.0f ? c : 1u;
  return c < top ? c : top;
}

// Four decoded values of the packed codes w of one lane; field as stored.
__device__ inline void decode_m4(uint32_t w, int field, float (&m)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    m[j] = ldexpf(bits_to_float((uint32_t)((int32_t)(w << (24 - 8 * j)) >> 4) & 0x87f00000u), field - 15);
  if (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((w >> (8 * j)) & 127u) == 127u) m[j] = bits_to_float(0x7fc00000u);
  }
}
__device__ inline void decode_r4(uint32_t w, int field, float (&r)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = ldexpf(bits_to_float(((w >> (8 * j)) & 255u) << 19), field - 15);
  if ((~w - 0x01010101u) & w & 0x80808080u) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((w >> (8 * j)) & 255u) == 255u) r[j] = bits_to_float(0x7fc00000u);
  }
}

// Codes and exponent fields of one block, four values a lane (the whole wave calls).
// h: 32 random bits per value (the upper half rounds m, the lower half r), or NULL for
// round to nearest even.
template <bool kStochastic>
__device__ inline void encode_block(const float (&m)[4], const float (&r)[4], const uint32_t (&h)[4], uint32_t& m8,
                                    uint32_t& r8, uint32_t& fields) {
  uint32_t mb[4], rb[4], mm = 0, rr = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mb[j] = float_to_bits(m[j]) & 0x7fffffffu;
    rb[j] = float_to_bits(r[j]) & 0x7fffffffu;
    mm = mm > mb[j] ? mm : mb[j];
    rr = rr > rb[j] ? rr : rb[j];
  }
  constexpr uint32_t kInf = 0x7f800000u;
  uint32_t wm = wave_max_u32(mm), wr = wave_max_u32(rr);
  const bool odd = wm >= kInf || wr >= kInf;  // uniform: something here is not finite
  if (odd) {
    mm = rr = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (mb[j] < kInf && mb[j] > mm) mm = mb[j];
      if (rb[j] < kInf && rb[j] > rr) rr = rb[j];
    }
    wm = wave_max_u32(mm);
    wr = wave_max_u32(rr);
  }
  const uint32_t fm = moment_field<3>(wm), fr = moment_field<4>(wr);
  fields = fm | (fr << 8);
  m8 = r8 = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t cm = moment_code<3>(bits_to_float(mb[j]), (int)fm, kStochastic ? (h[j] >> 16) << 4 : kNearest);
    uint32_t cr = moment_code<4>(bits_to_float(rb[j]), (int)fr, kStochastic ? (h[j] & 0xffffu) << 3 : kNearest);
    if (odd) {
      if (mb[j] >= kInf) cm = 127u;
      if (rb[j] >= kInf) cr = 255u;
    }
    cm |= (float_to_bits(m[j]) >> 24) & 128u;
    m8 |= cm << (8 * j);
    r8 |= cr << (8 * j);
  }
}

// 32 hashed bits of an element's place in the state: a Weyl step, one multiplication by an
// odd constant between two shifts.  key holds the seed and the step.
__device__ inline uint32_t place_hash(int64_t place, uint32_t key) {
  const uint32_t x = (uint32_t)place + (uint32_t)((uint64_t)place >> 32) * 0x632be5abu;
  uint32_t h = x * 0x9e3779b1u + key;
  h ^= h >> 15;
  h *= 0xd1b54a35u;
  return h ^ (h >> 13);
}

}  // namespace gs
