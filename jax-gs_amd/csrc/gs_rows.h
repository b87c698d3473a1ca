// Row masks over the elements of a tensor of rows x row_len, for the many-tensor operators.
#pragma once

#include "gs_common.h"

namespace gs {

// floor(2^64 / row_len) + 1 (0 for rows of one element): multiplied by an element's index, the
// upper 64 bits are its row, exactly for index * row_len < 2^64.
inline uint64_t row_magic(int64_t row_len) { return row_len > 1 ? ~(uint64_t)0 / (uint64_t)row_len + 1 : 0; }

constexpr int64_t kMaxRowLen = (int64_t)1 << 24;

// Mask bits of the n <= kVec elements from base + j on, j < 4096, base the same for the wave.
// The row of `base` is found once, in scalar registers; a lane's by a 32-bit reciprocal, for its
// distance from the row's start is below row_len + 4096.
template <int kVec>
__device__ inline uint32_t rows_on(const uint8_t* __restrict__ active, uint64_t magic, uint32_t row_len, int64_t base,
                                   uint32_t j, int n) {
  const uint64_t row0 = magic ? __umul64hi((uint64_t)base, magic) : (uint64_t)base;
  uint32_t e = (uint32_t)((uint64_t)base - row0 * row_len) + j;
  uint32_t q;
  if (row_len > 4096u) q = e >= row_len ? 1u : 0u;
  else q = magic ? __umulhi(e, (uint32_t)(magic >> 32) + 1u) : e;
  const uint8_t* a = active + row0;
  const uint32_t all = (1u << max(n, 0)) - 1u;
  if (n <= 0) return 0;
  // whole vectors within rows: bases are multiples of 256
  if (row_len % kVec == 0) return a[q] ? all : 0u;
  e -= q * row_len;
  if (row_len + 1 >= kVec) {  // at most two rows
    const uint32_t head = e + (uint32_t)n <= row_len ? all : (1u << (row_len - e)) - 1u;
    return (a[q] ? head : 0u) | (head != all && a[q + 1] ? all & ~head : 0u);
  }
  uint32_t on = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    if (i < n && a[q]) on |= 1u << i;
    if (++e == row_len) {
      e = 0;
      ++q;
    }
  }
  return on;
}

}  // namespace gs
