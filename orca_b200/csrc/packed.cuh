// Rows of 172 values held in 4 bits: 24 words of 32 bits, 96 bytes, three sectors of a cache line.
//   word 0       how columns 0..127 are held: step (bfloat16) in the low half, offset (bfloat16) in the high half
//   word 1       the same of columns 128..171
//   words 2..17  codes of columns 0..127, eight a word, the first column in the lowest bits
//   words 18..23 codes of columns 128..171 (the last word holds four)
// value = offset + step * code.  The split at column 128 fills sixteen whole words; two groups of 86 would err 2 % less on
// values of a normal distribution (its range in 86 draws against 128 and 44) and end inside words.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_math.cuh"
#include "common.cuh"

namespace orca {
namespace packed {

constexpr int WORDS = ORCA_PACKED_WORDS;      // 24
constexpr int BYTES = WORDS * 4;              // 96
constexpr int GROUP = 128;                    // columns of the first group
constexpr int TAIL = D - GROUP;               // 44 of the second
constexpr int PARTIAL = 1040;                 // floats of a part's result: 1032 sums, 2 maxima, 2 totals, flag

__device__ __forceinline__ float step_of(uint32_t how) { return __uint_as_float(how << 16); }
__device__ __forceinline__ float offset_of(uint32_t how) { return __uint_as_float(how & 0xffff0000u); }

// Nibbles 0..4 of a word as floats without a shift: or'ed into the mantissa under the exponent at which the nibble's lowest bit
// counts one, 2^e + code; e = 23, 19, 15, 11, 7.  Taking 2^e away is exact.
template <int I>
__device__ __forceinline__ float nibble_raw(uint32_t w) {
  static_assert(I >= 0 && I < 5, "a float has 23 bits of mantissa");
  return __uint_as_float((w & (0xfu << (4 * I))) | ((127u + 23u - 4u * I) << 23));
}
template <int I>
__device__ __forceinline__ constexpr float nibble_base() { return (float)(1 << (23 - 4 * I)); }

// columns 2 J and 2 J + 1 (of the nibbles I, I + 1): offset + step * code
template <int I>
__device__ __forceinline__ float2 decode_pair(uint32_t w, float2 step, float2 offset) {
  float2 c = make_float2(nibble_raw<I>(w), nibble_raw<I + 1>(w));
  c = add2(c, make_float2(-nibble_base<I>(), -nibble_base<I + 1>()));
  return fma2(c, step, offset);
}
// four columns from the low half of a word
__device__ __forceinline__ void decode4(uint32_t w, float2 step, float2 offset, float2 (&x)[2]) {
  x[0] = decode_pair<0>(w, step, offset);
  x[1] = decode_pair<2>(w, step, offset);
}
__device__ __forceinline__ void decode8(uint32_t w, float2 step, float2 offset, float2 (&x)[4]) {
  x[0] = decode_pair<0>(w, step, offset);
  x[1] = decode_pair<2>(w, step, offset);
  const uint32_t v = w >> 16;
  x[2] = decode_pair<0>(v, step, offset);
  x[3] = decode_pair<2>(v, step, offset);
}

}  // namespace packed
}  // namespace orca
