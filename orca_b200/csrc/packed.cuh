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
constexpr int PARTIAL = 1040;                 // floats of a part's result: 1032 sums, 2 references, 2 totals, flag

__device__ __forceinline__ float step_of(uint32_t how) { return __uint_as_float(how << 16); }
__device__ __forceinline__ float offset_of(uint32_t how) { return __uint_as_float(how & 0xffff0000u); }

// (a & b) | c in one instruction: with two constants the compiler makes two of it
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// A code moved to the top of a float's mantissa under the exponent of one: 1 + code / 16.
__device__ __forceinline__ float code_up(uint32_t shifted) { return __uint_as_float(and_or(shifted, 0x780000u, 0x3f800000u)); }
// Columns of a word: 16 step * (1 + code / 16) + (offset - 16 step), both twice for the packed instructions.  The product is exact; the
// difference is rounded once, which puts a value off by half a step of fp32 of 16 steps at most.
__device__ __forceinline__ void decode4(uint32_t w, float2 step16, float2 offset16, float2 (&x)[2]) {
  x[0] = fma2(make_float2(code_up(w << 19), code_up(w << 15)), step16, offset16);
  x[1] = fma2(make_float2(code_up(w << 11), code_up(w << 7)), step16, offset16);
}
__device__ __forceinline__ void decode8(uint32_t w, float2 step16, float2 offset16, float2 (&x)[4]) {
  x[0] = fma2(make_float2(code_up(w << 19), code_up(w << 15)), step16, offset16);
  x[1] = fma2(make_float2(code_up(w << 11), code_up(w << 7)), step16, offset16);
  x[2] = fma2(make_float2(code_up(w << 3), code_up(w >> 1)), step16, offset16);
  x[3] = fma2(make_float2(code_up(w >> 5), code_up(w >> 9)), step16, offset16);
}
// the same exactly as held: offset + step * code, rounded once
__device__ __forceinline__ float held(uint32_t code, float step, float offset) { return fmaf((float)code, step, offset); }

}  // namespace packed
}  // namespace orca
