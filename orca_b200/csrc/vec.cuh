// Rows of fp32, bf16 or fp16 read and written a piece at a time, and the kernel for a type and a piece.
#pragma once

#include <initializer_list>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace orca {

// VB bytes of a row at a time, as elements of T.
template <typename T, int VB>
struct Vec {
  static constexpr int N = VB / (int)sizeof(T);
  struct alignas(VB) Raw { T v[N]; };
  static __device__ __forceinline__ void load(const void *p, float (&x)[N]) {
    const Raw r = *reinterpret_cast<const Raw *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)r.v[i];
  }
  static __device__ __forceinline__ void store(void *p, const float (&x)[N], float scale) {
    Raw r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = (T)(x[i] * scale);
    *reinterpret_cast<Raw *>(p) = r;
  }
};

// Two values from a piece as words of 32 bits, and back.
template <typename T> struct Pair;
template <> struct Pair<float> {
  static constexpr int WORDS = 2;
  static __device__ __forceinline__ float2 of(const uint32_t *w) { return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])); }
  static __device__ __forceinline__ void to(uint32_t *w, float2 v) { w[0] = __float_as_uint(v.x), w[1] = __float_as_uint(v.y); }
};
template <> struct Pair<__nv_bfloat16> {
  static constexpr int WORDS = 1;
  static __device__ __forceinline__ float2 of(const uint32_t *w) { return make_float2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u)); }
  static __device__ __forceinline__ void to(uint32_t *w, float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    w[0] = *reinterpret_cast<const uint32_t *>(&h);
  }
};
template <> struct Pair<__half> {
  static constexpr int WORDS = 1;
  static __device__ __forceinline__ float2 of(const uint32_t *w) { return __half22float2(*reinterpret_cast<const __half2 *>(w)); }
  static __device__ __forceinline__ void to(uint32_t *w, float2 v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    w[0] = *reinterpret_cast<const uint32_t *>(&h);
  }
};

inline int size_of(int type) { return type == ORCA_F32 ? 4 : 2; }

// largest piece that rows can be read and written by
inline int piece(int64_t row_bytes, std::initializer_list<uint64_t> at) {
  uint64_t all = (uint64_t)row_bytes | 16;
  for (uint64_t a : at) all |= a;
  const int vb = (int)(all & (~all + 1));
  return vb > 16 ? 16 : vb;
}

template <typename F>
inline int by_type(int type, int vb, F &&f) {
  if (type == ORCA_F32) return vb == 16 ? f((float *)nullptr, std::integral_constant<int, 16>()) : vb == 8 ? f((float *)nullptr, std::integral_constant<int, 8>()) : f((float *)nullptr, std::integral_constant<int, 4>());
  if (type == ORCA_BF16)
    return vb == 16 ? f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 16>()) : vb == 8 ? f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 8>())
         : vb == 4 ? f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 4>()) : f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 2>());
  return vb == 16 ? f((__half *)nullptr, std::integral_constant<int, 16>()) : vb == 8 ? f((__half *)nullptr, std::integral_constant<int, 8>())
       : vb == 4 ? f((__half *)nullptr, std::integral_constant<int, 4>()) : f((__half *)nullptr, std::integral_constant<int, 2>());
}

}  // namespace orca
