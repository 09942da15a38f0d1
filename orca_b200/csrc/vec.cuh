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
