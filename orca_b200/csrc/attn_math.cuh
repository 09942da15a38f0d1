// What the gather-attention kernels share: packed fp32 arithmetic, time encodings of a slot, the sum of many values over a warp.
#pragma once

#include "common.cuh"

namespace orca {

constexpr int GA_P_ITERS = 3;                   // time-column pairs per lane (the third for lanes 0..21)

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 dup2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 lo2(const float4 &v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(const float4 &v) { return make_float2(v.z, v.w); }

// cos of two arguments below COS_SMALL at once: the reduction of cos_small in packed arithmetic with fewer steps.  The
// nearest integer k of x / 2pi comes from adding and subtracting 1.5 * 2^23, in one fused step, and 2pi is split in two:
// x - k * C1 is a multiple of 2^-22 below 4 (C1 has 24 bits, the last of them 2^-21), so the first difference is exact.
__device__ __forceinline__ float2 cos_small2(float2 x) {
  const float2 t = fma2(x, dup2(0.15915494309189535f), dup2(12582912.f));
  const float2 kk = add2(t, dup2(-12582912.f));
  float2 r = fma2(kk, dup2(-6.2831855f), x);
  r = fma2(kk, dup2(1.7484556e-07f), r);
  return make_float2(__cosf(r.x), __cosf(r.y));
}

// Arguments beyond the fixed-point range (or not finite) are rare: their cosine is a call, so that its long code does
// not stand in the loops six times over (the kernel has to stay within the instruction cache).
static __device__ __noinline__ float cos_far(float x) { return cos_any(x); }

// Time encodings of one slot for this lane's column pairs: the first nl pair groups (64 columns each) hold large
// arguments (fixed-point reduction), the others small ones (packed fp32 reduction); nl < 0: beyond both.  w decreases
// with the column, so "large" groups are always a prefix; nl is uniform over the warp.
__device__ __forceinline__ void time_terms(float dt, int nl, const float2 (&wt)[GA_P_ITERS], float2 (&te)[GA_P_ITERS]) {
#pragma unroll
  for (int i = 0; i < GA_P_ITERS; ++i) {
    const float2 x = mul2(dup2(dt), wt[i]);
    if (nl < 0) te[i] = make_float2(cos_far(x.x), cos_far(x.y));
    else if (i < nl) te[i] = make_float2(cos_fixed(x.x), cos_fixed(x.y));
    else te[i] = cos_small2(x);
  }
}

__device__ __forceinline__ float4 ldg4(const char *p) { return __ldg(reinterpret_cast<const float4 *>(p)); }

// Sums V values (V a power of two up to 32) over the warp: lane l returns the total of value l / (32 / V).
template <int V>
__device__ __forceinline__ float warp_sum_many(float (&v)[V], int lane) {
  constexpr unsigned FULL = 0xffffffffu;
  int o = 16;
#pragma unroll
  for (int n = V / 2; n > 0; n >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {   // a lane keeps the half of the values that its bit names and hands over the other
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(FULL, give, o);
    }
  }
  float s = v[0];
  for (; o > 0; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
  return s;
}

}  // namespace orca
