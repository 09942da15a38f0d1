// Layer norm over the last dimension, and its gradients.
//
//   m = mean of x, r = 1 / sqrt(mean of (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   with d = g w:  dx = r (d - mean(d) - h mean(d h)),  dw = sum over rows of g h,  db = sum over rows of g
//
// Bound by HBM: a row is read once and written once, backward two are read and one is written.  Nothing is kept from the forward pass: backward has x
// in its hands and finds m and r again, by the same steps.  Sums are of x - k with k near the mean: the rounding to 32 bits of a mean, or of a sum, misses by as
// much as a row varies where its mean is 2^24 times that.  k is the rounded mean, or, where one pass is to have all sums of a row, the
// mean of some of its values.  Where those are unlike the rest, variance and h are differences of larger numbers (a row of 8192 with k sixteen deviations from the
// mean: off by up to 5e-4): such rows of several warps are gone through once more at the end, around the mean.
// dw and db: each block sums its rows into a row of parts, in order, and another kernel adds up the parts: the same bits every time.
#include <algorithm>

#include <cooperative_groups.h>

#include "attn_math.cuh"
#include "common.cuh"
#include "context.cuh"
#include "vec.cuh"

namespace orca {
namespace norm {

struct Rows {            // of x, or of a gradient
  const char *p;
  int64_t stride;        // bytes
};
struct Stats {           // of a row: h = ((x - m) - c) * r
  float m, c, r;
};
struct Affine {          // of weights W; nullptr: one and zero
  const void *w, *b;
};

// r, NaN where the variance v has left the range of 32 bits (its inverse root is zero: the row would be the bias)
__device__ __forceinline__ float finite(float v, float r) { return fmaf(v, 0.f, r); }
__device__ __forceinline__ float inverse_root(float v) { return finite(v, rsqrtf(v)); }

template <typename W, int N> __device__ __forceinline__ void load_affine(const void *p, int64_t at, float otherwise, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = p == nullptr ? otherwise : (float)reinterpret_cast<const W *>(p)[at + i];
}

// ---------------------------------------------------------------------------------------------- rows of any width
// A block a row, which it goes through again for each sum: from L2 after the first time (2000 rows of 40 000 of bf16, forward: 128 us, 2.5 TB/s).  Few rows are
// shared by a cluster of blocks each (16 rows of a million: 633 us by a block each, 97 so).  Rows that lie as no wide load can take them go this way, too,
// a value at a time.
constexpr int ANY = 512, CLUSTER = 8;
struct Share {           // of a row: pieces first, first + step, ...
  int first, step, odd;
  __device__ Share() : odd(0) {
    const auto cluster = cooperative_groups::this_cluster();
    first = (int)cluster.block_rank() * blockDim.x + threadIdx.x;
    step = (int)cluster.num_blocks() * blockDim.x;
  }
  static __device__ __forceinline__ int blocks() { return (int)cooperative_groups::this_cluster().num_blocks(); }
  // Sums over the row, the same bits in every thread: of warps, then theirs in order, then the blocks'.
  template <int K> __device__ __forceinline__ void sum(float (&v)[K], float (*s)[2], float (*s_block)[2]) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
    __syncthreads();       // (s is read by the sums before)
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) s[warp][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = s[0][k];
    for (int w = 1; w < warps; ++w)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += s[w][k];
    const auto cluster = cooperative_groups::this_cluster();
    if (cluster.num_blocks() == 1) return;
    float *mine = s_block[odd];
    odd ^= 1;
    if (threadIdx.x == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) mine[k] = v[k];
    cluster.sync();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = 0.f;
    for (int r = 0; r < (int)cluster.num_blocks(); ++r)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += cluster.map_shared_rank(mine, r)[k];
  }
  // (a block stays until the others have read its sums)
  static __device__ __forceinline__ void end() {
    if (blocks() > 1) cooperative_groups::this_cluster().sync();
  }
};
struct Sums { float warps[ANY / 32][2], block[2][2]; };
template <typename T, int VB> __device__ __forceinline__ Stats any_stats(Share &share, Sums &s, const char *x, int nv, int width, float eps) {
  using X = Vec<T, VB>;
  float one[1] = {0.f}, two[2] = {0.f, 0.f};
  for (int v = share.first; v < nv; v += share.step) {
    float a[X::N];
    X::load(x + (int64_t)v * VB, a);
#pragma unroll
    for (int i = 0; i < X::N; ++i) one[0] += a[i];
  }
  share.sum(one, s.warps, s.block);
  Stats t;
  t.m = one[0] / (float)width;
  for (int v = share.first; v < nv; v += share.step) {
    float a[X::N];
    X::load(x + (int64_t)v * VB, a);
#pragma unroll
    for (int i = 0; i < X::N; ++i) {
      const float e = a[i] - t.m;
      two[0] += e;
      two[1] += e * e;
    }
  }
  share.sum(two, s.warps, s.block);
  t.c = two[0] / (float)width;
  const float v = relu(two[1] / (float)width - t.c * t.c) + eps;
  t.r = finite(v, 1.f / sqrtf(v));
  return t;
}

template <typename T, typename W, int VB>
__global__ void __launch_bounds__(ANY) any_kernel(Rows x, int64_t rows, int nv, int width, Affine a, float eps, char *__restrict__ y) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  __shared__ Sums s;
  Share share;
  for (int64_t row = blockIdx.x / Share::blocks(); row < rows; row += gridDim.x / Share::blocks()) {
    const char *p = x.p + row * x.stride;
    const Stats t = any_stats<T, VB>(share, s, p, nv, width, eps);
    for (int v = share.first; v < nv; v += share.step) {
      float e[X::N], w[X::N], b[X::N];
      X::load(p + (int64_t)v * VB, e);
      load_affine<W>(a.w, (int64_t)v * X::N, 1.f, w);
      load_affine<W>(a.b, (int64_t)v * X::N, 0.f, b);
#pragma unroll
      for (int i = 0; i < X::N; ++i) e[i] = fmaf(((e[i] - t.m) - t.c) * t.r, w[i], b[i]);
      X::store(y + (row * nv + v) * VB, e, 1.f);
    }
  }
  Share::end();
}

// dx where it is wanted; the rows' statistics for the sums over rows where those are.
template <typename T, typename W, int VB>
__global__ void __launch_bounds__(ANY) any_grad_kernel(Rows g, Rows x, int64_t rows, int nv, int width, Affine a, float eps, char *__restrict__ dx,
                                                       Stats *__restrict__ stats) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  __shared__ Sums s;
  Share share;
  for (int64_t row = blockIdx.x / Share::blocks(); row < rows; row += gridDim.x / Share::blocks()) {
    const char *px = x.p + row * x.stride, *pg = g.p + row * g.stride;
    const Stats t = any_stats<T, VB>(share, s, px, nv, width, eps);
    if (stats != nullptr && share.first == 0) stats[row] = t;
    if (dx == nullptr) continue;
    float sum[2] = {0.f, 0.f};
    for (int v = share.first; v < nv; v += share.step) {
      float e[X::N], d[X::N], w[X::N];
      X::load(px + (int64_t)v * VB, e);
      X::load(pg + (int64_t)v * VB, d);
      load_affine<W>(a.w, (int64_t)v * X::N, 1.f, w);
#pragma unroll
      for (int i = 0; i < X::N; ++i) {
        const float dw = d[i] * w[i];
        sum[0] += dw;
        sum[1] = fmaf(dw, ((e[i] - t.m) - t.c) * t.r, sum[1]);
      }
    }
    share.sum(sum, s.warps, s.block);
    const float c1 = sum[0] / (float)width, c2 = sum[1] / (float)width;
    for (int v = share.first; v < nv; v += share.step) {
      float e[X::N], d[X::N], w[X::N];
      X::load(px + (int64_t)v * VB, e);
      X::load(pg + (int64_t)v * VB, d);
      load_affine<W>(a.w, (int64_t)v * X::N, 1.f, w);
#pragma unroll
      for (int i = 0; i < X::N; ++i) e[i] = t.r * (fmaf(d[i], w[i], -c1) - ((e[i] - t.m) - t.c) * t.r * c2);
      X::store(dx + (row * nv + v) * VB, e, 1.f);
    }
  }
  Share::end();
}

// Parts of dw and db: a block has a strip of columns, a piece a thread, and `share` rows.  parts[blockIdx.y][2][width].
constexpr int STRIP = 128;
template <typename T, int VB>
__global__ void __launch_bounds__(STRIP) any_sums_kernel(Rows g, Rows x, int64_t rows, int64_t share, int nv, int width, const Stats *__restrict__ stats,
                                                         float *__restrict__ parts) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  const int v = blockIdx.x * STRIP + threadIdx.x;
  if (v >= nv) return;
  const int64_t first = blockIdx.y * share, end = min(first + share, rows);
  float dw[X::N] = {}, db[X::N] = {};
#pragma unroll 4
  for (int64_t row = first; row < end; ++row) {
    float e[X::N], d[X::N];
    const Stats t = stats[row];
    X::load(x.p + row * x.stride + (int64_t)v * VB, e);
    X::load(g.p + row * g.stride + (int64_t)v * VB, d);
#pragma unroll
    for (int i = 0; i < X::N; ++i) {
      dw[i] = fmaf(d[i], ((e[i] - t.m) - t.c) * t.r, dw[i]);
      db[i] += d[i];
    }
  }
  float *out = parts + (int64_t)blockIdx.y * 2 * width + (int64_t)v * X::N;
#pragma unroll
  for (int i = 0; i < X::N; ++i) {
    out[i] = dw[i];
    out[width + i] = db[i];
  }
}

// ---------------------------------------------------------------------------------------------- rows in registers
// 2^log_tpr threads a row, P pieces of VB bytes each (thread l has pieces l, l + tpr, ...), 16 values at most: x is read once, weights stay in registers while a
// block goes on to its next rows.  Those are on their way by asynchronous copies.  A thread copies what it reads itself, so nobody waits for a copy
// but its thread.  Rows that do not begin where wide loads can (SHIFT): pieces are those of memory, the first and last of a row hold values of its
// neighbours, which are masked; a thread's rows all begin at the same place within a piece, for the host makes the step between them whole pieces.
// Arithmetic on pairs of values, in packed instructions.
// s / n to the nearest (but for the rarest case), so that rows of one value have that as their pivot
__device__ __forceinline__ float quotient(float s, float n, float inverse) {
  const float q = s * inverse;
  return fmaf(fmaf(-q, n, s), inverse, q);
}

// Threads that share a row: 4 to 32 lanes of a warp, or several warps.  Sums take five shuffles whatever the team's size; a step that would leave the team
// takes the lane's own value instead, so that sums over teams of a warp come out `scale` times what they are (a power of two).
template <int THREADS, bool WIDE> struct Team {      // WIDE: several warps a row
  int log_tpr, lane, slot;       // thread in its row's team, team in the block
  int m[5];                      // lanes of the steps
  float scale;
  __device__ explicit Team(int log) : log_tpr(THREADS == 512 ? 9 : log), lane(threadIdx.x & ((1 << log_tpr) - 1)), slot(threadIdx.x >> log_tpr) {
    const int n = WIDE ? 32 : tpr();
#pragma unroll
    for (int k = 0; k < 5; ++k) m[k] = n >> (k + 1);
    scale = (float)(32 / n);
  }
  __device__ __forceinline__ int tpr() const { return 1 << log_tpr; }
  __device__ __forceinline__ int slots() const { return THREADS >> log_tpr; }
  // over the lanes of the team, or over the warp
  __device__ __forceinline__ float lanes_sum(float v) const {
#pragma unroll
    for (int k = 0; k < 5; ++k) v += __shfl_xor_sync(0xffffffffu, v, m[k]);
    return v;
  }
  // Barrier of a sum over several warps: of all threads of the block, or (ALONE) of the team, which has one by its number.
  template <bool ALONE> __device__ __forceinline__ void barrier() const {
    if (ALONE && THREADS != 512) asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(tpr()) : "memory");
    else __syncthreads();
  }
  // Over the team, the same bits in each thread.  Of several warps: all threads of the block call it (ALONE: of the team); s of two calls in turn.
  template <bool ALONE = false> __device__ __forceinline__ void sum(float (&v)[2], float (*s)[4]) const {
#pragma unroll
    for (int k = 0; k < 5; ++k) {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], m[k]);
      v[1] += __shfl_xor_sync(0xffffffffu, v[1], m[k]);
    }
    if (!WIDE) return;
    const int warp = threadIdx.x >> 5, warps = tpr() >> 5, from = warp & ~(warps - 1), w = threadIdx.x & 15;
    if ((threadIdx.x & 31) == 0) *reinterpret_cast<float2 *>(s[warp]) = make_float2(v[0], v[1]);
    barrier<ALONE>();
    const float2 q = w < warps ? *reinterpret_cast<const float2 *>(s[from + w]) : make_float2(0.f, 0.f);
    v[0] = q.x, v[1] = q.y;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      v[1] += __shfl_xor_sync(0xffffffffu, v[1], o);
    }
  }
  // Four at a time: lanes exchange two of them, then one, and a quarter of the lanes goes on with each: ten shuffles instead of twenty.
  template <bool ALONE = false> __device__ __forceinline__ void sum(float (&v)[4], float (*s)[4]) const {
    const int l = threadIdx.x & 31, n = WIDE ? 32 : tpr();
    const bool upper = l & m[0], second = l & m[1];
    const float a = __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], m[0]), b = __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], m[0]);
    const float c = (upper ? v[2] : v[0]) + a, d = (upper ? v[3] : v[1]) + b;
    float q = __shfl_xor_sync(0xffffffffu, second ? c : d, m[1]) + (second ? d : c);
#pragma unroll
    for (int k = 2; k < 5; ++k) q += __shfl_xor_sync(0xffffffffu, q, m[k]);
    if (WIDE) {
      const int warp = threadIdx.x >> 5, warps = tpr() >> 5, from = warp & ~(warps - 1), w = l & 7;
      if (w == 0) s[warp][l >> 3] = q;
      barrier<ALONE>();
      q = w < warps ? s[from + w][l >> 3] : 0.f;
      if (w + 8 < warps) q += s[from + w + 8][l >> 3];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    const int at = l & ~(n - 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __shfl_sync(0xffffffffu, q, at + k * m[1]);
  }
};

// Copies under way, in shared memory: stages of P pieces a thread of ARR arrays, and 32 values of its row a warp.
template <int VB> __device__ __forceinline__ void copy_async(uint32_t to, const char *from, int bytes = VB) {       // (zeros behind `bytes`)
  if constexpr (VB == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
template <int VB> __device__ __forceinline__ void read_shared(uint32_t at, uint32_t *w) {
  if constexpr (VB == 16) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
}
// As far ahead as 24 to 64 kB an SM: less is waited for (8192 of bf16, forward, 16 and 32 kB: 60 and 56 us), more is slower again (1.1 M rows of 172 of fp32, 36 and 72 kB: 246
// and 270 us; gradients of 8192 of fp32, 64 and 128 kB: 126 and 143 us).
template <typename T, int VB, int P, int ARR, int THREADS, int BLOCKS> struct Ring {
  static constexpr int STAGE = ARR * P * THREADS * VB, SAMPLES = THREADS * (int)sizeof(T), DEPTH = STAGE * BLOCKS <= 24576 ? 3 : 2, BYTES = DEPTH * (STAGE + SAMPLES);
  uint32_t pieces, samples;      // this thread's, its warp's
  __device__ explicit Ring(const char *shared) {
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(shared);
    pieces = base + threadIdx.x * VB;
    samples = base + DEPTH * STAGE + (threadIdx.x & ~31u) * (uint32_t)sizeof(T);
  }
  __device__ __forceinline__ uint32_t piece(int stage, int array, int k) const { return pieces + stage * STAGE + (array * P + k) * THREADS * VB; }
  __device__ __forceinline__ float sample(int stage) const {
    const uint32_t at = samples + stage * SAMPLES + (threadIdx.x & 31) * (uint32_t)sizeof(T);
    T v;
    if constexpr (sizeof(T) == 4) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    else asm volatile("ld.shared.u16 %0, [%1];" : "=h"(*reinterpret_cast<uint16_t *>(&v)) : "r"(at) : "memory");
    return (float)v;
  }
};

template <int H> __device__ __forceinline__ float sum_of(const float2 (&x)[H]) {      // two sums of every other pair
  float2 a = x[0], b = H > 1 ? x[H > 1] : make_float2(0.f, 0.f);
#pragma unroll
  for (int h = 2; h < H; ++h) (h & 1 ? b : a) = add2(h & 1 ? b : a, x[h]);
  if (H > 1) a = add2(a, b);
  return a.x + a.y;
}
template <int H> __device__ __forceinline__ float dot_of(const float2 (&x)[H], const float2 (&y)[H]) {
  float2 a = mul2(x[0], y[0]), b = H > 1 ? mul2(x[H > 1], y[H > 1]) : make_float2(0.f, 0.f);
#pragma unroll
  for (int h = 2; h < H; ++h) (h & 1 ? b : a) = fma2(x[h], y[h], h & 1 ? b : a);
  if (H > 1) a = add2(a, b);
  return a.x + a.y;
}

// (what follows from it is found again, not kept)
__device__ __forceinline__ int anew(int v) {
  asm volatile("" : "+r"(v));
  return v;
}

// A thread's pieces of a row.
template <typename T, int VB, int P, bool SHIFT> struct Slice {
  static constexpr int S = (int)sizeof(T), V = VB / S, E = V * P, H = E / 2, WORDS = VB / 4, PW = Pair<T>::WORDS;      // H: pairs of values
  // (16 values with masks fill the registers of gradients: where samples lie is found for each row, and far rows are noted in shared memory.  5003 rows of 7001 of bf16 97 us,
  // 88 so; of 8001 of fp32 137, 118.  Elsewhere, where there is room, the note costs 16 % at 8192.)
  static constexpr bool TIGHT = SHIFT && P == 4;
  static constexpr int SAMPLED = 32 / V, TOGETHER = 32 / VB;      // pieces that samples are, those that lie side by side: 32 bytes
  int first, step, width;        // column of the first value of piece 0 (negative: values of the row before), columns from piece to piece
  uint32_t mask;                 // of values that are the row's: whole pieces, but for SHIFT.  Only the last piece may have none.
  int to_samples;                // bytes from the first piece to what this lane copies of them
  // (SHIFT: pieces that may hold values of other rows are the first and the last, and the one before that where no thread has the last)
  static constexpr __host__ __device__ bool masked(int k) { return SHIFT && (k == 0 || k >= P - 2); }
  uint32_t words[SHIFT ? P * WORDS : 1];
  float2 one[SHIFT ? H : 1];     // where a value is the row's, else zero
  __device__ Slice(int lane, int tpr, int width, const char *row) : first(lane * V), step(tpr * V), width(width), mask(0) {
    if (SHIFT) first -= (int)((uintptr_t)row % VB) / S;
    to_samples = samples_from(lane, width);
#pragma unroll
    for (int i = 0; i < E; ++i) mask |= (uint32_t)(column(i) >= 0 && column(i) < width) << i;
    if (SHIFT) {
#pragma unroll
      for (int h = 0; h < H; ++h) one[h] = make_float2(mask >> 2 * h & 1u ? 1.f : 0.f, mask >> (2 * h + 1) & 1u ? 1.f : 0.f);
#pragma unroll
      for (int i = 0; i < P * WORDS; ++i) words[i] = 0;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (mask >> i & 1u) words[i * S / 4] |= S == 4 ? 0xffffffffu : 0xffffu << 16 * (i & 1);
    }
  }
  // (in the middle of each half, or quarter, of the row's pieces, from the second (SHIFT) or the first on)
  static __device__ __forceinline__ int samples_from(int lane, int width) {
    const int whole = (SHIFT ? width - V + 1 : width) / V, sample = threadIdx.x & (SAMPLED - 1), part = sample / TOGETHER;
    return (whole * (2 * part + 1) / (2 * SAMPLED / TOGETHER) + sample % TOGETHER + SHIFT - lane) * VB;
  }
  __device__ __forceinline__ int column(int i) const { return first + (i / V) * step + i % V; }
  __device__ __forceinline__ bool has(int i) const { return mask >> (SHIFT ? i : i / V * V) & 1u; }
  __device__ __forceinline__ uint32_t part(int k) const { return mask >> (k * V) & ((1u << V) - 1u); }
  __device__ __forceinline__ bool piece(int k) const { return k < P - 1 || part(k) != 0; }
  // Asks for the pieces of a row, the first of which is `at`.  SHIFT: `edge` where one may begin before, or end behind, the memory [begin, end) that may be read.
  template <typename R> __device__ __forceinline__ void fetch(const R &ring, int stage, int array, const char *at, bool edge, const char *begin, const char *end) const {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if (!piece(k)) continue;
      const char *p = at + k * step * S;
      const uint32_t to = ring.piece(stage, array, k);
      if (!SHIFT || !edge) {
        copy_async<VB>(to, p);
      } else if (p >= begin) {
        copy_async<VB>(to, p, (int)min((int64_t)VB, (int64_t)(end - p)));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (part(k) >> i & 1u) {
            if (S == 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + i * S), "r"(reinterpret_cast<const uint32_t *>(p)[i]) : "memory");
            else asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + i * S), "h"(reinterpret_cast<const uint16_t *>(p)[i]) : "memory");
          }
      }
    }
  }
  template <typename R> __device__ __forceinline__ void values(const R &ring, int stage, int array, float2 (&x)[H]) const {
    uint32_t w[P * WORDS];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if (k == P - 1)
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[k * WORDS + i] = 0;
      if (piece(k)) read_shared<VB>(ring.piece(stage, array, k), w + k * WORDS);
    }
#pragma unroll
    for (int i = 0; i < P * WORDS; ++i) w[i] = masked(i / WORDS) ? w[i] & words[i] : w[i];
#pragma unroll
    for (int h = 0; h < H; ++h) x[h] = Pair<T>::of(w + h * PW);
  }
  // The pivot of a team of a warp: the mean of its values; in 16 bits, where instructions count (66 001 rows of 172 forward: 11.9 us so, 10.1), that of each thread's first
  // (SHIFT, where that may be another row's: of its first piece), four deviations from the mean at most, for they are one of 16: h is off by 2e-6 then.
  // Larger teams: the mean of 32 values that lie in pieces over all of the row, which each warp copies for itself.
  static constexpr bool MEAN = sizeof(T) == 4;
  __device__ __forceinline__ float own_sample(const float2 (&x)[H]) const {
    if (MEAN) return sum_of(x);
    if (!SHIFT) return x[0].x;      // (zero where a thread has no piece)
    float v = x[0].x + x[0].y;
#pragma unroll
    for (int h = 1; h < V / 2; ++h) v += x[h].x + x[h].y;
    return v;
  }
  __device__ __forceinline__ float own_samples() const { return (float)(MEAN ? __popc(mask) : SHIFT ? __popc(part(0)) : has(0) ? 1 : 0); }
  template <typename R> __device__ __forceinline__ void fetch_samples(const R &ring, int stage, const char *at) const {
    const int lane = threadIdx.x & 31;
    if (lane < SAMPLED) copy_async<VB>(ring.samples + stage * R::SAMPLES + lane * VB, at + (TIGHT ? samples_from((first + V - 1) / V, anew(width)) : to_samples));
  }
  // x less m, zero where values are not the row's
  __device__ __forceinline__ void less(float2 (&x)[H], float m) const {
    const float2 whole = dup2(-m), last = dup2(piece(P - 1) ? -m : 0.f);
#pragma unroll
    for (int h = 0; h < H; ++h) x[h] = masked(2 * h / V) ? fma2(one[h], whole, x[h]) : add2(x[h], 2 * h / V < P - 1 ? whole : last);
  }
  __device__ __forceinline__ void store(char *at, const float2 (&x)[H]) const {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if (!piece(k)) continue;
      char *p = at + k * step * S;
      uint32_t w[WORDS];
#pragma unroll
      for (int h = 0; h < V / 2; ++h) Pair<T>::to(w + h * PW, x[k * (V / 2) + h]);
      if (!SHIFT || part(k) == (1u << V) - 1u) {
        if constexpr (VB == 16) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (part(k) >> i & 1u) {
            if (S == 4) reinterpret_cast<uint32_t *>(p)[i] = w[i];
            else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i / 2] >> 16 * (i & 1));
          }
      }
    }
  }
  __device__ __forceinline__ void affine(const void *p, bool fp32, float otherwise, float2 (&x)[H]) const {
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      v[i] = otherwise;
      if (p != nullptr && has(i)) v[i] = fp32 ? reinterpret_cast<const float *>(p)[column(i)] : (float)reinterpret_cast<const T *>(p)[column(i)];
    }
#pragma unroll
    for (int h = 0; h < H; ++h) x[h] = make_float2(v[2 * h], v[2 * h + 1]);
  }
};
// One array's rows of a team: the thread's first piece of the next one to ask for.
struct Walk {
  const char *at, *begin, *end;
  int64_t jump;
  __device__ Walk(const Rows &r, int64_t rows, int64_t row, int64_t step, int64_t row_bytes, int first)
      : at(r.p + row * r.stride + first), begin(r.p), end(r.p + (rows - 1) * r.stride + row_bytes), jump(step * r.stride) {}
};
// Rows at either end of an array whose pieces may be those of memory before or behind it: all of them where they are the same row.
__device__ __forceinline__ int64_t edge_rows(int vb, const Rows &r) { return r.stride > 0 ? 1 + vb / r.stride : INT64_MAX / 2; }

// A pivot is far from a row's mean where they are more than this many deviations apart (eight times what the mean of 32 normal values is off by).  A team
// of several warps that meets such a row goes through its rows again when it is done with all of them, which costs the others a comparison a row.  A branch for every row
// took up to 40 % (20 011 bf16 rows of 3000: 57 us forward, 78 with it), bits of a word for up to 31 rows up to 32 %, the second pass in the kernel's own registers
// up to 30 % of gradients; now 57 and 53 us, and kernels of their own for teams of a warp and of several are what the loop gained.  Odd widths lost
// some: 5003 rows of 6001 of fp32 47 / 76 us, 49 / 80 now, of 7001 of bf16 43 / 81, 42 / 88.
constexpr float FAR = 1.4142135f;

// What they measured (forward / gradients): 1.14 M rows of 172 of fp32 247 / 373 us, 6.4 / 6.3 TB/s, HBM; 8191 rows of 8192 of bf16 54 / 85 us, 5.0 / 4.8 TB/s, 66 001 of 172
// 10 / 20, 20 011 of 515 of fp16 18 / 36: 16 bits are bound by instructions (205 and 309 a warp that has 16 values a lane, every second cycle) and by waiting for a row's sums.
// Rows that are all far: 8191 of 8192 of bf16 174 / 232, 20 011 of 515 of fp16 53 / 90.
constexpr int SMS = 148;      // (a constant, so that the order of sums is that of the sizes whatever the device has)
template <int THREADS, bool SHIFT> constexpr int ROW_BLOCKS = THREADS == 512 ? 1 : SHIFT ? 2 : 3;      // an SM
template <int THREADS> constexpr int GRAD_BLOCKS = THREADS == 512 ? 1 : 2;
// (Gradients of rows between borders spill: with four pieces in 512 threads 28 to 36 bytes a thread stored and 56 to 108 loaded, with three of 16 bits in teams of a warp 16
// and 64; all the registers that so many threads can have are theirs.)

// The variance from the mean c of differences from a pivot and the sum of their squares.
// A mean of many values as the pivot (MEAN) may be a few steps off that of a row of one value, whose differences are all c: what their squares leave is rounding, far
// less than any other value would, a step away from them (c^2 over 9000 at least).  Such a row is `flat`: its variance is zero, and so is h.
template <bool MEAN> __device__ __forceinline__ float variance(float c, float sum, float inverse, bool &flat) {
  const float square = c * c, v = relu(fmaf(sum, inverse, -square));
  flat = MEAN && v < 1.5258789e-5f * square;       // 2^-16
  return flat ? 0.f : v;
}

// Rows of a team of several warps whose pivot is far: each is found as it was before, and gone through around the mean.  (A function of its own, for what it keeps in registers
// is not to be kept over the loops before it.)
template <typename T, int VB, int P, bool SHIFT, int THREADS>
__device__ __noinline__ void far_rows(Rows x, int64_t rows, int width, int log_tpr, Affine a, int fp32_weights, float eps, char *__restrict__ y) {
  using S = Slice<T, VB, P, SHIFT>;
  using R = Ring<T, VB, P, 1, THREADS, ROW_BLOCKS<THREADS, SHIFT>>;
  extern __shared__ __align__(16) char s_ring[];
  __shared__ __align__(16) float s_sum[2][THREADS / 32][4];
  const R ring(s_ring);
  const Team<THREADS, true> team(log_tpr);
  int64_t row = (int64_t)blockIdx.x * team.slots() + team.slot;
  const int64_t step = (int64_t)gridDim.x * team.slots();
  const S slice(team.lane, team.tpr(), width, x.p + row * x.stride);
  const char *end = x.p + (rows - 1) * x.stride + width * S::S;
  float2 w[S::H], b[S::H];
  slice.affine(a.w, fp32_weights, 1.f, w);
  slice.affine(a.b, fp32_weights, 0.f, b);
  const float inverse = 1.f / (float)width;
  for (; row < rows; row += step) {
    const char *at = x.p + row * x.stride + slice.first * S::S;
    slice.fetch(ring, 0, 0, at, SHIFT, x.p, end);
    slice.fetch_samples(ring, 0, at);
    copies_issued();
    copies_wait<0>();
    __syncwarp();
    float pivot = quotient(team.lanes_sum(ring.sample(0)), 32.f, 1.f / 32.f);
#pragma unroll 1
    for (int time = 0; time < 2; ++time) {
      float2 d[S::H];
      slice.values(ring, 0, 0, d);
      slice.less(d, pivot);
      float two[2] = {sum_of(d), dot_of(d, d)};
      team.template sum<true>(two, s_sum[time]);
      bool flat;
      const float c = two[0] * inverse, r = inverse_root(variance<false>(c, two[1], inverse, flat) + eps);
      const float2 rr = dup2(r), rc = dup2(-r * c);
      if (time == 0) {
        if (!(fabsf(rc.x) > FAR)) {
          team.template barrier<true>();       // (its sums are read)
          break;
        }
        pivot += c;
        continue;
      }
#pragma unroll
      for (int h = 0; h < S::H; ++h) d[h] = fma2(fma2(d[h], rr, rc), w[h], b[h]);
      slice.store(y + row * (width * S::S) + slice.first * S::S, d);
    }
  }
}
// The same for gradients.  What they change of dw goes to the block's sums, `out` (nullptr: not wanted), team by team; all threads of the block call it.
template <typename T, int VB, int P, bool SHIFT, int THREADS>
__device__ __noinline__ void far_rows_grad(Rows g, Rows x, int64_t rows, int width, int log_tpr, const void *weight, int fp32_weight, float eps, char *__restrict__ dx,
                                           float *out, bool far) {
  using S = Slice<T, VB, P, SHIFT>;
  using R = Ring<T, VB, P, 2, THREADS, GRAD_BLOCKS<THREADS>>;
  extern __shared__ __align__(16) char s_ring[];
  __shared__ __align__(16) float s_sum[2][THREADS / 32][4];
  const R ring(s_ring);
  const Team<THREADS, true> team(log_tpr);
  int64_t row = (int64_t)blockIdx.x * team.slots() + team.slot;
  const int64_t step = (int64_t)gridDim.x * team.slots();
  const S slice(team.lane, team.tpr(), width, x.p + row * x.stride);
  const char *end_x = x.p + (rows - 1) * x.stride + width * S::S, *end_g = g.p + (rows - 1) * g.stride + width * S::S;
  float2 w[S::H], dw[S::H];
  slice.affine(weight, fp32_weight, 1.f, w);
#pragma unroll
  for (int h = 0; h < S::H; ++h) dw[h] = make_float2(0.f, 0.f);
  const float inverse = 1.f / (float)width;
  for (; far && row < rows; row += step) {
    const char *at = x.p + row * x.stride + slice.first * S::S;
    slice.fetch(ring, 0, 0, at, SHIFT, x.p, end_x);
    slice.fetch(ring, 0, 1, g.p + row * g.stride + slice.first * S::S, SHIFT, g.p, end_g);
    slice.fetch_samples(ring, 0, at);
    copies_issued();
    copies_wait<0>();
    __syncwarp();
    float pivot = quotient(team.lanes_sum(ring.sample(0)), 32.f, 1.f / 32.f);
    float2 d[S::H];
    slice.values(ring, 0, 1, d);
#pragma unroll 1
    for (int time = 0; time < 2; ++time) {
      float2 e[S::H], t[S::H];
      slice.values(ring, 0, 0, e);
      slice.less(e, pivot);
#pragma unroll
      for (int h = 0; h < S::H; ++h) t[h] = mul2(d[h], w[h]);
      float four[4] = {sum_of(e), dot_of(e, e), sum_of(t), dot_of(t, e)};
      team.template sum<true>(four, s_sum[time]);
      bool flat;
      const float c = four[0] * inverse, c1 = four[2] * inverse, r = inverse_root(variance<false>(c, four[1], inverse, flat) + eps);
      const float2 rr = dup2(r), rc = dup2(-r * c);
      if (time == 0) {
        if (!(fabsf(rc.x) > FAR)) {
          team.template barrier<true>();       // (its sums are read)
          break;
        }
#pragma unroll
        for (int h = 0; h < S::H; ++h) dw[h] = fma2(make_float2(-d[h].x, -d[h].y), fma2(e[h], rr, rc), dw[h]);       // (as it was added)
        pivot += c;
        continue;
      }
      const float c2 = r * fmaf(-c, c1, four[3] * inverse);
      const float2 rc1 = dup2(-r * c1), rc2 = dup2(-r * c2);
#pragma unroll
      for (int h = 0; h < S::H; ++h) {
        e[h] = fma2(e[h], rr, rc);
        dw[h] = fma2(d[h], e[h], dw[h]);
        e[h] = fma2(e[h], rc2, fma2(mul2(d[h], w[h]), rr, rc1));
      }
      if (dx != nullptr) slice.store(dx + row * (width * S::S) + slice.first * S::S, e);
    }
  }
  for (int slot = 0; out != nullptr && slot < team.slots(); ++slot) {
    __syncthreads();
    if (!far || slot != team.slot) continue;
#pragma unroll
    for (int h = 0; h < S::H; ++h) {
      if (slice.has(2 * h)) out[slice.column(2 * h)] += dw[h].x;
      if (slice.has(2 * h + 1)) out[slice.column(2 * h + 1)] += dw[h].y;
    }
  }
}

template <typename T, int VB, int P, bool SHIFT, int THREADS, bool WIDE>
__global__ void __launch_bounds__(THREADS, ROW_BLOCKS<THREADS, SHIFT>) row_kernel(Rows x, int64_t rows, int width, int log_tpr, Affine a, int fp32_weights,
                                                                                         float eps, char *__restrict__ y) {
  dep_trigger();
  dep_wait();
  using S = Slice<T, VB, P, SHIFT>;
  using R = Ring<T, VB, P, 1, THREADS, ROW_BLOCKS<THREADS, SHIFT>>;
  extern __shared__ __align__(16) char s_ring[];
  __shared__ __align__(16) float s_sum[2][THREADS / 32][4];       // of rows in turn
  const R ring(s_ring);
  const Team<THREADS, WIDE> team(log_tpr);
  const int row_bytes = width * S::S;
  int64_t row = (int64_t)blockIdx.x * team.slots() + team.slot, ahead = row;
  const int64_t step = (int64_t)gridDim.x * team.slots();
  const S slice(team.lane, team.tpr(), width, x.p + row * x.stride);
  Walk from(x, rows, row, step, row_bytes, slice.first * S::S);
  char *to = y + row * row_bytes + slice.first * S::S;
  const int64_t jump = step * row_bytes, edge = SHIFT ? edge_rows(VB, x) : 0;
  auto fetch = [&](int stage) {
    if (ahead < rows) {
      slice.fetch(ring, stage, 0, from.at, SHIFT && (ahead < edge || ahead >= rows - edge), from.begin, from.end);
      if (WIDE) slice.fetch_samples(ring, stage, from.at);
    }
    copies_issued();
    from.at += from.jump, ahead += step;
  };
#pragma unroll
  for (int k = 0; k < R::DEPTH - 1; ++k) fetch(k);
  float2 w[S::H], b[S::H];
  slice.affine(a.w, fp32_weights, 1.f, w);
  slice.affine(a.b, fp32_weights, 0.f, b);
  const float inverse = 1.f / ((float)width * (WIDE ? 1.f : team.scale)), count = WIDE ? 32.f : team.lanes_sum(slice.own_samples()), inverse_count = 1.f / count;
  bool far = false;
  int stage = 0, odd = 0;
  for (int64_t base = (int64_t)blockIdx.x * team.slots(); base < rows; base += step) {
    copies_wait<R::DEPTH - 2>();
    if (WIDE) __syncwarp();
    float2 d[S::H];
    slice.values(ring, stage, 0, d);
    const float sample = WIDE ? ring.sample(stage) : slice.own_sample(d);
    fetch(stage == 0 ? R::DEPTH - 1 : stage - 1);
    stage = stage == R::DEPTH - 1 ? 0 : stage + 1;
    slice.less(d, quotient(team.lanes_sum(sample), count, inverse_count));
    float two[2] = {sum_of(d), dot_of(d, d)};
    team.sum(two, s_sum[odd]);
    odd ^= 1;
    bool flat;
    const float c = two[0] * inverse;
    float r = inverse_root(variance<!WIDE && S::MEAN>(c, two[1], inverse, flat) + eps);
    if (flat) r *= 0.f;       // (not a number where eps is zero)
    const float2 rr = dup2(r), rc = dup2(-r * c);
    if (WIDE) far |= fabsf(rc.x) > FAR;
#pragma unroll
    for (int h = 0; h < S::H; ++h) d[h] = fma2(fma2(d[h], rr, rc), w[h], b[h]);
    if (team.slots() == 1 || row < rows) slice.store(to, d);
    to += jump, row += step;
  }
  if (WIDE && far) far_rows<T, VB, P, SHIFT, THREADS>(x, rows, width, log_tpr, a, fp32_weights, eps, y);       // (the same in all threads of a team)
}

// The sums of a row are taken at once: those of e = x - k and its square, of t = g w and of t e; with c the mean of e, mean(t h) = r (mean(t e) - c mean(t)).
// Sums over rows stay in registers; a block's teams add theirs up in order.
template <typename T, int VB, int P, bool SHIFT, int THREADS, bool WIDE>
__global__ void __launch_bounds__(THREADS, GRAD_BLOCKS<THREADS>) row_grad_kernel(Rows g, Rows x, int64_t rows, int width, int log_tpr, const void *weight, int fp32_weight,
                                                                                  float eps, char *__restrict__ dx, float *__restrict__ parts) {
  dep_trigger();
  dep_wait();
  using S = Slice<T, VB, P, SHIFT>;
  using R = Ring<T, VB, P, 2, THREADS, GRAD_BLOCKS<THREADS>>;
  extern __shared__ __align__(16) char s_ring[];
  __shared__ __align__(16) float s_sum[2][THREADS / 32][4];       // of rows in turn
  __shared__ bool s_far[THREADS / 32];
  const R ring(s_ring);
  const Team<THREADS, WIDE> team(log_tpr);
  const int row_bytes = width * S::S;
  int64_t row = (int64_t)blockIdx.x * team.slots() + team.slot, ahead = row;
  const int64_t step = (int64_t)gridDim.x * team.slots();
  const S slice(team.lane, team.tpr(), width, x.p + row * x.stride);
  Walk from_x(x, rows, row, step, row_bytes, slice.first * S::S), from_g(g, rows, row, step, row_bytes, slice.first * S::S);
  char *to_dx = dx + row * row_bytes + slice.first * S::S;
  const int64_t jump = step * row_bytes, edge = SHIFT ? max(edge_rows(VB, x), edge_rows(VB, g)) : 0;
  auto fetch = [&](int stage) {
    if (ahead < rows) {
      const bool careful = SHIFT && (ahead < edge || ahead >= rows - edge);
      slice.fetch(ring, stage, 0, from_x.at, careful, from_x.begin, from_x.end);
      slice.fetch(ring, stage, 1, from_g.at, careful, from_g.begin, from_g.end);
      if (WIDE) slice.fetch_samples(ring, stage, from_x.at);
    }
    copies_issued();
    from_x.at += from_x.jump, from_g.at += from_g.jump, ahead += step;
  };
#pragma unroll
  for (int k = 0; k < R::DEPTH - 1; ++k) fetch(k);
  float2 w[S::H], dw[S::H], db[S::H];
  slice.affine(weight, fp32_weight, 1.f, w);
#pragma unroll
  for (int h = 0; h < S::H; ++h) dw[h] = db[h] = make_float2(0.f, 0.f);
  const float inverse = 1.f / ((float)width * (WIDE ? 1.f : team.scale)), count = WIDE ? 32.f : team.lanes_sum(slice.own_samples()), inverse_count = 1.f / count;
  bool far = false;
  if (S::TIGHT) s_far[threadIdx.x >> 5] = false;       // (a warp's own)
  int stage = 0, odd = 0;
  for (int64_t base = (int64_t)blockIdx.x * team.slots(); base < rows; base += step) {
    copies_wait<R::DEPTH - 2>();
    if (WIDE) __syncwarp();
    const bool there = team.slots() == 1 || row < rows;
    float2 e[S::H], d[S::H], t[S::H];
    slice.values(ring, stage, 0, e);
    slice.values(ring, stage, 1, d);
    float sample = WIDE ? ring.sample(stage) : slice.own_sample(e);
    if (!there) {       // (a team without a row goes along with the others' sums: zeros, and r is zero too)
      sample = 0.f;
#pragma unroll
      for (int h = 0; h < S::H; ++h) e[h] = d[h] = make_float2(0.f, 0.f);
    }
    fetch(stage == 0 ? R::DEPTH - 1 : stage - 1);
    stage = stage == R::DEPTH - 1 ? 0 : stage + 1;
    slice.less(e, quotient(team.lanes_sum(sample), count, inverse_count));
#pragma unroll
    for (int h = 0; h < S::H; ++h) t[h] = mul2(d[h], w[h]);
    float four[4] = {sum_of(e), dot_of(e, e), sum_of(t), dot_of(t, e)};
    team.sum(four, s_sum[odd]);
    odd ^= 1;
    const float c = four[0] * inverse, c1 = four[2] * inverse;
    bool flat;
    float r = inverse_root(variance<!WIDE && S::MEAN>(c, four[1], inverse, flat) + eps);
    if (!there) r = 0.f;
    const float c2 = r * fmaf(-c, c1, four[3] * inverse);
    const float to_h = flat ? r * 0.f : r;       // (not a number where eps is zero)
    const float2 rr = dup2(r), rh = dup2(to_h), rc = dup2(-to_h * c), rc1 = dup2(-r * c1), rc2 = dup2(-r * c2);
    if (S::TIGHT) {
      if (fabsf(rc.x) > FAR) s_far[threadIdx.x >> 5] = true;
    } else if (WIDE) {
      far |= fabsf(rc.x) > FAR;
    }
#pragma unroll
    for (int h = 0; h < S::H; ++h) {
      e[h] = fma2(e[h], rh, rc);
      dw[h] = fma2(d[h], e[h], dw[h]);
      db[h] = add2(db[h], d[h]);
      e[h] = fma2(e[h], rc2, fma2(mul2(d[h], w[h]), rr, rc1));
    }
    if (there && dx != nullptr) slice.store(to_dx, e);
    to_dx += jump, row += step;
  }
  float *const out = parts == nullptr ? nullptr : parts + (int64_t)blockIdx.x * 2 * width;
  if (out != nullptr) {
    // teams of a warp have the same columns, unless rows begin at places of their own
    int slot = team.slot, slots = team.slots();
    if (!SHIFT && team.tpr() < 32) {
      for (int o = team.tpr(); o < 32; o <<= 1)
#pragma unroll
        for (int h = 0; h < S::H; ++h) {
          dw[h] = add2(dw[h], make_float2(__shfl_xor_sync(0xffffffffu, dw[h].x, o), __shfl_xor_sync(0xffffffffu, dw[h].y, o)));
          db[h] = add2(db[h], make_float2(__shfl_xor_sync(0xffffffffu, db[h].x, o), __shfl_xor_sync(0xffffffffu, db[h].y, o)));
        }
      slots = THREADS / 32;
      slot = (threadIdx.x & 31) < team.tpr() ? (int)threadIdx.x >> 5 : -1;
    }
    copies_wait<0>();
    __syncthreads();
    float *const s_parts = reinterpret_cast<float *>(s_ring);       // [slots][2][width]
    static_assert(R::BYTES >= THREADS * S::E * 8, "room for the sums of a block's teams");
    float *to = slots == 1 ? out : s_parts + slot * 2 * width;
    if (slot >= 0)
#pragma unroll
      for (int h = 0; h < S::H; ++h) {
        const int c = slice.column(2 * h);
        if (!SHIFT && slice.has(2 * h)) {
          *reinterpret_cast<float2 *>(to + c) = dw[h];
          *reinterpret_cast<float2 *>(to + width + c) = db[h];
        } else if (SHIFT) {
          if (slice.has(2 * h)) to[c] = dw[h].x, to[width + c] = db[h].x;
          if (slice.has(2 * h + 1)) to[c + 1] = dw[h].y, to[width + c + 1] = db[h].y;
        }
      }
    if (slots > 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * width; i += THREADS) {
        float v = s_parts[i];
        for (int k = 1; k < slots; ++k) v += s_parts[k * 2 * width + i];
        out[i] = v;
      }
    }
  }
  if (S::TIGHT) far = s_far[threadIdx.x >> 5];
  if constexpr (WIDE)
    if (__syncthreads_or(far)) far_rows_grad<T, VB, P, SHIFT, THREADS>(g, x, rows, width, log_tpr, weight, fp32_weight, eps, dx, out, far);
}

// ---------------------------------------------------------------------------------------------- sums of parts
// 32 columns of [dw | db] a block; LANES threads a column take the parts in turn, their sums are added in order.
constexpr int LANES = 16;
template <typename W>
__global__ void __launch_bounds__(32 * LANES) join_kernel(const float *__restrict__ parts, int n_parts, int width, W *__restrict__ dw, W *__restrict__ db) {
  __shared__ float s_sum[LANES][32];
  dep_trigger();
  dep_wait();
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x, wide = 2ll * width;
  float sum = 0.f;
  if (col < wide)
#pragma unroll 4
    for (int k = threadIdx.y; k < n_parts; k += LANES) sum += parts[k * wide + col];
  s_sum[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || col >= wide) return;
  for (int k = 1; k < LANES; ++k) sum += s_sum[k][threadIdx.x];
  if (col < width) {
    if (dw != nullptr) dw[col] = (W)sum;
  } else if (db != nullptr) {
    db[col - width] = (W)sum;
  }
}

// ---------------------------------------------------------------------------------------------- host
constexpr int MOST_WIDTH = 1 << 24;
constexpr int MOST_PARTS = 4 * SMS;

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
struct Layout {
  int64_t parts, stats, total;            // bytes
};
// (a row of parts a piece of rows, 64 of them at least: fewer would write more parts than they read)
static int64_t most_parts(int64_t rows) { return std::min<int64_t>(MOST_PARTS, (rows + 63) / 64); }
// (rows in registers, which are of 8192 values at most, see plan: one of a block, which has a row at least, and eight blocks more or less; see blocks_of)
constexpr int MOST_IN_REGISTERS = 512 * 16;
static int64_t room_for_parts(int64_t rows, int width) {
  return width > MOST_IN_REGISTERS ? most_parts(rows) : std::max(most_parts(rows), std::min<int64_t>(SMS * GRAD_BLOCKS<256>, (rows + 7) / 8 * 8));
}
static Layout layout(int64_t rows, int width) {
  Layout l = {};
  l.stats = up256(room_for_parts(rows, width) * 2 * width * 4);
  l.total = l.stats + up256(rows * (int64_t)sizeof(Stats));
  return l;
}
static int is_type(int type) { return type == ORCA_F32 || type == ORCA_BF16 || type == ORCA_F16; }
// (weights are of the rows' type or fp32)
template <typename F> static int by_types(int type, int weight_type, int vb, F &&f) {
  return by_type(type, vb, [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (weight_type == ORCA_F32) return f(t, (float *)nullptr, v);
    return f(t, (T *)nullptr, v);
  });
}

// Blocks of a launch over rows of any width: clusters where that leaves SMs without a row else (and there is enough of a row for all of its blocks).
static cudaLaunchConfig_t any_launch(int64_t rows, int nv, cudaStream_t stream, cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t c = {};
  const int cluster = rows < SMS && nv >= 4 * ANY ? CLUSTER : 1;
  c.blockDim = std::min(ANY, (nv + 31) / 32 * 32);
  c.gridDim = (unsigned)(std::min<int64_t>(rows, 0x7fffffff / CLUSTER) * cluster);
  c.stream = stream;
  c.attrs = attr;
  if (cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    c.numAttrs = 1;
  }
  if (dependent_launch_enabled()) {
    attr[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[c.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  return c;
}

// How a row in registers is shared out: pieces of VB bytes, P a thread, 2^log_tpr threads; the fewest that have no part in it, then the fewest threads.  Not all rows of up to
// 8192 values fit: not those of fp32 with more than 4096 that lie on borders of 8 bytes alone, nor 8190 and 8191 in 16 bits, nor 8191 in fp32.
struct Plan {
  int vb, pieces, log_tpr, threads;      // pieces 0: the row does not fit
  bool shift;
  int slots() const { return threads >> log_tpr; }
};
static Plan plan(int width, int size, std::initializer_list<uint64_t> addresses, std::initializer_list<uint64_t> strides) {
  Plan p = {};
  const int64_t row = (int64_t)width * size;
  uint64_t all = (uint64_t)row, apart = 0;
  const uint64_t one = *addresses.begin();
  for (uint64_t a : addresses) all |= a, apart |= a ^ one;
  for (uint64_t a : strides) all |= a, apart |= a ^ (uint64_t)row;
  if (all % 16 == 0) p.vb = 16;
  else if (all % 8 == 0) p.vb = 8;
  else if (apart % (4 * size) == 0) p.vb = 4 * size, p.shift = true;       // (four values: wider pieces would leave half of the threads of 515 without)
  else return p;
  const int v = p.vb / size, nv = (width + v - 1 + (p.shift ? v - 1 : 0)) / v;
  const int most = v == 8 ? 2 : v == 4 ? 3 : 4;       // (four of four values do not fit the registers)
  int best = 0x7fffffff;
  for (int log = 2; log <= 8; ++log) {
    const int pieces = (nv + (1 << log) - 1) >> log;
    if (pieces > most || pieces << log >= best) continue;
    best = pieces << log;
    p.pieces = pieces, p.log_tpr = log, p.threads = 256;
  }
  if (p.pieces > 0) return p;
  const int pieces = (nv + 511) / 512;
  if (pieces <= std::min(4, 16 / v)) p.pieces = pieces, p.log_tpr = 9, p.threads = 512;
  return p;
}
// f(piece bytes, pieces, shift, threads, several warps a row) as constants
template <typename T, typename F> static int by_plan(const Plan &p, F &&f) {
  auto threads = [&](auto vb, auto pieces, auto shift) {
    constexpr int V = decltype(vb)::value / (int)sizeof(T), P = decltype(pieces)::value;
    if constexpr (P > (V == 2 ? 2 : 1)) {      // (256 threads have the others)
      if (p.threads == 512) return f(vb, pieces, shift, std::integral_constant<int, 512>(), std::true_type());
    }
    if constexpr (V != 4 || P < 4) {
      if (p.log_tpr > 5) return f(vb, pieces, shift, std::integral_constant<int, 256>(), std::true_type());
      return f(vb, pieces, shift, std::integral_constant<int, 256>(), std::false_type());
    }
    return set_error(ORCA_E_UNSUPPORTED, "%d pieces of %d bytes, %d threads", p.pieces, p.vb, p.threads);
  };
  auto pieces = [&](auto vb, auto shift) {
    if (p.pieces == 1) return threads(vb, std::integral_constant<int, 1>(), shift);
    if (p.pieces == 2) return threads(vb, std::integral_constant<int, 2>(), shift);
    if constexpr (decltype(vb)::value / (int)sizeof(T) <= 4) {
      if (p.pieces == 3) return threads(vb, std::integral_constant<int, 3>(), shift);
      if (p.pieces == 4) return threads(vb, std::integral_constant<int, 4>(), shift);
    }
    return set_error(ORCA_E_UNSUPPORTED, "%d pieces of %d bytes", p.pieces, p.vb);
  };
  if (p.shift) return pieces(std::integral_constant<int, 4 * (int)sizeof(T)>(), std::true_type());
  if (p.vb == 8) return pieces(std::integral_constant<int, 8>(), std::false_type());
  return pieces(std::integral_constant<int, 16>(), std::false_type());
}
// Blocks of a launch over `rows`, `most` at most; a multiple of what makes the step between a team's rows whole pieces.
static int64_t blocks_of(const Plan &p, int64_t rows, int64_t most) {
  if (p.shift) return std::min<int64_t>(most / 8, ((rows + p.slots() - 1) / p.slots() + 7) / 8) * 8;      // (four rows are whole pieces)
  return std::min<int64_t>(most, (rows + p.slots() - 1) / p.slots());
}

}  // namespace norm
}  // namespace orca

using namespace orca;
using namespace orca::norm;

extern "C" {

int orca_layer_norm(const void *d_x, int64_t x_stride, int64_t rows, int32_t width, int32_t type, const void *d_weight, const void *d_bias,
                    int32_t weight_type, float eps, void *d_out, void *stream) {
  ORCA_CHECK_ARG(rows >= 0 && width > 0 && width <= norm::MOST_WIDTH && x_stride >= 0 && eps >= 0.f && eps <= 3.402823466e38f);
  ORCA_CHECK_ARG(rows == 0 || (d_x && d_out));
  if (!is_type(type) || (weight_type != type && weight_type != ORCA_F32))
    return set_error(ORCA_E_UNSUPPORTED, "%s: rows of type %d, weights of type %d", __func__, type, weight_type);
  const int size = size_of(type), wsize = size_of(weight_type);
  ORCA_CHECK_ARG(((uintptr_t)d_x | (uintptr_t)d_out) % size == 0 && ((uintptr_t)d_weight | (uintptr_t)d_bias) % wsize == 0);
  if (rows == 0) return ORCA_OK;
  const Rows x = {(const char *)d_x, x_stride * size};
  const Affine a = {d_weight, d_bias};
  cudaStream_t s = (cudaStream_t)stream;
  const Plan p = plan(width, size, {(uint64_t)(uintptr_t)d_x, (uint64_t)(uintptr_t)d_out}, {(uint64_t)x.stride});
  if (p.pieces > 0)
    return by_type(type, 16, [&](auto *t, auto) {
      using T = std::remove_pointer_t<decltype(t)>;
      return by_plan<T>(p, [&](auto vb, auto pieces, auto shift, auto threads, auto wide) {
        constexpr int N = decltype(threads)::value;
        auto kernel = row_kernel<T, decltype(vb)::value, decltype(pieces)::value, decltype(shift)::value, N, decltype(wide)::value>;
        constexpr int BLOCKS = ROW_BLOCKS<N, decltype(shift)::value>, smem = Ring<T, decltype(vb)::value, decltype(pieces)::value, 1, N, BLOCKS>::BYTES;
        static std::atomic<uint64_t> ready;
        if (const int rc = allow_shared(kernel, smem, ready)) return rc;
        ORCA_CUDA(launch_dep(kernel, (unsigned)blocks_of(p, rows, SMS * BLOCKS), N, smem, s, x, rows, width, p.log_tpr, a,
                             (int)(weight_type == ORCA_F32), eps, (char *)d_out));
        ORCA_COUNT_LAUNCH();
        ORCA_LAUNCH_CHECK();
        return (int)ORCA_OK;
      });
    });
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_x, (uint64_t)(uintptr_t)d_out, (uint64_t)(x_stride * size)});
  return by_types(type, weight_type, vb, [&](auto *t, auto *w, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    constexpr int VB = decltype(v)::value;
    const int nv = width * size / VB;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t c = any_launch(rows, nv, s, attr);
    ORCA_CUDA(cudaLaunchKernelEx(&c, any_kernel<T, W, VB>, x, rows, nv, (int)width, a, eps, (char *)d_out));
    ORCA_COUNT_LAUNCH();
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

int64_t orca_layer_norm_grad_workspace_bytes(int64_t rows, int32_t width) {
  if (rows < 0 || rows > (1ll << 40) || width <= 0 || width > norm::MOST_WIDTH) return -1;
  return norm::layout(rows, width).total;
}

int orca_layer_norm_grad(const void *d_grad_out, int64_t grad_stride, const void *d_x, int64_t x_stride, int64_t rows, int32_t width, int32_t type,
                         const void *d_weight, int32_t weight_type, float eps, void *d_grad_x, void *d_grad_weight, void *d_grad_bias,
                         void *d_workspace, int64_t workspace_bytes, void *stream) {
  ORCA_CHECK_ARG(rows >= 0 && rows <= (1ll << 40) && width > 0 && width <= norm::MOST_WIDTH && x_stride >= 0 && grad_stride >= 0 && eps >= 0.f && eps <= 3.402823466e38f);
  ORCA_CHECK_ARG(rows == 0 || (d_x && d_grad_out));
  if (!is_type(type) || (weight_type != type && weight_type != ORCA_F32))
    return set_error(ORCA_E_UNSUPPORTED, "%s: rows of type %d, weights of type %d", __func__, type, weight_type);
  const int size = size_of(type), wsize = size_of(weight_type);
  ORCA_CHECK_ARG(((uintptr_t)d_x | (uintptr_t)d_grad_out | (uintptr_t)d_grad_x) % size == 0 &&
                 ((uintptr_t)d_weight | (uintptr_t)d_grad_weight | (uintptr_t)d_grad_bias) % wsize == 0);
  const bool sums = d_grad_weight != nullptr || d_grad_bias != nullptr;
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    if (d_grad_weight) ORCA_CUDA(cudaMemsetAsync(d_grad_weight, 0, (size_t)width * wsize, s));
    if (d_grad_bias) ORCA_CUDA(cudaMemsetAsync(d_grad_bias, 0, (size_t)width * wsize, s));
    return ORCA_OK;
  }
  if (!sums && d_grad_x == nullptr) return ORCA_OK;
  const norm::Layout L = norm::layout(rows, width);
  if (sums) {
    ORCA_CHECK_ARG(d_workspace && (uintptr_t)d_workspace % 256 == 0);
    if (workspace_bytes < L.total) return set_error(ORCA_E_BADARG, "%s: workspace of %lld bytes is too small", __func__, (long long)workspace_bytes);
  }
  float *parts = (float *)((char *)d_workspace + L.parts);
  Stats *stats = sums ? (Stats *)((char *)d_workspace + L.stats) : nullptr;
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_x, (uint64_t)(uintptr_t)d_grad_out, (uint64_t)(uintptr_t)d_grad_x,
                                               (uint64_t)(x_stride * size), (uint64_t)(grad_stride * size)});
  const Rows x = {(const char *)d_x, x_stride * size}, g = {(const char *)d_grad_out, grad_stride * size};
  const Plan p = plan(width, size, {(uint64_t)(uintptr_t)d_x, (uint64_t)(uintptr_t)d_grad_out, (uint64_t)(uintptr_t)(d_grad_x ? d_grad_x : d_x)},
                      {(uint64_t)x.stride, (uint64_t)g.stride});
  auto join = [&](auto *w, int64_t n_parts) {
    using W = std::remove_pointer_t<decltype(w)>;
    ORCA_CUDA(launch_dep(join_kernel<W>, (unsigned)((2ll * width + 31) / 32), dim3(32, LANES), 0, s, (const float *)parts, (int)n_parts, width,
                         (W *)d_grad_weight, (W *)d_grad_bias));
    ORCA_COUNT_LAUNCH();
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  };
  if (p.pieces > 0)
    return by_types(type, weight_type, 16, [&](auto *t, auto *w, auto) {
      using T = std::remove_pointer_t<decltype(t)>;
      using W = std::remove_pointer_t<decltype(w)>;
      const int64_t blocks = blocks_of(p, rows, SMS * (p.threads == 512 ? GRAD_BLOCKS<512> : GRAD_BLOCKS<256>));
      if (sums && blocks > room_for_parts(rows, width)) return set_error(ORCA_E_CAPACITY, "%s: %lld parts", "orca_layer_norm_grad", (long long)blocks);
      const int rc = by_plan<T>(p, [&](auto vb, auto pieces, auto shift, auto threads, auto wide) {
        constexpr int N = decltype(threads)::value;
        auto kernel = row_grad_kernel<T, decltype(vb)::value, decltype(pieces)::value, decltype(shift)::value, N, decltype(wide)::value>;
        constexpr int smem = Ring<T, decltype(vb)::value, decltype(pieces)::value, 2, N, GRAD_BLOCKS<N>>::BYTES;
        static std::atomic<uint64_t> ready;
        if (const int rc = allow_shared(kernel, smem, ready)) return rc;
        ORCA_CUDA(launch_dep(kernel, (unsigned)blocks, N, smem, s, g, x, rows, width, p.log_tpr, d_weight, (int)(weight_type == ORCA_F32), eps,
                             (char *)d_grad_x, sums ? parts : nullptr));
        ORCA_COUNT_LAUNCH();
        ORCA_LAUNCH_CHECK();
        return (int)ORCA_OK;
      });
      if (rc != ORCA_OK || !sums) return rc;
      return join(w, blocks);
    });
  return by_types(type, weight_type, vb, [&](auto *t, auto *w, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    constexpr int VB = decltype(v)::value;
    const int nv = width * size / VB;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t c = any_launch(rows, nv, s, attr);
    ORCA_CUDA(cudaLaunchKernelEx(&c, any_grad_kernel<T, W, VB>, g, x, rows, nv, (int)width, Affine{d_weight, nullptr}, eps, (char *)d_grad_x, stats));
    ORCA_COUNT_LAUNCH();
    if (sums) {
      const int strips = (nv + STRIP - 1) / STRIP;
      const int64_t want = std::max<int64_t>(1, std::min<int64_t>(most_parts(rows), 8 * MOST_PARTS / strips)), share = (rows + want - 1) / want;
      const int n_parts = (int)((rows + share - 1) / share);
      ORCA_CUDA(launch_dep(any_sums_kernel<T, VB>, dim3(strips, n_parts), STRIP, 0, s, g, x, rows, share, nv, width, (const Stats *)stats, parts));
      ORCA_COUNT_LAUNCH();
      return join(w, n_parts);
    }
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

}  // extern "C"
