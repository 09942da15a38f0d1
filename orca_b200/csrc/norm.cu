// Layer norm over the last dimension, and its gradients.
//
//   m = mean of x, r = 1 / sqrt(mean of (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   with d = g w:  dx = r (d - mean(d) - h mean(d h)),  dw = sum over rows of g h,  db = sum over rows of g
//
// Bound by HBM: a row is read once and written once, backward two are read and one is written.  Nothing is kept from the forward pass: backward has x
// in its hands and finds m and r again, by the same steps.  The mean is taken twice: what is left of the mean of x - m is taken off as well,
// because m rounded to 32 bits misses by as much as a row varies where its mean is 2^24 times that.
// dw and db: each block sums its rows into a row of parts, in order, and another kernel adds up the parts: the same bits every time.
#include <algorithm>

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

template <typename W, int N> __device__ __forceinline__ void load_affine(const void *p, int64_t at, float otherwise, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = p == nullptr ? otherwise : (float)reinterpret_cast<const W *>(p)[at + i];
}

// Sums over a block, the same bits in every thread: warps' sums, then theirs in order.
template <int THREADS, int K> __device__ __forceinline__ void block_sum(float (&v)[K], float (*s)[K]) {
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  __syncthreads();       // (s is read by the sums before)
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) s[warp][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) v[k] += s[w][k];
  }
}

// ---------------------------------------------------------------------------------------------- rows of any width
// A block a row, which it goes through again for each sum: from L2 after the first time.
constexpr int ANY = 512;
template <typename T, int VB> __device__ __forceinline__ Stats any_stats(const char *x, int nv, int width, float eps) {
  using X = Vec<T, VB>;
  __shared__ float s_one[ANY / 32][1], s_two[ANY / 32][2];
  float one[1] = {0.f}, two[2] = {0.f, 0.f};
  for (int v = threadIdx.x; v < nv; v += ANY) {
    float a[X::N];
    X::load(x + (int64_t)v * VB, a);
#pragma unroll
    for (int i = 0; i < X::N; ++i) one[0] += a[i];
  }
  block_sum<ANY>(one, s_one);
  Stats t;
  t.m = one[0] / (float)width;
  for (int v = threadIdx.x; v < nv; v += ANY) {
    float a[X::N];
    X::load(x + (int64_t)v * VB, a);
#pragma unroll
    for (int i = 0; i < X::N; ++i) {
      const float e = a[i] - t.m;
      two[0] += e;
      two[1] += e * e;
    }
  }
  block_sum<ANY>(two, s_two);
  t.c = two[0] / (float)width;
  t.r = 1.f / sqrtf(fmaxf(two[1] / (float)width - t.c * t.c, 0.f) + eps);
  return t;
}

template <typename T, typename W, int VB>
__global__ void __launch_bounds__(ANY) any_kernel(Rows x, int64_t rows, int nv, int width, Affine a, float eps, char *__restrict__ y) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const char *p = x.p + row * x.stride;
    const Stats t = any_stats<T, VB>(p, nv, width, eps);
    for (int v = threadIdx.x; v < nv; v += ANY) {
      float e[X::N], w[X::N], b[X::N];
      X::load(p + (int64_t)v * VB, e);
      load_affine<W>(a.w, (int64_t)v * X::N, 1.f, w);
      load_affine<W>(a.b, (int64_t)v * X::N, 0.f, b);
#pragma unroll
      for (int i = 0; i < X::N; ++i) e[i] = fmaf(((e[i] - t.m) - t.c) * t.r, w[i], b[i]);
      X::store(y + (row * nv + v) * VB, e, 1.f);
    }
  }
}

// dx where it is wanted; the rows' statistics for the sums over rows where those are.
template <typename T, typename W, int VB>
__global__ void __launch_bounds__(ANY) any_grad_kernel(Rows g, Rows x, int64_t rows, int nv, int width, Affine a, float eps, char *__restrict__ dx,
                                                       Stats *__restrict__ stats) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  __shared__ float s_sum[ANY / 32][2];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const char *px = x.p + row * x.stride, *pg = g.p + row * g.stride;
    const Stats t = any_stats<T, VB>(px, nv, width, eps);
    if (stats != nullptr && threadIdx.x == 0) stats[row] = t;
    if (dx == nullptr) continue;
    float sum[2] = {0.f, 0.f};
    for (int v = threadIdx.x; v < nv; v += ANY) {
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
    block_sum<ANY>(sum, s_sum);
    const float c1 = sum[0] / (float)width, c2 = sum[1] / (float)width;
    for (int v = threadIdx.x; v < nv; v += ANY) {
      float e[X::N], d[X::N], w[X::N];
      X::load(px + (int64_t)v * VB, e);
      X::load(pg + (int64_t)v * VB, d);
      load_affine<W>(a.w, (int64_t)v * X::N, 1.f, w);
#pragma unroll
      for (int i = 0; i < X::N; ++i) e[i] = t.r * (fmaf(d[i], w[i], -c1) - ((e[i] - t.m) - t.c) * t.r * c2);
      X::store(dx + (row * nv + v) * VB, e, 1.f);
    }
  }
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
constexpr int MOST_PARTS = 592;           // four blocks of sums an SM of 148

static int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
struct Layout {
  int64_t parts, stats, total;            // bytes
};
// (a row of parts a piece of rows, 64 of them at least: fewer would write more parts than they read)
static int64_t most_parts(int64_t rows) { return std::min<int64_t>(MOST_PARTS, (rows + 63) / 64); }
static Layout layout(int64_t rows, int width) {
  Layout l = {};
  l.stats = up256(most_parts(rows) * 2 * width * 4);
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
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_x, (uint64_t)(uintptr_t)d_out, (uint64_t)(x_stride * size)});
  return by_types(type, weight_type, vb, [&](auto *t, auto *w, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    constexpr int VB = decltype(v)::value;
    ORCA_CUDA(launch_dep(any_kernel<T, W, VB>, (unsigned)std::min<int64_t>(rows, 0x7fffffff), ANY, 0, (cudaStream_t)stream,
                         Rows{(const char *)d_x, x_stride * size}, rows, width * size / VB, width, Affine{d_weight, d_bias}, eps, (char *)d_out));
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
  return by_types(type, weight_type, vb, [&](auto *t, auto *w, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    constexpr int VB = decltype(v)::value;
    const int nv = width * size / VB;
    ORCA_CUDA(launch_dep(any_grad_kernel<T, W, VB>, (unsigned)std::min<int64_t>(rows, 0x7fffffff), ANY, 0, s, g, x, rows, nv, width,
                         Affine{d_weight, nullptr}, eps, (char *)d_grad_x, stats));
    ORCA_COUNT_LAUNCH();
    if (sums) {
      const int strips = (nv + STRIP - 1) / STRIP;
      const int64_t want = std::max<int64_t>(1, std::min<int64_t>(most_parts(rows), 8 * MOST_PARTS / strips)), share = (rows + want - 1) / want;
      const int n_parts = (int)((rows + share - 1) / share);
      ORCA_CUDA(launch_dep(any_sums_kernel<T, VB>, dim3(strips, n_parts), STRIP, 0, s, g, x, rows, share, nv, width, (const Stats *)stats, parts));
      ORCA_COUNT_LAUNCH();
      ORCA_CUDA(launch_dep(join_kernel<W>, (unsigned)((2ll * width + 31) / 32), dim3(32, LANES), 0, s, (const float *)parts, n_parts, width,
                           (W *)d_grad_weight, (W *)d_grad_bias));
      ORCA_COUNT_LAUNCH();
    }
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

}  // extern "C"
