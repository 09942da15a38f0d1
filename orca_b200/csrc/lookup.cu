// Rows of a trained table by id, times a scale, and the gradient of the table by sorted ids.
//
// Both are bound by HBM: a lookup reads and writes a row an id, the gradient reads a row an id and writes every row of the table
// once.  The gradient sorts (id, position) pairs, stably, so that a row's contributions lie side by side in the order of their positions; chunks
// of the sorted list are then summed by themselves.  A stretch of equal ids that lies in one chunk goes straight to its row; one that
// crosses a border leaves a sum on either side, which a second kernel adds in the order of the chunks.  No atomics: the same bits
// every time, and a hub that fills half of the list is spread over as many chunks as it needs.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "context.cuh"
#include "radix.cuh"

namespace orca {
namespace rows {

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

struct Ids {
  const void *p;
  int wide;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return wide ? reinterpret_cast<const int64_t *>(p)[i] : reinterpret_cast<const int32_t *>(p)[i];
  }
};

__device__ __forceinline__ int detail(int64_t i) { return (int)(i < 0x7fffffff ? i : 0x7fffffff); }

// tx threads a row (a power of two), nv pieces of VB bytes a row
template <typename T, int VB>
__global__ void __launch_bounds__(256) lookup_kernel(const char *__restrict__ table, int64_t n_rows, int64_t stride, int nv, int tx,
                                                     Ids ids, int64_t n, float scale, char *__restrict__ out, int32_t *status) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  const int t = threadIdx.x % tx;
  const int64_t i = (int64_t)blockIdx.x * (256 / tx) + threadIdx.x / tx;
  if (i >= n) return;
  const int64_t v = ids.at(i);
  const bool ok = v >= 0 && v < n_rows;
  if (!ok && t == 0) report(status, ORCA_E_BOUNDS, detail(i));
  for (int c = t; c < nv; c += tx) {
    float x[X::N] = {};
    if (ok) X::load(table + v * stride + (int64_t)c * VB, x);
    X::store(out + (i * nv + c) * VB, x, scale);
  }
}

// ---------------------------------------------------------------------------------------------- sorting
// key n_rows: an id that has no gradient
struct First {
  typedef uint2 Item;
  static constexpr int RUN = 256;
  Ids ids;
  int64_t n_rows, padding;
  int32_t *status;
  __device__ bool skip() const { return false; }
  __device__ Item load(int64_t i) const {
    const int64_t v = ids.at(i);
    if (v < 0 || v >= n_rows) report(status, ORCA_E_BOUNDS, detail(i));
    return make_uint2((uint32_t)(v < 0 || v >= n_rows || v == padding ? n_rows : v), (uint32_t)i);
  }
  __device__ int digit(Item x) const { return (int)(x.x & 0xff); }
};
struct Next {
  typedef uint2 Item;
  static constexpr int RUN = First::RUN;
  const uint2 *in;
  int shift;
  __device__ bool skip() const { return false; }
  __device__ Item load(int64_t i) const { return in[i]; }
  __device__ int digit(Item x) const { return (int)((x.x >> shift) & 0xff); }
};

// ---------------------------------------------------------------------------------------------- sums
constexpr int CHUNK = 32;      // sorted pairs a block sums

// Sums of chunk blockIdx.x.  The stretch that began in an earlier chunk goes to half 0 of the chunk's partial sums, the one that goes
// on into the next chunk (and began here) to half 1.
template <typename T, int VB>
__global__ void __launch_bounds__(256) sum_kernel(const char *__restrict__ g, int64_t stride, int nv, const uint2 *__restrict__ sorted,
                                                  int64_t n, int64_t n_rows, float scale, char *__restrict__ grad,
                                                  float *__restrict__ partial) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  constexpr int AHEAD = 8;
  __shared__ uint2 s_rec[CHUNK + 2];
  const int64_t beg = (int64_t)blockIdx.x * CHUNK;
  const int m = (int)(n - beg < CHUNK ? n - beg : CHUNK);
  // record 0: the one before the chunk, m + 1: the one behind it (a key that nothing has, at the ends)
  for (int i = threadIdx.x; i < m + 2; i += blockDim.x) {
    const int64_t at = beg + i - 1;
    s_rec[i] = at >= 0 && at < n ? sorted[at] : make_uint2(0xffffffffu, 0u);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < nv; c += blockDim.x) {
    float a[X::N] = {};
    bool before = s_rec[0].x == s_rec[1].x;
    for (int r0 = 0; r0 < m; r0 += AHEAD) {
      float x[AHEAD][X::N];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (r0 + u < m && s_rec[r0 + u + 1].x < n_rows) X::load(g + (int64_t)s_rec[r0 + u + 1].y * stride + (int64_t)c * VB, x[u]);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int r = r0 + u;
        const uint32_t key = s_rec[min(r, m - 1) + 1].x;
        if (r >= m || key >= n_rows) break;
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] += x[u][e];
        const bool goes_on = s_rec[r + 2].x == key;
        if (goes_on && r + 1 < m) continue;
        if (!before && !goes_on) {
          X::store(grad + ((int64_t)key * nv + c) * VB, a, scale);
        } else {
          float *p = partial + (((int64_t)blockIdx.x * 2 + (before ? 0 : 1)) * nv + c) * X::N;
#pragma unroll
          for (int e = 0; e < X::N; ++e) p[e] = a[e];
        }
        before = false;
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] = 0.f;
      }
    }
  }
}

// Stretches over several chunks: the block of the chunk where one begins adds its partial sums.  JOIN_Y threads a column take the
// chunks in turn.
constexpr int JOIN_Y = 4;
template <typename T, int VB>
__global__ void __launch_bounds__(256) join_kernel(int nv, const uint2 *__restrict__ sorted, int64_t n, int64_t n_rows, float scale,
                                                   char *__restrict__ grad, const float *__restrict__ partial) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  __shared__ float s_sum[JOIN_Y - 1][64][X::N];
  const int64_t beg = (int64_t)blockIdx.x * CHUNK, end = beg + CHUNK;
  if (end >= n) return;                            // the last chunk: nothing goes on
  const uint32_t key = sorted[end - 1].x;
  if (key >= n_rows || sorted[end].x != key) return;
  if (beg > 0 && sorted[beg].x == key && sorted[beg - 1].x == key) return;     // begun before this chunk
  int64_t lo = end, hi = n;                        // the stretch ends at the first larger key
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (sorted[mid].x > key) hi = mid;
    else lo = mid + 1;
  }
  const int64_t last = (lo - 1) / CHUNK;           // its last chunk
  const int t = threadIdx.x % 64, y = threadIdx.x / 64;
  for (int c0 = 0; c0 < nv; c0 += 64) {
    const int c = c0 + t;
    float a[X::N] = {};
    if (c < nv)
      for (int64_t k = blockIdx.x + y; k <= last; k += JOIN_Y) {
        const float *p = partial + ((k * 2 + (k == blockIdx.x ? 1 : 0)) * nv + c) * X::N;
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] += p[e];
      }
    if (y > 0)
#pragma unroll
      for (int e = 0; e < X::N; ++e) s_sum[y - 1][t][e] = a[e];
    __syncthreads();
    if (y == 0 && c < nv) {
      for (int k = 0; k < JOIN_Y - 1; ++k)
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] += s_sum[k][t][e];
      X::store(grad + ((int64_t)key * nv + c) * VB, a, scale);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- host
static int64_t up256(int64_t b) { return (b + 255) & ~255ll; }
static int size_of(int type) { return type == ORCA_F32 ? 4 : 2; }

struct Layout {
  int64_t a, b, counts, totals, partial, total;
  int blocks;
};
static Layout layout(int64_t n, int width) {
  Layout L;
  const int64_t tile = radix::WARPS * First::RUN;
  L.blocks = (int)((n + tile - 1) / tile);
  L.a = 0;
  L.b = up256(n * 8);
  L.counts = L.b + up256(n * 8);
  L.totals = L.counts + up256((int64_t)radix::BINS * L.blocks * 4);
  L.partial = L.totals + up256(radix::BINS * 4);
  L.total = L.partial + up256((n + CHUNK - 1) / CHUNK * 2 * width * 4);
  return L;
}

// largest piece that rows can be read and written by
static int piece(int64_t row_bytes, std::initializer_list<uint64_t> at) {
  uint64_t all = (uint64_t)row_bytes | 16;
  for (uint64_t a : at) all |= a;
  const int vb = (int)(all & (~all + 1));
  return vb > 16 ? 16 : vb;
}

template <typename F>
static int by_type(int type, int vb, F &&f) {
  if (type == ORCA_F32) return vb == 16 ? f((float *)nullptr, std::integral_constant<int, 16>()) : vb == 8 ? f((float *)nullptr, std::integral_constant<int, 8>()) : f((float *)nullptr, std::integral_constant<int, 4>());
  if (type == ORCA_BF16)
    return vb == 16 ? f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 16>()) : vb == 8 ? f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 8>())
         : vb == 4 ? f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 4>()) : f((__nv_bfloat16 *)nullptr, std::integral_constant<int, 2>());
  return vb == 16 ? f((__half *)nullptr, std::integral_constant<int, 16>()) : vb == 8 ? f((__half *)nullptr, std::integral_constant<int, 8>())
       : vb == 4 ? f((__half *)nullptr, std::integral_constant<int, 4>()) : f((__half *)nullptr, std::integral_constant<int, 2>());
}

}  // namespace rows
}  // namespace orca

using namespace orca;
using namespace orca::rows;

extern "C" {

int orca_rows_lookup(const void *d_table, int64_t n_rows, int64_t table_stride, int32_t width, int32_t type, const void *d_ids,
                     int32_t ids64, int64_t n, float scale, void *d_out, int32_t *d_status, void *stream) {
  ORCA_CHECK_ARG(n >= 0 && n_rows >= 0 && n_rows < 0x7fffffffll && width > 0 && table_stride >= width);
  ORCA_CHECK_ARG(n == 0 || (d_ids && d_out && (d_table || n_rows == 0)));
  if (type != ORCA_F32 && type != ORCA_BF16 && type != ORCA_F16) return set_error(ORCA_E_UNSUPPORTED, "%s: type %d", __func__, type);
  const int size = size_of(type);
  ORCA_CHECK_ARG((uintptr_t)d_table % size == 0 && (uintptr_t)d_out % size == 0 && (uintptr_t)d_ids % (ids64 ? 8 : 4) == 0);
  if (n == 0) return ORCA_OK;
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_table, (uint64_t)(uintptr_t)d_out, (uint64_t)(table_stride * size)});
  const int nv = width * size / vb;
  int tx = 1;
  while (tx < nv && tx < 256) tx *= 2;
  const int64_t blocks = (n + 256 / tx - 1) / (256 / tx);
  ORCA_CHECK_ARG(blocks <= 0x7fffffffll);
  return by_type(type, vb, [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    ORCA_CUDA(launch_dep(lookup_kernel<T, decltype(v)::value>, (unsigned)blocks, 256, 0, (cudaStream_t)stream, (const char *)d_table,
                         n_rows, table_stride * size, nv, tx, Ids{d_ids, ids64}, n, scale, (char *)d_out, d_status));
    ORCA_COUNT_LAUNCH();
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

int64_t orca_rows_grad_workspace_bytes(int64_t n, int64_t n_rows, int32_t width) {
  if (n < 0 || n >= 0x7fffffffll || n_rows < 0 || n_rows >= 0x7fffffffll || width <= 0) return -1;
  return layout(n, width).total;
}

int orca_rows_grad(const void *d_grad_out, int64_t grad_stride, int32_t width, int32_t type, const void *d_ids, int32_t ids64,
                   int64_t n, int64_t n_rows, float scale, int64_t padding, void *d_grad, int32_t *d_status, void *d_workspace,
                   int64_t workspace_bytes, void *stream) {
  ORCA_CHECK_ARG(n >= 0 && n < 0x7fffffffll && n_rows >= 0 && n_rows < 0x7fffffffll && width > 0 && (grad_stride >= width || grad_stride == 0));
  ORCA_CHECK_ARG((n == 0 || (d_grad_out && d_ids)) && (n_rows == 0 || d_grad));
  if (type != ORCA_F32 && type != ORCA_BF16 && type != ORCA_F16) return set_error(ORCA_E_UNSUPPORTED, "%s: type %d", __func__, type);
  const int size = size_of(type);
  ORCA_CHECK_ARG((uintptr_t)d_grad_out % size == 0 && (uintptr_t)d_grad % size == 0 && (uintptr_t)d_ids % (ids64 ? 8 : 4) == 0);
  cudaStream_t s = (cudaStream_t)stream;
  const Layout L = layout(n, width);
  if (n > 0 && n_rows > 0) {
    ORCA_CHECK_ARG(d_workspace && (uintptr_t)d_workspace % 256 == 0);
    if (workspace_bytes < L.total) return set_error(ORCA_E_BADARG, "%s: workspace of %lld bytes is too small", __func__, (long long)workspace_bytes);
  }
  if (n_rows > 0) ORCA_CUDA(cudaMemsetAsync(d_grad, 0, (size_t)n_rows * width * size, s));
  if (n == 0 || n_rows == 0) return ORCA_OK;
  char *w = (char *)d_workspace;
  int32_t *counts = (int32_t *)(w + L.counts), *totals = (int32_t *)(w + L.totals);
  uint2 *half[2] = {(uint2 *)(w + L.a), (uint2 *)(w + L.b)};
  int rc = radix::one_pass(First{{d_ids, ids64}, n_rows, padding, d_status}, n, half[0], counts, totals, nullptr, s);
  if (rc) return rc;
  int at = 0;
  for (int shift = 8; shift < 32 && (n_rows >> shift) != 0; shift += 8, at ^= 1) {
    rc = radix::one_pass(Next{half[at], shift}, n, half[at ^ 1], counts, totals, nullptr, s);
    if (rc) return rc;
  }
  const uint2 *sorted = half[at];
  float *partial = (float *)(w + L.partial);
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_grad_out, (uint64_t)(uintptr_t)d_grad, (uint64_t)(grad_stride * size)});
  const int nv = width * size / vb;
  const int threads = std::min(256, (nv + 31) / 32 * 32);
  const unsigned chunks = (unsigned)((n + CHUNK - 1) / CHUNK);
  return by_type(type, vb, [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int VB = decltype(v)::value;
    ORCA_CUDA(launch_dep(sum_kernel<T, VB>, chunks, threads, 0, s, (const char *)d_grad_out, grad_stride * size, nv, sorted, n, n_rows, scale,
                         (char *)d_grad, partial));
    ORCA_COUNT_LAUNCH();
    if (chunks > 1) {
      ORCA_CUDA(launch_dep(join_kernel<T, VB>, chunks, 64 * JOIN_Y, 0, s, nv, sorted, n, n_rows, scale, (char *)d_grad, (const float *)partial));
      ORCA_COUNT_LAUNCH();
    }
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

}  // extern "C"
