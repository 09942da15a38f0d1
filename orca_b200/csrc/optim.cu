// A step of AdamW over many tensors at once, gradients cut to a norm over all of them, moments in 32 or in 8 bits.
//
//   g' = g f, f = min(1, max_norm / norm) in 32 bits;  m' = b1 m + (1 - b1) g';  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
//
// Bound by HBM: 28 bytes an element of fp32 with moments in 32 bits, 16 with 8, 10 of bf16 with 8; the norm reads the gradients before.  One launch
// for all tensors of a type (their addresses are arguments of the kernel, so that a step needs no copy and can be captured), a block a chunk of a
// tensor.  Steps are counted on the device, a count a tensor: the last block of a launch to finish adds one to those of its tensors.
//
// Moments in 8 bits, by blocks of BLOCK elements of a tensor.  A block has an exponent E, that of its largest magnitude as a float, 33 at
// least (so that every value held is a normal number); 255 where that is not finite: the block is NaN then.  A mean is sign, 4 bits of exponent and
// 3 of mantissa, a square 5 bits of exponent and 3 of mantissa; the binade that E names has exponent TOP (one above is left to what rounds
// up into it), 0 is the subnormal one.  Bits of a float whose binade is moved there are positions on the scale of codes: 20 bits behind the point.
// Rounding adds 20 bits that follow from step and place (dither) and cuts: to the nearest, a square that moves by a thousandth a step
// would never leave its code, an eighth of a binade.  A square that is not zero has code 1 at least: a mean is never divided by a square
// that was lost while the mean was not; the smallest of either are 2^-16 and 2^-32 of the block's largest, so their ratio is that of the largest.
// Codes follow from m' and v' in 32 bits; products and sums that lead there are rounded as they are written (rn), whatever the compiler would make of them.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "context.cuh"
#include "vec.cuh"

namespace orca {
namespace optim {

constexpr int BLOCK = 256;                // elements that share an exponent
constexpr int TOP_MEAN = 14, TOP_SQUARE = 30;
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int CHUNK = 4096;               // elements of a tensor a block of threads takes
constexpr int MOST_GROUPS = 8;            // of a launch
constexpr int FEW = 48, MANY = 480;       // tensors of a launch: its arguments are copied with it, and end at 32 764 bytes
constexpr int PARTS = 592;                // blocks of the norm, four an SM

struct Entry {
  void *p;
  const void *g;
  void *m, *v;
  uint8_t *e;                             // [blocks][2], moments in 8 bits
  int32_t *step;
  int64_t n;
  uint32_t first;                         // chunk
  int32_t group;
};
template <int CAP> struct Table {
  int32_t count;
  uint32_t chunks;
  Entry of[CAP];
};
struct Group {
  double lr, b1, b2, eps, decay;
  const float *d_lr;                      // instead of lr
};
struct Groups { Group of[MOST_GROUPS]; };
struct Work {                             // of an optimiser, zero at first
  uint32_t ticket;
  uint32_t pad[15];
  double parts[PARTS];
};

template <int CAP> __device__ __forceinline__ int entry_of(const Table<CAP> &t, uint32_t chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.of[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------------------------- norm
// Squares are summed in 64 bits: the factor is the same whatever the tensors' order, but for one case in millions.
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double block_sum64(double v) {      // in every thread
  __shared__ double s_sum[WARPS];
  v = warp_sum64(v);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v += s_sum[w];
  return v;
}
template <typename T, int CAP>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ Table<CAP> t, Work *work, int add) {
  dep_trigger();
  dep_wait();
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const Entry &e = t.of[entry_of(t, chunk)];
    const int64_t first = (int64_t)(chunk - e.first) * CHUNK, end = min(first + CHUNK, e.n);
    for (int64_t i = first + threadIdx.x; i < end; i += THREADS) {
      const double x = (double)(float)reinterpret_cast<const T *>(e.g)[i];
      sum = fma(x, x, sum);
    }
  }
  sum = block_sum64(sum);
  if (threadIdx.x == 0) work->parts[blockIdx.x] = add ? work->parts[blockIdx.x] + sum : sum;
}

// ---------------------------------------------------------------------------------------------- 8 bits
__device__ __forceinline__ float bits(uint32_t b) { return __uint_as_float(b); }
// exponent of a block from the bits of its largest magnitude
__device__ __forceinline__ int exponent_of(uint32_t largest) { return max((int)(largest >> 23), 33); }
// x of a block with exponent e as a float whose binade e has exponent TOP: two products, for one power of two may be out of range
template <int TOP> __device__ __forceinline__ uint32_t position(float x, float up) { return __float_as_uint(__fmul_rn(__fmul_rn(x, up), bits((uint32_t)(TOP - 1) << 23))); }
__device__ __forceinline__ float up_of(int e) { return bits((uint32_t)(255 - e) << 23); }          // 2^(128 - e)
// and back: the block's power of two, NaN for a block that is not finite
__device__ __forceinline__ float down_of(int e) { return e == 255 ? bits(0x7fc00000u) : bits((uint32_t)e << 23); }   // 2^(e - 127)
template <int TOP> __device__ __forceinline__ float value(uint32_t code, float down) { return bits(code << 20) * bits((uint32_t)(254 - TOP) << 23) * down; }

// 20 bits for an element: the place's group of eight and the step through two rounds of multiplications (odd fractions of the golden ratio and
// of the roots of 2 and 3), then two steps an element of the linear congruence of Press et al., Numerical Recipes, 1992.
__device__ __forceinline__ uint32_t dither_of(int64_t eight, uint32_t step) {
  uint32_t x = (uint32_t)eight * 0x9e3779b1u + (uint32_t)(eight >> 32) * 0x6a09e667u + step * 0xbb67ae85u;
  x = (x ^ (x >> 16)) * 0x6a09e667u;
  x = (x ^ (x >> 15)) * 0xbb67ae85u;
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t next_dither(uint32_t &x) { return (x = x * 1664525u + 1013904223u) >> 12; }

// ---------------------------------------------------------------------------------------------- the step
struct Coefficients {
  float factor, b1, c1, b2, c2;           // c: one less b, rounded
  float size, root, eps, keep;            // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps, 1 - lr wd
  uint32_t step;
  bool skip;
};
__device__ __forceinline__ double power(double b, uint32_t t) {
  double r = 1.0;
  for (; t != 0; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}
__device__ __forceinline__ float next_mean(const Coefficients &c, float m, float g) { return __fmaf_rn(c.b1, m, __fmul_rn(c.c1, g)); }
__device__ __forceinline__ float next_square(const Coefficients &c, float v, float g) { return __fmaf_rn(c.b2, v, __fmul_rn(c.c2, __fmul_rn(g, g))); }
__device__ __forceinline__ float next_param(const Coefficients &c, float p, float m, float v) {
  return fmaf(p, c.keep, -c.size * m / fmaf(sqrtf(v), c.root, c.eps));
}

struct Norm {                             // max_norm below zero: none
  double max_norm;
  int parts;
  float *out;
};

template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(THREADS) step_kernel(const __grid_constant__ Table<CAP> t, const __grid_constant__ Groups groups, Norm norm, Work *work) {
  __shared__ Coefficients s_c;
  __shared__ int s_last;
  dep_trigger();
  dep_wait();
  const Entry &e = t.of[entry_of(t, blockIdx.x)];
  double total = 0.0;
  if (norm.max_norm >= 0.0) {
    for (int k = threadIdx.x; k < norm.parts; k += THREADS) total += work->parts[k];
    total = sqrt(block_sum64(total));
  }
  if (threadIdx.x == 0) {
    const Group &h = groups.of[e.group];
    Coefficients c;
    c.step = (uint32_t)*e.step + 1u;
    const double lr = h.d_lr != nullptr ? (double)*h.d_lr : h.lr;
    c.b1 = (float)h.b1, c.c1 = (float)(1.0 - h.b1), c.b2 = (float)h.b2, c.c2 = (float)(1.0 - h.b2);
    c.size = (float)(lr / (1.0 - power(h.b1, c.step)));
    c.root = (float)(1.0 / sqrt(1.0 - power(h.b2, c.step)));
    c.eps = (float)h.eps, c.keep = (float)(1.0 - lr * h.decay);
    c.factor = 1.f, c.skip = false;
    if (norm.max_norm >= 0.0) {
      c.skip = !isfinite(total);
      if (total > norm.max_norm) c.factor = (float)(norm.max_norm / total);
      if (blockIdx.x == 0) *norm.out = (float)total;
    }
    s_c = c;
  }
  __syncthreads();
  const Coefficients c = s_c;
  if (!c.skip) {
    const int64_t first = (int64_t)(blockIdx.x - e.first) * CHUNK, end = min(first + CHUNK, e.n);
    T *p = reinterpret_cast<T *>(e.p);
    const T *g = reinterpret_cast<const T *>(e.g);
    if constexpr (BITS == 32) {
      float *m = reinterpret_cast<float *>(e.m), *v = reinterpret_cast<float *>(e.v);
      for (int64_t i = first + threadIdx.x; i < end; i += THREADS) {
        const float gi = (float)g[i] * c.factor, mi = next_mean(c, m[i], gi), vi = next_square(c, v[i], gi);
        m[i] = mi, v[i] = vi;
        p[i] = (T)next_param(c, (float)p[i], mi, vi);
      }
    } else {
      uint8_t *m = reinterpret_cast<uint8_t *>(e.m), *v = reinterpret_cast<uint8_t *>(e.v);
      const int lane = threadIdx.x & 31;
      for (int64_t b = first + (threadIdx.x >> 5) * BLOCK; b < end; b += WARPS * BLOCK) {
        uint8_t *exponents = e.e + b / BLOCK * 2;
        const float down_m = down_of(exponents[0]), down_v = down_of(exponents[1]);
        const int64_t at = b + lane * 8;
        float mi[8], vi[8];
        uint32_t top_m = 0, top_v = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool in = at + k < end;
          const float gi = in ? __fmul_rn((float)g[at + k], c.factor) : 0.f;
          const uint32_t cm = in ? m[at + k] : 0u, cv = in ? v[at + k] : 0u;
          const float old = value<TOP_MEAN>(cm & 127u, down_m);
          mi[k] = in ? next_mean(c, cm > 127u ? -old : old, gi) : 0.f;
          vi[k] = in ? next_square(c, value<TOP_SQUARE>(cv, down_v), gi) : 0.f;
          if (in) p[at + k] = (T)next_param(c, (float)p[at + k], mi[k], vi[k]);
          top_m = max(top_m, __float_as_uint(mi[k]) & 0x7fffffffu);
          top_v = max(top_v, __float_as_uint(vi[k]) & 0x7fffffffu);
        }
        const int em = exponent_of(__reduce_max_sync(0xffffffffu, top_m)), ev = exponent_of(__reduce_max_sync(0xffffffffu, top_v));
        __syncwarp();
        if (lane == 0) exponents[0] = (uint8_t)em, exponents[1] = (uint8_t)ev;
        const float up_m = em == 255 ? 0.f : up_of(em), up_v = ev == 255 ? 0.f : up_of(ev);
        uint32_t x = dither_of(at >> 3, c.step);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t cm = (position<TOP_MEAN>(fabsf(mi[k]), up_m) + next_dither(x)) >> 20;
          uint32_t cv = (position<TOP_SQUARE>(vi[k], up_v) + next_dither(x)) >> 20;
          if (vi[k] > 0.f) cv = max(cv, 1u);
          if (at + k < end) {
            m[at + k] = (uint8_t)((cm & 127u) | (__float_as_uint(mi[k]) >> 31 << 7));
            v[at + k] = (uint8_t)cv;
          }
        }
      }
    }
  }
  // the last block to finish counts the step
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicInc(&work->ticket, gridDim.x - 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (s_last && !c.skip)
    for (int k = threadIdx.x; k < t.count; k += THREADS) *t.of[k].step += 1;
}

// ---------------------------------------------------------------------------------------------- values of moments
// p: the means' values, g: the squares' (bf16, which holds every value exactly)
template <int CAP>
__global__ void __launch_bounds__(THREADS) moments_kernel(const __grid_constant__ Table<CAP> t) {
  dep_trigger();
  dep_wait();
  const Entry &e = t.of[entry_of(t, blockIdx.x)];
  const int64_t first = (int64_t)(blockIdx.x - e.first) * CHUNK, end = min(first + CHUNK, e.n);
  const uint8_t *m = reinterpret_cast<const uint8_t *>(e.m), *v = reinterpret_cast<const uint8_t *>(e.v);
  __nv_bfloat16 *mean = reinterpret_cast<__nv_bfloat16 *>(e.p), *square = reinterpret_cast<__nv_bfloat16 *>(const_cast<void *>(e.g));
  for (int64_t i = first + threadIdx.x; i < end; i += THREADS) {
    const uint8_t *exponents = e.e + i / BLOCK * 2;
    const float x = value<TOP_MEAN>(m[i] & 127u, down_of(exponents[0]));
    mean[i] = __float2bfloat16_rn(m[i] > 127 ? -x : x);
    square[i] = __float2bfloat16_rn(value<TOP_SQUARE>(v[i], down_of(exponents[1])));
  }
}

// ---------------------------------------------------------------------------------------------- host
static int is_type(int type) { return type == ORCA_F32 || type == ORCA_BF16 || type == ORCA_F16; }

// (one of a tensor without elements: its step is counted)
static int64_t chunks_of(int64_t n) { return std::max<int64_t>(1, (n + CHUNK - 1) / CHUNK); }

// Calls run(table) with as many tensors at a time as fit: those of `type` (negative: of any), and of up to MOST_GROUPS groups.
// `groups` gets the numbers of the groups that the table's entries name.
template <int CAP, typename F>
static int tables(const orca_adamw_tensor_t *h, int n, int type, F &&run) {
  static thread_local Table<CAP> t;
  int numbers[MOST_GROUPS], n_groups = 0;
  t.count = 0, t.chunks = 0;
  auto flush = [&]() -> int {
    if (t.count == 0) return ORCA_OK;
    const int rc = run(t, numbers, n_groups);
    t.count = 0, t.chunks = 0, n_groups = 0;
    return rc;
  };
  for (int i = 0; i < n; ++i) {
    if (type >= 0 && h[i].type != type) continue;
    int g = 0;
    while (g < n_groups && numbers[g] != h[i].group) ++g;
    const uint32_t chunks = (uint32_t)chunks_of(h[i].n);
    if (t.count == CAP || g == MOST_GROUPS || t.chunks + (uint64_t)chunks > 0x7fffffffu) {
      if (const int rc = flush()) return rc;
      g = 0;
    }
    if (g == n_groups) numbers[n_groups++] = h[i].group;
    t.of[t.count++] = Entry{h[i].param, h[i].grad, h[i].mean, h[i].square, h[i].exponents, h[i].step, h[i].n, t.chunks, g};
    t.chunks += chunks;
  }
  return flush();
}
template <typename F> static int by_size(int n, F &&f) { return n <= FEW ? f(std::integral_constant<int, FEW>()) : f(std::integral_constant<int, MANY>()); }
template <typename F> static int each_type(F &&f) {
  int rc = f(ORCA_F32, (float *)nullptr);
  if (rc == ORCA_OK) rc = f(ORCA_BF16, (__nv_bfloat16 *)nullptr);
  return rc == ORCA_OK ? f(ORCA_F16, (__half *)nullptr) : rc;
}

static int check_tensors(const char *who, const orca_adamw_tensor_t *h, int n, int n_groups, int bits) {
  for (int i = 0; i < n; ++i) {
    const orca_adamw_tensor_t &t = h[i];
    if (!is_type(t.type)) return set_error(ORCA_E_UNSUPPORTED, "%s: tensor %d of type %d", who, i, t.type);
    const int size = size_of(t.type);
    if (t.n < 0 || t.n > (int64_t)0x7fffffff * CHUNK || t.group < 0 || t.group >= n_groups)
      return set_error(ORCA_E_BADARG, "%s: tensor %d: %lld elements, group %d of %d", who, i, (long long)t.n, t.group, n_groups);
    if (!t.step || (uintptr_t)t.step % 4 ||
        (t.n > 0 && (!t.param || !t.grad || !t.mean || !t.square || (bits == 8 && !t.exponents) || ((uintptr_t)t.param | (uintptr_t)t.grad) % size ||
                     (bits == 32 && ((uintptr_t)t.mean | (uintptr_t)t.square) % 4))))
      return set_error(ORCA_E_BADARG, "%s: tensor %d: a pointer is missing or not aligned to its type", who, i);
  }
  return ORCA_OK;
}

}  // namespace optim
}  // namespace orca

using namespace orca;
using namespace orca::optim;

extern "C" {

int64_t orca_adamw_work_bytes(void) { return sizeof(Work); }

int orca_adamw_step(const orca_adamw_tensor_t *h_tensors, int32_t n_tensors, const orca_adamw_group_t *h_groups, int32_t n_groups, int32_t bits,
                    double max_norm, float *d_norm, void *d_work, void *stream) {
  ORCA_CHECK_ARG(n_tensors >= 0 && n_groups >= 0 && (n_tensors == 0 || (h_tensors && h_groups)) && d_work && (uintptr_t)d_work % 64 == 0);
  ORCA_CHECK_ARG((bits == 32 || bits == 8) && !(max_norm != max_norm) && (max_norm < 0.0 || d_norm));
  if (const int rc = check_tensors(__func__, h_tensors, n_tensors, n_groups, bits)) return rc;
  for (int g = 0; g < n_groups; ++g) {
    const orca_adamw_group_t &h = h_groups[g];
    ORCA_CHECK_ARG(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0 && h.eps >= 0.0 && (uintptr_t)h.d_lr % 4 == 0);
  }
  cudaStream_t s = (cudaStream_t)stream;
  Work *work = (Work *)d_work;
  Norm norm = {max_norm, 0, d_norm};
  int64_t chunks = 0;
  for (int i = 0; i < n_tensors; ++i) chunks += chunks_of(h_tensors[i].n);
  if (max_norm >= 0.0 && chunks == 0) ORCA_CUDA(cudaMemsetAsync(d_norm, 0, 4, s));
  return by_size(n_tensors, [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    if (max_norm >= 0.0) {
      const int rc = each_type([&](int type, auto *of) {
        using T = std::remove_pointer_t<decltype(of)>;
        return tables<CAP>(h_tensors, n_tensors, type, [&](const Table<CAP> &t, const int *, int) {
          const int add = norm.parts > 0;      // (later launches add to the parts of the first)
          norm.parts = (int)std::min<int64_t>(PARTS, chunks);
          ORCA_CUDA(launch_dep(norm_kernel<T, CAP>, (unsigned)norm.parts, THREADS, 0, s, t, work, add));
          ORCA_COUNT_LAUNCH();
          return (int)ORCA_OK;
        });
      });
      if (rc != ORCA_OK) return rc;
    }
    return each_type([&](int type, auto *of) {
      using T = std::remove_pointer_t<decltype(of)>;
      return tables<CAP>(h_tensors, n_tensors, type, [&](const Table<CAP> &t, const int *numbers, int count) {
        Groups groups = {};
        for (int g = 0; g < count; ++g) {
          const orca_adamw_group_t &h = h_groups[numbers[g]];
          groups.of[g] = Group{h.lr, h.beta1, h.beta2, h.eps, h.weight_decay, h.d_lr};
        }
        if (bits == 8) ORCA_CUDA(launch_dep(step_kernel<T, 8, CAP>, t.chunks, THREADS, 0, s, t, groups, norm, work));
        else ORCA_CUDA(launch_dep(step_kernel<T, 32, CAP>, t.chunks, THREADS, 0, s, t, groups, norm, work));
        ORCA_COUNT_LAUNCH();
        ORCA_LAUNCH_CHECK();
        return (int)ORCA_OK;
      });
    });
  });
}

int orca_adamw_moments(const orca_adamw_tensor_t *h_tensors, int32_t n_tensors, void *stream) {
  ORCA_CHECK_ARG(n_tensors >= 0 && (n_tensors == 0 || h_tensors));
  for (int i = 0; i < n_tensors; ++i) {
    const orca_adamw_tensor_t &t = h_tensors[i];
    if (t.n < 0 || t.n > (int64_t)0x7fffffff * CHUNK || (t.n > 0 && (!t.param || !t.grad || !t.mean || !t.square || !t.exponents || ((uintptr_t)t.param | (uintptr_t)t.grad) % 2)))
      return set_error(ORCA_E_BADARG, "%s: tensor %d: %lld elements, or a pointer is missing or not aligned", __func__, i, (long long)t.n);
  }
  return by_size(n_tensors, [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    return tables<CAP>(h_tensors, n_tensors, -1, [&](const Table<CAP> &t, const int *, int) {
      ORCA_CUDA(launch_dep(moments_kernel<CAP>, t.chunks, THREADS, 0, (cudaStream_t)stream, t));
      ORCA_COUNT_LAUNCH();
      ORCA_LAUNCH_CHECK();
      return (int)ORCA_OK;
    });
  });
}

}  // extern "C"
