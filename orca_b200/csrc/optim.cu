// A step of AdamW over many tensors at once, gradients cut to a norm over all of them, moments in 32 or in 8 bits.
//
//   g' = g f, f = min(1, max_norm / norm) in 32 bits;  m' = b1 m + (1 - b1) g';  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
//
// Bound by HBM: 28 bytes an element of fp32 with moments in 32 bits, 16 with 8, 10 of bf16 with 8; the norm reads the gradients before.  One launch
// for all tensors of a type (their addresses are arguments of the kernel, so that a step needs no copy and can be captured), a block a chunk of a
// tensor.  Steps are counted on the device, a count a tensor: the block of a launch that is the last to read its tensor's count adds one to all of them.
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
#include <type_traits>

#include "attn_math.cuh"
#include "common.cuh"
#include "context.cuh"
#include "vec.cuh"

namespace orca {
namespace optim {

// (No kernel here calls dep_trigger: what follows would sit on the SMs beside the last blocks.  A step over the model's 32 tensors took 6.6 us with it and
// takes 5.2, one over 293 tensors 53 and 45.)

constexpr int BLOCK = 256;                // elements that share an exponent
constexpr int TOP_MEAN = 14, TOP_SQUARE = 30;
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int EACH = 8;                   // elements of a piece: one of a thread
constexpr int PIECES = 2;
constexpr int CHUNK = THREADS * EACH * PIECES;      // elements of a tensor a block of threads takes
constexpr int MOST_GROUPS = 8;            // of a launch
// Tensors of a launch: its arguments, 72 bytes each with the norm's, are copied by the host when it enqueues them (a step over 20 tensors with a norm takes it 15.9, 16.6 and 18.2 us
// with tables of 32, 128 and 320, over 128 tensors 29.5 with 128 and 31.3 with 320; the GPU, from a graph, 0.1 us more at most).  More than 320 take another launch.
constexpr int FEW = 32, SOME = 128, MANY = 320;
constexpr int PARTS = 1184;               // blocks of the norm, eight an SM

// What a kernel has of a tensor.  (`n` with the group's place in the launch in its top byte: arguments are copied, see FEW.)
struct NormEntry {
  const void *g;
  int64_t n;
  static NormEntry of(const orca_adamw_tensor_t &t, int) { return {t.grad, t.n}; }
};
template <int BITS> struct StepEntry {
  void *p;
  const void *g;
  void *m, *v;
  int32_t *step;
  int64_t n_group;
  static StepEntry of(const orca_adamw_tensor_t &t, int group) { return {t.param, t.grad, t.mean, t.square, t.step, t.n | (int64_t)group << 56}; }
  __device__ __forceinline__ int64_t n() const { return n_group & ((1ll << 56) - 1); }
  __device__ __forceinline__ int group() const { return (int)(n_group >> 56); }
  __device__ __forceinline__ uint8_t *exponents() const { return nullptr; }
};
template <> struct StepEntry<8> : StepEntry<32> {
  uint8_t *e;                             // [blocks][2]
  static StepEntry of(const orca_adamw_tensor_t &t, int group) { return {StepEntry<32>::of(t, group), t.exponents}; }
  __device__ __forceinline__ uint8_t *exponents() const { return e; }
};
struct MomentsEntry {
  __nv_bfloat16 *mean, *square;           // written
  const uint8_t *m, *v, *e;
  int64_t n;
  static MomentsEntry of(const orca_adamw_tensor_t &t, int) {
    return {(__nv_bfloat16 *)t.param, (__nv_bfloat16 *)const_cast<void *>(t.grad), (const uint8_t *)t.mean, (const uint8_t *)t.square, t.exponents, t.n};
  }
};
template <typename E, int CAP> struct Table {
  int32_t count;
  uint32_t chunks;
  uint32_t first[CAP];                    // chunk of each tensor: searched by every block, so side by side
  E of[CAP];
};
struct Group {
  double lr, b1, b2, eps, decay;
  const float *d_lr;                      // instead of lr
};
struct Groups { Group of[MOST_GROUPS]; };
struct Work {                             // of an optimiser, zero at first
  uint32_t ticket, norm_ticket;
  uint32_t pad[12];
  double norm;
  double parts[PARTS];
};

static_assert(sizeof(Table<StepEntry<8>, MANY>) + sizeof(Groups) + 64 <= 32764, "a launch's arguments");

template <typename E, int CAP> __device__ __forceinline__ int entry_of(const Table<E, CAP> &t, uint32_t chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------------------------- pieces
// EACH elements of type E (one, two or four bytes) from element i on as words, zero from `end` on; at once where they are all there and lie on a border.
template <int WORDS> __device__ __forceinline__ void load_words(const void *p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 8) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
  } else if constexpr (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  }
}
template <int WORDS> __device__ __forceinline__ void store_words(void *p, const uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 8)
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p) : "memory");
  else if constexpr (WORDS == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
}
template <int SIZE> struct Unsigned { using type = uint32_t; };
template <> struct Unsigned<1> { using type = uint8_t; };
template <> struct Unsigned<2> { using type = uint16_t; };
template <bool WHOLE = false, typename E, typename I, int WORDS>
__device__ __forceinline__ void load(const E *p, I i, I end, bool wide, uint32_t (&w)[WORDS]) {
  constexpr int S = (int)sizeof(E);
  static_assert(WORDS * 4 == EACH * S, "a piece");
  if (WHOLE || (wide && i + EACH <= end)) {
    load_words(p + i, w);
  } else {
#pragma unroll
    for (int k = 0; k < WORDS; ++k) w[k] = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if (i + k < end) w[k * S / 4] |= (uint32_t)reinterpret_cast<const typename Unsigned<S>::type *>(p)[i + k] << 8 * (k * S % 4);
  }
}
template <bool WHOLE = false, typename E, typename I, int WORDS>
__device__ __forceinline__ void store(E *p, I i, I end, bool wide, const uint32_t (&w)[WORDS]) {
  constexpr int S = sizeof(E);
  if (WHOLE || (wide && i + EACH <= end)) {
    store_words(p + i, w);
  } else {
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if (i + k < end) reinterpret_cast<typename Unsigned<S>::type *>(p)[i + k] = (typename Unsigned<S>::type)(w[k * S / 4] >> 8 * (k * S % 4));
  }
}

// ---------------------------------------------------------------------------------------------- norm
// Squares are summed as if in 64 bits, so that the factor does not depend on the order of sums but for one case in millions.  A thread's pieces
// are summed in 32 bits with what each rounding leaves (two sums, of even and odd elements), and that goes on in 64 bits: conversions of every
// element kept the pass at a third of the memory's rate (392 MB of bf16: 172 us, 80 so).  What a rounding leaves is found from the sum before and after, which is exact as
// long as the sum before is no smaller than the square: sums begin at a power of two that none of the thread's squares is above, and that is taken off again (exactly).
// The result is off by 2^-40 of it at most: eight remainders a sum, each rounded to 2^-24 of 2^-19 times the largest square.  (Begun at zero it is off by up to 2^-24, whenever a
// square is larger than the sum so far.)  Squares that leave the range of 32 bits are taken in 64.
__device__ __forceinline__ float largest3(float a, float b, float c) {       // of magnitudes, NaN if one is
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T, int W> __device__ __forceinline__ double squares(const uint32_t (&w)[PIECES][W]) {
  constexpr int H = EACH / 2, PW = Pair<T>::WORDS;
  float largest = 0.f;
#pragma unroll
  for (int k = 0; k < PIECES; ++k)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float2 x = Pair<T>::of(w[k] + h * PW);
      largest = largest3(largest, x.x, x.y);
    }
  if (largest == 0.f) return 0.0;
  const float binade = __uint_as_float(__float_as_uint(largest) & 0x7f800000u);
  if (binade >= 9.3132257e-10f && binade <= 2.8823038e+17f) {       // 2^-30, 2^58
    const float begin = 4.f * binade * binade;
    float2 sum = dup2(begin), rest = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float2 x = Pair<T>::of(w[k] + h * PW), next = fma2(x, x, sum), by = add2(next, make_float2(-sum.x, -sum.y));
        rest = add2(rest, fma2(x, x, make_float2(-by.x, -by.y)));
        sum = next;
      }
    return ((double)(sum.x - begin) + (double)(sum.y - begin)) + (double)(rest.x + rest.y);
  }
  double exact = 0.0;
#pragma unroll
  for (int k = 0; k < PIECES; ++k)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float2 x = Pair<T>::of(w[k] + h * PW);
      exact = fma((double)x.x, (double)x.x, exact);
      exact = fma((double)x.y, (double)x.y, exact);
    }
  return exact;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double block_sum64(double v) {      // in every thread
  __shared__ double s_sum[WARPS];
  v = warp_sum64(v);
  __syncthreads();          // (another sum's are read)
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v += s_sum[w];
  return v;
}
template <typename T, int CAP>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ Table<NormEntry, CAP> t, Work *work, int add, float *__restrict__ out) {
  dep_wait();
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const int at = entry_of(t, chunk);
    const NormEntry &e = t.of[at];
    const int64_t first = (int64_t)(chunk - t.first[at]) * CHUNK, end = min(first + CHUNK, e.n);
    const bool wide = (uintptr_t)e.g % (EACH * sizeof(T)) == 0;
    uint32_t g[PIECES][EACH * sizeof(T) / 4];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) load(reinterpret_cast<const T *>(e.g), first + (k * THREADS + threadIdx.x) * EACH, end, wide, g[k]);
    sum += squares<T>(g);
  }
  sum = block_sum64(sum);
  // The last block to finish adds the parts up, in their order.
  __shared__ int s_last;
  if (threadIdx.x == 0) {
    work->parts[blockIdx.x] = add ? work->parts[blockIdx.x] + sum : sum;
    __threadfence();
    s_last = atomicInc(&work->norm_ticket, gridDim.x - 1) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  sum = 0.0;
  for (int k = threadIdx.x; k < (int)gridDim.x; k += THREADS) sum += __ldcg(&work->parts[k]);
  sum = sqrt(block_sum64(sum));
  if (threadIdx.x == 0) work->norm = sum, *out = (float)sum;
}

// ---------------------------------------------------------------------------------------------- 8 bits
__device__ __forceinline__ float bits(uint32_t b) { return __uint_as_float(b); }
// exponent of a block from its largest magnitude
__device__ __forceinline__ int exponent_of(uint32_t largest) { return max((int)(largest >> 23), 33); }
// Values of a block with exponent e as floats whose binade e has exponent TOP, and back: by 2^(TOP - e) and 2^(e - TOP).  Those are floats themselves for blocks
// of values below 2^14 (SMALL), in two products for any: 2^(128 - e) and 2^(TOP - 128), 2^(127 - TOP) and 2^(e - 127); NaN for a block that is not finite.
constexpr int SMALL_E = 140;
template <int TOP, bool SMALL> __device__ __forceinline__ float up_of(int e) {
  return SMALL ? bits((uint32_t)(127 + TOP - e) << 23) : e == 255 ? 0.f : bits((uint32_t)(255 - e) << 23);
}
template <int TOP, bool SMALL> __device__ __forceinline__ float2 scaled(float2 x, float up) {
  const float2 y = mul2(x, dup2(up));
  return SMALL ? y : mul2(y, dup2(bits((uint32_t)(TOP - 1) << 23)));
}
template <int TOP, bool SMALL> __device__ __forceinline__ float down_of(int e) {
  return SMALL ? bits((uint32_t)(127 - TOP + e) << 23) : e == 255 ? bits(0x7fc00000u) : bits((uint32_t)e << 23);
}
template <int TOP, bool SMALL> __device__ __forceinline__ float2 values(uint32_t a, uint32_t b, float down) {
  const float2 y = make_float2(bits(a), bits(b));
  return mul2(SMALL ? y : mul2(y, dup2(bits((uint32_t)(254 - TOP) << 23))), dup2(down));
}
// The values of eight codes: byte j of a word to bits 20 to 27 (a mean's sign to bit 31).
template <bool SMALL> __device__ __forceinline__ void means_of(const uint32_t (&w)[2], int e, float2 (&x)[EACH / 2]) {
  const float down = down_of<TOP_MEAN, SMALL>(e);
#pragma unroll
  for (int h = 0; h < EACH / 2; ++h) {
    const uint32_t v = w[h / 2], a = v << (h & 1 ? 8 : 24), b = v << (h & 1 ? 0 : 16);
    x[h] = values<TOP_MEAN, SMALL>((uint32_t)((int)a >> 4) & 0x87f00000u, (uint32_t)((int)b >> 4) & 0x87f00000u, down);
  }
}
template <bool SMALL> __device__ __forceinline__ void squares_of(const uint32_t (&w)[2], int e, float2 (&x)[EACH / 2]) {
  const float down = down_of<TOP_SQUARE, SMALL>(e);
#pragma unroll
  for (int h = 0; h < EACH / 2; ++h) {
    const uint32_t v = w[h / 2];
    x[h] = values<TOP_SQUARE, SMALL>((h & 1 ? v << 4 : v << 20) & 0x0ff00000u, (h & 1 ? v >> 4 : v << 12) & 0x0ff00000u, down);
  }
}
// The top bytes of four words
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// 20 bits for an element: the place's group of eight and the step through two rounds of multiplications (odd fractions of the golden ratio and
// of the roots of 2 and 3), then two steps an element of the linear congruence of Press et al., Numerical Recipes, 1992.
__device__ __forceinline__ uint32_t dither_of(int64_t eight, uint32_t step) {
  uint32_t x = (uint32_t)eight * 0x9e3779b1u + (uint32_t)(eight >> 32) * 0x6a09e667u + step * 0xbb67ae85u;
  x = (x ^ (x >> 16)) * 0x6a09e667u;
  x = (x ^ (x >> 15)) * 0xbb67ae85u;
  return x ^ (x >> 16);
}
__device__ __forceinline__ uint32_t next_dither(uint32_t &x) { return (x = x * 1664525u + 1013904223u) >> 12; }

// A shift that stands by itself: (x + y) << 4 in C++ was folded with the selection of bytes behind it and lost for every other value (nvcc 12.9).
__device__ __forceinline__ uint32_t four_left(uint32_t x) {
  uint32_t y;
  asm("shl.b32 %0, %1, 4;" : "=r"(y) : "r"(x));
  return y;
}

// A thread's eight moments to two words of codes each.
template <bool SMALL>
__device__ __forceinline__ void codes_of(const float2 (&mean)[EACH / 2], const float2 (&square)[EACH / 2], int em, int ev, uint32_t x, uint32_t (&wm)[2], uint32_t (&wv)[2]) {
  const float up_m = up_of<TOP_MEAN, SMALL>(em), up_v = up_of<TOP_SQUARE, SMALL>(ev);
  uint32_t cm[EACH], cv[EACH];
#pragma unroll
  for (int h = 0; h < EACH / 2; ++h) {
    const float2 a = scaled<TOP_MEAN, SMALL>(mean[h], up_m), b = scaled<TOP_SQUARE, SMALL>(square[h], up_v);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      cm[2 * h + j] = four_left(__float_as_uint(j ? a.y : a.x) + next_dither(x));       // (never as far as the sign, which leaves here)
      uint32_t to = __float_as_uint(j ? b.y : b.x) + next_dither(x);
      if ((j ? square[h].y : square[h].x) > 0.f) to = max(to, 1u << 20);
      cv[2 * h + j] = four_left(to);
    }
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float2 a = mean[2 * q], b = mean[2 * q + 1];
    const uint32_t signs = top_bytes(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
    wm[q] = top_bytes(cm[4 * q], cm[4 * q + 1], cm[4 * q + 2], cm[4 * q + 3]) | (signs & 0x80808080u);
    wv[q] = top_bytes(cv[4 * q], cv[4 * q + 1], cv[4 * q + 2], cv[4 * q + 3]);
  }
}
// The exponents of a warp's block: of means and of squares.  Elements behind the end are zero.
__device__ __forceinline__ int2 exponents_of(const float2 (&mean)[EACH / 2], const float2 (&square)[EACH / 2]) {
  float top_m = 0.f, top_v = 0.f;
#pragma unroll
  for (int h = 0; h < EACH / 2; ++h) top_m = largest3(top_m, mean[h].x, mean[h].y), top_v = largest3(top_v, square[h].x, square[h].y);
  return make_int2(exponent_of(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m))), exponent_of(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v))));
}

// ---------------------------------------------------------------------------------------------- the step
struct Coefficients {
  float factor, b1, c1, b2, c2;           // c: one less b, rounded
  float size, root, eps, keep;            // -lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps, 1 - lr wd
  uint32_t step;
  int skip;
};
__device__ __forceinline__ double power(double b, uint32_t t) {
  double r = 1.0;
  for (; t != 0; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}
// Of a tensor, in every thread of the block, by two of them.  max_norm below zero: no norm was taken.  The first thread takes a ticket
// as soon as the step is read.
__device__ __forceinline__ Coefficients coefficients(const Group &h, const int32_t *step, double max_norm, Work *work, uint32_t &ticket) {
  __shared__ Coefficients s_c;
  if (threadIdx.x == 0 || threadIdx.x == 32) {
    const uint32_t t = (uint32_t)*step + 1u;
    const double b = threadIdx.x == 0 ? h.b1 : h.b2;
    const float rest = (float)(1.0 - power(b, t));
    if (threadIdx.x == 0) {
      const double lr = h.d_lr != nullptr ? (double)*h.d_lr : h.lr;
      s_c.step = t;
      s_c.b1 = (float)b, s_c.c1 = (float)(1.0 - b);
      s_c.size = -(float)lr / rest;
      s_c.keep = (float)(1.0 - lr * h.decay);
    } else {
      const double total = max_norm >= 0.0 ? work->norm : 0.0;
      s_c.b2 = (float)b, s_c.c2 = (float)(1.0 - b);
      s_c.root = rsqrtf(rest);
      s_c.eps = (float)h.eps;
      s_c.factor = max_norm >= 0.0 && total > max_norm ? (float)(max_norm / total) : 1.f;
      s_c.skip = !isfinite(total);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) ticket = atomicInc(&work->ticket, gridDim.x - 1);      // (both that read the step are here)
  return s_c;
}
// Moments and parameters of a pair.  Codes of 8 bits follow from these roundings: each product by itself but the last, which goes with the sum.
__device__ __forceinline__ float2 next_mean(const Coefficients &c, float2 m, float2 g) { return fma2(dup2(c.b1), m, mul2(dup2(c.c1), g)); }
__device__ __forceinline__ float2 next_square(const Coefficients &c, float2 v, float2 g) { return fma2(dup2(c.b2), v, mul2(dup2(c.c2), mul2(g, g))); }
// The root of a square; without SUBNORMAL of zero for one below 2^-126, which saves three of 44 instructions an element (196 M of bf16 with 8 bits 318 us, 331 with it).
template <bool SUBNORMAL> __device__ __forceinline__ float root(float x) {
  float y;
  if (SUBNORMAL) asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  else asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Whether that matters: such a root, over sqrt(1 - b2^t), is 2^-63 / sqrt(1 - b2) at most, and nothing beside an eps that is 2^25 times as large (any of 1.2e-10 and
// more with b2 = 0.999).
inline bool needs_subnormal(const orca_adamw_group_t &h) { return ldexp(1.0, -38) > h.eps * sqrt(1.0 - h.beta2); }
__device__ __forceinline__ float inverse(float x) {      // (eps is no subnormal number, and neither is the root of one)
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool SUBNORMAL> __device__ __forceinline__ float2 next_param(const Coefficients &c, float2 p, float2 m, float2 v) {
  const float2 low = fma2(make_float2(root<SUBNORMAL>(v.x), root<SUBNORMAL>(v.y)), dup2(c.root), dup2(c.eps));
  return fma2(p, dup2(c.keep), mul2(mul2(dup2(c.size), m), make_float2(inverse(low.x), inverse(low.y))));
}

// A block has a chunk, a thread N pieces of it at a time, whose loads are under way before the coefficients are known.  With 8 bits a warp's pieces are
// a block of BLOCK.  WHOLE: the chunk is full and lies where wide loads can begin.
// (Spills, bytes a thread stored and loaded: 8 bits of fp32 16 and 16 at 80 registers, of 16 bits 44 and 28 at 64.  Without them, one block an SM
// less: 134 M elements of fp32 330 us instead of 310, 196 M of bf16 347 instead of 318.)
// What it measured, us and TB/s: 196 M elements of fp32 799, 6.9; 134 M with 8 bits of fp32 307, 7.0, of bf16 217, 6.2 (44 instructions an element, three quarters of the
// cycles), with 32 bits of bf16 433, 6.8.  Blocks that go on to other chunks with the coefficients they have: 895 instead of 799, their loads do not overlap others' stores; all of
// a thread's 16 elements at once with 32 bits: as fast (797), but 293 tensors 55 instead of 51 with two blocks an SM instead of three.
template <typename T, int BITS> constexpr int AT_ONCE = BITS == 8 ? 2 : 1;
template <typename T, int BITS, bool SUBNORMAL, bool WHOLE>
__device__ __forceinline__ bool update(const StepEntry<BITS> &e, int64_t begin, const Group &h, double max_norm, Work *work, uint32_t &ticket) {
  using M = std::conditional_t<BITS == 8, uint8_t, float>;
  constexpr int PW = EACH * (int)sizeof(T) / 4, MW = EACH * (int)sizeof(M) / 4, H = EACH / 2, N = AT_ONCE<T, BITS>;
  T *p = reinterpret_cast<T *>(e.p) + begin;
  const T *g = reinterpret_cast<const T *>(e.g) + begin;
  M *m = reinterpret_cast<M *>(e.m) + begin, *v = reinterpret_cast<M *>(e.v) + begin;
  uint8_t *exponents = e.exponents() + begin / BLOCK * 2;
  const int end = WHOLE ? CHUNK : (int)min((int64_t)CHUNK, e.n() - begin);
  const bool wide = WHOLE || (((uintptr_t)p | (uintptr_t)g) % (EACH * sizeof(T)) == 0 && ((uintptr_t)m | (uintptr_t)v) % (EACH * sizeof(M)) == 0);
  Coefficients c;
#pragma unroll 1
  for (int first = threadIdx.x * EACH; first < CHUNK; first += N * THREADS * EACH) {
    uint32_t wp[N][PW], wg[N][PW], wm[N][MW], wv[N][MW], of[N] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = first + k * THREADS * EACH;
      load<WHOLE>(p, i, end, wide, wp[k]);
      load<WHOLE>(g, i, end, wide, wg[k]);
      load<WHOLE>(m, i, end, wide, wm[k]);
      load<WHOLE>(v, i, end, wide, wv[k]);
      if (BITS == 8 && (WHOLE || i / BLOCK * BLOCK < end)) of[k] = exponents[i / BLOCK * 2] | (uint32_t)exponents[i / BLOCK * 2 + 1] << 8;
    }
    if (first < N * THREADS * EACH) c = coefficients(h, e.step, max_norm, work, ticket);
    if (c.skip) return true;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = first + k * THREADS * EACH;
      if (BITS == 8 && !WHOLE && i / BLOCK * BLOCK >= end) break;          // (the warp as a whole)
      float2 mean[H], square[H];
      if constexpr (BITS == 8) {
        const int em = of[k] & 255u, ev = of[k] >> 8;
        if (max(em, ev) <= SMALL_E) means_of<true>(wm[k], em, mean), squares_of<true>(wv[k], ev, square);
        else means_of<false>(wm[k], em, mean), squares_of<false>(wv[k], ev, square);
      } else {
#pragma unroll
        for (int h = 0; h < H; ++h) mean[h] = Pair<float>::of(wm[k] + 2 * h), square[h] = Pair<float>::of(wv[k] + 2 * h);
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        constexpr int W = Pair<T>::WORDS;
        const float2 gh = mul2(Pair<T>::of(wg[k] + h * W), dup2(c.factor));
        mean[h] = next_mean(c, mean[h], gh);
        square[h] = next_square(c, square[h], gh);
        Pair<T>::to(wp[k] + h * W, next_param<SUBNORMAL>(c, Pair<T>::of(wp[k] + h * W), mean[h], square[h]));
      }
      store<WHOLE>(p, i, end, wide, wp[k]);
      if constexpr (BITS == 32) {
#pragma unroll
        for (int h = 0; h < H; ++h) Pair<float>::to(wm[k] + 2 * h, mean[h]), Pair<float>::to(wv[k] + 2 * h, square[h]);
      } else {
        const int2 now = exponents_of(mean, square);
        const uint32_t x = dither_of((begin + i) / EACH, c.step);
        if (max(now.x, now.y) <= SMALL_E) codes_of<true>(mean, square, now.x, now.y, x, wm[k], wv[k]);
        else codes_of<false>(mean, square, now.x, now.y, x, wm[k], wv[k]);
        if ((threadIdx.x & 31) == 0) exponents[i / BLOCK * 2] = (uint8_t)now.x, exponents[i / BLOCK * 2 + 1] = (uint8_t)now.y;
      }
      store<WHOLE>(m, i, end, wide, wm[k]);
      store<WHOLE>(v, i, end, wide, wv[k]);
    }
  }
  return false;
}

template <typename T, int BITS, bool SUBNORMAL, int CAP>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 ? 3 : 4)
    step_kernel(const __grid_constant__ Table<StepEntry<BITS>, CAP> t, const __grid_constant__ Groups groups, double max_norm, Work *work) {
  static_assert(32 * EACH == BLOCK, "a warp's pieces are a block");
  using M = std::conditional_t<BITS == 8, uint8_t, float>;
  dep_wait();
  // (the norm's pass ended with the last chunks, which may still be in L2)
  const uint32_t chunk = max_norm >= 0.0 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const int at = entry_of(t, chunk);
  const StepEntry<BITS> &e = t.of[at];
  const int64_t begin = (int64_t)(chunk - t.first[at]) * CHUNK;
  const bool whole = begin + CHUNK <= e.n() && ((uintptr_t)e.p | (uintptr_t)e.g) % (EACH * sizeof(T)) == 0 && ((uintptr_t)e.m | (uintptr_t)e.v) % (EACH * sizeof(M)) == 0;
  uint32_t ticket = 0;
  const Group &h = groups.of[e.group()];
  const bool skip = whole ? update<T, BITS, SUBNORMAL, true>(e, begin, h, max_norm, work, ticket) : update<T, BITS, SUBNORMAL, false>(e, begin, h, max_norm, work, ticket);
  // The block that was the last to read its tensor's step counts it, for all tensors.
  if (threadIdx.x < 32 && !skip && __shfl_sync(0xffffffffu, ticket, 0) == gridDim.x - 1)
    for (int k = threadIdx.x; k < t.count; k += 32) atomicAdd(t.of[k].step, 1);      // (nothing waits for it)
}

// ---------------------------------------------------------------------------------------------- values of moments
// (bf16 holds every value exactly)
template <int CAP>
__global__ void __launch_bounds__(THREADS) moments_kernel(const __grid_constant__ Table<MomentsEntry, CAP> t) {
  dep_wait();
  using B = __nv_bfloat16;
  const int at = entry_of(t, blockIdx.x);
  const MomentsEntry &e = t.of[at];
  const int64_t begin = (int64_t)(blockIdx.x - t.first[at]) * CHUNK, first = begin + threadIdx.x * EACH, end = min(begin + CHUNK, e.n);
  const bool wide = ((uintptr_t)e.mean | (uintptr_t)e.square) % (EACH * sizeof(B)) == 0 && ((uintptr_t)e.m | (uintptr_t)e.v) % EACH == 0;
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    const int64_t i = first + k * THREADS * EACH;
    if (i >= end) break;
    uint32_t wm[2], wv[2], out[4];
    load(e.m, i, end, wide, wm);
    load(e.v, i, end, wide, wv);
    float2 x[EACH / 2];
    means_of<false>(wm, e.e[i / BLOCK * 2], x);
#pragma unroll
    for (int h = 0; h < EACH / 2; ++h) Pair<B>::to(out + h, x[h]);
    store(e.mean, i, end, wide, out);
    squares_of<false>(wv, e.e[i / BLOCK * 2 + 1], x);
#pragma unroll
    for (int h = 0; h < EACH / 2; ++h) Pair<B>::to(out + h, x[h]);
    store(e.square, i, end, wide, out);
  }
}

// ---------------------------------------------------------------------------------------------- host
static int is_type(int type) { return type == ORCA_F32 || type == ORCA_BF16 || type == ORCA_F16; }

// (one of a tensor without elements: its step is counted)
static int64_t chunks_of(int64_t n) { return std::max<int64_t>(1, (n + CHUNK - 1) / CHUNK); }

// Calls run(table) with as many tensors at a time as fit: those of `type` (negative: of any), and of up to MOST_GROUPS groups.
// `groups` gets the numbers of the groups that the table's entries name.
template <typename E, int CAP, typename F>
static int tables(const orca_adamw_tensor_t *h, int n, int type, F &&run) {
  static thread_local Table<E, CAP> t;
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
    t.first[t.count] = t.chunks;
    t.of[t.count++] = E::of(h[i], g);
    t.chunks += chunks;
  }
  return flush();
}
template <typename F> static int by_size(int n, F &&f) {
  return n <= FEW ? f(std::integral_constant<int, FEW>()) : n <= SOME ? f(std::integral_constant<int, SOME>()) : f(std::integral_constant<int, MANY>());
}
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
  ORCA_CHECK_ARG((bits == 32 || bits == 8) && !(max_norm != max_norm) && (max_norm < 0.0 || (d_norm && (uintptr_t)d_norm % 4 == 0)));
  if (const int rc = check_tensors(__func__, h_tensors, n_tensors, n_groups, bits)) return rc;
  for (int g = 0; g < n_groups; ++g) {
    const orca_adamw_group_t &h = h_groups[g];
    ORCA_CHECK_ARG(h.beta1 >= 0.0 && h.beta1 < 1.0 && h.beta2 >= 0.0 && h.beta2 < 1.0 && (uintptr_t)h.d_lr % 4 == 0);
    ORCA_CHECK_ARG((float)h.eps == 0.f || ((float)h.eps >= 1.17549435e-38f && (float)h.eps <= 3.402823466e38f));
  }
  cudaStream_t s = (cudaStream_t)stream;
  Work *work = (Work *)d_work;
  int parts = 0;
  int64_t chunks = 0;
  for (int i = 0; i < n_tensors; ++i) chunks += chunks_of(h_tensors[i].n);
  if (max_norm >= 0.0 && chunks == 0) ORCA_CUDA(cudaMemsetAsync(d_norm, 0, 4, s));
  return by_size(n_tensors, [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    if (max_norm >= 0.0) {
      const int rc = each_type([&](int type, auto *of) {
        using T = std::remove_pointer_t<decltype(of)>;
        return tables<NormEntry, CAP>(h_tensors, n_tensors, type, [&](const auto &t, const int *, int) {
          const int add = parts > 0;      // (later launches add to the parts of the first)
          parts = (int)std::min<int64_t>(PARTS, chunks);
          ORCA_CUDA(launch_dep(norm_kernel<T, CAP>, (unsigned)parts, THREADS, 0, s, t, work, add, d_norm));
          ORCA_COUNT_LAUNCH();
          return (int)ORCA_OK;
        });
      });
      if (rc != ORCA_OK) return rc;
    }
    return each_type([&](int type, auto *of) {
      using T = std::remove_pointer_t<decltype(of)>;
      auto step = [&](auto of_bits) {
        constexpr int BITS = decltype(of_bits)::value;
        return tables<StepEntry<BITS>, CAP>(h_tensors, n_tensors, type, [&](const auto &t, const int *numbers, int count) {
          Groups groups = {};
          bool subnormal = false;
          for (int g = 0; g < count; ++g) {
            const orca_adamw_group_t &h = h_groups[numbers[g]];
            subnormal |= needs_subnormal(h);
            groups.of[g] = Group{h.lr, h.beta1, h.beta2, h.eps, h.weight_decay, h.d_lr};
          }
          ORCA_CUDA(launch_dep(subnormal ? step_kernel<T, BITS, true, CAP> : step_kernel<T, BITS, false, CAP>, t.chunks, THREADS, 0, s, t, groups, max_norm, work));
          ORCA_COUNT_LAUNCH();
          ORCA_LAUNCH_CHECK();
          return (int)ORCA_OK;
        });
      };
      return bits == 8 ? step(std::integral_constant<int, 8>()) : step(std::integral_constant<int, 32>());
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
    return tables<MomentsEntry, CAP>(h_tensors, n_tensors, -1, [&](const auto &t, const int *, int) {
      ORCA_CUDA(launch_dep(moments_kernel<CAP>, t.chunks, THREADS, 0, (cudaStream_t)stream, t));
      ORCA_COUNT_LAUNCH();
      ORCA_LAUNCH_CHECK();
      return (int)ORCA_OK;
    });
  });
}

}  // extern "C"
