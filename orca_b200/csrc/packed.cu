// Rows held in 4 bits (packed.cuh): put into a table, read from it, attended over.  Times are of a B200, which copies 6538 GB/s.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "context.cuh"
#include "packed.cuh"
#include "sampling.cuh"

namespace orca {
namespace packed {

constexpr unsigned FULL = 0xffffffffu;

// ---------------------------------------------------------------------------------------------- push and pull
// The last position of every id: record[id] = 1 + the largest position (0: none).
__global__ void __launch_bounds__(256) push_mark_kernel(const int32_t *__restrict__ ids, int n, int64_t n_rows,
                                                        int32_t *__restrict__ record, int32_t *status) {
  dep_trigger();
  dep_wait();
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
    const int v = ids[i];
    if (v < 0 || v >= n_rows) report(status, ORCA_E_BOUNDS, i);
    else atomicMax(&record[v], i + 1);
  }
}

__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}

// Whether a + b >= c, exactly (a + b and c within a factor of two of one another, or a + b - c exact).
__device__ __forceinline__ bool sum_reaches(float a, float b, float c) {
  const float s = a + b, bb = s - a;
  const float err = (a - (s - bb)) + (b - bb);      // s + err = a + b
  const float d = s - c;
  return d + err >= 0.f;
}
// How a group with these extremes is held (see packed.cuh): the offset rounded down, the step rounded up, so that 15 steps cover
// the group and a code is off by half a step at most.  15 * step is exact in 32 bits; the first bfloat16 from just below the
// quotient on that reaches the largest value is the step.
__device__ __forceinline__ uint32_t group_of(float lo, float hi) {
  const uint32_t b = __float_as_uint(lo);
  const uint32_t offset = ((int32_t)b < 0 && (b & 0xffffu) != 0 ? b + 0x10000u : b) & 0xffff0000u;
  const float off = __uint_as_float(offset), q = (hi - off) * (1.f / 15.f);
  const uint32_t at = __float_as_uint(q * (1.f - 1e-6f)) >> 16;      // (a subnormal quotient is off by a whole bfloat16 at most)
  uint32_t step = at > 0 ? at - 1 : 0;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (!sum_reaches(15.f * __uint_as_float(step << 16), off, hi)) ++step;
  return step | offset;
}
// The codes of N values, the nearest integers to (x - offset) / step, ties to even, four bits each.  Adding 2^23 rounds to an integer,
// which is then in the lowest bits.  A quotient in 32 bits is off by 15 * 4 * 2^-24 at most, so that it is wrong only next to a border
// between two codes; values there (values of 16 bits often lie on one) are held against the border itself: (k + 1/2) * step is exact, and
// so is the sign of x - (offset + (k + 1/2) * step) with the sum in two parts.
constexpr float ROUND = 8388608.f;
__device__ __noinline__ uint32_t code_of_tiny(float offset, float step, float x) {      // 1 / step overflows
  return step > 0.f ? (uint32_t)fmin(fmax(rint(((double)x - (double)offset) / (double)step), 0.0), 15.0) : 0u;
}
// (`row`: the values where they came from, for the few that are looked at again)
template <int N, typename T> __device__ __forceinline__ uint32_t codes_of(const float (&x)[N], const T *row, uint32_t how) {
  const float s = step_of(how), o = offset_of(how);
  float inv;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
  uint32_t c = 0, again = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float t = (x[j] - o) * inv, r = t + ROUND;
    if (!(fabsf(t - (r - ROUND)) < 0.49999f)) again |= 1u << j;
    c += __float_as_uint(r) << (4 * j);
  }
  c -= 0x4b000000u + (N > 1 ? 0xb0000000u : 0u);       // (what is left of the exponents of the first two; the others' are shifted out)
  if (how == 0x7fc07fc0u) return 0;
  const bool tiny = !(inv < 1e37f);
  if (tiny) again = (1u << N) - 1u;
  while (again != 0) {
    const int j = __ffs(again) - 1;
    again &= again - 1;
    const float v = (float)row[j];
    uint32_t right;
    if (tiny) {
      right = code_of_tiny(o, s, v);
    } else {
      const float t = (v - o) * inv, r = (t + ROUND) - ROUND, low = t > r ? r : r - 1.f, border = (low + 0.5f) * s;
      const float sum = o + border, bb = sum - o, err = (o - (sum - bb)) + (border - bb), above = (v - sum) - err;
      const uint32_t k = __float_as_uint(low + ROUND) & 15u;
      right = k + (above > 0.f || (above == 0.f && (k & 1u)) ? 1u : 0u);
    }
    c = (c & ~(15u << (4 * j))) | right << (4 * j);
  }
  return N < 8 ? c & ((1u << (4 * N % 32)) - 1u) : c;
}

// N neighbouring values of a row, by pieces of VB bytes.
template <int VB, int N, typename T>
__device__ __forceinline__ void load_values(const T *p, float (&x)[N]) {
  struct alignas(VB) Raw { T v[VB / sizeof(T)]; };
  constexpr int PER = VB / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < N / PER; ++i) {
    const Raw r = *reinterpret_cast<const Raw *>(p + i * PER);
#pragma unroll
    for (int j = 0; j < PER; ++j) x[i * PER + j] = (float)r.v[j];
  }
}
// smallest and largest, of which either is not a number where one of the two is none
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// the extremes of the values that N of each of sixteen lanes hold (`here`: this lane has some)
template <int N> __device__ __forceinline__ float2 extremes(const float (&x)[N], bool here) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int j = 1; j < N; ++j) lo = min_nan(lo, x[j]), hi = max_nan(hi, x[j]);
  if (!here) lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) lo = min_nan(lo, __shfl_xor_sync(FULL, lo, o)), hi = max_nan(hi, __shfl_xor_sync(FULL, hi, o));
  return make_float2(lo, hi);
}

// Bound by instructions, 195 a row of bf16 (185 of fp32): a group's extremes (four steps over sixteen lanes, of both groups), its step and offset,
// and 12 codes a lane.  73 % of what the schedulers can issue, DRAM at 18 % of its peak (fp32: 62 and 30, the rest waits for its rows).
// Two rows a warp let even lanes work out the first group's step and odd lanes the second's.
// 400 k rows of bf16 into a table of 1.14 M: 95 us, 1.9 TB/s; of fp32 101, 3.1.
// Sixteen lanes a row, two rows a warp: lane h packs columns 8 h .. 8 h + 7, a word, and, h < 11, columns 128 + 4 h .. + 3, half a word.
template <typename T, bool ALIGNED, bool FEW>
__global__ void __launch_bounds__(256) push_kernel(uint32_t *__restrict__ words, const T *__restrict__ x, int64_t x_stride,
                                                   const int32_t *__restrict__ ids, int n, int64_t n_rows,
                                                   int32_t *__restrict__ record, int32_t *status) {
  dep_trigger();
  dep_wait();
  const int h = threadIdx.x & 15;
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
  int64_t v = -1;
  if (i < n) {
    v = ids != nullptr ? ids[i] : i;
    if (v < 0 || v >= n_rows) v = -1;
  }
  if (FEW) {                        // no record: a later position of the same id shows that this one does not stay
    const int64_t id = v;
    if (i < n && v < 0 && h == 0) report(status, ORCA_E_BOUNDS, (int)i);
    bool later = false;
    for (int64_t j = i + 1 + h; j < n; j += 16) later |= ids[j] == id;
    const uint32_t any = __ballot_sync(FULL, later);
    if ((any >> (threadIdx.x & 16) & 0xffffu) != 0) v = -1;
  }
  // (the winner takes its record back; another position of the same id finds the winner's or none, never its own)
  if (record != nullptr && v >= 0 && *(volatile int32_t *)&record[v] != (int)i + 1) v = -1;
  __syncwarp();
  if (record != nullptr && v >= 0 && h == 0) record[v] = 0;
  if (!__any_sync(FULL, v >= 0)) return;
  const bool tail = h < TAIL / 4;
  float a[8] = {}, b[4] = {};
  const T *row = x + (v >= 0 ? i : 0) * x_stride;
  if (v >= 0) {
    constexpr int VB = ALIGNED ? (sizeof(T) == 4 ? 16 : 8) : (int)sizeof(T);
    load_values<VB>(row + 8 * h, a);
    if (tail) load_values<VB>(row + GROUP + 4 * h, b);
  }
  uint32_t how_a, how_b;
  {                                              // even lanes work the first group out, odd lanes the second
    constexpr float MOST = 8.507059173023462e37f;      // 2^126
    const float2 ea = extremes(a, true), eb = extremes(b, tail);
    const float lo = h & 1 ? eb.x : ea.x, hi = h & 1 ? eb.y : ea.y;
    const uint32_t how = lo > -MOST && hi < MOST ? group_of(lo, hi) : 0x7fc07fc0u;
    const uint32_t other = __shfl_xor_sync(FULL, how, 1);
    how_a = h & 1 ? other : how, how_b = h & 1 ? how : other;
  }
  if (v < 0) return;
  const uint32_t ca = codes_of(a, row + 8 * h, how_a), cb = tail ? codes_of(b, row + GROUP + 4 * h, how_b) : 0;
  uint32_t *out = words + v * WORDS;
  if (h == 0) *reinterpret_cast<uint2 *>(out) = make_uint2(how_a, how_b);
  out[2 + h] = ca;
  if (h < 12) reinterpret_cast<uint16_t *>(out + 18)[h] = tail ? (uint16_t)cb : 0;      // (the twelfth: four columns that are not there)
}

// Bound by HBM, 7 of 8 bytes are written, and by the way to a row, an id and then its words at a random place, which a warp waits for
// 24 of 31 cycles: 500 k rows 82 us, 4.8 TB/s.  The layout is for the writes: whole lines, a row's 43 pieces over whichever threads.
// A thread takes PULL_PIECES of the 43 pieces of four columns that a row has, 256 apart: whole lines are written.
constexpr int PULL_PIECES = 4, ROW_PIECES = D / 4;
__global__ void __launch_bounds__(256) pull_kernel(const uint32_t *__restrict__ words, int64_t n_rows,
                                                   const int32_t *__restrict__ ids, int64_t n, float *__restrict__ out,
                                                   int32_t *status) {
  dep_trigger();
  dep_wait();
  const int64_t p0 = (int64_t)blockIdx.x * (256 * PULL_PIECES), row0 = p0 / ROW_PIECES;
  const uint32_t skip = (uint32_t)(p0 - row0 * ROW_PIECES);
  uint32_t how[PULL_PIECES], w[PULL_PIECES];
  bool in[PULL_PIECES];
#pragma unroll
  for (int k = 0; k < PULL_PIECES; ++k) {
    const uint32_t p = skip + threadIdx.x + 256 * k, r = p / ROW_PIECES, c = p - r * ROW_PIECES;
    const int64_t i = row0 + r;
    in[k] = i < n;
    how[k] = w[k] = 0;
    if (in[k]) {
      const int v = ids[i];
      if (v >= 0 && v < n_rows) {
        const uint32_t *row = words + (int64_t)v * WORDS;
        how[k] = __ldg(row + (c >= GROUP / 4));
        w[k] = __ldg(reinterpret_cast<const uint16_t *>(row + 2) + c);
      } else if (c == 0) {
        report(status, ORCA_E_BOUNDS, (int)(i < 0x7fffffff ? i : 0x7fffffff));
      }
    }
  }
#pragma unroll
  for (int k = 0; k < PULL_PIECES; ++k) {
    const float s = step_of(how[k]), o = offset_of(how[k]);
    if (in[k])
      reinterpret_cast<float4 *>(out)[p0 + threadIdx.x + 256 * k] =
          make_float4(held(w[k] & 15u, s, o), held(w[k] >> 4 & 15u, s, o), held(w[k] >> 8 & 15u, s, o), held(w[k] >> 12, s, o));
  }
}

// ---------------------------------------------------------------------------------------------- attention
// Where the slots of the rows are.  A row's slots are cut into parts of `len`; a warp takes a part.
struct TableSlots {       // tables of k slots a row
  const int32_t *nbr, *eid;
  const float *delta;
  int64_t k;
  int parts;              // of a row
  int64_t len;            // slots of a part
};
struct ListSlots {        // the interactions of a node before a time, in the adjacency
  const int32_t *nbr, *eid;
  const double *ts, *time;
  const int64_t *beg;     // [rows]
  const int32_t *count;   // [rows]
  const int32_t *first;   // [rows + 1] number of the row's first part
  const int32_t *base;    // [rows] where the results of its parts go, if it has several
  const int32_t *head;    // slots of a part
};

struct Part {
  int row, at, of;        // part `at` of `of`
  int64_t beg;            // its slots
  int n;
  int64_t out;            // where its result goes, if of > 1
};
__device__ __forceinline__ bool part_of(const TableSlots &s, int rows, int64_t job, int, Part &p) {
  if (job >= (int64_t)rows * s.parts) return false;
  p.row = (int)job, p.at = 0, p.of = s.parts;
  if (s.parts > 1) p.row = (int)((uint32_t)job / (uint32_t)s.parts), p.at = (int)((uint32_t)job % (uint32_t)s.parts);
  p.beg = (int64_t)p.row * s.k + p.at * s.len;
  const int64_t left = s.k - p.at * s.len;
  p.n = (int)(left < 0 ? 0 : left < s.len ? left : s.len);
  p.out = job;
  return true;
}
__device__ __forceinline__ bool part_of(const ListSlots &s, int rows, int64_t job, int lane, Part &p) {
  if (job >= s.first[rows]) return false;
  int lo = 0, hi = rows;              // first[lo] <= job < first[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, q = lo + step * lane;
    const unsigned le = __ballot_sync(FULL, q < hi && s.first[q] <= job);
    const int k = 31 - __clz(le);     // (lane 0's holds always)
    lo += step * k;
    hi = min(hi, lo + step);
  }
  const int len = s.head[0];
  p.row = lo;
  p.at = (int)(job - s.first[lo]);
  p.of = s.first[lo + 1] - s.first[lo];
  const int64_t skip = (int64_t)p.at * len;
  const int64_t left = s.count[lo] - skip;
  p.beg = s.beg[lo] + skip;
  p.n = (int)(left < len ? left : len);
  p.out = (int64_t)s.base[lo] + p.at;
  return true;
}
struct Slot {
  int nbr, eid;
  float dt;
};
__device__ __forceinline__ Slot slot_of(const TableSlots &s, const Part &, int64_t i) { return {s.nbr[i], s.eid[i], s.delta[i]}; }
__device__ __forceinline__ Slot slot_of(const ListSlots &s, const Part &p, int64_t i) {
  return {s.nbr[i], s.eid[i], (float)(s.time[p.row] - (double)(float)s.ts[i])};
}

struct Tables {
  const uint32_t *rows, *edges;      // packed
  const float *edges32;              // or edge features in 32 bits
  int64_t n_rows, n_edges;
  const float *time_w;
};

struct __align__(16) Rec {           // what a step needs of a slot
  int nbr, eid;
  float dt;
  int kind;                          // which cosines its time encoding takes: 0 cos_small2, 1 cos_wide2 in the first 64 columns, 2 or 3 slow_terms in all (3: beyond 2^30)
};
// Cosines of two arguments below 2^30.  2pi is C1 + C2 + C3 to 72 bits.  First multiples of 512pi are taken away, K = the nearest integer
// to x / 512pi, below 2^20: x - K * 256 C1 is a multiple of 2^-13 below 2^10 and exact; what K * 256 C2 takes away on top (30 at most) is
// split into a part h that is a multiple of 2^-13 again and a rest.  Then k multiples of 2pi: h - k * C1 is exact; the small terms are
// added last.  Error of the reduction 1.2e-7 at most (a rounding of a value below 4), the remainder below 3.142.
__device__ __forceinline__ float2 cos_wide2(float2 x) {
  const float2 magic = dup2(12582912.f), demagic = dup2(-12582912.f);
  const float2 K = add2(fma2(x, dup2(0.00062169899f), magic), demagic);
  const float2 a = fma2(K, dup2(-256.f * 6.2831855f), x);
  const float2 h = add2(add2(fma2(K, dup2(4.4760464e-05f), a), dup2(1536.f)), dup2(-1536.f));
  float2 low = fma2(K, dup2(4.4760464e-05f), add2(a, make_float2(-h.x, -h.y)));
  const float2 k = add2(fma2(h, dup2(0.15915494309189535f), magic), demagic);
  low = fma2(k, dup2(1.7484556e-07f), low);
  low = fma2(K, dup2(1.7562875e-12f), low);
  const float2 r = add2(fma2(k, dup2(-6.2831855f), h), low);
  return make_float2(__cosf(r.x), __cosf(r.y));
}
// The time encodings of a step with arguments that are rare: a call, so that its code and what it does to the registers do not stand
// in the way of all others.
template <int GS>
__device__ __noinline__ void slow_terms(const float *time_w, const Rec *rec, int lane, float2 *out) {
#pragma unroll 1
  for (int u = 0; u < GS; ++u)
#pragma unroll 1
    for (int i = 0; i < GA_P_ITERS; ++i) {
      float2 c = make_float2(1.f, 1.f);
      if (i < 2 || lane < 22) {
        const float2 w = __ldg(reinterpret_cast<const float2 *>(time_w) + lane + 32 * i);
        c = make_float2(cos_any(rec[u].dt * w.x), cos_any(rec[u].dt * w.y));
      }
      out[u * GA_P_ITERS + i] = c;
    }
}

__device__ __forceinline__ void async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int AT_THREADS = 64, AT_WARPS = AT_THREADS / 32;
constexpr int AT_BLOCKS = 6;                               // an SM: 12 warps at 168 registers
constexpr int AT_SLOTS = 4;                                // of a step
constexpr int BATCH = 32;                                  // slots whose indices are read at a time, a lane each
constexpr float RESCALE = 8.f;
template <int GS, bool EDGE32> struct Stage {              // GS slots in shared memory: the neighbour's row, then the edge's
  static constexpr int EDGE = EDGE32 ? ROW_BYTES : BYTES, SLOT = BYTES + EDGE + (EDGE32 ? 16 : 0), SIZE = GS * SLOT;     // (fp32: and four zeros)
  static constexpr int COUNT = BATCH / GS;                 // stages of a batch
  static constexpr int DEPTH = EDGE32 ? COUNT / 2 : COUNT; // of which so many are under way
  struct Warp {
    char ring[DEPTH * SIZE];
    float4 qc[2][3][32];                                   // the lanes' columns of the heads' queries
    float4 qe[2][32];
    float2 qe2[2][32];
    float4 how[GS][2][2];                                  // [slot][table][group]: 16 step twice, offset - 16 step twice
    float4 p[GS];                                          // weights, head 0 twice, head 1 twice
    Rec rec[2][BATCH + GS - 1];
  };
};

// Results of the parts of rows that have several: PARTIAL floats a part [sums of both heads | what their weights are taken against | the
// weights' totals | whether there was a slot], and how many of a group have come, a word a level.
struct Parts {
  float *results;
  int32_t *come;       // [parts][LEVELS], zero at first
};
constexpr int FAN = 16, LEVELS = 4;
constexpr int JOIN_CHUNKS = (QT / 4 + 31) / 32;    // of 32 columns of four
// Joins the parts of a row, sixteen at a time: the warp whose part is the last of a group to come joins the group, always in the order
// of the parts, into the place of its first; so do the groups, until one is left.  No launch waits for the longest row to join the
// others (a kernel of its own took 12 us for 37 rows of two parts, 36 for three of 570, 65 for 4001 of three).
__device__ __noinline__ void join_parts(Parts s, int64_t first, int at, int of, float *ctx, uint8_t *valid, int lane) {
  int64_t stride = 1;
#pragma unroll 1
  for (int level = 0, n = of;; ++level, n = (n + FAN - 1) / FAN, at /= FAN, stride *= FAN) {
    const int g = at / FAN, members = min(FAN, n - g * FAN);
    const int64_t head = first + (int64_t)g * FAN * stride;
    if (members == 1) continue;                    // (is where it belongs already; never the last level)
    __threadfence();
    __syncwarp();
    int come = 0;
    if (lane == 0) come = atomicAdd(s.come + head * LEVELS + level, 1);
    if (__shfl_sync(FULL, come, 0) != members - 1) return;
    __threadfence();
    float *group = s.results + head * PARTIAL;
    const int64_t step = stride * PARTIAL;
    float4 st = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
    bool some = false;
    if (lane < members) {
      st = __ldcg(reinterpret_cast<const float4 *>(group + lane * step + QT));
      some = __ldcg(group + lane * step + QT + 4) != 0.f;
    }
    some = __any_sync(FULL, some);
    const float m0 = warp_max(st.x), m1 = warp_max(st.y);
    const float w0 = expf(st.x - (m0 == -INFINITY ? 0.f : m0)), w1 = expf(st.y - (m1 == -INFINITY ? 0.f : m1));      // (0 behind the last)
    const float t0 = warp_sum(lane < members ? w0 * st.z : 0.f), t1 = warp_sum(lane < members ? w1 * st.w : 0.f);
    const bool top = n <= FAN;
    float *out = top ? ctx : group;
    const float k0 = !top ? 1.f : some ? 1.f / t0 : 0.f, k1 = !top ? 1.f : some ? 1.f / t1 : 0.f;
    constexpr int CH = 3, AHEAD = 8;
#pragma unroll 1
    for (int c0 = 0; c0 < JOIN_CHUNKS; c0 += CH) {
      float4 a[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) a[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int j0 = 0; j0 < members; j0 += AHEAD) {
        float4 v[AHEAD][CH];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
          for (int c = 0; c < CH; ++c)
            if (j0 + u < members)
              v[u][c] = __ldcg(reinterpret_cast<const float4 *>(group + (j0 + u) * step) + min(32 * (c0 + c) + lane, QT / 4 - 1));
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (j0 + u >= members) break;
          const float x0 = __shfl_sync(FULL, w0, j0 + u), x1 = __shfl_sync(FULL, w1, j0 + u);
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const float w = 32 * (c0 + c) + lane >= KEY / 4 ? x1 : x0;            // (a head has 129 columns of four)
            a[c].x = fmaf(w, v[u][c].x, a[c].x), a[c].y = fmaf(w, v[u][c].y, a[c].y);
            a[c].z = fmaf(w, v[u][c].z, a[c].z), a[c].w = fmaf(w, v[u][c].w, a[c].w);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = 32 * (c0 + c) + lane;
        const float k = col >= KEY / 4 ? k1 : k0;
        if (col < QT / 4)
          reinterpret_cast<float4 *>(out)[col] = some ? make_float4(a[c].x * k, a[c].y * k, a[c].z * k, a[c].w * k) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if (top) {
      if (lane == 0) *valid = some;
      return;
    }
    __syncwarp();
    if (lane == 0) {
      *reinterpret_cast<float4 *>(group + QT) = make_float4(m0, m1, t0, t1);
      group[QT + 4] = some ? 1.f : 0.f;
    }
  }
}

// ctx_h = sum_j p_hj k_j, p_h = softmax_j(q_h . k_j), k_j = [row(nbr_j) | edge(eid_j) | cos(delta_j w)], 516 columns, two heads: one pass
// over the slots, with each key decoded once into registers for its logits and its weighted sum.
//
// A warp takes a part of a row's slots, GS at a time.  Lanes 0..15 hold what the neighbours' rows have, lanes 16..31 the edges':
// columns 8 h .. 8 h + 7 (a word of codes) and, h < 11, columns 128 + 4 h .. + 3 (half a word); all lanes hold column pairs
// l, l + 32, l + 64 of the time encoding.  Rows come by asynchronous copies into a ring of stages, a batch of 32 slots ahead.
// Weights are taken against a reference that only moves when a logit exceeds it by 8: up to e^8 they lose nothing in fp32, and the
// sums are rarely rescaled.
//
// Bound by instructions: a slot is 208 bytes in, but 2064 products and sums, 344 codes to decode and 172 cosines, 134 warp instructions
// (165 with edges in fp32), 46 of them packed ones that take the FMA pipe two cycles; in long lists 70 % of what the four schedulers can
// issue so.  1.2 M slots of three rows: 309 us, 0.8 TB/s, 8 TFLOP/s; in rows of twenty 348 us for 1.19 M; 12 warps an SM at 168
// registers.  Twice the slots a step spill, half of them halve what a step's latency is spread over; 16 warps at 128 registers spill.
// Decoding: codes go to the top of a mantissa by a shift and one logic instruction, and a packed multiplication and addition makes
// two values of two of them; conversions would queue for the unit that takes the cosines.  What was slower, us for the three long
// rows / 4001 of all lengths at a time when this took 341 / 580: codes as operands of matrix instructions (queries and weights cut into
// 16-bit pieces; a warp with 16 slots 427 / 983, eight warps with 64 410 / 717, two warps 349 / 685), a slot a lane 512 / 824.  Two queries a
// slot leave a matrix instruction three quarters empty, and its operands cost the decoding that it saves.
template <int GS, bool EDGE32, class S>
__global__ void __launch_bounds__(AT_THREADS, AT_BLOCKS) attend_kernel(const float *__restrict__ qt, Tables t, S slots, int rows,
                                                                       float *__restrict__ ctx, uint8_t *__restrict__ valid,
                                                                       Parts parts, int32_t *status) {
  using G = Stage<GS, EDGE32>;
  extern __shared__ __align__(128) char s_all[];
  int lane;                                    // (volatile: or it is read from its special register again in every step, 10 % of the time)
  asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));
  const int warp = __shfl_sync(FULL, threadIdx.x >> 5, 0);
  typename G::Warp &sm = reinterpret_cast<typename G::Warp *>(s_all)[warp];
  dep_trigger();
  dep_wait();
  Part p;
  if (!part_of(slots, rows, (int64_t)blockIdx.x * AT_WARPS + warp, lane, p)) return;
  const int side = lane >> 4, h = lane & 15;
  const bool has_tail = h < TAIL / 4, third = lane < 22;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(sm.ring);

  Slot next = {0, 0, 0.f};
  auto load_indices = [&](int at0) {
    next = {0, 0, 0.f};
    if (at0 + lane < p.n) next = slot_of(slots, p, p.beg + at0 + lane);
  };
  load_indices(0);
  float2 wt[GA_P_ITERS];
  float w_first, w_rest, w_last;               // the largest weights of the first 64 columns, of the others, of the last 44
  {
    uint32_t most[GA_P_ITERS];
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i) {
      wt[i] = (i < 2 || third) ? __ldg(reinterpret_cast<const float2 *>(t.time_w) + lane + 32 * i) : make_float2(0.f, 0.f);
      // (magnitudes are in the order of their bits; what is not a number is above them all)
      most[i] = __reduce_max_sync(FULL, max(__float_as_uint(wt[i].x) & 0x7fffffffu, __float_as_uint(wt[i].y) & 0x7fffffffu));
    }
    w_first = __uint_as_float(most[0]), w_rest = __uint_as_float(max(most[1], most[2])), w_last = __uint_as_float(most[2]);
  }
  // The slots of `next` that count, one behind the other, in record buffer b; behind them, up to a whole step, the first again (its
  // weight will be zero).  Returns their number.
  auto put_records = [&](int b) {
    Slot s = next;
    if (s.nbr != 0 && (s.nbr < 0 || s.nbr >= t.n_rows || s.eid < 0 || s.eid >= t.n_edges)) {      // (neighbour 0: no slot, whatever its edge)
      report(status, ORCA_E_BOUNDS, p.row);
      s.nbr = 0;
    }
    const unsigned used = __ballot_sync(FULL, s.nbr != 0);
    const int n_used = __popc(used);
    const float adt = fabsf(s.dt);
    const float rest = adt * w_rest, first = adt * w_first;
    const int kind = !(fmaxf(first, rest) < 1073741824.f) || !(adt < INFINITY) ? 3 : rest >= COS_SMALL ? 2
                     : first >= COS_SMALL || adt * w_last > 3.14f ? 1 : 0;
    const Rec r = {s.nbr, s.eid, s.dt, kind};
    const int place = __popc(used & ((1u << lane) - 1u));
    if (s.nbr != 0) sm.rec[b][place] = r;
    if (s.nbr != 0 && place == 0)
      for (int u = 0; u < GS - 1; ++u) sm.rec[b][n_used + u] = r;
    __syncwarp();
    return n_used;
  };
  // What a lane copies of a stage.  Packed edges: of its 12 GS pieces of 16 bytes number l and l + 32.  Edges in fp32: of every slot
  // piece l and, lanes 0..10, piece l + 32 of the edge, lanes 11..16 the six pieces of the neighbour's row.
  const char *src0, *src1;
  uint32_t dst0, dst1, id0, id1, mul1 = BYTES;
  bool on1;
  if (EDGE32) {
    src0 = reinterpret_cast<const char *>(t.edges32) + 16 * lane;
    dst0 = BYTES + 16 * lane, id0 = 1;
    const bool more = lane < 11;
    src1 = more ? src0 + 512 : reinterpret_cast<const char *>(t.rows) + 16 * (lane - 11);
    dst1 = more ? dst0 + 512 : 16 * (lane - 11), id1 = more ? 1 : 0, mul1 = more ? ROW_BYTES : BYTES;
    on1 = lane < 17;
  } else {
    auto piece = [&](int k, const char *&src, uint32_t &dst, uint32_t &id) {
      const int u = k / 12, part = k % 12;
      src = part < 6 ? reinterpret_cast<const char *>(t.rows) + 16 * part : reinterpret_cast<const char *>(t.edges) + 16 * (part - 6);
      dst = 16 * k, id = 4 * u + (part >= 6);      // (in words of the records)
    };
    piece(lane, src0, dst0, id0);
    piece(lane + 32, src1, dst1, id1);
    on1 = lane + 32 < 12 * GS;
  }
  // copies of stage j of the batch in record buffer b (a group of its own even when there is nothing to copy)
  auto fetch = [&](int b, int j, int n_used) {
    if (j * GS < n_used) {
      const int *rec = reinterpret_cast<const int *>(&sm.rec[b][j * GS]);
      const uint32_t dst = ring_at + (j % G::DEPTH) * G::SIZE;
      if (EDGE32) {
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          async16(dst + u * G::SLOT + dst0, src0 + (uint64_t)(uint32_t)rec[4 * u + 1] * ROW_BYTES);
          if (on1) async16(dst + u * G::SLOT + dst1, src1 + (uint64_t)(uint32_t)rec[4 * u + id1] * mul1);
        }
      } else {
        static_assert(12 * GS > 32 && 12 * GS <= 64, "two pieces a lane");
        async16(dst + dst0, src0 + (uint64_t)(uint32_t)rec[id0] * BYTES);
        if (on1) async16(dst + dst1, src1 + (uint64_t)(uint32_t)rec[id1] * BYTES);
      }
    }
    async_commit();
  };
  const int tail_at = has_tail ? 4 * GROUP + 16 * h : ROW_BYTES;
  if (EDGE32 && lane < G::DEPTH * GS) *reinterpret_cast<float4 *>(sm.ring + lane * G::SLOT + BYTES + ROW_BYTES) = make_float4(0.f, 0.f, 0.f, 0.f);
  static_assert(!EDGE32 || G::DEPTH * GS <= 32, "a slot a lane");
  int n_used = put_records(0), buf = 0;
#pragma unroll 1
  for (int j = 0; j < G::DEPTH; ++j) fetch(0, j, n_used);
  if (p.n > BATCH) load_indices(BATCH);

#pragma unroll
  for (int g = 0; g < 2; ++g) {                // this lane's columns of the two heads' queries
    const float *qh = qt + (int64_t)p.row * QT_LD + g * QT_HEAD, *qr = qh + side * D;
    sm.qc[g][0][lane] = ldg4(reinterpret_cast<const char *>(qr + 8 * h));
    sm.qc[g][1][lane] = ldg4(reinterpret_cast<const char *>(qr + 8 * h + 4));
    sm.qc[g][2][lane] = has_tail ? ldg4(reinterpret_cast<const char *>(qr + GROUP + 4 * h)) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float2 *qe = reinterpret_cast<const float2 *>(qh + 2 * D) + lane;
    const float2 a = __ldg(qe), b = __ldg(qe + 32);
    sm.qe[g][lane] = make_float4(a.x, a.y, b.x, b.y);
    sm.qe2[g][lane] = third ? __ldg(qe + 64) : make_float2(0.f, 0.f);
  }
  float2 ac[2][6], ae[2][GA_P_ITERS];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
#pragma unroll
    for (int j = 0; j < 6; ++j) ac[g][j] = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i) ae[g][i] = make_float2(0.f, 0.f);
  }
  float psum = 0.f, ref = -INFINITY;                 // of this lane's head: its slots' weights, what they are taken against
  bool any_valid = false;
  constexpr int V = 2 * GS, LPV = 32 / V;
  for (int at0 = 0; at0 < p.n; at0 += BATCH) {
    any_valid |= n_used > 0;
    const bool more = at0 + BATCH < p.n;
    int n_next = 0;
    for (int j = 0; j < G::COUNT; ++j) {
      if (j * GS >= n_used && !more) break;
      async_wait<G::DEPTH - 1>();
      __syncwarp();
      if (j * GS < n_used) {
        const Rec *rec = &sm.rec[buf][j * GS];
        const char *stage = sm.ring + (j % G::DEPTH) * G::SIZE;
        {                                            // the groups of the stage, a lane each
          constexpr int TABLES = EDGE32 ? 1 : 2;
          const int u = lane / (2 * TABLES), k = lane % (2 * TABLES);
          if (lane < GS * 2 * TABLES) {
            const uint32_t how = *reinterpret_cast<const uint32_t *>(stage + u * G::SLOT + (k >> 1) * BYTES + (k & 1) * 4);
            const float s = 16.f * step_of(how), o = offset_of(how) - s;
            sm.how[u][k >> 1][k & 1] = make_float4(s, s, o, o);
          }
          __syncwarp();
        }
        int kind = 0;
        float2 x[GS][6], te[GS][GA_P_ITERS];
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          const float2 r = *reinterpret_cast<const float2 *>(&rec[u].dt);
          kind = max(kind, __float_as_int(r.y));
          te[u][0] = mul2(dup2(r.x), wt[0]), te[u][1] = mul2(dup2(r.x), wt[1]), te[u][2] = mul2(dup2(r.x), wt[2]);
          const char *row = stage + u * G::SLOT + (EDGE32 ? 0 : side * BYTES);
          const uint32_t w = *reinterpret_cast<const uint32_t *>(row + 8 + 4 * h);
          const uint32_t v = *reinterpret_cast<const uint16_t *>(row + 72 + 2 * min(h, 11));      // (lanes without a tail: times queries of zero)
          const float4 g0 = sm.how[u][EDGE32 ? 0 : side][0], g1 = sm.how[u][EDGE32 ? 0 : side][1];
          float2 c8[4], c4[2];
          decode8(w, lo2(g0), hi2(g0), c8);
          decode4(v, lo2(g1), hi2(g1), c4);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u][i] = c8[i];
          x[u][4] = c4[0], x[u][5] = c4[1];
          if (EDGE32 && side) {                      // (over what was decoded: three loads, no branch around the decoding)
            const char *edge = stage + u * G::SLOT + BYTES;
            const float4 a = *reinterpret_cast<const float4 *>(edge + 32 * h), b = *reinterpret_cast<const float4 *>(edge + 32 * h + 16);
            const float4 c = *reinterpret_cast<const float4 *>(edge + tail_at);
            x[u][0] = lo2(a), x[u][1] = hi2(a), x[u][2] = lo2(b), x[u][3] = hi2(b), x[u][4] = lo2(c), x[u][5] = hi2(c);
          }
        }
        if (kind == 0) {
#pragma unroll
          for (int u = 0; u < GS; ++u) {
            te[u][0] = cos_small2(te[u][0]), te[u][1] = cos_small2(te[u][1]);
            te[u][2] = make_float2(__cosf(te[u][2].x), __cosf(te[u][2].y));       // (below pi)
          }
        } else if (kind == 1) {
#pragma unroll
          for (int u = 0; u < GS; ++u) te[u][0] = cos_wide2(te[u][0]), te[u][1] = cos_small2(te[u][1]), te[u][2] = cos_small2(te[u][2]);
        } else {
          float2 slow[GS * GA_P_ITERS];
          slow_terms<GS>(t.time_w, rec, lane, slow);
#pragma unroll
          for (int u = 0; u < GS; ++u)
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) te[u][i] = slow[u * GA_P_ITERS + i];
        }
        float v[V];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const float4 q0 = sm.qc[g][0][lane], q1 = sm.qc[g][1][lane], q2 = sm.qc[g][2][lane], q3 = sm.qe[g][lane];
          const float2 q4 = sm.qe2[g][lane];
#pragma unroll
          for (int u = 0; u < GS; ++u) {
            float2 a = mul2(x[u][0], lo2(q0));
            a = fma2(x[u][1], hi2(q0), a);
            a = fma2(x[u][2], lo2(q1), a);
            a = fma2(x[u][3], hi2(q1), a);
            a = fma2(x[u][4], lo2(q2), a);
            a = fma2(x[u][5], hi2(q2), a);
            a = fma2(te[u][0], lo2(q3), a);
            a = fma2(te[u][1], hi2(q3), a);
            a = fma2(te[u][2], q4, a);
            v[2 * u + g] = a.x + a.y;
          }
        }
        // lane l holds value l / LPV = 2 * slot + head
        float lg = warp_sum_many<V>(v, lane);
        const bool on = j * GS + lane / (2 * LPV) < n_used;
        if (!on) lg = -INFINITY;
        float top = lg;
#pragma unroll
        for (int o = 2 * LPV; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
        const bool moves = top > ref + RESCALE || (ref == -INFINITY && top > ref);
        if (__any_sync(FULL, moves)) {
          const float k = moves ? expf(ref - top) : 1.f;            // (0 the first time: nothing has been added)
          if (moves) ref = top;
          psum *= k;
          const float2 k0 = dup2(__shfl_sync(FULL, k, 0)), k1 = dup2(__shfl_sync(FULL, k, LPV));
#pragma unroll
          for (int i = 0; i < 6; ++i) ac[0][i] = mul2(k0, ac[0][i]), ac[1][i] = mul2(k1, ac[1][i]);
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) ae[0][i] = mul2(k0, ae[0][i]), ae[1][i] = mul2(k1, ae[1][i]);
        }
        const float w = on ? expf(lg - (ref == -INFINITY ? 0.f : ref)) : 0.f;      // (logits of minus infinity only: weights of zero)
        psum += w;
        // [slot][head] weights, each twice (operands of the packed instructions)
        reinterpret_cast<float2 *>(sm.p)[lane / LPV] = dup2(w);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          // (a slot that is there twice has weight zero the second time; infinities of its edge make their columns NaN the first time)
          const float4 w4 = sm.p[u];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float2 k = g ? hi2(w4) : lo2(w4);
#pragma unroll
            for (int i = 0; i < 6; ++i) ac[g][i] = fma2(k, x[u][i], ac[g][i]);
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) ae[g][i] = fma2(k, te[u][i], ae[g][i]);
          }
        }
        __syncwarp();
      }
      // the stage is free: what comes DEPTH stages later goes there
      if (j + G::DEPTH < G::COUNT) {
        fetch(buf, j + G::DEPTH, n_used);
      } else if (more) {
        if (j + G::DEPTH == G::COUNT) {
          n_next = put_records(buf ^ 1);
          if (at0 + 2 * BATCH < p.n) load_indices(at0 + 2 * BATCH);
        }
        fetch(buf ^ 1, j + G::DEPTH - G::COUNT, n_next);
      } else {
        async_commit();
      }
    }
    n_used = n_next;
    buf ^= 1;
  }
  async_wait<0>();
#pragma unroll
  for (int o = 2 * LPV; o < 32; o <<= 1) psum += __shfl_xor_sync(FULL, psum, o);
  const float sum0 = __shfl_sync(FULL, psum, 0), sum1 = __shfl_sync(FULL, psum, LPV);
  const float m0 = __shfl_sync(FULL, ref, 0), m1 = __shfl_sync(FULL, ref, LPV);
  const bool whole = p.of == 1;
  float *out = whole ? ctx + (int64_t)p.row * QT : parts.results + p.out * PARTIAL;
  const float k0 = !any_valid ? 0.f : whole ? 1.f / sum0 : 1.f, k1 = !any_valid ? 0.f : whole ? 1.f / sum1 : 1.f;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float2 k = dup2(g ? k1 : k0);
    float *o = out + g * KEY;
    float4 *oc = reinterpret_cast<float4 *>(o + side * D);
    float2 r[6];
#pragma unroll
    for (int j = 0; j < 6; ++j) r[j] = mul2(k, ac[g][j]);
    oc[2 * h] = make_float4(r[0].x, r[0].y, r[1].x, r[1].y);
    oc[2 * h + 1] = make_float4(r[2].x, r[2].y, r[3].x, r[3].y);
    if (has_tail) oc[GROUP / 4 + h] = make_float4(r[4].x, r[4].y, r[5].x, r[5].y);
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i)
      if (i < 2 || third) reinterpret_cast<float2 *>(o + 2 * D)[lane + 32 * i] = mul2(k, ae[g][i]);
  }
  if (lane == 0) {
    if (whole) {
      valid[p.row] = any_valid;
    } else {
      *reinterpret_cast<float4 *>(out + QT) = make_float4(m0, m1, sum0, sum1);
      out[QT + 4] = any_valid ? 1.f : 0.f;
    }
  }
  if (!whole) join_parts(parts, p.out - p.at, p.at, p.of, ctx + (int64_t)p.row * QT, valid + p.row, lane);
}

constexpr int MOST_SLOTS = 1 << 30;      // of a list: positions in it stay below 2^31 with what is added to them
// Where a row's list lies: the interactions of its node before its time, the last `last` of them (0: all).
struct Bounds {
  const int64_t *indptr;
  const double *ts;
  int64_t n_nodes;
  const int32_t *nodes;
  const double *time;
  int64_t last;
  int64_t *beg;
  int32_t *count, *status;
};
__device__ __forceinline__ void bounds_of(const Bounds &b, int r, int lane) {
  const int v = b.nodes[r];
  long long lo = 0, hi = 0;
  if (v >= 0 && v < b.n_nodes) lo = b.indptr[v], hi = b.indptr[v + 1];
  else if (lane == 0) report(b.status, ORCA_E_BOUNDS, r);
  const long long end = lower_bound_group<32>(b.ts, lo, hi, b.time[r], lane, FULL, 0);
  if (b.last > 0 && end - lo > b.last) lo = end - b.last;
  const bool fits = end - lo <= MOST_SLOTS;
  if (lane == 0 && !fits) report(b.status, ORCA_E_BOUNDS, r);
  if (lane == 0) b.beg[r] = lo, b.count[r] = fits ? (int32_t)(end - lo) : 0;
}
// A warp a row: a search by 32 probes at a time, four rounds in a list of a million.  Bound by their latency.
__global__ void __launch_bounds__(256) list_bounds_kernel(Bounds b, int rows) {
  dep_trigger();
  dep_wait();
  const int r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (r < rows) bounds_of(b, r, threadIdx.x & 31);
}

// Cuts the lists into parts: about `target` of them over all rows, none shorter than `least` slots but a row's last; sets the words that
// count how many of a group have come to zero.  Where the rows are few, it looks the lists up itself.  One block, bound by latency: 5 us.
__global__ void __launch_bounds__(1024) list_parts_kernel(Bounds bounds, bool look_up, int rows, int target, int least,
                                                          int32_t *__restrict__ first, int32_t *__restrict__ base,
                                                          int32_t *__restrict__ head, int4 *__restrict__ come) {
  __shared__ unsigned long long s_warp[32];
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t *count = bounds.count;
  if (look_up) {
    for (int r = warp; r < rows; r += 32) bounds_of(bounds, r, lane);
    __syncthreads();
  }
  constexpr int KEPT = 4;             // counts of a thread that are kept
  int kept[KEPT];
  unsigned long long total = 0;
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    const int r = threadIdx.x + 1024 * k;
    kept[k] = r < rows ? count[r] : 0;
    total += kept[k];
  }
  for (int r = threadIdx.x + 1024 * KEPT; r < rows; r += 1024) total += count[r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
  if (lane == 0) s_warp[warp] = total;
  __syncthreads();
  total = s_warp[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
  __syncthreads();
  const unsigned long long want = ((total + target - 1) / target + AT_SLOTS - 1) / AT_SLOTS * AT_SLOTS;
  const int len = (int)(want < (unsigned)least ? least : want < MOST_SLOTS ? want : MOST_SLOTS);
  // summed together: parts (low half), and parts of rows of several
  unsigned long long carry = 0;
  for (int r0 = 0, k = 0; r0 < rows; r0 += 1024, ++k) {
    const int r = r0 + threadIdx.x;
    const int n = k < KEPT ? (k == 0 ? kept[0] : k == 1 ? kept[1] : k == 2 ? kept[2] : kept[3]) : r < rows ? count[r] : 0;
    const unsigned parts = r < rows ? max(1, (int)(((long long)n + len - 1) / len)) : 0;
    const unsigned long long mine = parts > 1 ? parts | (unsigned long long)parts << 32 : parts;
    unsigned long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(FULL, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    unsigned long long sums = s_warp[lane];       // of the warps: every warp sums them for itself
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(FULL, sums, o);
      if (lane >= o) sums += up;
    }
    const unsigned long long before_warp = __shfl_sync(FULL, sums, max(warp - 1, 0));
    const unsigned long long before = carry + incl - mine + (warp > 0 ? before_warp : 0);
    carry += __shfl_sync(FULL, sums, 31);
    if (r < rows) {
      first[r] = (int32_t)(unsigned)before;
      base[r] = (int32_t)(before >> 32);
    }
    __syncthreads();
  }
  static_assert(LEVELS == 4, "int4");
  for (int i = threadIdx.x; i < (int)(carry >> 32); i += 1024) come[i] = make_int4(0, 0, 0, 0);
  if (threadIdx.x == 0) first[rows] = (int32_t)(unsigned)carry, head[0] = len;
}

// ---------------------------------------------------------------------------------------------- host
// Parts that the slots of all rows are cut into.  A few long rows come in equal parts: as many as run at a time.  Rows of all lengths
// come in parts of all lengths, and the launch ends when the last one does: eight times as many.  (us, 12 / 24 / 36 parts an SM: three
// rows of 1.2 M slots 309 / 317 / 316; 64 / 96 / 160: 4001 rows of 1.7 M slots 519 / 508 / 516.)
constexpr int FEW_ROWS = 64;
// No part but a row's last is shorter.  Short lists of few rows are cut finer, for the GPU is empty beside them (37 rows of 33 slots: 19.6 us
// in parts of 8, 17.6 of 12 or 16, 18.2 of 20, 20 of 32).  Many long rows want long parts, for each costs what
// a step does to begin and end, and its joining (1201 lists of 253, 16 / 24 / 32 / 48 / 64: 155 / 155 / 145 / 140 / 136 us, edges in 4 bits 138 / 138 / 128 / 122 / 116; lists
// of 4001 rows are cut by `parts_wanted` alone).  In between 64 is too long, and the rule does not know it: 500 lists of 103 42 / 41 / 36 / 41 / 47,
// of 34 26 / 29 / 28 / 33 / 37, 65 lists of 31 18 / 19 / 20 / 24 / 28, a table's row of 200 16 / 16 / 17 / 19 / 21, of 64 12 / 14 / 15 / 15 / 16.
constexpr int LEAST_PART = 64, LEAST_OF_FEW = 16;
constexpr int LOOK_UP = 128;          // rows that list_parts_kernel looks up itself, four a warp: a launch less
// Pushed without marking: the rows look through the ids behind theirs (device us, so / marked: 600 ids 3.2 / 3.3, 1024 3.8 / 3.3; the host is
// spared a launch of 2).
constexpr int FEW_IDS = 1024;
static int sms();
static int least_of_list(int rows) { return rows <= FEW_ROWS ? LEAST_OF_FEW : LEAST_PART; }
static int parts_wanted(int rows) { return sms() * (rows <= FEW_ROWS ? AT_BLOCKS * AT_WARPS : 96); }

static int sms() {
  Ctx *c = cur();
  return c != nullptr ? c->sm_count : 148;
}
static int64_t up256(int64_t b) { return (b + 255) & ~255ll; }

// parts of a row of a table: one, unless there are too few rows to fill the GPU
static int table_parts(int rows, int64_t k) {
  const int64_t by_rows = rows > 0 ? parts_wanted(rows) / rows : 1;
  const int64_t by_len = (k + LEAST_PART - 1) / LEAST_PART;
  return (int)std::max<int64_t>(1, std::min(by_rows, by_len));
}

struct ListLayout {
  int64_t beg, count, first, base, head, come, partial, total;
  int target;
};
static ListLayout list_layout(int rows, int64_t last) {
  ListLayout L;
  L.target = parts_wanted(rows);
  // parts of rows of several: all but the rows' last are full, and so is half of them at least
  int64_t parts = L.target + (int64_t)std::min(L.target, rows);
  if (last > 0) {                     // no list is longer, no part but a list's last shorter than `least`
    const int64_t least = least_of_list(rows), of_row = (std::min<int64_t>(last, MOST_SLOTS) + least - 1) / least;
    parts = of_row == 1 ? 0 : std::min(parts, rows * of_row);
  }
  L.beg = 0;
  L.count = up256((int64_t)rows * 8);
  L.first = L.count + up256((int64_t)rows * 4);
  L.base = L.first + up256((int64_t)rows * 4 + 4);
  L.head = L.base + up256((int64_t)rows * 4);
  L.come = L.head + 256;
  L.partial = L.come + up256(parts * LEVELS * 4);
  L.total = L.partial + up256(parts * PARTIAL * 4);
  return L;
}
// of a row: FAN^LEVELS parts can be joined
static_assert(FAN * FAN * FAN * FAN == 65536 && LEVELS == 4, "levels");

template <class S>
static int launch_attend(const float *d_qt, const Tables &t, const S &slots, int rows, int64_t jobs, float *d_ctx,
                         uint8_t *d_valid, const Parts &parts, int32_t *d_status, cudaStream_t s) {
  const unsigned grid = (unsigned)((jobs + AT_WARPS - 1) / AT_WARPS);
  using G = Stage<AT_SLOTS, true>;
  using P = Stage<AT_SLOTS, false>;
  const int smem = AT_WARPS * (t.edges32 != nullptr ? sizeof(typename G::Warp) : sizeof(typename P::Warp));
  static_assert(AT_BLOCKS * (AT_WARPS * sizeof(typename P::Warp) + 1024) <= 228 * 1024 && AT_BLOCKS * (AT_WARPS * sizeof(typename G::Warp) + 1024) <= 228 * 1024,
                "blocks an SM");
  auto kernel = t.edges32 != nullptr ? attend_kernel<AT_SLOTS, true, S> : attend_kernel<AT_SLOTS, false, S>;
  static std::atomic<uint64_t> ready[2];
  if (const int rc = allow_shared(kernel, smem, ready[t.edges32 != nullptr])) return rc;
  ORCA_CUDA(launch_dep(kernel, grid, AT_THREADS, smem, s, d_qt, t, slots, rows, d_ctx, d_valid, parts, d_status));
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

}  // namespace packed
}  // namespace orca

using namespace orca;
using namespace orca::packed;

#define CHECK_TABLES()                                                                                                  \
  ORCA_CHECK_ARG(d_words && n_rows > 0 && n_rows <= 0x7fffffffll && d_edges && n_edges > 0 && n_edges <= 0x7fffffffll);  \
  ORCA_CHECK_ARG((uintptr_t)d_words % 16 == 0 && (uintptr_t)d_edges % 16 == 0 && (uintptr_t)d_qt % 16 == 0 && (uintptr_t)d_ctx % 16 == 0); \
  ORCA_CHECK_ARG(edges_packed == 0 || edges_packed == 1);                                                               \
  ORCA_CHECK_ARG((uintptr_t)d_time_w % 8 == 0)

extern "C" {

int orca_packed_push(uint32_t *d_words, int64_t n_rows, const void *d_x, int32_t type, int64_t x_stride, const int32_t *d_ids, int32_t n,
                     int32_t *d_record, int32_t *d_status, void *stream) {
  ORCA_CHECK_ARG(d_words && n_rows > 0 && n >= 0 && (n == 0 || d_x) && x_stride >= D);
  ORCA_CHECK_ARG((d_ids != nullptr) == (d_record != nullptr));
  ORCA_CHECK_ARG(d_ids != nullptr || n <= n_rows);
  ORCA_CHECK_ARG((uintptr_t)d_words % 16 == 0);
  if (type != ORCA_F32 && type != ORCA_BF16 && type != ORCA_F16) return set_error(ORCA_E_UNSUPPORTED, "%s: type %d", __func__, type);
  ORCA_CHECK_ARG((uintptr_t)d_x % (type == ORCA_F32 ? 4 : 2) == 0);
  if (n == 0) return ORCA_OK;
  cudaStream_t s = (cudaStream_t)stream;
  const bool few = d_ids != nullptr && n <= FEW_IDS;
  if (d_ids != nullptr && !few) {
    ORCA_CUDA(launch_dep(push_mark_kernel, std::min((n + 255) / 256, sms() * 8), 256, 0, s, d_ids, (int)n, n_rows, d_record, d_status));
    ORCA_COUNT_LAUNCH();
  }
  const unsigned grid = (unsigned)((n + 15) / 16);
  const int size = type == ORCA_F32 ? 4 : 2, wide = type == ORCA_F32 ? 16 : 8;
  const bool aligned = (uintptr_t)d_x % wide == 0 && x_stride * size % wide == 0;
  auto go = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto kernel = few ? (aligned ? push_kernel<T, true, true> : push_kernel<T, false, true>)
                      : (aligned ? push_kernel<T, true, false> : push_kernel<T, false, false>);
    ORCA_CUDA(launch_dep(kernel, grid, 256, 0, s, d_words, (const T *)d_x, x_stride, d_ids, (int)n, n_rows, few ? nullptr : d_record, d_status));
    ORCA_COUNT_LAUNCH();
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  };
  return type == ORCA_F32 ? go((float *)nullptr) : type == ORCA_BF16 ? go((__nv_bfloat16 *)nullptr) : go((__half *)nullptr);
}

int orca_packed_pull(const uint32_t *d_words, int64_t n_rows, const int32_t *d_ids, int64_t n, float *d_out, int32_t *d_status,
                     void *stream) {
  ORCA_CHECK_ARG(d_words && n_rows > 0 && n >= 0 && (n == 0 || (d_ids && d_out)));
  ORCA_CHECK_ARG((uintptr_t)d_words % 16 == 0 && (uintptr_t)d_out % 16 == 0 && n < 0x7fffffffll);
  if (n == 0) return ORCA_OK;
  ORCA_CUDA(launch_dep(pull_kernel, (unsigned)((n * ROW_PIECES + 256 * PULL_PIECES - 1) / (256 * PULL_PIECES)), 256, 0, (cudaStream_t)stream, d_words, n_rows, d_ids, n, d_out, d_status));
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

int64_t orca_packed_attend_workspace_bytes(int32_t n_rows, int64_t k) {
  if (n_rows < 0 || k < 0) return -1;
  const int parts = table_parts(n_rows, k);
  return parts > 1 ? up256((int64_t)n_rows * parts * LEVELS * 4) + (int64_t)n_rows * parts * PARTIAL * 4 : 0;
}

int orca_packed_attend(const float *d_qt, const uint32_t *d_words, int64_t n_rows, const void *d_edges, int64_t n_edges,
                       int32_t edges_packed, const float *d_time_w, const int32_t *d_nbr, const int32_t *d_eid, const float *d_delta,
                       int64_t k, int32_t n_query, float *d_ctx, uint8_t *d_valid, int32_t *d_status, void *d_workspace,
                       int64_t workspace_bytes, void *stream) {
  ORCA_CHECK_ARG(n_query >= 0 && k >= 0 && k <= MOST_SLOTS);
  if (n_query == 0) return ORCA_OK;
  ORCA_CHECK_ARG(d_qt && d_time_w && (k == 0 || (d_nbr && d_eid && d_delta)) && d_ctx && d_valid);
  CHECK_TABLES();
  const int parts = table_parts(n_query, k);
  if (parts > 1) {
    ORCA_CHECK_ARG(d_workspace && (uintptr_t)d_workspace % 256 == 0);
    if (workspace_bytes < orca_packed_attend_workspace_bytes(n_query, k))
      return set_error(ORCA_E_BADARG, "%s: workspace of %lld bytes is too small", __func__, (long long)workspace_bytes);
  }
  cudaStream_t s = (cudaStream_t)stream;
  const Tables t = {d_words, edges_packed ? (const uint32_t *)d_edges : nullptr, edges_packed ? nullptr : (const float *)d_edges, n_rows,
                    n_edges, d_time_w};
  const TableSlots slots = {d_nbr, d_eid, d_delta, k, parts, (k + parts - 1) / parts};
  const int64_t jobs = (int64_t)n_query * parts, counters = jobs * LEVELS * 4;
  const Parts results = {(float *)((char *)d_workspace + up256(counters)), (int32_t *)d_workspace};
  if (parts > 1) ORCA_CUDA(cudaMemsetAsync(d_workspace, 0, (size_t)counters, s));
  return launch_attend(d_qt, t, slots, n_query, jobs, d_ctx, d_valid, results, d_status, s);
}

int64_t orca_packed_attend_lists_workspace_bytes(int32_t n_query) { return n_query < 0 ? -1 : list_layout(n_query, 0).total; }
int64_t orca_packed_attend_last_workspace_bytes(int32_t n_query, int64_t last) {
  return n_query < 0 || last < 0 ? -1 : list_layout(n_query, last).total;
}

int orca_packed_attend_lists(const float *d_qt, const uint32_t *d_words, int64_t n_rows, const void *d_edges, int64_t n_edges,
                             int32_t edges_packed, const float *d_time_w, const int64_t *d_indptr, const int32_t *d_adj_nbr,
                             const int32_t *d_adj_eid, const double *d_adj_ts, int64_t n_nodes, const int32_t *d_nodes, const double *d_ts,
                             int64_t last, int32_t n_query, float *d_ctx, uint8_t *d_valid, int32_t *d_status, void *d_workspace,
                             int64_t workspace_bytes, void *stream) {
  ORCA_CHECK_ARG(n_query >= 0 && last >= 0);
  if (n_query == 0) return ORCA_OK;
  ORCA_CHECK_ARG(d_qt && d_time_w && d_indptr && d_adj_nbr && d_adj_eid && d_adj_ts && n_nodes > 0 && d_nodes && d_ts && d_ctx && d_valid);
  CHECK_TABLES();
  ORCA_CHECK_ARG(d_workspace && (uintptr_t)d_workspace % 256 == 0);
  const ListLayout L = list_layout(n_query, last);
  if (workspace_bytes < L.total) return set_error(ORCA_E_BADARG, "%s: workspace of %lld bytes is too small", __func__, (long long)workspace_bytes);
  cudaStream_t s = (cudaStream_t)stream;
  char *w = (char *)d_workspace;
  int64_t *beg = (int64_t *)(w + L.beg);
  int32_t *count = (int32_t *)(w + L.count), *first = (int32_t *)(w + L.first), *base = (int32_t *)(w + L.base);
  int32_t *head = (int32_t *)(w + L.head);
  const Parts results = {(float *)(w + L.partial), (int32_t *)(w + L.come)};
  const Bounds bounds = {d_indptr, d_adj_ts, n_nodes, d_nodes, d_ts, last, beg, count, d_status};
  const bool look_up = n_query <= LOOK_UP;
  if (!look_up) {
    ORCA_CUDA(launch_dep(list_bounds_kernel, (unsigned)((n_query + 7) / 8), 256, 0, s, bounds, (int)n_query));
    ORCA_COUNT_LAUNCH();
  }
  ORCA_CUDA(launch_dep(list_parts_kernel, 1, 1024, 0, s, bounds, look_up, (int)n_query, L.target, least_of_list(n_query), first, base, head,
                       (int4 *)results.come));
  ORCA_COUNT_LAUNCH();
  const Tables t = {d_words, edges_packed ? (const uint32_t *)d_edges : nullptr, edges_packed ? nullptr : (const float *)d_edges, n_rows,
                    n_edges, d_time_w};
  const ListSlots slots = {d_adj_nbr, d_adj_eid, d_adj_ts, d_ts, beg, count, first, base, head};
  return launch_attend(d_qt, t, slots, n_query, (int64_t)n_query + L.target, d_ctx, d_valid, results, d_status, s);
}

}  // extern "C"
