// Rows held in 4 bits (packed.cuh): put into a table, read from it, attended over.
#include <algorithm>
#include <type_traits>

#include "context.cuh"
#include "packed.cuh"
#include "sampling.cuh"

namespace orca {
namespace packed {

#ifndef ORCA_GS
#define ORCA_GS 4
#endif
#ifndef ORCA_TGS
#define ORCA_TGS 0
#endif
#ifndef ORCA_LB
#define ORCA_LB 6
#endif
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
// How a group with these extremes is held (see packed.cuh): the offset rounded down, the step rounded up, so that 16 steps cover
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
// The code of x: the nearest integer to (x - offset) / step, ties to even.  A quotient in 32 bits is wrong only next to a border
// between two codes (it is off by 15 * 3 * 2^-24 at most); there 64 bits decide, in which x - offset - (k + 1/2) step has the right sign.
__device__ __noinline__ uint32_t code_at_border(float x, float offset, float step) {
  return (uint32_t)fmin(fmax(rint(((double)x - (double)offset) / (double)step), 0.0), 15.0);
}
__device__ __forceinline__ uint32_t code_of(float x, float offset, float step, float inv) {
  const float t = (x - offset) * inv;
  const float c = rintf(t);
  if (fabsf(fabsf(t - c) - 0.5f) < 1e-5f || !(inv < 1e37f)) return step > 0.f ? code_at_border(x, offset, step) : 0;
  return (uint32_t)fminf(c, 15.f);         // (t is not below 0: no value is below the offset)
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
template <int N> __device__ __forceinline__ uint32_t codes_of(const float (&x)[N], uint32_t how) {
  const float s = step_of(how), o = offset_of(how), inv = 1.f / s;
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) c |= code_of(x[j], o, s, inv) << (4 * j);
  return how == 0x7fc07fc0u ? 0 : c;
}
// extremes over the sixteen lanes of a row; `fine`: all magnitudes below 2^126
template <int N> __device__ __forceinline__ uint32_t how_of(const float (&x)[N], bool here) {
  constexpr float MOST = 8.507059173023462e37f;   // 2^126
  float lo = INFINITY, hi = -INFINITY;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < N; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]), fine &= fabsf(x[j]) < MOST;
  if (!here) lo = INFINITY, hi = -INFINITY, fine = true;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) lo = fminf(lo, __shfl_xor_sync(FULL, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(FULL, hi, o));
  const uint32_t bad = __ballot_sync(FULL, !fine);
  return (bad >> (threadIdx.x & 16) & 0xffffu) != 0 ? 0x7fc07fc0u : group_of(lo, hi);
}

// Sixteen lanes a row, two rows a warp: lane h packs columns 8 h .. 8 h + 7, a word, and, h < 11, columns 128 + 4 h .. + 3, half a word.
// Bound by instructions: some 110 a row, most of them for the codes.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) push_kernel(uint32_t *__restrict__ words, const T *__restrict__ x, int64_t x_stride,
                                                   const int32_t *__restrict__ ids, int n, int64_t n_rows,
                                                   int32_t *__restrict__ record) {
  dep_trigger();
  dep_wait();
  const int h = threadIdx.x & 15;
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
  int64_t v = -1;
  if (i < n) {
    v = ids != nullptr ? ids[i] : i;
    if (v < 0 || v >= n_rows) v = -1;
  }
  // (the winner takes its record back; another position of the same id finds the winner's or none, never its own)
  if (record != nullptr && v >= 0 && *(volatile int32_t *)&record[v] != (int)i + 1) v = -1;
  __syncwarp();
  if (record != nullptr && v >= 0 && h == 0) record[v] = 0;
  if (!__any_sync(FULL, v >= 0)) return;
  const bool tail = h < TAIL / 4;
  float a[8] = {}, b[4] = {};
  if (v >= 0) {
    constexpr int VB = ALIGNED ? (sizeof(T) == 4 ? 16 : 8) : (int)sizeof(T);
    const T *row = x + i * x_stride;
    load_values<VB>(row + 8 * h, a);
    if (tail) load_values<VB>(row + GROUP + 4 * h, b);
  }
  const uint32_t how_a = how_of(a, true), how_b = how_of(b, tail);
  const uint32_t ca = codes_of(a, how_a), cb = codes_of(b, how_b);
  if (v < 0) return;
  uint32_t *out = words + v * WORDS;
  if (h == 0) *reinterpret_cast<uint2 *>(out) = make_uint2(how_a, how_b);
  out[2 + h] = ca;
  if (h < 12) reinterpret_cast<uint16_t *>(out + 18)[h] = tail ? (uint16_t)cb : 0;      // (the twelfth: four columns that are not there)
}

// Sixteen lanes a row, PULL_ROWS rows of a thread side by side.
constexpr int PULL_ROWS = 4;
__global__ void __launch_bounds__(256) pull_kernel(const uint32_t *__restrict__ words, int64_t n_rows,
                                                   const int32_t *__restrict__ ids, int64_t n, float *__restrict__ out,
                                                   int32_t *status) {
  dep_trigger();
  dep_wait();
  const int h = threadIdx.x & 15;
  const bool tail = h < TAIL / 4;
  const int64_t i0 = (int64_t)blockIdx.x * (16 * PULL_ROWS) + (threadIdx.x >> 4);
  uint2 how[PULL_ROWS];
  uint32_t w[PULL_ROWS], u[PULL_ROWS];
#pragma unroll
  for (int r = 0; r < PULL_ROWS; ++r) {
    const int64_t i = i0 + 16 * r;
    how[r] = make_uint2(0, 0), w[r] = u[r] = 0;
    if (i < n) {
      const int v = ids[i];
      if (v >= 0 && v < n_rows) {
        const uint32_t *row = words + (int64_t)v * WORDS;
        how[r] = __ldg(reinterpret_cast<const uint2 *>(row));
        w[r] = __ldg(row + 2 + h);
        if (tail) u[r] = __ldg(reinterpret_cast<const uint16_t *>(row + 18) + h);
      } else if (h == 0) {
        report(status, ORCA_E_BOUNDS, (int)(i < 0x7fffffff ? i : 0x7fffffff));
      }
    }
  }
#pragma unroll
  for (int r = 0; r < PULL_ROWS; ++r) {
    const int64_t i = i0 + 16 * r;
    if (i >= n) break;
    float2 x[4], y[2];
    decode8(w[r], dup2(step_of(how[r].x)), dup2(offset_of(how[r].x)), x);
    decode4(u[r], dup2(step_of(how[r].y)), dup2(offset_of(how[r].y)), y);
    float4 *o = reinterpret_cast<float4 *>(out + i * D);
    o[2 * h] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
    o[2 * h + 1] = make_float4(x[2].x, x[2].y, x[3].x, x[3].y);
    if (tail) o[GROUP / 4 + h] = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
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
  const int32_t *head;    // {slots of a part, rows of several parts}
};

struct Part {
  int row, at, of;        // part `at` of `of`
  int64_t beg;            // its slots
  int n;
  int64_t out;            // where its result goes, if of > 1
};
__device__ __forceinline__ bool part_of(const TableSlots &s, int rows, int64_t job, int, Part &p) {
  if (job >= (int64_t)rows * s.parts) return false;
  p.row = (int)(job / s.parts);
  p.at = (int)(job % s.parts);
  p.of = s.parts;
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
  int kind;                          // which cosines its time encoding takes: 0 cos_small2, 1 cos_wide2 in the first 64 columns, 2 in all, 3 cos_far
};
__device__ __noinline__ float2 cos_slow2(float2 x, int kind) {
  return kind == 3 ? make_float2(cos_far(x.x), cos_far(x.y)) : cos_wide2(x);
}

__device__ __forceinline__ void async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int AT_THREADS = 64, AT_WARPS = AT_THREADS / 32;
constexpr int BATCH = 32;                                  // slots whose indices are read at a time, a lane each
template <int GS, bool EDGE32> struct Stage {              // GS slots in shared memory: the neighbour's row, then the edge's
  static constexpr int EDGE = EDGE32 ? ROW_BYTES : BYTES, SLOT = BYTES + EDGE, SIZE = GS * SLOT;
  static constexpr int COUNT = BATCH / GS;                 // stages of a batch
  static constexpr int DEPTH = EDGE32 ? COUNT / 2 : COUNT; // of which so many are under way
  static constexpr int WARP = DEPTH * SIZE;
};

// A warp takes a part of a row's slots, GS at a time.  Lanes 0..15 hold what the neighbours' rows have, lanes 16..31 the edges':
// columns 8 h .. 8 h + 7 (a word of codes) and, h < 11, columns 128 + 4 h .. + 3 (half a word); all lanes hold column pairs
// l, l + 32, l + 64 of the time encoding.  Rows come by asynchronous copies into a ring of stages, a batch of 32 slots ahead.
template <int GS, bool EDGE32, class S>
__global__ void __launch_bounds__(AT_THREADS, ORCA_LB) attend_kernel(const float *__restrict__ qt, Tables t, S slots, int rows,
                                                               float *__restrict__ ctx, uint8_t *__restrict__ valid,
                                                               float *__restrict__ partial, int32_t *status) {
  using G = Stage<GS, EDGE32>;
  extern __shared__ __align__(128) char s_ring[];
  __shared__ Rec s_rec[AT_WARPS][2][BATCH + GS - 1];
  __shared__ __align__(16) float s_p[AT_WARPS][4 * GS + 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  dep_trigger();
  dep_wait();
  Part p;
  if (!part_of(slots, rows, (int64_t)blockIdx.x * AT_WARPS + warp, lane, p)) return;
  const int side = lane >> 4, h = lane & 15;
  const bool has_tail = h < TAIL / 4, third = lane < 22;
  char *const ring = s_ring + warp * G::WARP;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  float *const pbuf = s_p[warp];

  Slot next = {0, 0, 0.f};
  auto load_indices = [&](int at0) {
    next = {0, 0, 0.f};
    if (at0 + lane < p.n) next = slot_of(slots, p, p.beg + at0 + lane);
  };
  load_indices(0);
  float2 wt[GA_P_ITERS];
  float w_most[GA_P_ITERS];
#pragma unroll
  for (int i = 0; i < GA_P_ITERS; ++i) {
    wt[i] = (i < 2 || third) ? __ldg(reinterpret_cast<const float2 *>(t.time_w) + lane + 32 * i) : make_float2(0.f, 0.f);
    w_most[i] = warp_max(fmaxf(fabsf(wt[i].x), fabsf(wt[i].y)));
  }
  // The slots of `next` that count, one behind the other, in record buffer b; behind them, up to a whole step, the first again (its
  // weight will be zero).  Returns their number.
  auto put_records = [&](int b) {
    Slot s = next;
    if (s.nbr < 0 || s.nbr >= t.n_rows || s.eid < 0 || s.eid >= t.n_edges) {
      report(status, ORCA_E_BOUNDS, p.row);
      s.nbr = 0;
    }
    const unsigned used = __ballot_sync(FULL, s.nbr != 0);
    const int n_used = __popc(used);
    const float adt = fabsf(s.dt);
    const float rest = adt * fmaxf(w_most[1], w_most[2]), first = adt * w_most[0];
    const int kind = !(fmaxf(first, rest) < 1073741824.f) || !(adt < INFINITY) ? 3 : rest >= COS_SMALL ? 2 : first >= COS_SMALL ? 1 : 0;
    const Rec r = {s.nbr, s.eid, s.dt, kind};
    const int place = __popc(used & ((1u << lane) - 1u));
    if (s.nbr != 0) s_rec[warp][b][place] = r;
    if (s.nbr != 0 && place == 0)
      for (int u = 0; u < GS - 1; ++u) s_rec[warp][b][n_used + u] = r;
    __syncwarp();
    return n_used;
  };
  // copies of stage j of the batch in record buffer b (a group of its own even when there is nothing to copy)
  auto fetch = [&](int b, int j, int n_used) {
    if (j * GS < n_used) {
      const Rec *rec = &s_rec[warp][b][j * GS];
      const uint32_t dst = ring_at + (j % G::DEPTH) * G::SIZE;
      if (EDGE32) {
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          const char *nbr = reinterpret_cast<const char *>(t.rows) + (int64_t)rec[u].nbr * BYTES;
          const char *edge = reinterpret_cast<const char *>(t.edges32) + (int64_t)rec[u].eid * ROW_BYTES;
          async16(dst + u * G::SLOT + BYTES + 16 * lane, edge + 16 * lane);
          if (lane < 11) async16(dst + u * G::SLOT + BYTES + 512 + 16 * lane, edge + 512 + 16 * lane);
          else if (lane < 17) async16(dst + u * G::SLOT + 16 * (lane - 11), nbr + 16 * (lane - 11));
        }
      } else {
#pragma unroll
        for (int i = 0; i < (GS * 12 + 31) / 32; ++i) {
          const int piece = lane + 32 * i, u = piece / 12, part = piece % 12;
          if (piece < GS * 12) {
            const char *src = part < 6 ? reinterpret_cast<const char *>(t.rows) + (int64_t)rec[u].nbr * BYTES + 16 * part
                                       : reinterpret_cast<const char *>(t.edges) + (int64_t)rec[u].eid * BYTES + 16 * (part - 6);
            async16(dst + 16 * piece, src);
          }
        }
      }
    }
    async_commit();
  };
  int n_used = put_records(0), buf = 0;
#pragma unroll 1
  for (int j = 0; j < G::DEPTH; ++j) fetch(0, j, n_used);
  if (p.n > BATCH) load_indices(BATCH);

  float2 qc[2][6], qe[2][GA_P_ITERS];          // this lane's columns of the two heads' queries
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float *qh = qt + (int64_t)p.row * QT_LD + g * QT_HEAD + side * D;
#pragma unroll
    for (int j = 0; j < 4; ++j) qc[g][j] = __ldg(reinterpret_cast<const float2 *>(qh + 8 * h) + j);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      qc[g][4 + j] = has_tail ? __ldg(reinterpret_cast<const float2 *>(qh + GROUP + 4 * h) + j) : make_float2(0.f, 0.f);
    const float *qe_h = qt + (int64_t)p.row * QT_LD + g * QT_HEAD + 2 * D;
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i)
      qe[g][i] = (i < 2 || third) ? __ldg(reinterpret_cast<const float2 *>(qe_h) + lane + 32 * i) : make_float2(0.f, 0.f);
  }
  float2 ac[2][6], ae[2][GA_P_ITERS];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
#pragma unroll
    for (int j = 0; j < 6; ++j) ac[g][j] = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i) ae[g][i] = make_float2(0.f, 0.f);
  }
  float sum0 = 0.f, sum1 = 0.f, m = -INFINITY;       // m: running maximum of this lane's head
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
        const Rec *rec = &s_rec[warp][buf][j * GS];
        const char *stage = ring + (j % G::DEPTH) * G::SIZE + side * BYTES;
        int kind = 0;
        float2 x[GS][6], te[GS][GA_P_ITERS];
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          const float2 r = *reinterpret_cast<const float2 *>(&rec[u].dt);
          kind = max(kind, __float_as_int(r.y));
          te[u][0] = mul2(dup2(r.x), wt[0]), te[u][1] = mul2(dup2(r.x), wt[1]), te[u][2] = mul2(dup2(r.x), wt[2]);
          if (EDGE32 && side) {
            const float4 *row = reinterpret_cast<const float4 *>(stage + u * G::SLOT);
            const float4 a = row[2 * h], b = row[2 * h + 1], c = has_tail ? row[GROUP / 4 + h] : make_float4(0.f, 0.f, 0.f, 0.f);
            x[u][0] = lo2(a), x[u][1] = hi2(a), x[u][2] = lo2(b), x[u][3] = hi2(b), x[u][4] = lo2(c), x[u][5] = hi2(c);
          } else {
            const char *row = stage + u * G::SLOT;
            const uint2 how = *reinterpret_cast<const uint2 *>(row);
            const uint32_t w = *reinterpret_cast<const uint32_t *>(row + 8 + 4 * h);
            const uint32_t v = has_tail ? *reinterpret_cast<const uint16_t *>(row + 72 + 2 * h) : 0;
            float2 c8[4], c4[2];
            decode8(w, dup2(step_of(how.x)), dup2(offset_of(how.x)), c8);
            decode4(v, dup2(step_of(how.y)), dup2(offset_of(how.y)), c4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][i] = c8[i];
            x[u][4] = c4[0], x[u][5] = c4[1];        // (lanes without a tail multiply what is there by queries of zero)
          }
        }
        if (kind == 0) {
#pragma unroll
          for (int u = 0; u < GS; ++u)
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) te[u][i] = cos_small2(te[u][i]);
        } else if (kind == 1) {
#pragma unroll
          for (int u = 0; u < GS; ++u) {
            te[u][0] = cos_wide2(te[u][0]);
#pragma unroll
            for (int i = 1; i < GA_P_ITERS; ++i) te[u][i] = cos_small2(te[u][i]);
          }
        } else {
#pragma unroll
          for (int u = 0; u < GS; ++u)
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) te[u][i] = cos_slow2(te[u][i], kind);
        }
        float v[V];
#pragma unroll
        for (int u = 0; u < GS; ++u)
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float2 a = mul2(x[u][0], qc[g][0]);
#pragma unroll
            for (int i = 1; i < 6; ++i) a = fma2(x[u][i], qc[g][i], a);
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) a = fma2(te[u][i], qe[g][i], a);
            v[2 * u + g] = a.x + a.y;
          }
        // lane l holds value l / LPV = 2 * slot + head
        float lg = warp_sum_many<V>(v, lane);
        if (j * GS + lane / (2 * LPV) >= n_used) lg = -INFINITY;
        float top = lg;
#pragma unroll
        for (int o = 2 * LPV; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
        const float m_new = fmaxf(m, top);
        const float from = m_new == -INFINITY ? 0.f : m_new;      // (logits of minus infinity only: weights of zero so far)
        // even lanes: the slot's weight; odd lanes: what the sums so far are scaled by (0 the first time)
        const float w = expf((lane & 1 ? m : lg) - from);
        m = m_new;
        // [slot][head] weights, [head] scales, each twice (operands of the packed instructions)
        const int where = lane & 1 ? 2 * GS + (lane / LPV & 1) : lane / LPV;
        reinterpret_cast<float2 *>(pbuf)[where] = dup2(w);
        __syncwarp();
        const float4 scale = *reinterpret_cast<const float4 *>(pbuf + 4 * GS);
        sum0 *= scale.x, sum1 *= scale.z;
        if (scale.x != 1.f || scale.z != 1.f) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float2 k = g ? hi2(scale) : lo2(scale);
#pragma unroll
            for (int i = 0; i < 6; ++i) ac[g][i] = mul2(k, ac[g][i]);
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) ae[g][i] = mul2(k, ae[g][i]);
          }
        }
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          if (j * GS + u >= n_used) break;     // (a slot that is there twice adds nothing, not even what is not a number)
          const float4 w4 = *reinterpret_cast<const float4 *>(pbuf + 4 * u);
          sum0 += w4.x, sum1 += w4.z;
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
  const bool whole = p.of == 1;
  float *out = whole ? ctx + (int64_t)p.row * QT : partial + p.out * PARTIAL;
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
  const float m0 = __shfl_sync(FULL, m, 0), m1 = __shfl_sync(FULL, m, LPV);
  if (lane == 0) {
    if (whole) {
      valid[p.row] = any_valid;
    } else {
      *reinterpret_cast<float4 *>(out + QT) = make_float4(m0, m1, sum0, sum1);
      out[QT + 4] = any_valid ? 1.f : 0.f;
    }
  }
}

// ---- packed edges: products on the tensor cores
// A warp takes a part, sixteen slots (a tile) at a time.  The codes of the tile's rows are whole numbers up to 15, exact in bf16:
// they are written out once to shared memory, sixteen slots by 2 x 176 columns, and read from there as the left operand of both
// products (m16n8k16):
//   logits   [16 slots x columns] . [columns x 6]: the query's two heads, each as three bf16 parts, which hold all 24 bits
//   sums     [16 columns x 16 slots] . [16 slots x 6]: the slots' weights times their steps, in three parts again
// What the steps and offsets of a row add is worked out apart: logit = sum over the groups of step * (q . codes) + middle * (sum of q),
// and sum p x = sum (p step) codes + sum p middle, where codes are less 8 and middle = offset + 8 step: sums of codes of either sign stay
// small, which matters to long sums, since the tensor core cuts off what it adds.  Queries are scaled by 2^-16 meanwhile, so that
// only what overflows a logit overflows a sum.  The time encoding stays in fp32 on the lanes that compute it, a pair of columns each,
// GS slots at a time.  Columns lie in the order of the nibbles that come out of a word together: 0 4 1 5 2 6 3 7.
//
// Weights are taken against a reference that only moves when a logit exceeds it by 8: up to e^8 they lose nothing in fp32, and
// the accumulators are rarely rescaled.
constexpr int TILE = 16;
constexpr int ROW16 = 2 * 22 * 16;                 // bytes of a slot's codes in bf16
constexpr int ROW16_LD = ROW16 + 16;               // (eight rows on different banks)
constexpr int TK_DEPTH = 3;                        // tiles under way
constexpr int RAW = 2 * BYTES;                     // a slot as it comes
constexpr int TK_TILE = TILE * RAW;
constexpr float RESCALE = 8.f;
constexpr float Q_SCALE = 1.f / 65536.f;
__device__ __forceinline__ float middle_of(uint32_t how) { return fmaf(8.f, step_of(how), offset_of(how)); }
struct TileWarp {                                  // shared memory of a warp
  char raw[TK_DEPTH][TK_TILE];
  char codes[TILE * ROW16_LD];                     // (at the end: the sums, [352][8] floats)
  char q[7 * ROW16_LD];                            // rows 2 part + head; row 6 is zero
  uint16_t ps[4][2][8][8];                         // [group][slots 0..7 | 8..15][column][slot]: weight times step
  float2 dt[TK_DEPTH][TILE];                       // time difference, kind
  float4 p[TILE];                                  // weights, head 0 twice, head 1 twice
  float2 lg[TILE];                                 // what the rows add to the logits
  float qsum[8];                                   // sum of the query's columns: [head][table][group]
  float osum[8];                                   // sum of weight times middle: [head][group of a table, neighbour's first]
};
static_assert(TILE * ROW16_LD >= 352 * 8 * 4, "room for the sums");

__device__ __forceinline__ uint32_t smem_at(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// codes i and i + 4 of a word shifted down by 4 i, less 8, as two bf16: or'ed under the exponent of 128, then 136 taken away
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  const uint32_t raw = (w & 0x000f000fu) | 0x43004300u, base = 0x43084308u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&raw), *reinterpret_cast<const __nv_bfloat162 *>(&base));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint4 code_word(uint32_t w) {
  return make_uint4(code_pair(w), code_pair(w >> 4), code_pair(w >> 8), code_pair(w >> 12));
}
// the parts of two values: x = hi + mid + lo, each a bf16 (the first value in the low half)
__device__ __forceinline__ void three_parts(float a, float b, uint32_t (&part)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    part[i] = *reinterpret_cast<const uint32_t *>(&h);
    a -= __uint_as_float(part[i] << 16);
    b -= __uint_as_float(part[i] & 0xffff0000u);
  }
}

template <int GS, class S>
__global__ void __launch_bounds__(AT_THREADS, 4) attend_tile_kernel(const float *__restrict__ qt, Tables t, S slots, int rows,
                                                                    float *__restrict__ ctx, uint8_t *__restrict__ valid,
                                                                    float *__restrict__ partial, int32_t *status) {
  extern __shared__ __align__(128) char s_all[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  TileWarp &sm = reinterpret_cast<TileWarp *>(s_all)[warp];
  dep_trigger();
  dep_wait();
  Part p;
  if (!part_of(slots, rows, (int64_t)blockIdx.x * AT_WARPS + warp, lane, p)) return;
  const bool third = lane < 22;

  Slot next = {0, 0, 0.f};
  auto load_indices = [&](int tile) {
    next = {0, 0, 0.f};
    const int at = tile * TILE + lane;
    if (lane < TILE && at < p.n) next = slot_of(slots, p, p.beg + at);
  };
  const int n_tiles = (p.n + TILE - 1) / TILE;
  load_indices(0);
  float2 wt[GA_P_ITERS];
  float w_most[GA_P_ITERS];
#pragma unroll
  for (int i = 0; i < GA_P_ITERS; ++i) {
    wt[i] = (i < 2 || third) ? __ldg(reinterpret_cast<const float2 *>(t.time_w) + lane + 32 * i) : make_float2(0.f, 0.f);
    // (magnitudes are in the order of their bits; what is not a number is above them all)
    w_most[i] = __uint_as_float(__reduce_max_sync(FULL, max(__float_as_uint(wt[i].x) & 0x7fffffffu, __float_as_uint(wt[i].y) & 0x7fffffffu)));
  }
  uint32_t masks = 0, masks_hi = 0;             // slots in use of the tiles under way: bits 16 * (tile % 3)
  auto mask_of = [&](int slot) { return slot == 2 ? masks_hi : (masks >> (16 * slot)) & 0xffffu; };
  // the rows of the tile whose indices are in `next` go to stage `at`
  auto fetch = [&](int at) {
    Slot s = next;
    if (s.nbr < 0 || s.nbr >= t.n_rows || s.eid < 0 || s.eid >= t.n_edges) {
      report(status, ORCA_E_BOUNDS, p.row);
      s.nbr = 0;
    }
    const uint32_t used = __ballot_sync(FULL, s.nbr != 0);
    if (at == 2) masks_hi = used;
    else masks = at == 1 ? (masks & 0xffffu) | (used << 16) : (masks & 0xffff0000u) | used;
    if (lane < TILE) {
      const float adt = fabsf(s.dt);
      const float first = adt * w_most[0], rest = adt * fmaxf(w_most[1], w_most[2]);
      const int kind = !(fmaxf(first, rest) < 1073741824.f) || !(adt < INFINITY) ? 3 : rest >= COS_SMALL ? 2
                       : first >= COS_SMALL || adt * w_most[2] > 3.14f ? 1 : 0;
      sm.dt[at][lane] = make_float2(s.dt, __int_as_float(s.nbr != 0 ? kind : 0));
    }
    const uint32_t dst = smem_at(sm.raw[at]);
#pragma unroll
    for (int i = 0; i < TILE * 12 / 32; ++i) {
      const int piece = lane + 32 * i, u = piece / 12, part = piece % 12;
      const int nbr = __shfl_sync(FULL, s.nbr, u), eid = __shfl_sync(FULL, s.eid, u);
      const char *src = part < 6 ? reinterpret_cast<const char *>(t.rows) + (int64_t)nbr * BYTES + 16 * part
                                 : reinterpret_cast<const char *>(t.edges) + (int64_t)eid * BYTES + 16 * (part - 6);
      if (nbr != 0) async16(dst + 16 * piece, src);
    }
  };
#pragma unroll 1
  for (int k = 0; k < TK_DEPTH; ++k) {
    if (k < n_tiles) {
      fetch(k);
      if (k + 1 < n_tiles) load_indices(k + 1);
    }
    async_commit();
  }

  // the query: its columns over the tables in three parts, its time columns on the lanes
  const float *q_row = qt + (int64_t)p.row * QT_LD;
  {
    float sums[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      const int g = i / 6, table = (i / 3) & 1, it = i % 3;          // two rounds of 32 pairs of columns, then 24
      const int r = it * 32 + lane, w = r / 4, j = r % 4;
      if (it < 2 || lane < 24) {
        const float *src = q_row + g * QT_HEAD + table * D + 8 * w + j;
        const float a = __ldg(src) * Q_SCALE, b = w < 21 ? __ldg(src + 4) * Q_SCALE : 0.f;
        uint32_t part[3];
        three_parts(a, b, part);
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t *>(sm.q + (2 * k + g) * ROW16_LD + (table * 22 + w) * 16 + 4 * j) = part[k];
        sums[g * 4 + table * 2 + (it == 2)] += a + b;
      }
    }
    const float total = warp_sum_many<8>(sums, lane);
    if (lane % 4 == 0) sm.qsum[lane / 4] = total;
    for (int i = lane; i < ROW16_LD / 4; i += 32) reinterpret_cast<uint32_t *>(sm.q + 6 * ROW16_LD)[i] = 0;
    // (columns 6 and 7 of the weights stay zero)
    for (int i = lane; i < 4 * 2 * 2 * 4; i += 32) reinterpret_cast<uint32_t *>(&sm.ps[i / 16][i / 8 % 2][6][0])[i % 8] = 0;
  }
  float2 qe[2][GA_P_ITERS], ae[2][GA_P_ITERS];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i) {
      qe[g][i] = (i < 2 || third) ? __ldg(reinterpret_cast<const float2 *>(q_row + g * QT_HEAD + 2 * D) + lane + 32 * i) : make_float2(0.f, 0.f);
      ae[g][i] = make_float2(0.f, 0.f);
    }
  float acc[22][4];                              // sums of 16 columns by 8: head 0 and 1 of the first part, of the second, third, nothing
#pragma unroll
  for (int i = 0; i < 22; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  float osum[4] = {0.f, 0.f, 0.f, 0.f};          // lane = 2 slot + head: weight times middle, by group
  float psum = 0.f, ref = -INFINITY;             // of this lane's head: sum of weights, what they are taken against
  bool any_valid = false;
  constexpr int V = 2 * GS, LPV = 32 / V;
  const uint32_t codes_at = smem_at(sm.codes), q_at = smem_at(sm.q), ps_at = smem_at(sm.ps);
  const uint32_t a_at = codes_at + (lane & 15) * ROW16_LD + (lane >> 4) * 16;                            // slots l % 16, columns 8 (l / 16)
  const uint32_t b_at = q_at + min(lane & 7, 6) * ROW16_LD + (lane >> 3) * 16;
  const uint32_t at_at = codes_at + ((lane & 7) + (lane >> 4) * 8) * ROW16_LD + ((lane >> 3) & 1) * 16;   // transposed: columns by slots
  const int side = lane >> 4, h = lane & 15;
  int stage = 0;
  for (int tile = 0; tile < n_tiles; ++tile) {
    async_wait<TK_DEPTH - 1>();
    __syncwarp();
    const uint32_t used = mask_of(stage);
    if (used != 0) {
      any_valid = true;
      const char *raw = sm.raw[stage];
      // codes to shared memory: sixteen words of either row a slot, then the six last ones, two slots at a time
#pragma unroll
      for (int s = 0; s < TILE; ++s)
        *reinterpret_cast<uint4 *>(sm.codes + s * ROW16_LD + side * (ROW16 / 2) + 16 * h) =
            code_word(*reinterpret_cast<const uint32_t *>(raw + s * RAW + side * BYTES + 8 + 4 * h));
      if (lane < 24) {
        const int s0 = lane / 12, table = lane / 6 % 2, w = 16 + lane % 6;
#pragma unroll
        for (int s = 0; s < TILE; s += 2)
          *reinterpret_cast<uint4 *>(sm.codes + (s + s0) * ROW16_LD + table * (ROW16 / 2) + 16 * w) =
              code_word(*reinterpret_cast<const uint32_t *>(raw + (s + s0) * RAW + table * BYTES + 8 + 4 * w));
      }
      sm.p[lane & 15] = make_float4(0.f, 0.f, 0.f, 0.f);
      __syncwarp();
      {
        float c[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) c[i][j] = 0.f;
#pragma unroll
        for (int k = 0; k < 22; k += 2) {        // steps of sixteen columns: eight of a first group, three of a second, twice
          uint32_t a[4], b[4];
          ldsm4(b, b_at + k * 32);
          ldsm4(a, a_at + k * 32);
          mma_bf16(c[k / 11 * 2 + (k % 11 >= 8)], a, b[0], b[1]);
          ldsm4(a, a_at + (k + 1) * 32);
          mma_bf16(c[(k + 1) / 11 * 2 + ((k + 1) % 11 >= 8)], a, b[2], b[3]);
        }
        // this thread: slots l / 4 and l / 4 + 8, heads of part l % 4
        const float4 qs0 = *reinterpret_cast<const float4 *>(sm.qsum), qs1 = *reinterpret_cast<const float4 *>(sm.qsum + 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int s = lane / 4 + 8 * i;
          const uint2 hn = *reinterpret_cast<const uint2 *>(raw + s * RAW), he = *reinterpret_cast<const uint2 *>(raw + s * RAW + BYTES);
          float l0 = step_of(hn.x) * c[0][2 * i] + step_of(hn.y) * c[1][2 * i] + step_of(he.x) * c[2][2 * i] + step_of(he.y) * c[3][2 * i];
          float l1 = step_of(hn.x) * c[0][2 * i + 1] + step_of(hn.y) * c[1][2 * i + 1] + step_of(he.x) * c[2][2 * i + 1] +
                     step_of(he.y) * c[3][2 * i + 1];
          l0 += __shfl_xor_sync(FULL, l0, 1), l1 += __shfl_xor_sync(FULL, l1, 1);
          l0 += __shfl_xor_sync(FULL, l0, 2), l1 += __shfl_xor_sync(FULL, l1, 2);
          l0 += middle_of(hn.x) * qs0.x + middle_of(hn.y) * qs0.y + middle_of(he.x) * qs0.z + middle_of(he.y) * qs0.w;
          l1 += middle_of(hn.x) * qs1.x + middle_of(hn.y) * qs1.y + middle_of(he.x) * qs1.z + middle_of(he.y) * qs1.w;
          if (lane % 4 == 0) sm.lg[s] = make_float2(l0 * (1.f / Q_SCALE), l1 * (1.f / Q_SCALE));
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int s0 = 0; s0 < TILE; s0 += GS) {
        if (((used >> s0) & ((1u << GS) - 1u)) == 0) continue;
        float2 te[GS][GA_P_ITERS];
        int kind = 0;
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          const float2 r = sm.dt[stage][s0 + u];
          kind = max(kind, __float_as_int(r.y));
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) te[u][i] = mul2(dup2(r.x), wt[i]);
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
#pragma unroll
          for (int u = 0; u < GS; ++u)
#pragma unroll
            for (int i = 0; i < GA_P_ITERS; ++i) te[u][i] = cos_slow2(te[u][i], kind);
        }
        float v[V];
#pragma unroll
        for (int u = 0; u < GS; ++u)
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float2 a = mul2(te[u][0], qe[g][0]);
            a = fma2(te[u][1], qe[g][1], a);
            a = fma2(te[u][2], qe[g][2], a);
            v[2 * u + g] = a.x + a.y;
          }
        // lane l holds value l / LPV = 2 * slot + head
        float lg = warp_sum_many<V>(v, lane);
        const int su = s0 + lane / (2 * LPV), head = lane / LPV & 1;
        lg += reinterpret_cast<const float *>(&sm.lg[su])[head];
        if (!(used >> su & 1u)) lg = -INFINITY;
        float top = lg;
#pragma unroll
        for (int o = 2 * LPV; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
        const bool moves = top > ref + RESCALE || (ref == -INFINITY && top > ref);
        if (__any_sync(FULL, moves)) {
          const float scale = moves ? expf(ref - top) : 1.f;       // (0 the first time: nothing has been added)
          if (moves) ref = top;
          psum *= scale;
          const float k0 = __shfl_sync(FULL, scale, 0), k1 = __shfl_sync(FULL, scale, LPV);
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) ae[0][i] = mul2(dup2(k0), ae[0][i]), ae[1][i] = mul2(dup2(k1), ae[1][i]);
#pragma unroll
          for (int i = 0; i < 22; ++i) acc[i][0] *= k0, acc[i][1] *= k1, acc[i][2] *= k0, acc[i][3] *= k1;
#pragma unroll
          for (int i = 0; i < 4; ++i) osum[i] *= lane & 1 ? k1 : k0;
          if (lane < TILE) {                     // weights of this tile that are there already
            const float4 w = sm.p[lane];
            sm.p[lane] = make_float4(w.x * k0, w.y * k0, w.z * k1, w.w * k1);
          }
          __syncwarp();
        }
        const float w = expf(lg - (ref == -INFINITY ? 0.f : ref));      // (logits of minus infinity only: weights of zero)
        psum += w;
        reinterpret_cast<float2 *>(&sm.p[su])[head] = dup2(w);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < GS; ++u) {
          if (!(used >> (s0 + u) & 1u)) continue;      // (nothing of a slot that is not there, not even what is not a number)
          const float4 w4 = sm.p[s0 + u];
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) ae[0][i] = fma2(lo2(w4), te[u][i], ae[0][i]), ae[1][i] = fma2(hi2(w4), te[u][i], ae[1][i]);
        }
        __syncwarp();
      }
      {
        // this lane: slot l / 2, head l % 2: weight times step in three parts, weight times middle
        const int s = lane / 2, head = lane & 1;
        const float w = reinterpret_cast<const float *>(&sm.p[s])[2 * head];
        const uint2 hn = *reinterpret_cast<const uint2 *>(raw + s * RAW), he = *reinterpret_cast<const uint2 *>(raw + s * RAW + BYTES);
        const uint32_t how[4] = {hn.x, hn.y, he.x, he.y};
        const bool on = used >> s & 1u;
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          uint32_t part[3];
          three_parts(on ? w * step_of(how[g]) : 0.f, on ? w * step_of(how[g + 1]) : 0.f, part);
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            sm.ps[g][s / 8][2 * k + head][s % 8] = (uint16_t)part[k];
            sm.ps[g + 1][s / 8][2 * k + head][s % 8] = (uint16_t)(part[k] >> 16);
          }
          if (on) osum[g] = fmaf(w, middle_of(how[g]), osum[g]), osum[g + 1] = fmaf(w, middle_of(how[g + 1]), osum[g + 1]);
        }
        __syncwarp();
        uint32_t b[2][4];
        ldsm4(b[0], ps_at + lane * 16);
        ldsm4(b[1], ps_at + 512 + lane * 16);
#pragma unroll
        for (int i = 0; i < 22; ++i) {
          uint32_t a[4];
          ldsm4t(a, at_at + i * 32);
          const int second = i % 11 >= 8;
          mma_bf16(acc[i], a, b[i / 11][2 * second], b[i / 11][2 * second + 1]);
        }
      }
    }
    __syncwarp();
    if (tile + TK_DEPTH < n_tiles) {
      fetch(stage);
      if (tile + TK_DEPTH + 1 < n_tiles) load_indices(tile + TK_DEPTH + 1);
    }
    async_commit();
    stage = stage == TK_DEPTH - 1 ? 0 : stage + 1;
  }
  async_wait<0>();
  // the result
#pragma unroll
  for (int o = 2 * LPV; o < 32; o <<= 1) psum += __shfl_xor_sync(FULL, psum, o);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int o = 2; o < 32; o <<= 1) osum[i] += __shfl_xor_sync(FULL, osum[i], o);
  if (lane < 2) *reinterpret_cast<float4 *>(sm.osum + 4 * lane) = make_float4(osum[0], osum[1], osum[2], osum[3]);
  float *const sums = reinterpret_cast<float *>(sm.codes);      // [column][part and head]
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 22; ++i) {
    *reinterpret_cast<float2 *>(sums + (16 * i + lane / 4) * 8 + 2 * (lane % 4)) = make_float2(acc[i][0], acc[i][1]);
    *reinterpret_cast<float2 *>(sums + (16 * i + lane / 4 + 8) * 8 + 2 * (lane % 4)) = make_float2(acc[i][2], acc[i][3]);
  }
  __syncwarp();
  const float sum0 = __shfl_sync(FULL, psum, 0), sum1 = __shfl_sync(FULL, psum, LPV);
  const float m0 = __shfl_sync(FULL, ref, 0), m1 = __shfl_sync(FULL, ref, LPV);
  const bool whole = p.of == 1;
  float *out = whole ? ctx + (int64_t)p.row * QT : partial + p.out * PARTIAL;
  const float k0 = !any_valid ? 0.f : whole ? 1.f / sum0 : 1.f, k1 = !any_valid ? 0.f : whole ? 1.f / sum1 : 1.f;
#pragma unroll
  for (int table = 0; table < 2; ++table)
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const int c = lane + 32 * i, j = c % 8;
      if (c < D) {
        const float *v = sums + (table * 176 + c - j + (j < 4 ? 2 * j : 2 * j - 7)) * 8;
        const float4 a = *reinterpret_cast<const float4 *>(v);
        const float2 b = *reinterpret_cast<const float2 *>(v + 4);
        const int g = table * 2 + (i >= GROUP / 32);
        out[table * D + c] = (a.x + a.z + b.x + sm.osum[g]) * k0;
        out[KEY + table * D + c] = (a.y + a.w + b.y + sm.osum[4 + g]) * k1;
      }
    }
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int i = 0; i < GA_P_ITERS; ++i)
      if (i < 2 || third) reinterpret_cast<float2 *>(out + g * KEY + 2 * D)[lane + 32 * i] = mul2(dup2(g ? k1 : k0), ae[g][i]);
  if (lane == 0) {
    if (whole) {
      valid[p.row] = any_valid;
    } else {
      *reinterpret_cast<float4 *>(out + QT) = make_float4(m0, m1, sum0, sum1);
      out[QT + 4] = any_valid ? 1.f : 0.f;
    }
  }
}

// Joins the parts of rows that have several.  A block takes 32 columns of four of a row at a time; its warps take parts in turn,
// and their sums are added in the order of the warps.
constexpr int JOIN_COLS = (QT / 4 + 31) / 32;      // 9 blocks of columns
template <int JOIN_WARPS>
__global__ void __launch_bounds__(32 * JOIN_WARPS) join_kernel(const float *__restrict__ partial, const int32_t *__restrict__ several,
                                                               const int32_t *__restrict__ d_n, int n_rows, int parts,
                                                               const int32_t *__restrict__ first, const int32_t *__restrict__ base,
                                                               float *__restrict__ ctx, uint8_t *__restrict__ valid) {
  __shared__ float4 s_sum[JOIN_WARPS][32];
  __shared__ float s_top[JOIN_WARPS][2], s_total[JOIN_WARPS][2];
  __shared__ int s_valid[JOIN_WARPS];
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = d_n != nullptr ? *d_n : n_rows;
  for (int64_t item = blockIdx.x; item < (int64_t)n * JOIN_COLS; item += gridDim.x) {
    const int i = (int)(item / JOIN_COLS), col = (int)(item % JOIN_COLS) * 32 + lane;
    const int row = several != nullptr ? several[i] : i;
    const int of = first != nullptr ? first[row + 1] - first[row] : parts;
    const float *p0 = partial + (first != nullptr ? (int64_t)base[row] : (int64_t)row * parts) * PARTIAL;
    float m0 = -INFINITY, m1 = -INFINITY;
    bool some = false;
    for (int j = threadIdx.x; j < of; j += blockDim.x) {
      const float *p = p0 + (int64_t)j * PARTIAL + QT;
      m0 = fmaxf(m0, p[0]), m1 = fmaxf(m1, p[1]);
      some |= p[4] != 0.f;
    }
    m0 = warp_max(m0), m1 = warp_max(m1);
    some = __any_sync(FULL, some);
    if (lane == 0) s_top[warp][0] = m0, s_top[warp][1] = m1, s_valid[warp] = some;
    __syncthreads();
    some = false;
    for (int w = 0; w < JOIN_WARPS; ++w) m0 = fmaxf(m0, s_top[w][0]), m1 = fmaxf(m1, s_top[w][1]), some |= s_valid[w] != 0;
    if (m0 == -INFINITY) m0 = 0.f;
    if (m1 == -INFINITY) m1 = 0.f;
    const bool second = col >= KEY / 4;            // (a head has 129 columns of four)
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float total0 = 0.f, total1 = 0.f;
    constexpr int AHEAD = 4;
    for (int j0 = warp; j0 < of; j0 += AHEAD * JOIN_WARPS) {
      float4 st[AHEAD], v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int j = j0 + u * JOIN_WARPS;
        const float *p = p0 + (int64_t)min(j, of - 1) * PARTIAL;
        st[u] = *reinterpret_cast<const float4 *>(p + QT);
        v[u] = reinterpret_cast<const float4 *>(p)[min(col, QT / 4 - 1)];
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (j0 + u * JOIN_WARPS >= of) break;
        const float w0 = expf(st[u].x - m0), w1 = expf(st[u].y - m1);
        total0 += w0 * st[u].z, total1 += w1 * st[u].w;
        const float w = second ? w1 : w0;
        a.x = fmaf(w, v[u].x, a.x), a.y = fmaf(w, v[u].y, a.y), a.z = fmaf(w, v[u].z, a.z), a.w = fmaf(w, v[u].w, a.w);
      }
    }
    s_sum[warp][lane] = a;
    if (lane == 0) s_total[warp][0] = total0, s_total[warp][1] = total1;
    __syncthreads();
    if (warp == 0 && col < QT / 4) {
      float total = 0.f;
      a = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < JOIN_WARPS; ++w) {
        const float4 v = s_sum[w][lane];
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        total += s_total[w][second];
      }
      const float k = some ? 1.f / total : 0.f;
      reinterpret_cast<float4 *>(ctx + (int64_t)row * QT)[col] = some ? make_float4(a.x * k, a.y * k, a.z * k, a.w * k)
                                                                     : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (threadIdx.x == 0 && col == 0) valid[row] = some;
    __syncthreads();
  }
}

// Where a row's list lies: the interactions of its node before its time, the last `last` of them (0: all).
__global__ void __launch_bounds__(256) list_bounds_kernel(const int64_t *__restrict__ indptr, const double *__restrict__ ts,
                                                          int64_t n_nodes, const int32_t *__restrict__ nodes,
                                                          const double *__restrict__ time, int64_t last, int rows,
                                                          int64_t *__restrict__ beg, int32_t *__restrict__ count, int32_t *status) {
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int v = nodes[r];
  long long lo = 0, hi = 0;
  if (v >= 0 && v < n_nodes) lo = indptr[v], hi = indptr[v + 1];
  else if (lane == 0) report(status, ORCA_E_BOUNDS, r);
  const long long end = lower_bound_group<32>(ts, lo, hi, time[r], lane, FULL, 0);
  if (last > 0 && end - lo > last) lo = end - last;
  if (lane == 0) beg[r] = lo, count[r] = (int32_t)(end - lo);
}

// Cuts the lists into parts: about `target` of them over all rows, none shorter than `least` slots but a row's last.
__global__ void __launch_bounds__(1024) list_parts_kernel(const int32_t *__restrict__ count, int rows, int target, int least,
                                                          int32_t *__restrict__ first, int32_t *__restrict__ base,
                                                          int32_t *__restrict__ several, int32_t *__restrict__ head) {
  __shared__ unsigned long long s_warp[32];
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
  const unsigned long long want = ((total + target - 1) / target + 31) / 32 * 32;
  const int len = (int)(want < (unsigned)least ? least : want > 0x7fffffe0ull ? 0x7fffffe0 : want);
  // summed together: parts (32 bits), parts of rows of several (16: twice the target at most), such rows (16)
  unsigned long long carry = 0;
  for (int r0 = 0, k = 0; r0 < rows; r0 += 1024, ++k) {
    const int r = r0 + threadIdx.x;
    const int n = k < KEPT ? (k == 0 ? kept[0] : k == 1 ? kept[1] : k == 2 ? kept[2] : kept[3]) : r < rows ? count[r] : 0;
    const unsigned parts = r < rows ? max(1, (int)(((long long)n + len - 1) / len)) : 0;
    const unsigned long long mine = parts > 1 ? parts | (unsigned long long)parts << 32 | 1ull << 48 : parts;
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
      base[r] = (int32_t)(before >> 32 & 0xffff);
      if (parts > 1) several[before >> 48] = r;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) first[rows] = (int32_t)(unsigned)carry, head[0] = len, head[1] = (int32_t)(carry >> 48);
}

// ---------------------------------------------------------------------------------------------- host
constexpr int PARTS_PER_SM = 16;      // parts that the slots of few rows are cut into, for every SM
constexpr int LEAST_PART = 64;        // slots

static int sms() {
  Ctx *c = cur();
  return c != nullptr ? c->sm_count : 148;
}
static int64_t up256(int64_t b) { return (b + 255) & ~255ll; }

// parts of a row of a table: one, unless there are too few rows to fill the GPU
static int table_parts(int rows, int64_t k) {
  const int64_t by_rows = rows > 0 ? (int64_t)sms() * PARTS_PER_SM / rows : 1;
  const int64_t by_len = (k + LEAST_PART - 1) / LEAST_PART;
  return (int)std::max<int64_t>(1, std::min(by_rows, by_len));
}

struct ListLayout {
  int64_t beg, count, first, base, several, head, partial, total;
  int target;
};
static ListLayout list_layout(int rows) {
  ListLayout L;
  L.target = sms() * PARTS_PER_SM;
  L.beg = 0;
  L.count = up256((int64_t)rows * 8);
  L.first = L.count + up256((int64_t)rows * 4);
  L.base = L.first + up256((int64_t)rows * 4 + 4);
  L.several = L.base + up256((int64_t)rows * 4);
  L.head = L.several + up256((int64_t)rows * 4);
  L.partial = L.head + 256;
  // a part of a row of several is at least half full on average: no more than twice as many as the target
  L.total = L.partial + up256((int64_t)2 * L.target * PARTIAL * 4);
  return L;
}

template <class S>
static int launch_attend(const float *d_qt, const Tables &t, const S &slots, int rows, int64_t jobs, float *d_ctx, uint8_t *d_valid,
                         float *partial, int32_t *d_status, cudaStream_t s) {
  const unsigned grid = (unsigned)((jobs + AT_WARPS - 1) / AT_WARPS);
  if (ORCA_TGS == 0 && t.edges32 == nullptr) {
    constexpr int smem = AT_WARPS * Stage<ORCA_GS, false>::WARP;
    ORCA_CUDA(launch_dep(attend_kernel<ORCA_GS, false, S>, grid, AT_THREADS, smem, s, d_qt, t, slots, rows, d_ctx, d_valid, partial, d_status));
  } else if (t.edges32 != nullptr) {
    constexpr int smem = AT_WARPS * Stage<ORCA_GS, true>::WARP;
    static_assert(smem + 4096 < 227 * 1024 / 6, "six blocks an SM");
    ORCA_CUDA(launch_dep(attend_kernel<ORCA_GS, true, S>, grid, AT_THREADS, smem, s, d_qt, t, slots, rows, d_ctx, d_valid, partial, d_status));
  } else {
    constexpr int smem = AT_WARPS * (int)sizeof(TileWarp);
    static_assert(4 * (smem + 1024) <= 228 * 1024, "four blocks an SM");
    auto kernel = attend_tile_kernel<ORCA_TGS == 0 ? 4 : ORCA_TGS, S>;
    ORCA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ORCA_CUDA(launch_dep(kernel, grid, AT_THREADS, smem, s, d_qt, t, slots, rows, d_ctx, d_valid, partial, d_status));
  }
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

// Few rows have many parts each: 32 warps to a row's columns then (three rows of 790 parts 51 us with eight).
static int launch_join(int n_query, int n_rows, const float *partial, const int32_t *several, const int32_t *d_n, int parts,
                       const int32_t *first, const int32_t *base, float *d_ctx, uint8_t *d_valid, cudaStream_t s) {
  const bool few = n_query <= 64;
  const int64_t items = (int64_t)n_query * JOIN_COLS;
  ORCA_CUDA(launch_dep(few ? join_kernel<32> : join_kernel<8>, (unsigned)std::min<int64_t>(items, (int64_t)sms() * 8), few ? 1024 : 256, 0, s,
                       partial, several, d_n, n_rows, parts, first, base, d_ctx, d_valid));
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
  if (n == 0) return ORCA_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (d_ids != nullptr) {
    ORCA_CUDA(launch_dep(push_mark_kernel, std::min((n + 255) / 256, sms() * 8), 256, 0, s, d_ids, (int)n, n_rows, d_record, d_status));
    ORCA_COUNT_LAUNCH();
  }
  const unsigned grid = (unsigned)((n + 15) / 16);
  const int size = type == ORCA_F32 ? 4 : 2, wide = type == ORCA_F32 ? 16 : 8;
  ORCA_CHECK_ARG((uintptr_t)d_x % size == 0);
  const bool aligned = (uintptr_t)d_x % wide == 0 && x_stride * size % wide == 0;
  auto go = [&](auto *t) {
    using T = std::remove_pointer_t<decltype(t)>;
    ORCA_CUDA(launch_dep(aligned ? push_kernel<T, true> : push_kernel<T, false>, grid, 256, 0, s, d_words, (const T *)d_x, x_stride, d_ids,
                         (int)n, n_rows, d_record));
    ORCA_COUNT_LAUNCH();
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  };
  return type == ORCA_F32 ? go((float *)nullptr) : type == ORCA_BF16 ? go((__nv_bfloat16 *)nullptr) : go((__half *)nullptr);
}

int orca_packed_pull(const uint32_t *d_words, int64_t n_rows, const int32_t *d_ids, int64_t n, float *d_out, int32_t *d_status,
                     void *stream) {
  ORCA_CHECK_ARG(d_words && n_rows > 0 && n >= 0 && (n == 0 || (d_ids && d_out)));
  ORCA_CHECK_ARG((uintptr_t)d_words % 16 == 0 && (uintptr_t)d_out % 16 == 0 && n / (16 * PULL_ROWS) < 0x7fffffffll);
  if (n == 0) return ORCA_OK;
  ORCA_CUDA(launch_dep(pull_kernel, (unsigned)((n + 16 * PULL_ROWS - 1) / (16 * PULL_ROWS)), 256, 0, (cudaStream_t)stream, d_words, n_rows, d_ids, n, d_out, d_status));
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

int64_t orca_packed_attend_workspace_bytes(int32_t n_rows, int64_t k) {
  if (n_rows < 0 || k < 0) return -1;
  const int parts = table_parts(n_rows, k);
  return parts > 1 ? (int64_t)n_rows * parts * PARTIAL * 4 : 0;
}

int orca_packed_attend(const float *d_qt, const uint32_t *d_words, int64_t n_rows, const void *d_edges, int64_t n_edges,
                       int32_t edges_packed, const float *d_time_w, const int32_t *d_nbr, const int32_t *d_eid, const float *d_delta,
                       int64_t k, int32_t n_query, float *d_ctx, uint8_t *d_valid, int32_t *d_status, void *d_workspace,
                       int64_t workspace_bytes, void *stream) {
  ORCA_CHECK_ARG(n_query >= 0 && k >= 0 && k <= 0x7fffffffll);
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
  const int rc = launch_attend(d_qt, t, slots, n_query, (int64_t)n_query * parts, d_ctx, d_valid, (float *)d_workspace, d_status, s);
  if (rc || parts == 1) return rc;
  return launch_join(n_query, n_query, (const float *)d_workspace, nullptr, nullptr, parts, nullptr, nullptr, d_ctx, d_valid, s);
}

int64_t orca_packed_attend_lists_workspace_bytes(int32_t n_query) { return n_query < 0 ? -1 : list_layout(n_query).total; }

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
  const ListLayout L = list_layout(n_query);
  if (workspace_bytes < L.total) return set_error(ORCA_E_BADARG, "%s: workspace of %lld bytes is too small", __func__, (long long)workspace_bytes);
  cudaStream_t s = (cudaStream_t)stream;
  char *w = (char *)d_workspace;
  int64_t *beg = (int64_t *)(w + L.beg);
  int32_t *count = (int32_t *)(w + L.count), *first = (int32_t *)(w + L.first), *base = (int32_t *)(w + L.base);
  int32_t *several = (int32_t *)(w + L.several), *head = (int32_t *)(w + L.head);
  float *partial = (float *)(w + L.partial);
  ORCA_CUDA(launch_dep(list_bounds_kernel, (unsigned)((n_query + 7) / 8), 256, 0, s, d_indptr, d_adj_ts, n_nodes, d_nodes, d_ts, last,
                       (int)n_query, beg, count, d_status));
  ORCA_COUNT_LAUNCH();
  ORCA_CUDA(launch_dep(list_parts_kernel, 1, 1024, 0, s, (const int32_t *)count, (int)n_query, L.target, LEAST_PART, first, base, several, head));
  ORCA_COUNT_LAUNCH();
  const Tables t = {d_words, edges_packed ? (const uint32_t *)d_edges : nullptr, edges_packed ? nullptr : (const float *)d_edges, n_rows,
                    n_edges, d_time_w};
  const ListSlots slots = {d_adj_nbr, d_adj_eid, d_adj_ts, d_ts, beg, count, first, base, head};
  const int rc = launch_attend(d_qt, t, slots, n_query, (int64_t)n_query + L.target, d_ctx, d_valid, partial, d_status, s);
  if (rc) return rc;
  return launch_join(n_query, 0, partial, several, head + 1, 0, first, base, d_ctx, d_valid, s);
}

}  // extern "C"
