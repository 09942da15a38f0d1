// Rows held in 4 bits (packed.cuh): put into a table, read from it, attended over.
#include <algorithm>

#include "context.cuh"
#include "packed.cuh"
#include "sampling.cuh"

namespace orca {
namespace packed {

constexpr unsigned FULL = 0xffffffffu;

// ---------------------------------------------------------------------------------------------- push and pull
template <typename T> __device__ __forceinline__ float as_float(T v) { return (float)v; }

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

// How a group with these extremes is held (see packed.cuh): the offset rounded down, the step rounded up, so that 16 steps cover
// the group and a code is off by half a step at most.  The division is exact to 53 bits: what it gives decides between two bfloat16.
__device__ __forceinline__ uint32_t group_of(float lo, float hi) {
  const uint32_t b = __float_as_uint(lo);
  const uint32_t offset = ((int32_t)b < 0 && (b & 0xffffu) != 0 ? b + 0x10000u : b) & 0xffff0000u;
  const uint32_t s = __float_as_uint(__double2float_ru(((double)hi - (double)__uint_as_float(offset)) / 15.0));
  return ((s + 0xffffu) >> 16) | offset;
}
// The code of x: the nearest integer to (x - offset) / step, ties to even.  A quotient in 32 bits is wrong only next to a border
// between two codes (it is off by 15 * 3 * 2^-24 at most); there 64 bits decide, in which x - offset - (k + 1/2) step has the right sign.
__device__ __forceinline__ uint32_t code_of(float x, float offset, float step, float inv) {
  if (!(step > 0.f)) return 0;
  const float t = (x - offset) * inv;
  const float k = floorf(t);
  const float f = t - k;
  uint32_t c = (uint32_t)fminf(fmaxf(rintf(t), 0.f), 15.f);
  if (fabsf(f - 0.5f) < 1e-5f || !(inv < 1e37f)) {
    const double q = ((double)x - (double)offset) / (double)step;
    c = (uint32_t)fmin(fmax(rint(q), 0.0), 15.0);
  }
  return c;
}

// A warp a row: lane l packs columns 4 l .. 4 l + 3 of the first group, lanes 0..10 four columns of the second.
template <typename T>
__global__ void __launch_bounds__(256) push_kernel(uint32_t *__restrict__ words, const T *__restrict__ x, int64_t x_stride,
                                                   const int32_t *__restrict__ ids, int n, int64_t n_rows,
                                                   int32_t *__restrict__ record) {
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= n) return;
  const int v = ids != nullptr ? ids[i] : i;
  if (v < 0 || v >= n_rows) return;
  if (record != nullptr) {
    // (the winner takes its record back; another position of the same id finds the winner's or none, never its own)
    const int last = __shfl_sync(FULL, lane == 0 ? *(volatile int32_t *)&record[v] : 0, 0);
    if (last != i + 1) return;
    if (lane == 0) record[v] = 0;
  }
  const T *row = x + (int64_t)i * x_stride;
  const bool tail = lane < TAIL / 4;
  float a[4], b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = as_float(row[4 * lane + j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = tail ? as_float(row[GROUP + 4 * lane + j]) : 0.f;
  constexpr float MOST = 8.507059173023462e37f;   // 2^126
  bool fine_a = true, fine_b = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) fine_a &= fabsf(a[j]) < MOST, fine_b &= fabsf(b[j]) < MOST;
  fine_a = __all_sync(FULL, fine_a), fine_b = __all_sync(FULL, fine_b);
  const float lo_a = warp_min(fminf(fminf(a[0], a[1]), fminf(a[2], a[3])));
  const float hi_a = warp_max(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
  const float lo_b = warp_min(tail ? fminf(fminf(b[0], b[1]), fminf(b[2], b[3])) : INFINITY);
  const float hi_b = warp_max(tail ? fmaxf(fmaxf(b[0], b[1]), fmaxf(b[2], b[3])) : -INFINITY);
  // lanes 0 and 1 work the two groups out
  uint32_t how = 0;
  if (lane < 2) how = (lane == 0 ? fine_a : fine_b) ? group_of(lane == 0 ? lo_a : lo_b, lane == 0 ? hi_a : hi_b) : 0x7fc07fc0u;
  const uint32_t how_a = __shfl_sync(FULL, how, 0), how_b = __shfl_sync(FULL, how, 1);
  uint32_t ca = 0, cb = 0;
  {
    const float s = step_of(how_a), o = offset_of(how_a), inv = 1.f / s;
#pragma unroll
    for (int j = 0; j < 4; ++j) ca |= code_of(a[j], o, s, inv) << (4 * j);
  }
  if (tail) {
    const float s = step_of(how_b), o = offset_of(how_b), inv = 1.f / s;
#pragma unroll
    for (int j = 0; j < 4; ++j) cb |= code_of(b[j], o, s, inv) << (4 * j);
  }
  uint32_t *out = words + (int64_t)v * WORDS;
  if (lane < 2) out[lane] = how;
  uint16_t *half = reinterpret_cast<uint16_t *>(out + 2);
  half[lane] = (uint16_t)ca;
  if (lane < 12) half[32 + lane] = (uint16_t)cb;      // (the twelfth: four columns that are not there)
}

// A warp a row.
__global__ void __launch_bounds__(256) pull_kernel(const uint32_t *__restrict__ words, int64_t n_rows,
                                                   const int32_t *__restrict__ ids, int64_t n, float *__restrict__ out,
                                                   int32_t *status) {
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= n) return;
  const int v = ids[i];
  float2 x[2], y[2];
  x[0] = x[1] = y[0] = y[1] = make_float2(0.f, 0.f);
  const bool tail = lane < TAIL / 4;
  if (v >= 0 && v < n_rows) {
    const uint32_t *row = words + (int64_t)v * WORDS;
    const uint2 how = __ldg(reinterpret_cast<const uint2 *>(row));
    const uint16_t *half = reinterpret_cast<const uint16_t *>(row + 2);
    decode4(__ldg(half + lane), dup2(step_of(how.x)), dup2(offset_of(how.x)), x);
    if (tail) decode4(__ldg(half + 32 + lane), dup2(step_of(how.y)), dup2(offset_of(how.y)), y);
  } else if (lane == 0) {
    report(status, ORCA_E_BOUNDS, (int)(i < 0x7fffffff ? i : 0x7fffffff));
  }
  float4 *o = reinterpret_cast<float4 *>(out + i * D);
  o[lane] = make_float4(x[0].x, x[0].y, x[1].x, x[1].y);
  if (tail) o[32 + lane] = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
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
  int large;                         // pair groups of its time encoding with large arguments (time_terms)
};

constexpr int AT_THREADS = 64, AT_WARPS = AT_THREADS / 32;

// A warp takes a part of a row's slots, GS at a time.  Lanes 0..15 hold what the neighbours' rows have, lanes 16..31 the edges':
// columns 8 h .. 8 h + 7 (a word of codes) and, h < 11, columns 128 + 4 h .. + 3 (half a word); all lanes hold column pairs
// l, l + 32, l + 64 of the time encoding.
template <int GS, bool EDGE32, class S>
__global__ void __launch_bounds__(AT_THREADS) attend_kernel(const float *__restrict__ qt, Tables t, S slots, int rows,
                                                            float *__restrict__ ctx, uint8_t *__restrict__ valid,
                                                            float *__restrict__ partial, int32_t *status) {
  __shared__ Rec s_rec[AT_WARPS][32 + GS - 1];
  __shared__ __align__(16) float s_p[AT_WARPS][4 * GS + 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  dep_trigger();
  dep_wait();
  Part p;
  if (!part_of(slots, rows, (int64_t)blockIdx.x * AT_WARPS + warp, lane, p)) return;
  const int side = lane >> 4, h = lane & 15;
  const bool has_tail = h < TAIL / 4, third = lane < 22;
  const float *q = qt + (int64_t)p.row * QT_LD + side * D;
  float2 qc[2][6], qe[2][GA_P_ITERS];          // this lane's columns of the two heads' queries
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float *qh = q + g * QT_HEAD;
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
  float2 wt[GA_P_ITERS];
  float w_most[GA_P_ITERS], w_least[GA_P_ITERS];
#pragma unroll
  for (int i = 0; i < GA_P_ITERS; ++i) {
    const bool has = i < 2 || third;
    wt[i] = has ? __ldg(reinterpret_cast<const float2 *>(t.time_w) + lane + 32 * i) : make_float2(0.f, 0.f);
    w_most[i] = warp_max(fmaxf(fabsf(wt[i].x), fabsf(wt[i].y)));
    w_least[i] = warp_min(has ? fminf(fabsf(wt[i].x), fabsf(wt[i].y)) : INFINITY);
  }
  // cos_fixed wants arguments of 2^-8 and more: weights of the usual falling kind give them to every group in front of one
  // that holds an argument of 2^24
  bool falling = true;
#pragma unroll
  for (int i = 0; i < GA_P_ITERS; ++i)
#pragma unroll
    for (int j = i; j < GA_P_ITERS; ++j) falling &= w_least[i] * 1073741824.f >= w_most[j];

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
  Rec *const rec = s_rec[warp];
  float *const pbuf = s_p[warp];
  constexpr int V = 2 * GS, LPV = 32 / V;
  for (int at0 = 0; at0 < p.n; at0 += 32) {
    Slot s = {0, 0, 0.f};
    if (at0 + lane < p.n) {
      s = slot_of(slots, p, p.beg + at0 + lane);
      if (s.nbr < 0 || s.nbr >= t.n_rows || s.eid < 0 || s.eid >= t.n_edges) {
        report(status, ORCA_E_BOUNDS, p.row);
        s.nbr = 0;
      }
    }
    const unsigned used = __ballot_sync(FULL, s.nbr != 0);
    const int n_used = __popc(used);
    if (n_used == 0) continue;
    any_valid = true;
    {
      const float adt = fabsf(s.dt);
      int large = adt * w_most[2] >= COS_SMALL ? 3 : adt * w_most[1] >= COS_SMALL ? 2 : adt * w_most[0] >= COS_SMALL ? 1 : 0;
      const float far = adt * fmaxf(w_most[0], fmaxf(w_most[1], w_most[2]));
      if (!(far < 1073741824.f) || (large != 0 && !falling)) large = -1;
      const Rec r = {s.nbr, s.eid, s.dt, large};
      const int place = __popc(used & ((1u << lane) - 1u));
      __syncwarp();
      if (s.nbr != 0) rec[place] = r;
      if (s.nbr != 0 && place == 0)       // behind the last, up to a whole step, the first again with weight zero
        for (int u = 0; u < GS - 1; ++u) rec[n_used + u] = r;
      __syncwarp();
    }
    for (int at = 0; at < n_used; at += GS) {
      float2 x[GS][6], te[GS][GA_P_ITERS];
#pragma unroll
      for (int u = 0; u < GS; ++u) {
        const Rec r = rec[at + u];
        if (EDGE32 && side) {
          const float4 *row = reinterpret_cast<const float4 *>(t.edges32 + (int64_t)r.eid * D);
          const float4 a = __ldg(row + 2 * h), b = __ldg(row + 2 * h + 1);
          const float4 c = has_tail ? __ldg(row + GROUP / 4 + h) : make_float4(0.f, 0.f, 0.f, 0.f);
          x[u][0] = lo2(a), x[u][1] = hi2(a), x[u][2] = lo2(b), x[u][3] = hi2(b), x[u][4] = lo2(c), x[u][5] = hi2(c);
        } else {
          const uint32_t *row = side ? t.edges + (int64_t)r.eid * WORDS : t.rows + (int64_t)r.nbr * WORDS;
          const uint2 how = __ldg(reinterpret_cast<const uint2 *>(row));
          const uint32_t w = __ldg(row + 2 + h);
          const uint32_t v = has_tail ? __ldg(reinterpret_cast<const uint16_t *>(row + 18) + h) : 0;
          float2 c8[4], c4[2];
          decode8(w, dup2(step_of(how.x)), dup2(offset_of(how.x)), c8);
          decode4(v, dup2(step_of(how.y)), dup2(offset_of(how.y)), c4);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[u][j] = c8[j];
          x[u][4] = has_tail ? c4[0] : make_float2(0.f, 0.f);
          x[u][5] = has_tail ? c4[1] : make_float2(0.f, 0.f);
        }
        time_terms(r.dt, r.large, wt, te[u]);
      }
      float v[V];
#pragma unroll
      for (int u = 0; u < GS; ++u)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          float2 a = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 6; ++j) a = fma2(x[u][j], qc[g][j], a);
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) a = fma2(te[u][i], qe[g][i], a);
          v[2 * u + g] = a.x + a.y;
        }
      // lane l holds value l / LPV = 2 * slot + head
      float lg = warp_sum_many<V>(v, lane);
      if (at + lane / (2 * LPV) >= n_used) lg = -INFINITY;
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
          for (int j = 0; j < 6; ++j) ac[g][j] = mul2(k, ac[g][j]);
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) ae[g][i] = mul2(k, ae[g][i]);
        }
      }
#pragma unroll
      for (int u = 0; u < GS; ++u) {
        if (at + u >= n_used) break;         // (a slot that is there twice adds nothing, not even what is not a number)
        const float4 w4 = *reinterpret_cast<const float4 *>(pbuf + 4 * u);
        sum0 += w4.x, sum1 += w4.z;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const float2 k = g ? hi2(w4) : lo2(w4);
#pragma unroll
          for (int j = 0; j < 6; ++j) ac[g][j] = fma2(k, x[u][j], ac[g][j]);
#pragma unroll
          for (int i = 0; i < GA_P_ITERS; ++i) ae[g][i] = fma2(k, te[u][i], ae[g][i]);
        }
      }
      __syncwarp();
    }
  }
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

// Joins the parts of rows that have several.  A block takes 32 columns of four of a row at a time; its warps take parts in turn,
// and their sums are added in the order of the warps.
constexpr int JOIN_WARPS = 8, JOIN_COLS = (QT / 4 + 31) / 32;      // 9 blocks of columns
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
    for (int j = warp; j < of; j += JOIN_WARPS) {
      const float *p = p0 + (int64_t)j * PARTIAL;
      const float4 st = *reinterpret_cast<const float4 *>(p + QT);
      const float w0 = expf(st.x - m0), w1 = expf(st.y - m1);
      total0 += w0 * st.z, total1 += w1 * st.w;
      if (col < QT / 4) {
        const float4 v = reinterpret_cast<const float4 *>(p)[col];
        const float w = second ? w1 : w0;
        a.x = fmaf(w, v.x, a.x), a.y = fmaf(w, v.y, a.y), a.z = fmaf(w, v.z, a.z), a.w = fmaf(w, v.w, a.w);
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
  __shared__ long long s_total[32];
  __shared__ int s_scan[3][32];
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long total = 0;
  for (int r = threadIdx.x; r < rows; r += 1024) total += count[r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
  if (lane == 0) s_total[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < 32; ++w) total += s_total[w];
  long long want = (total + target - 1) / target;
  want = (want + 31) / 32 * 32;
  const int len = (int)(want < least ? least : want > 0x7fffffe0ll ? 0x7fffffe0ll : want);
  int carry[3] = {0, 0, 0};                       // parts, parts of rows of several, such rows
  for (int r0 = 0; r0 < rows; r0 += 1024) {
    const int r = r0 + threadIdx.x;
    const int parts = r < rows ? max(1, (int)(((long long)count[r] + len - 1) / len)) : 0;
    const int mine[3] = {parts, parts > 1 ? parts : 0, parts > 1 ? 1 : 0};
    int incl[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      incl[k] = mine[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(FULL, incl[k], o);
        if (lane >= o) incl[k] += up;
      }
      if (lane == 31) s_scan[k][warp] = incl[k];
    }
    __syncthreads();
    int before[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      before[k] = carry[k] + incl[k] - mine[k];
      for (int w = 0; w < 32; ++w) {
        if (w < warp) before[k] += s_scan[k][w];
        carry[k] += s_scan[k][w];
      }
    }
    if (r < rows) {
      first[r] = before[0];
      base[r] = before[1];
      if (mine[2]) several[before[2]] = r;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) first[rows] = carry[0], head[0] = len, head[1] = carry[2];
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
  constexpr int GS = 4;
  auto kernel = t.edges32 != nullptr ? attend_kernel<GS, true, S> : attend_kernel<GS, false, S>;
  ORCA_CUDA(launch_dep(kernel, (unsigned)((jobs + AT_WARPS - 1) / AT_WARPS), AT_THREADS, 0, s, d_qt, t, slots, rows, d_ctx, d_valid,
                       partial, d_status));
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
  const unsigned grid = (unsigned)((n + 7) / 8);
  if (type == ORCA_F32)
    ORCA_CUDA(launch_dep(push_kernel<float>, grid, 256, 0, s, d_words, (const float *)d_x, x_stride, d_ids, (int)n, n_rows, d_record));
  else if (type == ORCA_BF16)
    ORCA_CUDA(launch_dep(push_kernel<__nv_bfloat16>, grid, 256, 0, s, d_words, (const __nv_bfloat16 *)d_x, x_stride, d_ids, (int)n, n_rows, d_record));
  else
    ORCA_CUDA(launch_dep(push_kernel<__half>, grid, 256, 0, s, d_words, (const __half *)d_x, x_stride, d_ids, (int)n, n_rows, d_record));
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

int orca_packed_pull(const uint32_t *d_words, int64_t n_rows, const int32_t *d_ids, int64_t n, float *d_out, int32_t *d_status,
                     void *stream) {
  ORCA_CHECK_ARG(d_words && n_rows > 0 && n >= 0 && (n == 0 || (d_ids && d_out)));
  ORCA_CHECK_ARG((uintptr_t)d_words % 16 == 0 && (uintptr_t)d_out % 16 == 0 && (n + 7) / 8 <= 0x7fffffffll);
  if (n == 0) return ORCA_OK;
  ORCA_CUDA(launch_dep(pull_kernel, (unsigned)((n + 7) / 8), 256, 0, (cudaStream_t)stream, d_words, n_rows, d_ids, n, d_out, d_status));
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
  const int64_t items = (int64_t)n_query * JOIN_COLS;
  ORCA_CUDA(launch_dep(join_kernel, (unsigned)std::min<int64_t>(items, (int64_t)sms() * 8), 32 * JOIN_WARPS, 0, s,
                       (const float *)d_workspace, (const int32_t *)nullptr, (const int32_t *)nullptr, (int)n_query, parts,
                       (const int32_t *)nullptr, (const int32_t *)nullptr, d_ctx, d_valid));
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
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
  ORCA_CUDA(launch_dep(join_kernel, (unsigned)(sms() * 4), 32 * JOIN_WARPS, 0, s, (const float *)partial, (const int32_t *)several,
                       (const int32_t *)(head + 1), 0, 0, (const int32_t *)first, (const int32_t *)base, d_ctx, d_valid));
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

}  // extern "C"
