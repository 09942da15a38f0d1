// Rows of a trained table by id, times a scale, and the gradient of the table by sorted ids.
//
// Both are bound by HBM: a lookup reads and writes a row an id, the gradient reads a row an id and writes every row of the table
// once.  The gradient sorts (id, position) pairs, stably, so that a row's contributions lie side by side in the order of their positions;
// chunks of the sorted list are then summed by themselves.  A stretch of equal ids that lies in one chunk goes straight to its row; one that
// crosses a border leaves a sum on either side, which another kernel adds in the order of the chunks.  No atomics on values: the same bits
// every time, and a hub that fills half of the list is spread over as many chunks as it needs.  Rows that no id names are written zero by
// blocks that go along with the sort, whose launches leave the memory idle; no row is written twice.
// Few ids (SMALL) are not sorted: the block of an id that no earlier one equals finds the later ones by looking at all.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "context.cuh"
#include "vec.cuh"

namespace orca {
namespace rows {

struct Ids {
  const void *p;
  int wide;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return wide ? reinterpret_cast<const int64_t *>(p)[i] : reinterpret_cast<const int32_t *>(p)[i];
  }
};

__device__ __forceinline__ int detail(int64_t i) { return (int)(i < 0x7fffffff ? i : 0x7fffffff); }

// 400 k rows of 688 bytes: 91 us, 6.0 TB/s.  Four loads of a thread are under way before the first store.
// A thread takes PIECES pieces of VB bytes, 256 apart, of the n * nv that the rows have; nv by multiplication (Divide).
struct Divide {                       // by an invariant divisor: Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994
  uint32_t d, mul, shift;
  static Divide by(uint32_t d) {      // q = (x * mul >> 32) + x >> shift for x below 2^31
    Divide v = {d, 0, 0};
    while ((1ull << v.shift) < d) ++v.shift;
    v.mul = (uint32_t)(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
    return v;
  }
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return (__umulhi(x, mul) + x) >> shift; }
};
constexpr int PIECES = 4;
template <typename T, int VB>
__global__ void __launch_bounds__(256) lookup_kernel(const char *__restrict__ table, int64_t n_rows, int64_t stride, Divide nv,
                                                     Ids ids, int64_t n, float scale, char *__restrict__ out, int32_t *status) {
  dep_trigger();
  dep_wait();
  using X = Vec<T, VB>;
  // rows of this block from `row0`, pieces counted from its first (a block's share is below 2^31 pieces)
  const int64_t p0 = (int64_t)blockIdx.x * (256 * PIECES), row0 = p0 / nv.d;
  const uint32_t skip = (uint32_t)(p0 - row0 * nv.d);
  float x[PIECES][X::N] = {};
  bool in[PIECES];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    const uint32_t p = skip + threadIdx.x + 256 * k, r = nv.of(p), c = p - r * nv.d;
    const int64_t i = row0 + r;
    in[k] = i < n;
    if (in[k]) {
      const int64_t v = ids.at(i);
      if (v >= 0 && v < n_rows) X::load(table + v * stride + (int64_t)c * VB, x[k]);
      else if (c == 0) report(status, ORCA_E_BOUNDS, detail(i));
    }
  }
#pragma unroll
  for (int k = 0; k < PIECES; ++k)
    if (in[k]) X::store(out + (p0 + threadIdx.x + 256 * k) * VB, x[k], scale);
}

// ---------------------------------------------------------------------------------------------- few ids
// Latency: n^2 comparisons of ids against the sort's launches (gradient of 9 k rows, us: 600 ids 6.1, 2048 21, 3000 36, 4096 58; sorted 32 for
// any such number).  Of ids that hardly repeat, or a tenth of which are one (7.1, 20): a hub is one block's to sum, and ids that are all
// the same take 20 (600), 31 (1024) or 58 (2048), sorted 29.
constexpr int SMALL = 2048;
// Block i: the row of id i, if no earlier position has the same id.  64 threads a column of pieces, SMALL_Y of them take the
// positions of the id in turn; their sums are added in order.
constexpr int SMALL_Y = 4;
template <typename T, int VB>
__global__ void __launch_bounds__(64 * SMALL_Y) small_kernel(const char *__restrict__ g, int64_t stride, int nv, Ids ids, int n, int64_t n_rows,
                                                             int64_t padding, float scale, char *__restrict__ grad, int32_t *status) {
  using X = Vec<T, VB>;
  __shared__ float s_sum[SMALL_Y - 1][64][X::N];
  __shared__ uint32_t s_mask[SMALL / 32];
  __shared__ int s_before;
  __shared__ int16_t s_list[SMALL];
  dep_trigger();
  dep_wait();
  const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const int64_t v = ids.at(i);
  if (v < 0 || v >= n_rows) {
    if (tid == 0) report(status, ORCA_E_BOUNDS, i);
    return;
  }
  if (v == padding) return;
  if (tid == 0) s_before = 0;
  __syncthreads();
  const int words = (n + 31) / 32;
  for (int w = tid >> 5; w < words; w += 2 * SMALL_Y) {
    const int j = 32 * w + lane;
    const uint32_t same = __ballot_sync(0xffffffffu, j < n && ids.at(j < n ? j : 0) == v);
    if (lane == 0) {
      s_mask[w] = same;
      if (32 * w < i && (same & (i - 32 * w >= 32 ? 0xffffffffu : (1u << (i - 32 * w)) - 1u)) != 0) s_before = 1;
    }
  }
  __syncthreads();
  if (s_before) return;
  // the positions in order
  int count = 0;
  for (int w = 0; w < words; ++w) {
    const uint32_t same = s_mask[w];
    if (tid < 32 && (same >> lane & 1u)) s_list[count + __popc(same & ((1u << lane) - 1u))] = (int16_t)(32 * w + lane);
    count += __popc(same);
  }
  __syncthreads();
  const int t = tid % 64, y = tid / 64;
  for (int c0 = 0; c0 < nv; c0 += 64) {
    const int c = c0 + t;
    float a[X::N] = {};
    if (c < nv)
#pragma unroll 4
      for (int k = y; k < count; k += SMALL_Y) {
        float x[X::N];
        X::load(g + (int64_t)s_list[k] * stride + (int64_t)c * VB, x);
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] += x[e];
      }
    if (y > 0)
#pragma unroll
      for (int e = 0; e < X::N; ++e) s_sum[y - 1][t][e] = a[e];
    __syncthreads();
    if (y == 0 && c < nv) {
      for (int k = 0; k < SMALL_Y - 1; ++k)
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] += s_sum[k][t][e];
      X::store(grad + (v * nv + c) * VB, a, scale);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- sorting
// A stable radix sort by digits of up to eleven bits, two passes up to four million rows.  A pass: digits counted by tile (by the pass before,
// as it puts a pair into its tile), the counts of every digit summed over the tiles before, pairs put at their places.  A warp walks its run of the tile 32 pairs at a time; lanes of
// equal digit find one another with match.any.  Key n_rows: an id that has no gradient.
constexpr int S_THREADS = 256, S_WARPS = S_THREADS / 32, S_RUN = 256, S_TILE = S_WARPS * S_RUN;
constexpr int MOST_BITS = 11;

struct Source {          // of a pass: the ids themselves (first), or pairs
  Ids ids;
  int64_t n_rows, padding;
  uint8_t *named;        // [n_rows], set for rows that have a gradient
  int32_t *status;
  const uint2 *pairs;    // nullptr: the first pass
  // the pairs first, first + 32, ... of a run; MARK: marks rows that are named and reports ids outside the table
  template <bool MARK, int N> __device__ __forceinline__ void load(int64_t first, int64_t n, uint2 (&x)[N]) const {
    if (!MARK && pairs != nullptr) {
#pragma unroll
      for (int u = 0; u < N; ++u) x[u] = first + 32 * u < n ? pairs[first + 32 * u] : make_uint2(0u, 0u);
      return;
    }
    int64_t v[N];
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = first + 32 * u < n ? ids.at(first + 32 * u) : -1;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int64_t i = first + 32 * u;
      const bool inside = v[u] >= 0 && v[u] < n_rows, counts = inside && v[u] != padding;
      if (MARK && counts) named[v[u]] = 1;
      if (MARK && !inside && i < n) report(status, ORCA_E_BOUNDS, detail(i));
      x[u] = make_uint2((uint32_t)(counts ? v[u] : n_rows), (uint32_t)i);
    }
  }
};

struct Next {             // where a pass counts for the one behind it, whose tiles its pairs go to
  int32_t *counts;         // nullptr: there is none
  int shift, tiles;
};
template <bool SCATTER, bool MARK = false>
__device__ __forceinline__ void walk(const Source &s, uint2 *out, int64_t first, int64_t n, int shift, int mask, int32_t *count, const Next &next = {}) {
  const int lane = threadIdx.x & 31;
  const uint32_t lower = (1u << lane) - 1u;
  uint2 x[S_RUN / 32];
  s.template load<MARK>(first + lane, n, x);
#pragma unroll
  for (int u = 0; u < S_RUN / 32; ++u) {
    const bool there = first + 32 * u + lane < n;
    const int d = there ? (int)(x[u].x >> shift) & mask : mask + 1 + lane;       // (lanes past the end group with nobody)
    const uint32_t group = __match_any_sync(0xffffffffu, d);
    if (SCATTER && there) {
      const int at = count[d] + __popc(group & lower);
      out[at] = x[u];
      if (next.counts != nullptr) atomicAdd(next.counts + ((int64_t)(x[u].x >> next.shift & mask) * next.tiles + at / S_TILE), 1);
    }
    __syncwarp();
    if (there && (group & lower) == 0) count[d] += __popc(group);
    __syncwarp();
  }
}

// Zeros for rows that have no gradient, ZERO_ROWS of the table a block: a share of the blocks of the passes' last launches, which leave most of the memory's bandwidth unused (400 k ids of 1.14 M rows of 688 bytes: the gradient 275 us, 189
// without the 0.65 GB of zeros, which take 99 by themselves at the copy's rate).
constexpr int ZERO_ROWS = 64;
struct Zero {
  char *grad;
  int64_t row_bytes, n_rows;
  const uint8_t *named;
  int64_t first;           // tile of rows of the launch's first such block
  int piece;               // bytes that rows can be written by
};
template <typename V> __device__ __forceinline__ void zero_tile(const Zero &z, int64_t tile) {
  const int64_t r0 = tile * ZERO_ROWS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int nv = (int)(z.row_bytes / (int64_t)sizeof(V));
  static_assert(ZERO_ROWS / (S_THREADS / 32) <= 32, "a warp's rows, a lane each");
  const int64_t mine = r0 + warp + (int64_t)lane * warps;        // all flags at once: nothing waits between the rows
  uint32_t todo = __ballot_sync(0xffffffffu, lane < ZERO_ROWS / warps && mine < z.n_rows && z.named[mine < z.n_rows ? mine : 0] == 0);
  while (todo != 0) {
    const int k = __ffs(todo) - 1;
    todo &= todo - 1;
    V *row = reinterpret_cast<V *>(z.grad + (r0 + warp + k * warps) * z.row_bytes);
    for (int c = lane; c < nv; c += 32) row[c] = V{};
  }
}
__device__ __forceinline__ void zero_rows(const Zero &z, int64_t tile) {
  tile += z.first;
  if (z.piece == 16) zero_tile<uint4>(z, tile);
  else if (z.piece == 8) zero_tile<uint2>(z, tile);
  else if (z.piece == 4) zero_tile<uint32_t>(z, tile);
  else zero_tile<uint16_t>(z, tile);
}

// The first pass: counts[digit * tiles + tile].  Marks the rows that are named and reports ids outside the table.
__global__ void __launch_bounds__(S_THREADS) count_kernel(Source s, int64_t n, int bits, int tiles, int32_t *__restrict__ counts) {
  extern __shared__ int32_t s_count[];         // [S_WARPS][bins]
  dep_trigger();
  dep_wait();
  const int bins = 1 << bits, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < S_WARPS * bins; i += S_THREADS) s_count[i] = 0;
  __syncthreads();
  const int64_t beg = (int64_t)blockIdx.x * S_TILE;
  walk<false, true>(s, nullptr, beg + warp * S_RUN, n, 0, bins - 1, s_count + warp * bins);
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += S_THREADS) {
    int total = 0;
    for (int w = 0; w < S_WARPS; ++w) total += s_count[w * bins + d];
    counts[(int64_t)d * tiles + blockIdx.x] = total;
  }
}

// a warp a digit: its counts summed over the tiles before, in place; totals[digit]
__global__ void __launch_bounds__(256) scan_kernel(int32_t *__restrict__ counts, int tiles, int bins, int32_t *__restrict__ totals) {
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, d = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (d >= bins) return;
  int32_t *c = counts + (int64_t)d * tiles;
  int carry = 0;
  for (int i0 = 0; i0 < tiles; i0 += 32) {
    const int v = i0 + lane < tiles ? c[i0 + lane] : 0;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (i0 + lane < tiles) c[i0 + lane] = carry + incl - v;
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) totals[d] = carry;
}

__global__ void __launch_bounds__(S_THREADS) scatter_kernel(Source s, int64_t n, int shift, int bits, const int32_t *__restrict__ before,
                                                            const int32_t *__restrict__ totals, uint2 *__restrict__ out, int tiles, Next next,
                                                            Zero zero) {
  extern __shared__ int32_t s_count[];
  __shared__ int32_t s_warp[S_WARPS];
  dep_trigger();
  dep_wait();
  if ((int)blockIdx.x >= tiles) return zero_rows(zero, blockIdx.x - tiles);
  const int bins = 1 << bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < S_WARPS * bins; i += S_THREADS) s_count[i] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * S_TILE + warp * S_RUN;
  walk<false>(s, nullptr, first, n, shift, bins - 1, s_count + warp * bins);
  __syncthreads();
  // where a digit starts: behind all lower digits, the tiles and the warps before
  int32_t carry = 0;
  for (int d0 = 0; d0 < bins; d0 += S_THREADS) {
    const int d = d0 + threadIdx.x;
    const int32_t v = d < bins ? totals[d] : 0;
    int32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int32_t at = carry + incl - v;
    for (int w = 0; w < S_WARPS; ++w) {
      if (w < warp) at += s_warp[w];
      carry += s_warp[w];
    }
    __syncthreads();
    if (d < bins) {
      at += before[(int64_t)d * tiles + blockIdx.x];
      for (int w = 0; w < S_WARPS; ++w) {
        const int32_t c = s_count[w * bins + d];
        s_count[w * bins + d] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  walk<true>(s, out, first, n, shift, bins - 1, s_count + warp * bins, next);
}

// ---------------------------------------------------------------------------------------------- sums
// Bound by HBM, whole rows at random places: 400 k rows of 688 bytes 106 us for 0.32 GB read and 0.19 GB written, 4.8 TB/s; 60 k of 344 bytes 12.  A
// warp waits for its rows 14 of 20 cycles, at 39 % of the warps that an SM holds (68 registers, blocks of 64 threads).  Eight rows of a
// thread's columns are under way at a time, loaded without conditions (with them 24).  The chunk's size matters little (16 / 32 / 64 rows:
// gradient of 60 k ids 52 / 53 / 54 us; 32 / 64 / 128: of 400 k 274 / 275 / 276).
constexpr int CHUNK = 32;
// A block sums a chunk of the sorted pairs.  The stretch that began in an earlier chunk goes to half 0 of the chunk's partial sums, the
// one that goes on into the next chunk (and began here) to half 1.
template <typename T, int VB>
__global__ void __launch_bounds__(256) sum_kernel(const char *__restrict__ g, int64_t stride, int nv, const uint2 *__restrict__ sorted,
                                                  int64_t n, int64_t n_rows, float scale, char *__restrict__ grad,
                                                  float *__restrict__ partial) {
  using X = Vec<T, VB>;
  constexpr int AHEAD = 8;
  __shared__ uint2 s_rec[CHUNK + 2];
  dep_trigger();
  dep_wait();
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
        X::load(g + (int64_t)s_rec[min(r0 + u, m - 1) + 1].y * stride + (int64_t)c * VB, x[u]);
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

// Stretches over several chunks.  A warp looks at a chunk: whether a stretch begins in it that goes on, and to which chunk it reaches.  It
// adds the partial sums of a short one itself; long ones are left to the whole block, whose warps take their chunks in turn and whose sums
// are added in order.
constexpr int JOIN_WARPS = 8, JOIN_LONG = 16;
template <typename T, int VB>
__global__ void __launch_bounds__(32 * JOIN_WARPS) join_kernel(int nv, const uint2 *__restrict__ sorted, int64_t n, int64_t n_rows, float scale,
                                                               char *__restrict__ grad, const float *__restrict__ partial) {
  using X = Vec<T, VB>;
  __shared__ float s_sum[JOIN_WARPS][32][X::N];
  __shared__ int s_parts[JOIN_WARPS];
  __shared__ uint32_t s_key[JOIN_WARPS];
  dep_trigger();
  dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chunk = (int64_t)blockIdx.x * JOIN_WARPS + warp, beg = chunk * CHUNK, end = beg + CHUNK;
  int parts = 0;
  uint32_t key = 0;
  if (end < n) {
    key = sorted[end - 1].x;
    const uint32_t behind = sorted[end].x, head = sorted[beg].x, before = beg > 0 ? sorted[beg - 1].x : 0xffffffffu;
    if (key < n_rows && behind == key && !(head == key && before == key)) {
      parts = 2;                     // and as many more as begin with the same key
      for (;;) {
        const int64_t at = (chunk + parts + lane) * CHUNK;
        const uint32_t same = __ballot_sync(0xffffffffu, at < n && sorted[at < n ? at : 0].x == key);
        const int more = __ffs(~same) - 1;      // (-1: all 32)
        parts += more < 0 ? 32 : more;
        if (more >= 0) break;
      }
    }
  }
  auto part_of = [&](int64_t first, int k) { return partial + (((first + k) * 2 + (k == 0 ? 1 : 0)) * nv) * X::N; };
  if (parts > 0 && parts <= JOIN_LONG) {
    for (int c = lane; c < nv; c += 32) {
      float a[X::N] = {};
#pragma unroll 4
      for (int k = 0; k < parts; ++k) {
        const float *p = part_of(chunk, k) + c * X::N;
#pragma unroll
        for (int e = 0; e < X::N; ++e) a[e] += p[e];
      }
      X::store(grad + ((int64_t)key * nv + c) * VB, a, scale);
    }
  }
  if (lane == 0) s_parts[warp] = parts > JOIN_LONG ? parts : 0, s_key[warp] = key;
  __syncthreads();
  for (int w = 0; w < JOIN_WARPS; ++w) {
    const int all = s_parts[w];
    if (all == 0) continue;
    const int64_t first = (int64_t)blockIdx.x * JOIN_WARPS + w;
    for (int c0 = 0; c0 < nv; c0 += 32) {
      const int c = c0 + lane;
      float a[X::N] = {};
      if (c < nv)
#pragma unroll 8
        for (int k = warp; k < all; k += JOIN_WARPS) {
          const float *p = part_of(first, k) + c * X::N;
#pragma unroll
          for (int e = 0; e < X::N; ++e) a[e] += p[e];
        }
#pragma unroll
      for (int e = 0; e < X::N; ++e) s_sum[warp][lane][e] = a[e];
      __syncthreads();
      if (warp == 0 && c < nv) {
        for (int k = 1; k < JOIN_WARPS; ++k)
#pragma unroll
          for (int e = 0; e < X::N; ++e) a[e] += s_sum[k][lane][e];
        X::store(grad + ((int64_t)s_key[w] * nv + c) * VB, a, scale);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
constexpr int MOST_WIDTH = 1 << 24;
static int64_t up256(int64_t b) { return (b + 255) & ~255ll; }

struct Layout {
  int64_t a, b, totals, counts, pass_counts, named, partial, total;
  int tiles, passes, bits;
};
static Layout layout(int64_t n, int64_t n_rows, int width) {
  Layout L = {};
  if (n <= SMALL) return L;
  int key_bits = 1;
  while ((n_rows >> key_bits) != 0) ++key_bits;
  L.passes = (key_bits + MOST_BITS - 1) / MOST_BITS;
  L.bits = (key_bits + L.passes - 1) / L.passes;
  L.tiles = (int)((n + S_TILE - 1) / S_TILE);
  L.a = 0;
  L.b = up256(n * 8);
  L.pass_counts = up256(((int64_t)L.tiles << L.bits) * 4);
  L.totals = L.b + up256(n * 8);
  L.counts = L.totals + up256((int64_t)4 << L.bits);        // of every pass; all but the first's are zero at first, as are the flags behind them
  L.named = L.counts + L.passes * L.pass_counts;
  L.partial = L.named + up256(n_rows);
  L.total = L.partial + up256((n + CHUNK - 1) / CHUNK * 2 * width * 4);
  return L;
}

}  // namespace rows
}  // namespace orca

using namespace orca;
using namespace orca::rows;

extern "C" {

int orca_rows_lookup(const void *d_table, int64_t n_rows, int64_t table_stride, int32_t width, int32_t type, const void *d_ids,
                     int32_t ids64, int64_t n, float scale, void *d_out, int32_t *d_status, void *stream) {
  ORCA_CHECK_ARG(n >= 0 && n_rows >= 0 && n_rows < 0x7fffffffll && width > 0 && width <= MOST_WIDTH && table_stride >= width);
  ORCA_CHECK_ARG(n == 0 || (d_ids && d_out && (d_table || n_rows == 0)));
  if (type != ORCA_F32 && type != ORCA_BF16 && type != ORCA_F16) return set_error(ORCA_E_UNSUPPORTED, "%s: type %d", __func__, type);
  const int size = size_of(type);
  ORCA_CHECK_ARG((uintptr_t)d_table % size == 0 && (uintptr_t)d_out % size == 0 && (uintptr_t)d_ids % (ids64 ? 8 : 4) == 0);
  if (n == 0) return ORCA_OK;
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_table, (uint64_t)(uintptr_t)d_out, (uint64_t)(table_stride * size)});
  const int nv = width * size / vb;
  const int64_t per = 256 * PIECES;
  ORCA_CHECK_ARG(n <= 0x7fffffffll * per / nv - 1);
  const int64_t blocks = (n * nv + per - 1) / per;
  return by_type(type, vb, [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    ORCA_CUDA(launch_dep(lookup_kernel<T, decltype(v)::value>, (unsigned)blocks, 256, 0, (cudaStream_t)stream, (const char *)d_table,
                         n_rows, table_stride * size, Divide::by(nv), Ids{d_ids, ids64}, n, scale, (char *)d_out, d_status));
    ORCA_COUNT_LAUNCH();
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

int64_t orca_rows_grad_workspace_bytes(int64_t n, int64_t n_rows, int32_t width) {
  if (n < 0 || n >= 0x7fffffffll || n_rows < 0 || n_rows >= 0x7fffffffll || width <= 0 || width > MOST_WIDTH) return -1;
  return layout(n, n_rows, width).total;
}

int orca_rows_grad(const void *d_grad_out, int64_t grad_stride, int32_t width, int32_t type, const void *d_ids, int32_t ids64,
                   int64_t n, int64_t n_rows, float scale, int64_t padding, void *d_grad, int32_t *d_status, void *d_workspace,
                   int64_t workspace_bytes, void *stream) {
  ORCA_CHECK_ARG(n >= 0 && n < 0x7fffffffll && n_rows >= 0 && n_rows < 0x7fffffffll && width > 0 && width <= MOST_WIDTH && (grad_stride >= width || grad_stride == 0));
  ORCA_CHECK_ARG((n == 0 || (d_grad_out && d_ids)) && (n_rows == 0 || d_grad));
  if (type != ORCA_F32 && type != ORCA_BF16 && type != ORCA_F16) return set_error(ORCA_E_UNSUPPORTED, "%s: type %d", __func__, type);
  const int size = size_of(type);
  ORCA_CHECK_ARG((uintptr_t)d_grad_out % size == 0 && (uintptr_t)d_grad % size == 0 && (uintptr_t)d_ids % (ids64 ? 8 : 4) == 0);
  cudaStream_t s = (cudaStream_t)stream;
  const Layout L = layout(n, n_rows, width);
  if (L.total > 0 && n_rows > 0) {
    ORCA_CHECK_ARG(d_workspace && (uintptr_t)d_workspace % 256 == 0);
    if (workspace_bytes < L.total) return set_error(ORCA_E_BADARG, "%s: workspace of %lld bytes is too small", __func__, (long long)workspace_bytes);
  }
  if (n_rows == 0) return ORCA_OK;
  const int vb = piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_grad_out, (uint64_t)(uintptr_t)d_grad, (uint64_t)(grad_stride * size)});
  const int nv = width * size / vb;
  const Ids ids{d_ids, ids64};
  if (L.total == 0) {
    ORCA_CUDA(cudaMemsetAsync(d_grad, 0, (size_t)n_rows * width * size, s));
    if (n == 0) return ORCA_OK;
    return by_type(type, vb, [&](auto *t, auto v) {
      using T = std::remove_pointer_t<decltype(t)>;
      ORCA_CUDA(launch_dep(small_kernel<T, decltype(v)::value>, (unsigned)n, 64 * SMALL_Y, 0, s, (const char *)d_grad_out, grad_stride * size,
                           nv, ids, (int)n, n_rows, padding, scale, (char *)d_grad, d_status));
      ORCA_COUNT_LAUNCH();
      ORCA_LAUNCH_CHECK();
      return (int)ORCA_OK;
    });
  }
  char *w = (char *)d_workspace;
  int32_t *totals = (int32_t *)(w + L.totals);
  uint2 *half[2] = {(uint2 *)(w + L.a), (uint2 *)(w + L.b)};
  uint8_t *named = (uint8_t *)(w + L.named);
  ORCA_CUDA(cudaMemsetAsync(w + L.counts + L.pass_counts, 0, (size_t)(L.named - L.counts - L.pass_counts + n_rows), s));
  const int smem = S_WARPS * 4 << L.bits, bins = 1 << L.bits;
  static_assert((S_WARPS * 4 << MOST_BITS) <= 99 * 1024, "two blocks of a pass an SM");
  static std::atomic<uint64_t> count_ready, scatter_ready;
  int rc = allow_shared(count_kernel, S_WARPS * 4 << MOST_BITS, count_ready);
  if (rc == ORCA_OK) rc = allow_shared(scatter_kernel, S_WARPS * 4 << MOST_BITS, scatter_ready);
  if (rc) return rc;
  // blocks of zeros go along with the passes' last launches, which know the rows that are named
  const int64_t zero_tiles = (n_rows + ZERO_ROWS - 1) / ZERO_ROWS, share = (zero_tiles + L.passes - 1) / L.passes;
  Zero zero = {(char *)d_grad, (int64_t)width * size, n_rows, named, 0, piece((int64_t)width * size, {(uint64_t)(uintptr_t)d_grad})};
  auto counts_of = [&](int pass) { return (int32_t *)(w + L.counts + pass * L.pass_counts); };
  for (int pass = 0; pass < L.passes; ++pass) {
    const Source src{ids, n_rows, padding, named, d_status, pass == 0 ? nullptr : half[(pass - 1) & 1]};
    int32_t *counts = counts_of(pass);
    if (pass == 0) {
      ORCA_CUDA(launch_dep(count_kernel, (unsigned)L.tiles, S_THREADS, smem, s, src, n, L.bits, L.tiles, counts));
      ORCA_COUNT_LAUNCH();
    }
    ORCA_CUDA(launch_dep(scan_kernel, (bins + 7) / 8, 256, 0, s, counts, L.tiles, bins, totals));
    ORCA_COUNT_LAUNCH();
    const Next next = {pass + 1 < L.passes ? counts_of(pass + 1) : nullptr, (pass + 1) * L.bits, L.tiles};
    zero.first = pass * share;
    const int64_t more = std::max<int64_t>(0, std::min(share, zero_tiles - zero.first));
    ORCA_CUDA(launch_dep(scatter_kernel, (unsigned)(L.tiles + more), S_THREADS, smem, s, src, n, pass * L.bits, L.bits, (const int32_t *)counts,
                         (const int32_t *)totals, half[pass & 1], L.tiles, next, zero));
    ORCA_COUNT_LAUNCH();
  }
  const uint2 *sorted = half[(L.passes - 1) & 1];
  float *partial = (float *)(w + L.partial);
  const int threads = std::min(256, (nv + 31) / 32 * 32);
  return by_type(type, vb, [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int VB = decltype(v)::value;
    const int chunks = (int)((n + CHUNK - 1) / CHUNK);
    auto sum = sum_kernel<T, VB>;
    auto join = join_kernel<T, VB>;
    ORCA_CUDA(launch_dep(sum, chunks, threads, 0, s, (const char *)d_grad_out, grad_stride * size, nv, sorted, n, n_rows, scale,
                         (char *)d_grad, partial));
    ORCA_COUNT_LAUNCH();
    if (chunks > 1) {
      ORCA_CUDA(launch_dep(join, (unsigned)((chunks + JOIN_WARPS - 1) / JOIN_WARPS), 32 * JOIN_WARPS, 0, s, nv, sorted, n, n_rows, scale,
                           (char *)d_grad, (const float *)partial));
      ORCA_COUNT_LAUNCH();
    }
    ORCA_LAUNCH_CHECK();
    return (int)ORCA_OK;
  });
}

}  // extern "C"
