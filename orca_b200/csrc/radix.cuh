// One pass of a stable radix sort by eight bits, for what sorts by a few bytes of an id or a time.  A sorter S says what it sorts:
//   typedef Item; static constexpr int RUN (records a warp takes); bool skip(); Item load(int64_t i); int digit(Item).
// One pass = a per-block digit histogram, a scan of the counts of every digit over the blocks (one block per digit),
// and a stable scatter.  Inside a block every warp owns a contiguous run of the tile and walks it 32 records at a
// time (eight loads in flight); lanes with the same digit find one another with match.any, so a record's rank among
// its digit is the warp's running count plus the number of lower lanes in its group.
#pragma once

#include "common.cuh"

namespace orca {
namespace radix {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int BINS = 256;
constexpr int UNROLL = 8;            // loads in flight per lane

// Walks the warp's run, advancing the warp's digit counts; SCATTER: writes every item at its digit's count.
template <bool SCATTER, class S>
__device__ __forceinline__ void walk_run(const S &s, typename S::Item *out, int64_t first, int64_t n,
                                         int32_t *count /* [BINS] of this warp */) {
  const int lane = threadIdx.x & 31;
  const uint32_t lower = (1u << lane) - 1u;
  for (int r = 0; r < S::RUN && first + r < n; r += 32 * UNROLL) {
    typename S::Item x[UNROLL];
    int d[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int64_t i = first + r + 32 * u + lane;
      if (i < n) x[u] = s.load(i);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)   // lanes past the end group with nobody
      d[u] = first + r + 32 * u + lane < n ? s.digit(x[u]) : BINS + lane;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const uint32_t group = __match_any_sync(0xffffffffu, d[u]);
      const bool valid = d[u] < BINS;
      if (SCATTER && valid) out[count[d[u]] + __popc(group & lower)] = x[u];
      __syncwarp();
      if (valid && (group & lower) == 0) count[d[u]] += __popc(group);
      __syncwarp();
    }
  }
}

// counts[digit * n_blocks + block] = items of the block's tile with that digit
template <class S>
__global__ void __launch_bounds__(THREADS) digit_count_kernel(S s, int64_t n, int32_t *counts, int n_blocks) {
  __shared__ int32_t count[WARPS][BINS];
  if (s.skip()) return;
  for (int i = threadIdx.x; i < WARPS * BINS; i += THREADS) (&count[0][0])[i] = 0;
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  walk_run<false>(s, (typename S::Item *)nullptr, (int64_t)blockIdx.x * (WARPS * S::RUN) + (int64_t)warp * S::RUN, n, count[warp]);
  __syncthreads();
  int total = 0;
  for (int w = 0; w < WARPS; ++w) total += count[w][threadIdx.x];
  counts[(int64_t)threadIdx.x * n_blocks + blockIdx.x] = total;
}

__device__ __forceinline__ int32_t block_scan(int32_t v, int32_t *warp_sum, int32_t &total) {   // exclusive, THREADS threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int32_t before = 0;
  total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  __syncthreads();
  return before + incl - v;
}

// exclusive scan of one digit's counts over the blocks, in place; totals[digit] = their sum
static __global__ void __launch_bounds__(THREADS) digit_scan_kernel(int32_t *counts, int n_blocks, int32_t *totals,
                                                             const int32_t *unsorted) {
  __shared__ int32_t warp_sum[WARPS];
  if (unsorted != nullptr && *unsorted == 0) return;
  int32_t *c = counts + (int64_t)blockIdx.x * n_blocks;
  int32_t carry = 0;
  for (int base = 0; base < n_blocks; base += 4 * THREADS) {
    const int i = base + 4 * (int)threadIdx.x;
    int32_t v[4], mine = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) mine += v[j] = i + j < n_blocks ? c[i + j] : 0;
    int32_t run = carry + block_scan(mine, warp_sum, total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i + j < n_blocks) c[i + j] = run;
      run += v[j];
    }
    carry += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// stable scatter of the block's tile: a digit's items of this block start behind all lower digits and behind the
// same digit's items of the blocks before
template <class S>
__global__ void __launch_bounds__(THREADS) digit_scatter_kernel(S s, int64_t n, typename S::Item *out,
                                                                const int32_t *offsets, const int32_t *totals,
                                                                int n_blocks) {
  __shared__ int32_t count[WARPS][BINS];
  __shared__ int32_t warp_sum[WARPS];
  if (s.skip()) return;
  for (int i = threadIdx.x; i < WARPS * BINS; i += THREADS) (&count[0][0])[i] = 0;
  int32_t all;
  int32_t at = block_scan(totals[threadIdx.x], warp_sum, all) + offsets[(int64_t)threadIdx.x * n_blocks + blockIdx.x];
  const int warp = threadIdx.x >> 5;
  const int64_t first = (int64_t)blockIdx.x * (WARPS * S::RUN) + (int64_t)warp * S::RUN;
  walk_run<false>(s, (typename S::Item *)nullptr, first, n, count[warp]);
  __syncthreads();
  for (int w = 0; w < WARPS; ++w) {
    const int32_t c = count[w][threadIdx.x];
    count[w][threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
  walk_run<true>(s, out, first, n, count[warp]);
}

template <class S>
static int one_pass(const S &s, int64_t n, typename S::Item *out, int32_t *counts, int32_t *totals,
                    const int32_t *unsorted, cudaStream_t stream) {
  const int blocks = (int)((n + WARPS * S::RUN - 1) / (WARPS * S::RUN));
  digit_count_kernel<S><<<blocks, THREADS, 0, stream>>>(s, n, counts, blocks);
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  digit_scan_kernel<<<BINS, THREADS, 0, stream>>>(counts, blocks, totals, unsorted);
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  digit_scatter_kernel<S><<<blocks, THREADS, 0, stream>>>(s, n, out, counts, totals, blocks);
  ORCA_COUNT_LAUNCH();
  ORCA_LAUNCH_CHECK();
  return ORCA_OK;
}

}  // namespace radix
}  // namespace orca
