// Ragged groups of rows: group e covers rows offsets[e] .. offsets[e + 1] of a matrix, with the offsets in device memory
// (whoever assigned the rows to experts wrote them there), so that every CTA finds its own tile.
//
// Offsets are not trusted: they are clamped to [0, rows] and made non-decreasing by a running maximum, so no access
// leaves the matrix and no two groups share a row whatever they hold; a call whose offsets needed that reports
// CB200_ERR_INVALID in the stream's status word, which cb200_stream_sync returns.
#pragma once
#include "common.cuh"

namespace groups {

enum { MAX_EXPERTS = 4096, STATUS_BAD_OFFSETS = 600 };

struct Tile { int expert, lo, hi, index; };   // rows [lo, hi) of the group; index: which row tile of the group this is

// max(v, 0) that keeps a NaN
template <typename T> __device__ __forceinline__ T relu(T v) { return v <= (T)0 ? (T)0 : v; }

__device__ __forceinline__ void report_bad(int* status) {
  if (atomicCAS(status, 0, 1 /* CB200_ERR_INVALID */) == 0) status[1] = STATUS_BAD_OFFSETS;
}

// The whole warp: which group owns row tile `t` when every group's rows are cut into tiles of `tile_rows`.
// False where there are fewer tiles.
__device__ __forceinline__ bool find_tile(const int* offsets, int experts, int rows, int tile_rows, int t, int* status,
                                          Tile& out) {
  const int lane = threadIdx.x & 31;
  int carry_max = 0, carry_tiles = 0;
  bool found = false, bad = false;
  for (int base = 0; base < experts && !found; base += 32) {
    const int e = base + lane;
    int lo = 0, hi = 0;
    if (e < experts) {
      const int raw_lo = offsets[e], raw_hi = offsets[e + 1];
      lo = min(max(raw_lo, 0), rows);
      hi = min(max(raw_hi, 0), rows);
      bad = bad || lo != raw_lo || hi != raw_hi || hi < lo;
    }
    hi = max(hi, lo);
    int run = hi;                                  // running maximum of everything up to this group's end
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, d);
      if (lane >= d) run = max(run, up);
    }
    run = max(run, carry_max);
    int before = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) before = carry_max;
    lo = max(lo, before);
    hi = max(hi, lo);
    int tiles = e < experts ? (hi - lo + tile_rows - 1) / tile_rows : 0, sum = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    sum += carry_tiles;
    const unsigned mine = __ballot_sync(0xffffffffu, t < sum && t >= sum - tiles);
    if (mine) {
      const int src = __ffs(mine) - 1;
      out.expert = base + src;
      out.lo = __shfl_sync(0xffffffffu, lo, src);
      out.hi = __shfl_sync(0xffffffffu, hi, src);
      out.index = t - __shfl_sync(0xffffffffu, sum - tiles, src);
      found = true;
    }
    carry_max = __shfl_sync(0xffffffffu, run, 31);
    carry_tiles = __shfl_sync(0xffffffffu, sum, 31);
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) report_bad(status);
  return found;
}

// A search for a tile stops at the 32 groups around its own, and sees bad offsets no further.  One for a tile that there is not
// sees all, and there is one unless as many tiles as there can be -- of `tile_rows` rows, a row each -- lie before the last groups.
__host__ __device__ __forceinline__ bool all_may_be_found(int rows, int experts, int tile_rows) { return rows <= tile_rows && experts > 32; }

// The whole CTA: looks over all offsets and reports bad ones.
__device__ __forceinline__ void check_offsets(const int* offsets, int experts, int rows, int* status) {
  bool bad = false;
#pragma unroll 4
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    const int lo = offsets[e], hi = offsets[e + 1];
    bad = bad || lo < 0 || hi > rows || hi < lo;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) report_bad(status);
}

// The whole warp: the rows of group `e`.
__device__ __forceinline__ void group_rows(const int* offsets, int rows, int e, int* status, int& lo, int& hi) {
  const int lane = threadIdx.x & 31;
  int m = 0;
  bool bad = false;
  for (int i = lane; i <= e; i += 32) {
    const int raw = offsets[i], v = min(max(raw, 0), rows);
    bad = bad || v != raw;
    m = max(m, v);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  const int own = min(max(offsets[e], 0), rows), raw_hi = offsets[e + 1], next = min(max(raw_hi, 0), rows);
  bad = bad || own != m || next != raw_hi || next < m;
  lo = m;
  hi = max(next, m);
  if (__any_sync(0xffffffffu, bad) && lane == 0) report_bad(status);
}

}  // namespace groups
