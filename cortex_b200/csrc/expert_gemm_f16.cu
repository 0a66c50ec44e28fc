// Large fp32 products grouped by expert at twice the rate of 3xTF32: operands as pairs of scaled halves.
//
// The tensor core multiplies fp16 at twice the rate of tf32 with the same 11-bit significands, so the split
//   x * s = h1 + h2,   h1 = half(x * s),  h2 = half(x * s - h1),   s = a power of two per operand row
// carries 22 bits like hi + lo of 3xTF32 does, and the three products h1 h1, h1 h2, h2 h1 cost half of what they cost
// there.  What tf32 has and fp16 lacks is range: s puts a row's largest value into [2^14, 2^15), values down to 2^-17 of
// it keep their 22 bits, smaller ones an absolute error of 2^-25 (scaled).  Down to 2^-20 of the largest that is at most
// 2^-19 of the value, 2^-18 of the sum of |a||b| in every element of a result.  What the halves leave of values below that
// (2.3 in a million of normal data; of values below TINY all) is written to lists, and elements of the result in which it could show -- whose sum is not
// far above what can be missing: next to none of dense data -- get it, times what it meets, in a small launch behind the
// product.  So every element is good, whatever it is made of.  Where there are too many such values (in all or in one row),
// where a row's largest value is outside [2^-48, 2^60] or a scaled value below 2^-100, and where there is an infinity or a NaN,
// a flag is raised in device memory; the kernels here then do nothing more and the 3xTF32 kernel launched behind them, which
// otherwise does nothing, does the work.
// (Measured against a check that let 1 in 64 values of a row lie low and bounded no element, us: 8000 rows over 32 experts of
// 2048 x 1024 206 -> 212 forward, 225 -> 226 input gradient, 211 -> 209 weight gradient; a piece that needs remainders costs
// the call about 6 more.  A proof from counts of low values per row and column instead of the lists: 211, 230 and 214, but 490
// for ReLU'd or rarely used features and 2000 for pruned matrices, which it had to send to 3xTF32.)
//
// Steps of a call: group bounds and the table of tiles (one warp); the operands' halves, K-contiguous, with their scales
// and lists (HBM-bound; operands whose reduction axis is not contiguous get a pass for the column maxima first); the product;
// remainders; the guarded 3xTF32 kernel.
//
// The product runs on CTA pairs (tcgen05.mma.cta_group::2, 256 lanes x up to 256 columns per pair), persistent, three
// pipeline stages of 64 KB (128-byte rows), as the pre-split layer GEMM: every TMA load is a plain one into the issuing CTA, completing on
// the leader's barrier.  Output features (expert_gemm) or input features (expert_gemm_weights) lie in the lanes, so a warp
// stores 128 consecutive bytes; the ragged rows (or output features) lie in the columns, in multiples of 32.
// All three products go to one accumulator of 256 columns, so TMEM holds two: the tensor cores fill one while the epilogue
// warps empty the other.  (With the cross terms in an accumulator of their own, scaled by 2^11 for range, there was room
// for one tile, and the read-out and its hand-shakes cost 5 us per tile where the product of a weight gradient takes 3:
// 125 us against 117 for 8000 rows over 32 experts,
// 2048 x 1024.)  The tensor core adds with truncation: every 256 values of
// k -- 48 additions -- the accumulator is added into registers, rounded to nearest, and the other one takes over.  (Error of
// normal data against 64 bits, and time of 16384 rows over 8 experts of 4096 x 4096: every 512 1.8e-6 and 1.376 ms, 256
// 0.93e-6 and 1.382 ms, 128 0.49e-6 and 1.456 ms.)
#include "gemm3x_common.cuh"
#include "expert_groups.cuh"
#include <cuda_fp16.h>
#include <math.h>
#include <mutex>
#include <type_traits>

using namespace sm100;
using namespace gemm3x;

namespace {

constexpr int BM = 128, BN = 256, BK = 64;               // per CTA: 128 lanes, 256 columns of the pair, 64 halves of k
constexpr int POS = 32;                                  // padded positions that the column pass writes at a time
constexpr int EPI_WARPS = 8;
constexpr int THREADS = (EPI_WARPS + 4) * 32;            // three warpgroups; the last warp only gives its registers up
constexpr int L_TILE = BM * BK * 2, R_TILE = BN / 2 * BK * 2;       // 16 KiB each
constexpr int R_BOX = 64;                                // rows of one box of the column operand
constexpr int RAW = L_TILE + R_TILE, STAGE = 2 * RAW, STAGES = 196608 / STAGE;
constexpr int WHERE = 16384;                             // places for remainders (normal data: a few hundred are taken), two bits each
constexpr int WHERE_BYTES = WHERE / 4 + WHERE * 4;
constexpr int SCALES = EPI_WARPS * (BN / 2) * 4;           // a column-scale list per epilogue warp
constexpr int SMEM = STAGES * STAGE + 1024 + 256 + SCALES + WHERE / 4;
constexpr int TMEM_COLS = 2 * BN;
constexpr int DRAIN = 256 / BK;                         // stages per accumulator filling

// what one warp works out at the start of a call, in device memory
struct Plan {
  int flag;                    // 1: the operands do not fit scaled halves
  int tiles;                   // expert_gemm: row tiles in the table
  int padded;                  // expert_gemm_weights: padded positions in use
  int first_row, end_row;      // rows outside are in no group
  int later;                   // pieces in the list for add_rests_kernel
  int unused[2];
};
// What an expert's operands have for the lists; all zero at the start of a call.  (A line each: the counts are atomics.)
struct alignas(128) Fit {
  int bad;                     // something does not fit scaled halves, or its list
  int listed[2];               // remainders of the lanes' operand, of the columns'
  int most;                    // no more of them than this in one lane or column
};
// What the two halves leave of a scaled value below SMALL: of lane or column `at` (of the expert's matrix; a row of the batch; a
// column of a weight gradient's operand), at position k of the halves.
struct alignas(16) Rest { int at, k; float rest; int unused; };
// A value below TINY is left to the list as a whole: the tensor core adds products of halves whose first half is not normal with as
// many bits less as that has leading zeros (three of either operand at TINY: 18 left; 10 at 2^-24).
constexpr float SMALL = 1.f / 64, TINY = 0x1p-17f, LEAST = 0x1p-100f;
constexpr int MOST_RESTS = 8;            // in a lane or column (they are added one after another; normal data: 4 in the largest calls)
// An operand's lists, `cap` for every expert.  Both operands': by where remainders are, hashed, two bits -- a lane or a column without
// the lower has none, one with the higher has values below TINY -- and (behind the bits) the number of remainders.
struct Rests { Rest* list; uint32_t* where; int cap, side; };
__device__ __forceinline__ int where_of(int side, int expert, int at) {
  return (int)(((unsigned)at * 2u + (unsigned)side + (unsigned)expert * 0x9e3779b1u) * 0x85ebca6bu >> 18);
}
struct Entry { int expert, lo, hi, first; };   // expert_gemm: rows [lo, hi); expert_gemm_weights: rows and first padded position

// bounds -> table.  WEIGHTS: entry e per expert (+ one behind the last, whose `first` ends the positions); otherwise an
// entry per tile of BN rows.
// (CTA 0, one warp; the other CTAs zero the words that the next kernels take maxima into)
__global__ void __launch_bounds__(128) plan_kernel(Plan* plan, Entry* table, int* owner, int* begins, const int* offsets, int experts,
                                                   int rows, int weights, int* status, uint32_t* zero, long long zero_n) {
  if (blockIdx.x > 0) {
    for (long long i = (blockIdx.x - 1LL) * 128 + threadIdx.x; i < zero_n; i += (gridDim.x - 1LL) * 128) zero[i] = 0;
    return;
  }
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  int carry_max = 0, carry = 0, first_row = rows;
  bool bad = false;
  for (int base = 0; base < experts; base += 32) {
    const int e = base + lane;
    int lo = 0, hi = 0;
    if (e < experts) {
      const int raw_lo = offsets[e], raw_hi = offsets[e + 1];
      lo = min(max(raw_lo, 0), rows);
      hi = min(max(raw_hi, 0), rows);
      bad = bad || lo != raw_lo || hi != raw_hi || hi < lo;
    }
    hi = max(hi, lo);
    int run = hi;
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
    if (e < experts && begins) begins[e] = lo;
    if (e < experts && hi > lo) first_row = min(first_row, lo);
    const int mine = e < experts ? (weights ? (hi - lo + BK - 1) / BK * BK : (hi - lo + BN - 1) / BN) : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    sum += carry;
    if (e < experts) {
      if (weights) {
        table[e] = {e, lo, hi, sum - mine};
        for (int i = 0; i < mine; i += POS) owner[(sum - mine + i) / POS] = e;      // whose the next 32 positions are
      } else for (int i = 0; i < mine; ++i) table[sum - mine + i] = {e, lo + i * BN, hi, 0};
    }
    carry_max = __shfl_sync(0xffffffffu, run, 31);
    carry = __shfl_sync(0xffffffffu, sum, 31);
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) groups::report_bad(status);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) first_row = min(first_row, __shfl_xor_sync(0xffffffffu, first_row, d));
  if (lane == 0) {
    plan->flag = plan->later = 0;
    plan->tiles = plan->padded = carry;
    plan->first_row = first_row;
    plan->end_row = carry_max;
    if (weights) table[experts] = {experts, 0, 0, carry};
  }
}

// The kernels of a call are launched so that each may be set up while its predecessor ends; nothing of the predecessors'
// results is touched before this.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- scaled halves ---------------------------------------------------------------------------------------------
// Scale of a row (or column) whose largest magnitude has these bits: 2^up; its inverse; false: outside the range.
__device__ __forceinline__ bool scale_of(uint32_t max_bits, float& up, float& down) {
  if (max_bits == 0) { up = down = 1.f; return true; }
  const int ex = (int)(max_bits >> 23) - 127;
  const bool ok = ex >= -48 && ex <= 60;                   // (two inverse scales multiply to a normal number)
  const int e = ok ? 14 - ex : 0;
  up = __uint_as_float((uint32_t)(127 + e) << 23);
  down = __uint_as_float((uint32_t)(127 - e) << 23);
  return ok;
}
__device__ __forceinline__ void split_half(float y, __half& h1, __half& h2) {
  h1 = __float2half_rn(y);
  h2 = __float2half_rn(y - __half2float(h1));
}
union Half8 { __half h[8]; __half2 h2[4]; uint4 v; };

// Eight values times `up` as halves; bit j: value j is below SMALL, and not 0.
__device__ __forceinline__ uint32_t split8(const float (&w)[8], float up, Half8& a, Half8& b) {
  __half2 least = __float2half2_rn(65504.f);               // two at a time
  uint32_t small = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) split_half(w[j] * up, a.h[j], b.h[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) least = __hmin2(least, __habs2(a.h2[j]));
  if (__half2float(__hmin(__low2half(least), __high2half(least))) < SMALL)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (w[j] != 0.f && fabsf(w[j] * up) < SMALL) {
        small |= 1u << j;
        if (fabsf(w[j] * up) < TINY) a.h[j] = b.h[j] = __float2half_rn(0.f);
      }
  return small;
}
// Are there so many that lists are no use?  (Data of a wide range would queue up at the counts: 2048 x 1024 values over 60 powers
// of two for each of 32 experts 100 ms.)
__device__ __forceinline__ bool too_many(Fit* fit, int expert, uint32_t small) {
  const unsigned lanes = __activemask();
  const bool many = __popc(__ballot_sync(lanes, small != 0)) > MOST_RESTS || __popc(small) > 2;
  if (many) fit[expert].bad = 1;
  return many || __ldcg(&fit[expert].bad) != 0;
}
__device__ __forceinline__ void keep_rest(Fit* fit, const Rests& rests, int expert, int at, int k, float y) {
  Fit* f = fit + expert;
  if (!(fabsf(y) >= LEAST)) f->bad = 1;
  __half h1, h2;
  split_half(y, h1, h2);
  const bool tiny = fabsf(y) < TINY;
  const float rest = tiny ? y : (y - __half2float(h1)) - __half2float(h2);      // both differences are exact
  if (rest == 0.f) return;
  const int i = atomicAdd(&f->listed[rests.side], 1), h = where_of(rests.side, expert, at);
  atomicOr(rests.where + (h >> 4), (tiny ? 3u : 1u) << 2 * (h & 15));
  const int here = (int)atomicAdd(rests.where + WHERE / 16 + h, 1u) + 1;
  atomicMax(&f->most, here);
  if (i >= rests.cap || here > MOST_RESTS) f->bad = 1;
  else rests.list[(long long)expert * rests.cap + i] = {at, k, rest, 0};
}

__device__ __forceinline__ void load8(const float* p, int left, bool vec, float (&v)[8]) {
  if (vec && left >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
  }
}

// One row of scaled halves: TPR threads per row, 8 values per thread and step, the first HOLD steps in registers between the
// maximum and the split (longer rows are read again, from L2).  hi / lo: pitch kp (a multiple of 8).
//   RAGGED = 0  the experts' matrices: row r at x + (r / rows_per) * stride + (r % rows_per) * ld
//   RAGGED = 3  the same, of rows that run across the reduction; a row of zeros gets the inverse scale 0
//   RAGGED = 1  the ragged rows: rows in no group become zeros
//   RAGGED = 2  the same, every value multiplied by 2^14 fold[expert of the row][column] first: the inverse scales of a matrix
//               whose rows run across the reduction, which cannot be taken out of the sum behind it
template <int TPR, int RAGGED>
__global__ void __launch_bounds__(256, 4) split_rows_kernel(__half* hi, __half* lo, float* down_out, const float* x, long long ld,
                                                         long long stride, int rows_per, long long rows, int cols, int kp,
                                                         const Plan* plan, Fit* fit, Rests rests, const float* fold, const int* begins,
                                                         int experts) {
  constexpr int HOLD = 4;
  constexpr bool MATRICES = RAGGED == 0 || RAGGED == 3;
  wait_for_previous_kernel();
  __shared__ uint32_t part_max[8];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, warp = threadIdx.x >> 5;
  const long long r = (long long)blockIdx.x * (256 / TPR) + sub;
  const bool live = r < rows, grouped = MATRICES || (r >= plan->first_row && r < plan->end_row);
  const float* src = live ? (!MATRICES ? x + r * ld : x + (r / rows_per) * stride + (r % rows_per) * ld) : x;
  const bool vec = ((uintptr_t)src & 15) == 0;
  const int n = live ? cols : 0;
  auto expert_of_row = [&]() {
    if (MATRICES) return (int)(r / rows_per);
    int a = 0, z = experts;                                // the last group that begins at or before this row
    while (z - a > 1) {
      const int mid = (a + z) >> 1;
      if (begins[mid] <= r) a = mid; else z = mid;
    }
    return a;
  };
  const float* scales = nullptr;
  if (RAGGED == 2 && live && grouped) scales = fold + (long long)expert_of_row() * cols;
  auto fetch = [&](int c, float (&w)[8]) {
    if (!MATRICES && !grouped) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = 0.f;
      return;
    }
    load8(src + c, n - c, vec, w);
    if (RAGGED == 2) {
      float f[8];
      load8(scales + c, n - c, ((uintptr_t)scales & 15) == 0, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= 16384.f * f[j];
    }
  };
  float v[HOLD][8];
  uint32_t m = 0;
#pragma unroll
  for (int it = 0; it < HOLD; ++it) {
    const int c = (it * TPR + t) * 8;
    if (c < n) fetch(c, v[it]);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[it][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[it][j]) & 0x7fffffffu);
  }
  for (int c = (HOLD * TPR + t) * 8; c < n; c += TPR * 8) {
    float w[8];
    fetch(c, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(w[j]) & 0x7fffffffu);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) m = max(m, part_max[sub * (TPR / 32) + w]);
  }
  float up, down;
  const bool ok = scale_of(m, up, down);
  if (!ok) up = 0.f;
  auto put = [&](int c, const float (&w)[8]) {
    Half8 a, b;
    uint32_t small = split8(w, up, a, b);
    *reinterpret_cast<uint4*>(hi + r * kp + c) = a.v;      // pitch and position are multiples of 8 halves
    *reinterpret_cast<uint4*>(lo + r * kp + c) = b.v;
    if (!ok || (small && too_many(fit, expert_of_row(), small))) small = 0;
    for (; small; small &= small - 1) {
      const int at = c + __ffs(small) - 1, row = (int)(MATRICES ? r % rows_per : r);
      const float y = (RAGGED == 2 ? src[at] * (16384.f * scales[at]) : src[at]) * up;
      keep_rest(fit, rests, expert_of_row(), RAGGED == 3 ? at : row, RAGGED == 3 ? row : at, y);
    }
  };
#pragma unroll
  for (int it = 0; it < HOLD; ++it) {
    const int c = (it * TPR + t) * 8;
    if (c < n) put(c, v[it]);
  }
  for (int c = (HOLD * TPR + t) * 8; c < n; c += TPR * 8) {
    float w[8];
    fetch(c, w);
    put(c, w);
  }
  if (t == 0 && live) {
    // (a scale of 0 that is folded into the other operand takes what meets a row of zeros out of its row's maximum, but for
    // infinities and NaN)
    down_out[r] = RAGGED == 3 && m == 0 ? 0.f : down;
    if (!ok) fit[expert_of_row()].bad = 1;
  }
}

// Operands whose reduction runs down their columns, in ragged groups of rows: table[g].lo .. hi.
// maxima[g][c] = bits of the largest magnitude in column c of group g.  A CTA: 128 columns of up to 64 rows of one group at a
// time, four rows side by side and (where the rows are 16-byte aligned) four columns per thread.  `sums`, where given, gets
// those rows' column sums, in row b + g for the rows of block b that belong to group g (a pair of its own for every such row).
template <int V>
__global__ void __launch_bounds__(128) column_max_kernel(uint32_t* maxima, float* sums, const float* x, long long ld, const Entry* table,
                                                         int groups_n, int rows, int cols) {
  constexpr int LANES = 128 / V, SIDE = 128 / LANES;       // threads per row, rows side by side
  wait_for_previous_kernel();
  struct alignas(4 * V) Pack { float e[V]; };
  __shared__ uint32_t part[SIDE][128];
  __shared__ float part_sum[SIDE][128];
  const int tx = threadIdx.x % LANES, ty = threadIdx.x / LANES, c = blockIdx.x * 128 + tx * V;
  const bool live = c < cols;                              // V = 4: cols is a multiple of 4
  auto reduce = [&](long long b, int g, int a, int z) {    // rows a .. z - 1 of block b, all of group g
    uint32_t m[V];
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { m[j] = 0; s[j] = 0.f; }
    if (live) {
#pragma unroll 4
      for (int r = a + ty; r < z; r += SIDE) {
        const Pack v = *reinterpret_cast<const Pack*>(x + (long long)r * ld + c);
#pragma unroll
        for (int j = 0; j < V; ++j) { m[j] = max(m[j], __float_as_uint(v.e[j]) & 0x7fffffffu); s[j] += v.e[j]; }
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) { part[ty][tx * V + j] = m[j]; part_sum[ty][tx * V + j] = s[j]; }
    __syncthreads();
    uint32_t all = part[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < SIDE; ++i) all = max(all, part[i][threadIdx.x]);
    const int at = blockIdx.x * 128 + threadIdx.x;
    if (at < cols) atomicMax(maxima + (long long)g * cols + at, all);
    if (sums && at < cols) {
      float sum = part_sum[0][threadIdx.x];
#pragma unroll
      for (int i = 1; i < SIDE; ++i) sum += part_sum[i][threadIdx.x];
      sums[(b + g) * cols + at] = sum;
    }
    __syncthreads();
  };
  for (long long b = blockIdx.y; b * 64 < rows; b += gridDim.y) {
    const int r0 = (int)(b * 64), r1 = min(rows, r0 + 64);
    int g = 0, end = groups_n;                              // the last group that begins at or before r0
    while (end - g > 1) {
      const int mid = (g + end) >> 1;
      if (table[mid].lo <= r0) g = mid; else end = mid;
    }
    for (; g < groups_n && table[g].lo < r1; ++g) {
      const int a = max(r0, table[g].lo), z = min(r1, table[g].hi);
      if (z > a) reduce(b, g, a, z);
    }
  }
}

// bias_gradient[g, c] = alpha * (the sums of group g's rows, block by block) + beta * bias_gradient[g, c]
__global__ void __launch_bounds__(128) column_sum_kernel(float* out, const float* sums, const Entry* table, int cols, float alpha, float beta) {
  wait_for_previous_kernel();
  const int c = blockIdx.x * 128 + threadIdx.x, g = blockIdx.y;
  if (c >= cols) return;
  const Entry e = table[g];
  float s = 0.f;
  if (e.hi > e.lo) {
    const long long first = e.lo / 64, last = (e.hi - 1) / 64;
#pragma unroll 8
    for (long long b = first; b <= last; ++b) s += sums[(b + g) * cols + c];
  }
  float* to = out + (long long)g * cols + c;
  float v = alpha * s;
  if (beta != 0.f) v += beta * (*to);
  *to = v;
}

// hi / lo [cols][positions]: 32 positions x 64 columns at a time through shared memory.  Groups start at a multiple of 64
// positions and are padded with zeros (owner: which group the next 32 positions belong to).  A CTA takes two neighbouring
// blocks of 64 columns.
__global__ void __launch_bounds__(256) split_columns_kernel(__half* hi, __half* lo, float* down_out, const uint32_t* maxima, const float* x,
                                                            long long ld, const Entry* table, const int* owner, int cols, long long kp,
                                                            const Plan* plan, Fit* fit, Rests rests) {
  __shared__ float tile[2][32][65];
  wait_for_previous_kernel();
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int blocks = plan->padded / POS;
  for (int b = blockIdx.y; b < blocks; b += gridDim.y) {
    const int g = owner[b];
    const Entry e = table[g];
    const long long pos = (long long)b * POS;              // first position written
    const int r0 = e.lo + (int)(pos - e.first), end = e.hi;
    const bool begins = pos == e.first;                    // these are the group's first positions
    __syncthreads();
    uint32_t m[2] = {0, 0};
    const int col = threadIdx.x >> 2, p8 = (threadIdx.x & 3) * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mine = blockIdx.x * 128 + h * 64 + col;
      if (mine < cols) m[h] = maxima[(long long)g * cols + mine];
      const int c = blockIdx.x * 128 + h * 64 + tx;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + ty + 4 * i;
        tile[h][ty + 4 * i][tx] = (r < end && c < cols) ? x[(long long)r * ld + c] : 0.f;
      }
    }
    __syncthreads();
    // a thread: 8 positions of one column of each block
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = blockIdx.x * 128 + h * 64 + col;
      if (c >= cols) continue;
      float up, down, w[8];
      const bool ok = scale_of(m[h], up, down);
      Half8 a, z;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = tile[h][p8 + j][col];
      uint32_t small = split8(w, up, a, z);
      *reinterpret_cast<uint4*>(hi + c * kp + pos + p8) = a.v;             // kp is a multiple of 64
      *reinterpret_cast<uint4*>(lo + c * kp + pos + p8) = z.v;
      if (p8 == 0 && begins) down_out[(long long)g * cols + c] = down;
      if (!ok) {
        fit[g].bad = 1;
        small = 0;
      }
      if (small && too_many(fit, g, small)) small = 0;
      for (; small; small &= small - 1) {
        const int j = __ffs(small) - 1;
        keep_rest(fit, rests, g, c, (int)pos + p8 + j, tile[h][p8 + j][col] * up);
      }
    }
  }
}

// ---- the product -----------------------------------------------------------------------------------------------
struct PairArgs {
  float* C;                     // element (column c, lane l) of a tile at C + c * ldc + l
  long long ldc, c_stride;
  const float* l_down; const float* r_down;      // inverse scales (l_down null: the lanes' ones were folded into the columns' values)
  const float* bias;
  Plan* plan;
  const Fit* fit;               // per expert
  Rests l_rests, r_rests;
  int4* later;                  // pieces that wait for their remainders: expert, first lane, first column, columns
  // the halves: the lane operand's element (expert, lane, k) at expert * l_expert + lane * l_lane + k * l_k, the column operand's
  // (row, k) at row * r_pitch + k
  const __half* l_hi; const __half* l_lo; const __half* r_hi; const __half* r_lo;
  long long l_expert, l_lane, l_k, r_pitch;
  const Entry* table;
  int* status;
  int lanes, cols;              // extents: lanes of one expert's matrix; WEIGHTS: columns of one result
  int K;                        // expert_gemm: reduction length
  int l_mn;                     // the lanes are contiguous in the lane operand ([k][lane], 64-lane boxes)
  int experts, weights, act;
  float alpha, beta;
};

struct Unit { int expert, l0, r0, cols, l_row, kb, nkb; };

// The table entry of a unit: requested one unit ahead, so that its latency is not between two tiles.
__device__ __forceinline__ Entry entry_of(const PairArgs& p, int unit, int n_units) {
  const int tiles_l = (p.lanes + 2 * BM - 1) / (2 * BM);
  int row = min(unit, n_units - 1) / tiles_l;
  if (p.weights) row /= (p.cols + BN - 1) / BN;
  const int4 v = __ldg(reinterpret_cast<const int4*>(p.table) + row);
  return {v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ Unit unit_of(const PairArgs& p, int unit, const Entry& e) {
  const int tiles_l = (p.lanes + 2 * BM - 1) / (2 * BM);
  Unit u;
  const int row = unit / tiles_l;
  u.expert = e.expert;
  u.l0 = (unit - row * tiles_l) * 2 * BM;
  if (p.weights) {
    const int tiles_r = (p.cols + BN - 1) / BN;
    u.r0 = (row - e.expert * tiles_r) * BN;
    u.cols = min(BN, p.cols - u.r0);
    u.l_row = u.l0;
    u.kb = e.first / BK;
    u.nkb = (e.hi - e.lo + BK - 1) / BK;
  } else {
    u.r0 = e.lo;
    u.cols = min(BN, e.hi - e.lo);
    u.l_row = p.l_mn ? u.l0 : e.expert * p.lanes + u.l0;
    u.kb = 0;
    u.nkb = (p.K + BK - 1) / BK;
  }
  return u;
}

__device__ __forceinline__ void mma_f16_pair_words(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                                   uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// instruction descriptor of kind::f16 with half operands and fp32 accumulation (the fields of make_idesc_tf32)
__host__ __device__ __forceinline__ uint32_t make_idesc_f16(int m, int n, int a_mn_major) {
  return (1u << 4) | ((uint32_t)(a_mn_major & 1) << 15) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// The next of n remainders in the order of (at, k) -- whatever order they were written in -- with at in [first, end), by the
// whole warp; returns how many there are from it on.  `key` starts as 0.
__device__ __forceinline__ int next_rest(const Rest* list, int n, int first, int end, unsigned long long& key, int& at, int& k, float& rest) {
  const int lane = threadIdx.x & 31;
  unsigned long long best = ~0ull;
  int count = 0;
  rest = 0.f;
#pragma unroll 2
  for (int i = lane; i < n; i += 32) {
    const int4 v = __ldg(reinterpret_cast<const int4*>(list) + i);
    const unsigned long long own = ((unsigned long long)(unsigned)v.x << 32 | (unsigned)v.y) + 1;
    if (v.x >= first && v.x < end && own > key) {
      ++count;
      if (own < best) { best = own; rest = __int_as_float(v.z); }
    }
  }
  count = (int)__reduce_add_sync(0xffffffffu, (unsigned)count);
  if (count == 0) return 0;
  const unsigned high = __reduce_min_sync(0xffffffffu, (unsigned)(best >> 32));
  const unsigned low = __reduce_min_sync(0xffffffffu, (unsigned)(best >> 32) == high ? (unsigned)best : 0xffffffffu);
  const unsigned owner = __ballot_sync(0xffffffffu, best == ((unsigned long long)high << 32 | low));
  rest = __shfl_sync(0xffffffffu, rest, __ffs(owner) - 1);
  key = (unsigned long long)high << 32 | low;
  at = (int)((key - 1) >> 32);
  k = (int)(key - 1);
  return count;
}

// The pieces (32 lanes, up to 128 columns) that the product has left for later: what the halves leave out of the operands' small
// values -- remainders of the lanes times the columns' values (these with their own remainders), those of the columns times the
// lanes' halves -- and the activation.  A CTA a piece, a warp 16 columns of it.  (Most calls have a piece or none: loops are kept
// short, since fetching their code is what takes the time.)
__global__ void __launch_bounds__(256) add_rests_kernel(const __grid_constant__ PairArgs p) {
  constexpr int OWN = BN / 2 / 8;
  __shared__ float sums[8][OWN][32];
  wait_for_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pieces = p.plan->later;
#pragma unroll 1
  for (int i = blockIdx.x; i < pieces; i += gridDim.x) {
    const int4 piece = p.later[i];
    const int expert = piece.x, l = piece.y + lane, r_first = piece.z + warp * OWN, cols = min(OWN, piece.w - warp * OWN);
    if (cols <= 0) continue;
    const Fit f = p.fit[expert];
    float (&sum)[OWN][32] = sums[warp];
#pragma unroll 1
    for (int j = 0; j < cols; ++j) sum[j][lane] = 0.f;
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      const Rest* list = (side ? p.r_rests.list : p.l_rests.list) + (long long)expert * (side ? p.r_rests.cap : p.l_rests.cap);
      const int first = side ? r_first : piece.y, end = side ? r_first + cols : piece.y + 32;
      unsigned long long key = 0;
      int at, k;
      float rest;
#pragma unroll 1
      while (next_rest(list, f.listed[side], first, end, key, at, k, rest)) {
        const long long r_at = (long long)(side ? at : r_first + lane) * p.r_pitch + k, l_at = expert * p.l_expert + l * p.l_lane + k * p.l_k;
        const bool there = side ? l < p.lanes : lane < cols;
        float x = there ? __half2float((side ? p.l_hi : p.r_hi)[side ? l_at : r_at]) + __half2float((side ? p.l_lo : p.r_lo)[side ? l_at : r_at]) : 0.f;
        if (side) {
          sum[at - r_first][lane] = fmaf(rest, x, sum[at - r_first][lane]);
          continue;
        }
        const Rest* of_r = p.r_rests.list + (long long)expert * p.r_rests.cap;
#pragma unroll 1
        for (int b = 0; b < f.listed[1]; b += 32) {
          const int4 v = b + lane < f.listed[1] ? __ldg(reinterpret_cast<const int4*>(of_r) + b + lane) : make_int4(-1, -1, 0, 0);
#pragma unroll 1
          for (unsigned hit = __ballot_sync(0xffffffffu, v.y == k && v.x >= r_first && v.x < r_first + cols); hit; hit &= hit - 1) {
            const int c = __shfl_sync(0xffffffffu, v.x, __ffs(hit) - 1) - r_first;
            const float its = __int_as_float(__shfl_sync(0xffffffffu, v.z, __ffs(hit) - 1));
            if (c == lane) x += its;
          }
        }
        __syncwarp();
        if (lane < cols) sum[lane][at - piece.y] = fmaf(rest, x, sum[lane][at - piece.y]);
        __syncwarp();
      }
    }
    const float r_scale = lane < cols ? p.r_down[(p.weights ? (long long)expert * p.cols : 0) + r_first + lane] : 0.f;
    float l_scale = 0.f, old[OWN];
    float* c = p.C + (p.weights ? expert * p.c_stride : 0) + (long long)r_first * p.ldc + l;
    if (l < p.lanes) {
      l_scale = p.l_down ? p.l_down[(long long)expert * p.lanes + l] : 1.f / 16384.f;
#pragma unroll
      for (int j = 0; j < OWN; ++j) old[j] = j < cols ? c[(long long)j * p.ldc] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < OWN; ++j) {
      const float scale = l_scale * __shfl_sync(0xffffffffu, r_scale, j);
      if (j < cols) old[j] = fmaf(sum[j][lane] * scale, p.alpha, old[j]);
    }
    if (l < p.lanes) {
#pragma unroll
      for (int j = 0; j < OWN; ++j)
        if (j < cols) sum[j][lane] = old[j];
#pragma unroll 1
      for (int j = 0; j < cols; ++j) {
        float v = sum[j][lane];
        if (p.act == CB200_ACT_RELU) v = groups::relu(v);
        else if (p.act != CB200_ACT_NONE) v = apply_act_transcendental(v, p.act);
        c[(long long)j * p.ldc] = v;
      }
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(THREADS, 1)
expert_pair_kernel(const __grid_constant__ CUtensorMap tmL, const __grid_constant__ CUtensorMap tmLlo, const __grid_constant__ CUtensorMap tmR,
                   const __grid_constant__ CUtensorMap tmRlo, const __grid_constant__ PairArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = (uint64_t*)(smem + STAGES * STAGE);
  // bars[0..S) full (the leader's copy: its two producers arrive, both CTAs' loads complete bytes), [S..2S) empty,
  // [2S..2S+2) accumulator 0 / 1 is filled (each CTA's own), [2S+2..2S+4) it has been read out (the leader's: one arrival
  // per epilogue warp of both CTAs), [2S+4] unwinding only: every MMA issued so far has retired
  uint32_t* tmem_slot = (uint32_t*)(bars + 2 * STAGES + 5);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_clusters = (int)gridDim.x >> 1, cluster_id = (int)blockIdx.x >> 1;

  wait_for_previous_kernel();
  uint32_t* where = reinterpret_cast<uint32_t*>(smem + STAGES * STAGE + 256 + SCALES);
  int* most_rests = reinterpret_cast<int*>(smem + STAGES * STAGE + 248);
  if (threadIdx.x < WHERE / 64) reinterpret_cast<uint4*>(where)[threadIdx.x] = reinterpret_cast<const uint4*>(p.l_rests.where)[threadIdx.x];
  int no_fit = 0, most = 0;
  for (int e = threadIdx.x; e < p.experts; e += THREADS) {
    const Fit f = p.fit[e];
    no_fit |= f.bad;
    most = max(most, f.most);
  }
  if (threadIdx.x == 0) *most_rests = 0;
  __syncthreads();
  if (most > 0) atomicMax(most_rests, most);
  if (__syncthreads_or(no_fit)) {         // every CTA comes to the same: nothing has been set up yet
    if (threadIdx.x == 0) p.plan->flag = 1;
    return;
  }
  const int tiles_l = (p.lanes + 2 * BM - 1) / (2 * BM);
  const int n_units = (p.weights ? p.experts * ((p.cols + BN - 1) / BN) : p.plan->tiles) * tiles_l;

  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + STAGES), bar_filled = smem_u32(bars + 2 * STAGES),
                 bar_drained = bar_filled + 16, bar_retired = bar_filled + 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 2);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_filled + 8 * b, 1);
      mbar_init(bar_drained + 8 * b, 2 * EPI_WARPS);
    }
    mbar_init(bar_retired, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == EPI_WARPS + 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish_pair();
  }
  if (lane == 0 && warp == EPI_WARPS) { tma_prefetch_desc(&tmL); tma_prefetch_desc(&tmLlo); }
  if (lane == 0 && warp == EPI_WARPS + 2) { tma_prefetch_desc(&tmR); tma_prefetch_desc(&tmRlo); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();     // the peer's barriers exist before anything is signalled across the pair
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Registers: 384 threads are launched with 168 each; an epilogue thread holds 128 accumulators and wants more than the
  // 40 that leaves, and the third warpgroup needs few: 2 x 216 + 72 = 3 x 168.
  if (warp >= EPI_WARPS) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == EPI_WARPS || warp == EPI_WARPS + 2) {
    // ---------------- TMA producers (each CTA, its own tiles) ----------------
    if (lane == 0) {
      const bool is_l = warp == EPI_WARPS;
      const CUtensorMap* hi_map = is_l ? &tmL : &tmR;
      const CUtensorMap* lo_map = is_l ? &tmLlo : &tmRlo;
      const uint32_t tile_off = is_l ? 0u : (uint32_t)L_TILE;
      const uint32_t leader_full = mapa(bar_full, 0);
      long long issued = 0;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const bool withhold = (p.status[3] & 1) != 0;     // host-injected fault: arm nothing, load nothing
      for (int unit = cluster_id; ok && unit < n_units; unit += n_clusters) {
        const Unit u = unit_of(p, unit, entry_of(p, unit, n_units));
        const int n_half = (u.cols + 31) / 32 * 16;     // columns of the pair's MMA that this CTA stages
        const int row0 = is_l ? u.l_row + (int)rank * BM : u.r0 + (int)rank * n_half;
        const int boxes = (n_half + R_BOX - 1) / R_BOX;
        const uint32_t bytes = 4u * (is_l ? (uint32_t)L_TILE : (uint32_t)(boxes * R_BOX * BK * 2));      // hi and lo, this CTA's and the peer's
        for (int i = 0; i < u.nkb; ++i) {
          if (!mbar_wait_cluster(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 500 + s)) { ok = false; break; }
          const uint32_t dst = smem_base + s * STAGE + tile_off;
          const int k0 = (u.kb + i) * BK;
          if (!withhold) {
            if (leader) mbar_arrive_expect_tx(bar_full + 8 * s, bytes);
            if (is_l && p.l_mn) {
              // [k][lane]: 64 k x 64 lanes per box; k rows behind the expert's meet zeros of the other operand
              const int k_row = u.expert * p.K + k0;
              for (int h = 0; h < 2; ++h) {
                tma_load_2d_pair(dst + h * (L_TILE / 2), hi_map, row0 + 64 * h, k_row, leader_full + 8 * s);
                tma_load_2d_pair(dst + RAW + h * (L_TILE / 2), lo_map, row0 + 64 * h, k_row, leader_full + 8 * s);
              }
            } else if (is_l) {
              tma_load_2d_pair(dst, hi_map, k0, row0, leader_full + 8 * s);
              tma_load_2d_pair(dst + RAW, lo_map, k0, row0, leader_full + 8 * s);
            } else {
              for (int h = 0; h < boxes; ++h) {
                tma_load_2d_pair(dst + h * (R_BOX * BK * 2), hi_map, k0, row0 + h * R_BOX, leader_full + 8 * s);
                tma_load_2d_pair(dst + RAW + h * (R_BOX * BK * 2), lo_map, k0, row0 + h * R_BOX, leader_full + 8 * s);
              }
            }
            ++issued;
          }
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      }
      if (leader && *abort_flag) {
        // loads in flight complete on the leader's full barriers: give them (bounded) time before leaving
        for (long long i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
          for (int spin = 0; spin < (1 << 16); ++spin)
            if (mbar_try_wait(bar_full + 8 * (int)(i % STAGES), (uint32_t)((i / STAGES) & 1))) break;
      }
    }
  } else if (warp == EPI_WARPS + 1) {
    // ---------------- MMA issuer (leader CTA only) ----------------
    if (leader && lane == 0) {
      // K-major: 128-byte rows, 8-row groups SBO apart, 32 B per k-step.  Lanes contiguous: 64-lane blocks (boxes) LBO apart,
      // 8-k groups of 128-byte rows SBO apart, 2048 B per k-step.
      const uint64_t d_a = p.l_mn ? make_smem_desc(smem_base, L_TILE / 2, 1024, SWZ_128B) : make_smem_desc(smem_base, 16, 8 * BK * 2, SWZ_128B);
      const uint32_t a_step = p.l_mn ? 2048u >> 4 : 32u >> 4;
      const uint64_t d_b = make_smem_desc(smem_base + L_TILE, 16, 8 * BK * 2, SWZ_128B);
      const uint32_t a_hiw = (uint32_t)(d_a >> 32), b_hiw = (uint32_t)(d_b >> 32);
      const uint32_t a_low0 = (uint32_t)d_a, b_low0 = (uint32_t)d_b;
      constexpr uint32_t LO_TILE = RAW >> 4, STAGE_STEP = STAGE >> 4;
      const uint32_t peer_empty = mapa(bar_empty, 1), peer_filled = mapa(bar_filled, 1);
      int s = 0;
      uint32_t ph = 0, stage_off = 0, fill = 0;            // fill: accumulator fillings so far; filling n goes to accumulator n & 1
      bool ok = true;
      Entry next = n_units > 0 ? entry_of(p, cluster_id, n_units) : Entry{0, 0, 0, 0};
      for (int unit = cluster_id; ok && unit < n_units; unit += n_clusters) {
        const Unit u = unit_of(p, unit, next);
        next = entry_of(p, unit + n_clusters, n_units);
        const uint32_t idesc = make_idesc_f16(2 * BM, (u.cols + 31) / 32 * 32, p.l_mn);
        for (int i0 = 0; ok && i0 < u.nkb; i0 += DRAIN, ++fill) {      // (a group without rows: nothing to multiply)
          const int end = min(u.nkb, i0 + DRAIN);
          const uint32_t acc = tmem_base + (fill & 1) * BN;
          // the filling before the last one must have been read out of this accumulator (the first two pass at once)
          if (!mbar_wait_cluster(bar_drained + 8 * (fill & 1), ((fill >> 1) & 1) ^ 1, abort_flag, p.status, 750)) { ok = false; break; }
          for (int i = i0; i < end; ++i) {
            if (!mbar_wait_cluster(bar_full + 8 * s, ph, abort_flag, p.status, 700 + s)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              const uint32_t al = a_low0 + stage_off + kk * a_step, bl = b_low0 + stage_off + kk * 2;
              mma_f16_pair_words(acc, al + LO_TILE, a_hiw, bl, b_hiw, idesc, (i > i0 || kk) ? 1u : 0u);
              mma_f16_pair_words(acc, al, a_hiw, bl + LO_TILE, b_hiw, idesc, 1);
              mma_f16_pair_words(acc, al, a_hiw, bl, b_hiw, idesc, 1);
            }
            mma_commit_pair(bar_empty + 8 * s);         // stage free in the leader ...
            mma_commit_pair(peer_empty + 8 * s);        // ... and in the peer
            if (++s == STAGES) { s = 0; ph ^= 1; stage_off = 0; } else { stage_off += STAGE_STEP; }
          }
          if (!ok) break;
          mma_commit_pair(bar_filled + 8 * (fill & 1));
          mma_commit_pair(peer_filled + 8 * (fill & 1));
        }
      }
      if (*abort_flag) {
        mma_commit_pair(bar_retired);
        for (int spin = 0; spin < (1 << 20); ++spin)
          if (mbar_try_wait(bar_retired, 0)) break;
      }
    }
  }
  } else {
    // ---------------- epilogue warps: this CTA's 128 lanes, 128 columns per warp ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int q = warp & 3, half = warp >> 2;
    const uint32_t leader_drained = mapa(bar_drained, 0);
    const uint32_t tmem_lane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * (BN / 2));
    float* scales = reinterpret_cast<float*>(smem + STAGES * STAGE + 256) + warp * (BN / 2);
    float acc[BN / 2];
    uint32_t fill = 0;
    bool ok = true;
    Entry next = n_units > 0 ? entry_of(p, cluster_id, n_units) : Entry{0, 0, 0, 0};
    for (int unit = cluster_id; ok && unit < n_units; unit += n_clusters) {
      const Unit u = unit_of(p, unit, next);
      next = entry_of(p, unit + n_clusters, n_units);
      const int ncc = min(BN / 2 / 32, max(0, (u.cols - half * (BN / 2) + 31) / 32));    // 32-column pieces of this thread
      const bool none = u.nkb == 0;                        // a group without rows: zeros, and no scales
      const int l = u.l0 + (int)rank * BM + q * 32 + lane, left = u.cols - half * (BN / 2);
      // the scales of this thread's lane and (spread over the warp's lanes) of its columns, requested before the wait
      const float* r_down = (p.weights ? p.r_down + (long long)u.expert * p.cols : p.r_down) + u.r0 + half * (BN / 2);
      float col_scale[BN / 2 / 32], l_scale = 1.f, b = 0.f;
#pragma unroll
      for (int cc = 0; cc < BN / 2 / 32; ++cc) col_scale[cc] = (!none && cc * 32 + lane < left) ? r_down[cc * 32 + lane] : 1.f;
      if (l < p.lanes) {
        if (!none && p.l_down) l_scale = p.l_down[(long long)u.expert * p.lanes + l];
        else if (!none) l_scale = 1.f / 16384.f;           // (2^14 of the folded scales)
        if (p.bias) b = p.bias[(long long)u.expert * p.lanes + l];
      }
      const int r_first = u.r0 + half * (BN / 2);
      auto rests_at = [&](int side, int at) {
        const int h = where_of(side, u.expert, at);
        return where[h >> 4] >> 2 * (h & 15) & 3;            // 0: none
      };
      unsigned with_rests = l < p.lanes ? rests_at(0, l) : 0u;       // (before the wait)
#pragma unroll
      for (int i = 0; i < BN / 64; ++i)
        if (i * 32 + lane < left) with_rests |= rests_at(1, r_first + i * 32 + lane);
      with_rests = __reduce_or_sync(0xffffffffu, none ? 0u : with_rests);
#pragma unroll
      for (int j = 0; j < BN / 2; ++j) acc[j] = 0.f;
#pragma unroll 1
      for (int i0 = 0; i0 < u.nkb; i0 += DRAIN, ++fill) {
        ok = mbar_wait_cluster(bar_filled + 8 * (fill & 1), (fill >> 1) & 1, abort_flag, p.status, 850);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int cc = 0; cc < BN / 2 / 32; ++cc) {
          if (cc < ncc) {
            uint32_t r[32];
            tmem_ld_32x32(tmem_lane + (fill & 1) * BN + cc * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[cc * 32 + j] += __uint_as_float(r[j]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_drained + 8 * (fill & 1));
      }
      if (!ok) break;
      // What the halves have left out, in the lanes and columns with remainders: one is at most 2^-25 and meets at most 2^15, so
      // where a sum itself is 2^8 times their number, all of them together are below 2^-18 of it (normal data: hardly anywhere
      // not).  Other pieces, and those with values below TINY, are left to add_rests_kernel, with the activation.
      bool later = (with_rests & 2) != 0;
      if (with_rests) {
        const bool of_lane = rests_at(0, l) != 0 && l < p.lanes;
        unsigned of_columns[BN / 64];
#pragma unroll
        for (int i = 0; i < BN / 64; ++i) of_columns[i] = __ballot_sync(0xffffffffu, i * 32 + lane < left && rests_at(1, r_first + i * 32 + lane) != 0);
        const float bound = 512.f * (float)*most_rests;      // (an element has those of its lane and those of its column)
        if (__any_sync(0xffffffffu, of_lane)) {
          float least = INFINITY;
#pragma unroll
          for (int j = 0; j < BN / 2; ++j) least = fminf(least, j < left ? fabsf(acc[j]) : INFINITY);
          later = later || (of_lane && least < bound);
        }
#pragma unroll
        for (int i = 0; i < BN / 64; ++i)
          if (of_columns[i]) {
#pragma unroll
            for (int j = 0; j < 32; ++j) later = later || ((of_columns[i] >> j & 1) && fabsf(acc[i * 32 + j]) < bound && l < p.lanes);
          }
        later = __any_sync(0xffffffffu, later);
        if (later && lane == 0) p.later[atomicAdd(&p.plan->later, 1)] = make_int4(u.expert, l, r_first, min(left, BN / 2));
      }
      // out of registers, while the tensor cores work on the pair's next tile
      float* c = p.C + (p.weights ? u.expert * p.c_stride : 0) + (long long)(u.r0 + half * (BN / 2)) * p.ldc + l;
      const bool live = l < p.lanes, relu = p.act == CB200_ACT_RELU && !later;
      // whole warps of whole tiles without a beta: about 9 instructions per value (24 with predicates, shuffles and the
      // three factors apart, which held the epilogue to 9 us per tile where the product takes 3)
      const bool whole = left >= BN / 2 && __all_sync(0xffffffffu, live) && p.beta == 0.f;
#pragma unroll
      for (int cc = 0; cc < BN / 2 / 32; ++cc) scales[cc * 32 + lane] = col_scale[cc];
      __syncwarp();
      auto store_whole = [&](auto with_relu) {
        constexpr bool RELU = decltype(with_relu)::value;
        float* to = c;
#pragma unroll
        for (int j0 = 0; j0 < BN / 2; j0 += 4) {
          const float4 d = *reinterpret_cast<const float4*>(scales + j0);
          float v[4] = {acc[j0] * (l_scale * d.x), acc[j0 + 1] * (l_scale * d.y), acc[j0 + 2] * (l_scale * d.z),
                        acc[j0 + 3] * (l_scale * d.w)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = fmaf(v[j], p.alpha, b);
            if (RELU) v[j] = groups::relu(v[j]);
            *to = v[j];
            to += p.ldc;
          }
        }
      };
      if (whole && relu) {
        store_whole(std::true_type{});
      } else if (whole) {
        store_whole(std::false_type{});
      } else {
        float* to = c;
#pragma unroll
        for (int j0 = 0; j0 < BN / 2; j0 += 8) {
          if (j0 < left) {
            float old[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) old[j] = 0.f;
            if (p.beta != 0.f) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (live && j0 + j < left) old[j] = to[(long long)j * p.ldc];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float v = fmaf(acc[j0 + j] * (l_scale * scales[j0 + j]), p.alpha, b);
              if (p.beta != 0.f) v += p.beta * old[j];
              if (relu) v = groups::relu(v);
              if (live && j0 + j < left) *to = v;
              to += p.ldc;
            }
          }
        }
      }
      __syncwarp();                                        // the list is rewritten for the next tile
      if (p.act > CB200_ACT_RELU && live && !later) {
        // tanh / logistic over what was just stored: a call among 128 live accumulators would spill them
        const int n = min(left, BN / 2);
#pragma unroll 1
        for (int j0 = 0; j0 < n; j0 += 8) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = j0 + j < n ? c[(long long)j * p.ldc] : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j0 + j < n) c[(long long)j * p.ldc] = apply_act_transcendental(v[j], p.act);
          c += 8 * p.ldc;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();     // neither CTA leaves (or frees TMEM) while the pair's MMAs may still touch it
  if (warp == EPI_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ---- host side -------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)f;
  });
  return fn;
}

int half_map(CUtensorMap* tm, const __half* base, long long rows, long long cols, long long pitch, int box_cols, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) { cb200_set_error("cuTensorMapEncodeTiled is not available from this driver"); return CB200_ERR_CUDA; }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { cb200_set_error("cuTensorMapEncodeTiled failed with %d", (int)r); return CB200_ERR_CUDA; }
  return CB200_OK;
}

// Launch `kernel` behind what the stream holds, set up while its predecessor ends (it waits by itself).
template <typename... P, typename... A>
int launch_next(cb200_stream* s, void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  if (e != cudaSuccess) return cb200_cuda_fail(e, "cudaLaunchKernelEx(expert product)", __FILE__, __LINE__);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

template <int RAGGED>
int split_rows(cb200_stream* s, __half* hi, __half* lo, float* down, const float* x, long long ld, long long stride, int rows_per,
               long long rows, int cols, int kp, const Plan* plan, Fit* fit, const Rests& rests, const int* begins, int experts,
               const float* fold) {
  const int rows_a_cta = cols <= 1024 ? 8 : (cols <= 4096 ? 2 : 1);
  auto* kernel = cols <= 1024 ? split_rows_kernel<32, RAGGED> : (cols <= 4096 ? split_rows_kernel<128, RAGGED> : split_rows_kernel<256, RAGGED>);
  return launch_next(s, kernel, dim3((unsigned)((rows + rows_a_cta - 1) / rows_a_cta)), 256, 0, 1, hi, lo, down, x, ld, stride, rows_per, rows,
                     cols, kp, plan, fit, rests, fold, begins, experts);
}

// `sums` (may be null): workspace for the column sums of 64-row blocks, ((rows + 63) / 64 + groups_n) x cols
int split_columns(cb200_stream* s, __half* hi, __half* lo, float* down, uint32_t* maxima, float* sums, const float* x, long long ld,
                  const Entry* table, const int* owner, int groups_n, int rows, int cols, long long kp, const Plan* plan, Fit* fit,
                  const Rests& rests) {
  const long long chunks = (rows + 63) / 64, blocks = kp / POS;
  const dim3 grid_max((unsigned)((cols + 127) / 128), (unsigned)(chunks < 65535 ? chunks : 65535));
  const bool vec = ((uintptr_t)x & 15) == 0 && ld % 4 == 0 && cols % 4 == 0;
  int rc = launch_next(s, vec ? column_max_kernel<4> : column_max_kernel<1>, grid_max, 128, 0, 1, maxima, sums, x, ld, table, groups_n, rows, cols);
  if (rc) return rc;
  return launch_next(s, split_columns_kernel, dim3((unsigned)((cols + 127) / 128), (unsigned)(blocks < 65535 ? blocks : 65535)), 256, 0, 1, hi,
                     lo, down, maxima, x, ld, table, owner, cols, kp, plan, fit, rests);
}

int launch_pair(cb200_stream* s, const __half* l_hi, const __half* l_lo, long long l_rows, long long l_cols, long long l_pitch,
                const __half* r_hi, const __half* r_lo, long long r_rows, long long r_cols, long long r_pitch, const PairArgs& a,
                long long units) {
  static std::once_flag once[64];
  static cudaError_t result[64];
  const int dev = s->device & 63;
  std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(expert_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
  if (result[dev] != cudaSuccess) return cb200_cuda_fail(result[dev], "cudaFuncSetAttribute", __FILE__, __LINE__);
  CUtensorMap tmL, tmLlo, tmR, tmRlo;
  int rc;
  const int l_box = a.l_mn ? BK : BM;                      // 64 halves wide either way
  if ((rc = half_map(&tmL, l_hi, l_rows, l_cols, l_pitch, 64, l_box)) || (rc = half_map(&tmLlo, l_lo, l_rows, l_cols, l_pitch, 64, l_box)) ||
      (rc = half_map(&tmR, r_hi, r_rows, r_cols, r_pitch, 64, R_BOX)) || (rc = half_map(&tmRlo, r_lo, r_rows, r_cols, r_pitch, 64, R_BOX)))
    return rc;
  const long long clusters = units < s->sm_count / 2 ? units : s->sm_count / 2;
  if ((rc = launch_next(s, expert_pair_kernel, dim3((unsigned)(2 * clusters)), THREADS, SMEM, 2, tmL, tmLlo, tmR, tmRlo, a))) return rc;
  return launch_next(s, add_rests_kernel, dim3((unsigned)(2 * s->sm_count)), 256, 0, 1, a);
}

// pieces of 32 lanes x 128 columns that `units` of the product consist of, which may all have to wait for their remainders
constexpr int PIECES = 2 * BM / 32 * 2;

inline long long up8(long long v) { return (v + 7) / 8 * 8; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Pieces of the stream's workspace, each on a 256-byte boundary.
struct Carve {
  char* base;
  size_t used;
  template <typename T> T* take(size_t n) {
    T* p = (T*)(base + used);
    used += up256(n * sizeof(T));
    return p;
  }
};

// Room in an expert's list of remainders for `values` of an operand: six times what normal data bring (2.4 in a million)
long long rests_room(double values) { return 64 + (long long)(values / 65536 < 4032 ? values / 65536 : 4032); }

constexpr size_t MOST_WORKSPACE = (size_t)2 << 30;

}  // namespace

// Is this product better off here?  Both sides' times by the sizes, in microseconds (the split reads and writes the operands
// once).  Measured, here / 3xTF32: 8 experts of 2048 x 1024 with 96, 256, 1024 rows each 56, 75, 122 / 60, 87, 203; 32 of 512 x
// 512 43, 56, 97 / 41, 53, 119; weight gradients of 8 experts of 1024 x 4096 with 96, 256, 512 rows 81, 107, 164 / 81, 146, 229;
// 32 of 512 x 512 52, 79, 119 / 48, 72, 134.
bool cb200_expert_f16_ok(cb200_stream* s, long long rows, long long K, long long N, long long experts) {
  if (s->opt_gemm_auto_presplit == 1) return false;
  const double l = (double)experts * N * K, r = (double)rows * K;
  if ((l + r) * 4 > (double)MOST_WORKSPACE - (64 << 20) || experts * N > 2000000000LL || experts * K > 2000000000LL) return false;
  if (s->opt_gemm_auto_presplit == 2) return true;
  const double flops = 2.0 * rows * N * K;
  // (halves that do not stay in L2 between the split and the product are read from memory)
  const double beyond = l + r > 60e6 ? l + r - 60e6 : 0.0;
  // (whole reductions: a tile of 256 x 256 takes 0.85 us per 64 values of k, fewer rows less, on a pair of SMs)
  const double even = (double)rows / experts, tiles = (double)((N + 255) / 256) * (rows / 256 + experts / 2 + 1), waves = ceil(tiles / (s->sm_count / 2));
  const double tile = K * (0.85 / 64) * (even < 256 ? even / 256 : 1.0), product = waves * tile > flops / 590e6 ? waves * tile : flops / 590e6;
  const double here = 25.0 + (l + r) * 1.7e-6 + beyond * 2.3e-6 + product, there = 15.0 + l * 1.2e-6 + flops / 120e6;
  return rows >= 96 * experts && here < there;
}
bool cb200_expert_weights_f16_ok(cb200_stream* s, long long rows, long long M, long long N, long long experts) {
  if (s->opt_gemm_auto_presplit == 1) return false;
  const double operands = (double)(rows + BK * experts) * (M + N);
  if (operands * 4 > (double)MOST_WORKSPACE - (64 << 20) || experts * (M + N) > 500000000LL) return false;
  if (s->opt_gemm_auto_presplit == 2) return true;
  const double flops = 2.0 * rows * N * M, results = (double)experts * N * M;
  const double here = 28.0 + operands * 1.85e-6 + results * 0.67e-6 + flops / 300e6, there = 12.0 + results * 1e-6 + flops / 125e6;
  return rows >= 96 * experts && here < there;
}

// The flag that the guarded 3xTF32 launch reads is returned through `guard_out`, which is left alone where there is no room for
// the workspace (CB200_ERR_NOMEM; nothing has been launched then).
int cb200_expert_rows_f16(cb200_stream* s, float* C, long long ldc, int trans_b, float alpha, const float* A, int rows, int K,
                          long long lda, const float* B, int experts, int N, long long b_stride, long long ldb, float beta,
                          const int* offsets, const float* bias, int act, const int** guard_out) {
  DeviceGuard guard(s->device);
  // the matrices' rows as they are stored: [N, K] reduces along them, [K, N] (the gradient of the input) across them
  const int l_per = trans_b ? N : K, l_cols = trans_b ? K : N;
  const long long kp = up8(K), lp = up8(l_cols), l_rows = (long long)experts * l_per;
  // (groups up to 16 times the average have room enough)
  Rests l_rests = {nullptr, nullptr, (int)rests_room((double)N * K), 0}, r_rests = {nullptr, nullptr, (int)rests_room(16.0 * rows * K / experts), 1};
  const size_t tiles = (size_t)((rows + BN - 1) / BN + (experts < rows ? experts : rows));
  const long long units = (long long)tiles * ((N + 2 * BM - 1) / (2 * BM));
  const size_t bytes = up256(sizeof(Plan)) + up256((size_t)units * PIECES * sizeof(int4)) + up256((tiles + 1) * sizeof(Entry)) + up256((size_t)experts * 4) + up256((size_t)experts * sizeof(Fit) + WHERE_BYTES) +
                       up256((size_t)experts * l_rests.cap * sizeof(Rest)) + up256((size_t)experts * r_rests.cap * sizeof(Rest)) +
                       2 * up256((size_t)l_rows * lp * 2) + 2 * up256((size_t)rows * kp * 2) + up256((size_t)l_rows * 4) +
                       up256((size_t)rows * 4);
  void* ws = nullptr;
  int rc = cb200_scratch(s, bytes, &ws);
  if (rc) return rc;
  Carve w = {(char*)ws, 0};
  Plan* plan = w.take<Plan>(1);
  *guard_out = &plan->flag;
  Entry* table = w.take<Entry>(tiles + 1);
  int* begins = w.take<int>((size_t)experts);
  char* zeroed = w.take<char>((size_t)experts * sizeof(Fit) + WHERE_BYTES);
  Fit* fit = (Fit*)zeroed;
  l_rests.where = r_rests.where = (uint32_t*)(fit + experts);
  l_rests.list = w.take<Rest>((size_t)experts * l_rests.cap);
  r_rests.list = w.take<Rest>((size_t)experts * r_rests.cap);
  __half* l_hi = w.take<__half>((size_t)l_rows * lp);
  __half* l_lo = w.take<__half>((size_t)l_rows * lp);
  __half* r_hi = w.take<__half>((size_t)rows * kp);
  __half* r_lo = w.take<__half>((size_t)rows * kp);
  float* l_down = w.take<float>((size_t)l_rows);
  float* r_down = w.take<float>((size_t)rows);
  plan_kernel<<<65, 128, 0, s->stream>>>(plan, table, nullptr, begins, offsets, experts, rows, 0, s->status_dev, (uint32_t*)zeroed,
                                                       (long long)experts * (sizeof(Fit) / 4) + WHERE_BYTES / 4);
  CB_LAUNCH_CHECK(s);
  rc = trans_b ? split_rows<0>(s, l_hi, l_lo, l_down, B, ldb, b_stride, l_per, l_rows, l_cols, (int)lp, plan, fit, l_rests, begins, experts, nullptr)
               : split_rows<3>(s, l_hi, l_lo, l_down, B, ldb, b_stride, l_per, l_rows, l_cols, (int)lp, plan, fit, l_rests, begins, experts, nullptr);
  if (rc) return rc;
  rc = trans_b ? split_rows<1>(s, r_hi, r_lo, r_down, A, lda, 0, rows, rows, K, (int)kp, plan, fit, r_rests, begins, experts, nullptr)
               : split_rows<2>(s, r_hi, r_lo, r_down, A, lda, 0, rows, rows, K, (int)kp, plan, fit, r_rests, begins, experts, l_down);
  if (rc) return rc;
  PairArgs a;
  a.later = w.take<int4>((size_t)units * PIECES);
  a.C = C; a.ldc = ldc; a.c_stride = 0; a.l_down = trans_b ? l_down : nullptr; a.r_down = r_down; a.bias = bias; a.plan = plan;
  a.fit = fit; a.l_rests = l_rests; a.r_rests = r_rests; a.l_hi = l_hi; a.l_lo = l_lo; a.r_hi = r_hi; a.r_lo = r_lo;
  a.l_expert = l_per * lp; a.l_lane = trans_b ? lp : 1; a.l_k = trans_b ? 1 : lp; a.r_pitch = kp;
  a.table = table; a.status = s->status_dev; a.lanes = N; a.cols = 0; a.K = K; a.l_mn = trans_b ? 0 : 1; a.experts = experts;
  a.weights = 0; a.act = act; a.alpha = alpha; a.beta = beta;
  return launch_pair(s, l_hi, l_lo, l_rows, l_cols, lp, r_hi, r_lo, rows, K, kp, a, units);
}

int cb200_expert_weights_f16(cb200_stream* s, float* C, long long c_stride, long long ldc, float alpha, const float* A, int rows, int M,
                             long long lda, const float* B, int N, long long ldb, int experts, float beta, const int* offsets,
                             float* bias_gradient, const int** guard_out) {
  DeviceGuard guard(s->device);
  // C_e[m, n] = sum A[r, m] B[r, n]: n in the lanes, m in the columns
  const long long kp = ((long long)rows + (BK - 1LL) * (experts < rows ? experts : rows) + BK - 1) / BK * BK;
  Rests l_rests = {nullptr, nullptr, (int)rests_room(16.0 * rows * N / experts), 0}, r_rests = {nullptr, nullptr, (int)rests_room(16.0 * rows * M / experts), 1};
  const size_t sums_n = bias_gradient ? ((size_t)(rows + 63) / 64 + experts) * M : 0;
  const long long units = (long long)experts * ((M + BN - 1) / BN) * ((N + 2 * BM - 1) / (2 * BM));
  const size_t bytes = up256(sizeof(Plan)) + up256((size_t)units * PIECES * sizeof(int4)) + up256(((size_t)experts + 1) * sizeof(Entry)) + 2 * up256((size_t)N * kp * 2) +
                       2 * up256((size_t)M * kp * 2) + up256((size_t)(kp / POS) * 4) + up256((size_t)experts * N * 4) + up256((size_t)experts * M * 4) +
                       up256(((size_t)experts * (M + N) + (size_t)experts * (sizeof(Fit) / 4)) * 4 + WHERE_BYTES) +
                       up256((size_t)experts * l_rests.cap * sizeof(Rest)) + up256((size_t)experts * r_rests.cap * sizeof(Rest)) + up256(sums_n * 4);
  void* ws = nullptr;
  int rc = cb200_scratch(s, bytes, &ws);
  if (rc) return rc;
  Carve w = {(char*)ws, 0};
  Plan* plan = w.take<Plan>(1);
  *guard_out = &plan->flag;
  Entry* table = w.take<Entry>((size_t)experts + 1);
  int* owner = w.take<int>((size_t)(kp / POS));
  __half* l_hi = w.take<__half>((size_t)N * kp);
  __half* l_lo = w.take<__half>((size_t)N * kp);
  __half* r_hi = w.take<__half>((size_t)M * kp);
  __half* r_lo = w.take<__half>((size_t)M * kp);
  float* l_down = w.take<float>((size_t)experts * N);
  float* r_down = w.take<float>((size_t)experts * M);
  // (one block, so that it is zeroed in one go)
  const size_t l_n = (size_t)experts * N, r_n = (size_t)experts * M, fit_words = (size_t)experts * (sizeof(Fit) / 4) + WHERE_BYTES / 4;
  uint32_t* zeroed = w.take<uint32_t>(l_n + r_n + fit_words);
  Fit* fit = (Fit*)zeroed;
  l_rests.where = r_rests.where = zeroed + (size_t)experts * (sizeof(Fit) / 4);
  uint32_t* l_max = zeroed + fit_words;
  uint32_t* r_max = l_max + l_n;
  l_rests.list = w.take<Rest>((size_t)experts * l_rests.cap);
  r_rests.list = w.take<Rest>((size_t)experts * r_rests.cap);
  float* sums = bias_gradient ? w.take<float>(sums_n) : nullptr;
  plan_kernel<<<129, 128, 0, s->stream>>>(plan, table, owner, nullptr, offsets, experts, rows, 1, s->status_dev, zeroed,
                                          (long long)(l_n + r_n + fit_words));
  CB_LAUNCH_CHECK(s);
  if ((rc = split_columns(s, l_hi, l_lo, l_down, l_max, nullptr, B, ldb, table, owner, experts, rows, N, kp, plan, fit, l_rests))) return rc;
  if ((rc = split_columns(s, r_hi, r_lo, r_down, r_max, sums, A, lda, table, owner, experts, rows, M, kp, plan, fit, r_rests))) return rc;
  if (bias_gradient && (rc = launch_next(s, column_sum_kernel, dim3((unsigned)((M + 127) / 128), (unsigned)experts), 128, 0, 1, bias_gradient,
                                         sums, table, M, alpha, beta)))
    return rc;
  PairArgs a;
  a.later = w.take<int4>((size_t)units * PIECES);
  a.C = C; a.ldc = ldc; a.c_stride = c_stride; a.l_down = l_down; a.r_down = r_down; a.bias = nullptr; a.plan = plan; a.fit = fit; a.table = table;
  a.status = s->status_dev; a.lanes = N; a.cols = M; a.K = 0; a.l_mn = 0; a.experts = experts; a.weights = 1; a.act = CB200_ACT_NONE;
  a.alpha = alpha; a.beta = beta;
  a.l_rests = l_rests; a.r_rests = r_rests; a.l_hi = l_hi; a.l_lo = l_lo; a.r_hi = r_hi; a.r_lo = r_lo;
  a.l_expert = 0; a.l_lane = kp; a.l_k = 1; a.r_pitch = kp;
  return launch_pair(s, l_hi, l_lo, N, kp, kp, r_hi, r_lo, M, kp, kp, a,
                     units);
}
