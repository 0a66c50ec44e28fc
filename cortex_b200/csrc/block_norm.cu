// The normalisations around a residual block, fused with its gate and the residual add.  With N(x) = x_hat,
//   rms:    x_hat = x / sqrt(mean(x^2) + eps)          layer:  x_hat = (x - mean(x)) / sqrt(mean((x - mean)^2) + eps)
// per row of cols values,
//   u      = N(block) * after_scale + after_bias       (u = block without an `after` normalisation)
//   total  = residual + residual_scale * gate * u      (total = residual without a block)
//   output = N(total) * before_scale + before_bias     (no output without a `before` normalisation)
// and, given output_gradient (dy) and total_gradient (dt, the gradient that reaches the sum by the residual path),
//   N'(x, d) = (d - x_hat * mean(d * x_hat) [- mean(d)]) / std                       [layer only]
//   residual_gradient = r = dt + N'(total, dy * before_scale)
//   gate_gradient     = sum over the rows that share the gate row of residual_scale * r * u
//   du                = residual_scale * gate * r
//   block_gradient    = N'(block, du * after_scale)     (du without an `after` normalisation)
//   {before,after}_scale_gradient = column sums of dy * N(total), du * N(block);  bias gradients: of dy, du.
// The row statistics are recomputed from the rows, which the gradients read anyway: nothing is kept between the calls.
// Sums and statistics are held in the element type (32 bits at least) as trees over a row, column sums over blocks of
// rows and then over the blocks in order: no atomics, the same bits on every run.
#include "common.cuh"
#include <math.h>
#include <initializer_list>
#include <mutex>

namespace {

enum { KIND_RMS = 0, KIND_LAYER = 1 };

template <typename T> struct Forward {
  T* out; long long ld_out;
  T* total; long long ld_total;
  const T* block; long long ld_block;
  const T* residual; long long ld_residual;
  const T* gate; const T* after_w; const T* after_b; const T* before_w; const T* before_b;
  int layer;
  T eps, scale;
  long long rows, cols, rows_per_gate;
};

template <typename T> struct Backward {
  T* block_g; long long ld_block_g;
  T* residual_g; long long ld_residual_g;
  T* gate_g; T* after_w_g; T* after_b_g; T* before_w_g; T* before_b_g;
  const T* out_g; long long ld_out_g;
  const T* total_g; long long ld_total_g;
  const T* total; long long ld_total;
  const T* block; long long ld_block;
  const T* gate; const T* after_w; const T* after_b; const T* before_w;
  int layer;
  T eps, scale;
  long long rows, cols, rows_per_gate;
};

__device__ __forceinline__ float rsqrt_of(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double rsqrt_of(double v) { return 1.0 / sqrt(v); }

constexpr int WIDE_THREADS = 512;

// sums over the CTA of two values at once; every thread gets both
template <typename T>
__device__ __forceinline__ void block_sum2(T& a, T& b) {
  __shared__ T part[2][WIDE_THREADS / 32];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, d);
    b += __shfl_xor_sync(0xffffffffu, b, d);
  }
  if ((threadIdx.x & 31) == 0) { part[0][threadIdx.x >> 5] = a; part[1][threadIdx.x >> 5] = b; }
  __syncthreads();
  a = part[0][0];
  b = part[1][0];
#pragma unroll
  for (int w = 1; w < WIDE_THREADS / 32; ++w) { a += part[0][w]; b += part[1][w]; }
  __syncthreads();
}

// mean and 1 / std of the n values f(0) .. f(n - 1)
template <typename T, typename F>
__device__ __forceinline__ void row_stats(F f, long long n, int layer, T eps, T& mean, T& rstd) {
  mean = (T)0;
  if (layer) {
    T s = (T)0, unused = (T)0;
    for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) s += f(i);
    block_sum2(s, unused);
    mean = s / (T)n;
  }
  T q = (T)0, unused = (T)0;
  for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) { const T v = f(i) - mean; q += v * v; }
  block_sum2(q, unused);
  rstd = rsqrt_of(q / (T)n + eps);
}

// ---- rows of any width: one CTA per row, the row read again for every pass over it ---------------------------------
template <typename T>
__global__ void __launch_bounds__(WIDE_THREADS) forward_wide_kernel(Forward<T> p) {
  const long long r = blockIdx.x, n = p.cols;
  const T* x = p.block ? p.block + r * p.ld_block : nullptr;
  const T* res = p.residual + r * p.ld_residual;
  const T* gate = p.gate ? p.gate + (r / p.rows_per_gate) * n : nullptr;
  T* total = p.total ? p.total + r * p.ld_total : nullptr;
  T mean_a = (T)0, rstd_a = (T)1;
  if (x && p.after_w) row_stats([&](long long i) { return x[i]; }, n, p.layer, p.eps, mean_a, rstd_a);
  if (x) {
    for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) {
      T u = x[i];
      if (p.after_w) u = (u - mean_a) * rstd_a * p.after_w[i] + (p.after_b ? p.after_b[i] : (T)0);
      if (gate) u *= gate[i];
      total[i] = res[i] + p.scale * u;
    }
  } else if (total && total != res) {
    for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) total[i] = res[i];
  }
  if (!p.out) return;
  const T* h = total ? total : res;                 // each thread reads back what it wrote itself
  T mean, rstd;
  row_stats([&](long long i) { return h[i]; }, n, p.layer, p.eps, mean, rstd);
  T* out = p.out + r * p.ld_out;
  for (long long i = threadIdx.x; i < n; i += WIDE_THREADS)
    out[i] = (h[i] - mean) * rstd * p.before_w[i] + (p.before_b ? p.before_b[i] : (T)0);
}

// stats: per row mean and 1 / std of total, then of block (for the column sums)
template <typename T>
__global__ void __launch_bounds__(WIDE_THREADS) backward_wide_kernel(Backward<T> p, T* stats) {
  const long long r = blockIdx.x, n = p.cols;
  const T* h = p.total ? p.total + r * p.ld_total : nullptr;
  const T* dy = p.out_g ? p.out_g + r * p.ld_out_g : nullptr;
  const T* dt = p.total_g ? p.total_g + r * p.ld_total_g : nullptr;
  const T* x = p.block ? p.block + r * p.ld_block : nullptr;
  const long long g = r / p.rows_per_gate;
  const T* gate = p.gate ? p.gate + g * n : nullptr;
  T* rg = p.residual_g + r * p.ld_residual_g;
  T mean = (T)0, rstd = (T)1, dot = (T)0, sum = (T)0;
  if (dy) {
    row_stats([&](long long i) { return h[i]; }, n, p.layer, p.eps, mean, rstd);
    for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) {
      const T d = dy[i] * p.before_w[i];
      dot += d * ((h[i] - mean) * rstd);
      sum += d;
    }
    block_sum2(dot, sum);
    dot /= (T)n;
    sum = p.layer ? sum / (T)n : (T)0;
  }
  for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) {
    T v = dt ? dt[i] : (T)0;
    if (dy) v += (dy[i] * p.before_w[i] - (h[i] - mean) * rstd * dot - sum) * rstd;
    rg[i] = v;
  }
  T mean_a = (T)0, rstd_a = (T)1;
  if (x) {
    T* xg = p.block_g + r * p.ld_block_g;
    T* gg = (p.gate_g && p.rows_per_gate == 1) ? p.gate_g + g * n : nullptr;
    if (p.after_w) row_stats([&](long long i) { return x[i]; }, n, p.layer, p.eps, mean_a, rstd_a);
    T dot_a = (T)0, sum_a = (T)0;
    for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) {
      const T s = p.scale * rg[i];
      const T hat = (x[i] - mean_a) * rstd_a;
      T du = gate ? s * gate[i] : s;
      if (gg) gg[i] = s * (p.after_w ? hat * p.after_w[i] + (p.after_b ? p.after_b[i] : (T)0) : x[i]);
      if (p.after_w) {
        du *= p.after_w[i];
        dot_a += du * hat;
        sum_a += du;
      } else {
        xg[i] = du;
      }
    }
    if (p.after_w) {
      block_sum2(dot_a, sum_a);
      dot_a /= (T)n;
      sum_a = p.layer ? sum_a / (T)n : (T)0;
      for (long long i = threadIdx.x; i < n; i += WIDE_THREADS) {
        const T du = p.scale * rg[i] * (gate ? gate[i] : (T)1) * p.after_w[i];
        xg[i] = (du - (x[i] - mean_a) * rstd_a * dot_a - sum_a) * rstd_a;
      }
    }
  }
  if (threadIdx.x == 0) {
    stats[4 * r] = mean;
    stats[4 * r + 1] = rstd;
    stats[4 * r + 2] = mean_a;
    stats[4 * r + 3] = rstd_a;
  }
}

// ---- column sums: blocks of consecutive rows, then the blocks in order -----------------------------------------------
// Row block b of P covers rows [b * rows / P, (b + 1) * rows / P).  The rows that share a gate row may start and end
// inside blocks: a group that lies in one block is summed there; of the others every block keeps at most two partial
// rows, the one that begins at the block's first row in slot 2b and the one that begins later in slot 2b + 1.
__host__ __device__ inline long long block_begin(long long rows, int blocks, int b) { return rows * b / blocks; }
__host__ __device__ inline int block_of(long long rows, int blocks, long long r) {
  int b = (int)(((r + 1) * blocks - 1) / rows);          // the largest b with rows * b / blocks <= r
  return b;
}

enum { SUM_BEFORE_W = 0, SUM_BEFORE_B = 1, SUM_AFTER_W = 2, SUM_AFTER_B = 3, SUMS = 4 };

// parts: [blocks][SUMS][cols], gate_parts: [2 * blocks][cols]
template <typename T>
__global__ void __launch_bounds__(128) column_sums_kernel(Backward<T> p, const T* stats, T* parts, T* gate_parts, int blocks) {
  const long long c = (long long)blockIdx.x * 128 + threadIdx.x;
  if (c >= p.cols) return;
  const int b = blockIdx.y;
  const long long r0 = block_begin(p.rows, blocks, b), r1 = block_begin(p.rows, blocks, b + 1);
  const bool gates = p.gate_g && p.rows_per_gate > 1;
  const T aw = p.after_w ? p.after_w[c] : (T)1, ab = p.after_b ? p.after_b[c] : (T)0;
  T s[SUMS] = {(T)0, (T)0, (T)0, (T)0};
  T gs = (T)0;
  // the rows that share a gate row make a segment; without such groups the whole block does
  const long long per = p.rows_per_gate;
  const bool grouped = p.gate && per > 1;
  const long long gate_step = p.gate && per == 1 ? p.cols : 0;
  for (long long r = r0; r < r1;) {
    const long long g = grouped ? r / per : 0, end = grouped ? (g + 1) * per : r1, stop = end < r1 ? end : r1;
    const T* gate = p.gate ? p.gate + (grouped ? g : (per == 1 ? r : 0)) * p.cols + c : nullptr;
    const long long first = r;
#pragma unroll 4
    for (; r < stop; ++r) {
      if (p.out_g) {
        const T dy = p.out_g[r * p.ld_out_g + c];
        s[SUM_BEFORE_W] += dy * ((p.total[r * p.ld_total + c] - stats[4 * r]) * stats[4 * r + 1]);
        s[SUM_BEFORE_B] += dy;
      }
      if (p.block) {
        const T d = p.scale * p.residual_g[r * p.ld_residual_g + c];
        const T x = p.block[r * p.ld_block + c];
        const T hat = (x - stats[4 * r + 2]) * stats[4 * r + 3];
        const T du = gate ? d * gate[(r - first) * gate_step] : d;
        s[SUM_AFTER_W] += du * hat;
        s[SUM_AFTER_B] += du;
        gs += d * (p.after_w ? hat * aw + ab : x);
      }
    }
    if (gates) {
      const bool whole = first == g * per && r == end;
      T* to = whole ? p.gate_g + g * p.cols : gate_parts + (2LL * b + (first != r0)) * p.cols;
      to[c] = gs;
    }
    gs = (T)0;
  }
#pragma unroll
  for (int k = 0; k < SUMS; ++k) parts[((long long)b * SUMS + k) * p.cols + c] = s[k];
}

// The sum over n rows first, first + pitch, ... of one column: COLUMNS columns x blockDim.x / COLUMNS threads each, added in order.
template <typename T, int COLUMNS, int THREADS>
__device__ __forceinline__ void add_rows(const T* first, long long pitch, int n, T* to, bool live) {
  constexpr int DEEP = THREADS / COLUMNS;
  __shared__ T part[DEEP][COLUMNS + 1];
  const int tx = threadIdx.x % COLUMNS, ty = threadIdx.x / COLUMNS;
  const int a = (int)((long long)n * ty / DEEP), z = (int)((long long)n * (ty + 1) / DEEP);
  T s = (T)0;
  if (live) {
#pragma unroll 8
    for (int i = a; i < z; ++i) s += first[(long long)i * pitch];
  }
  __syncthreads();
  part[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && live) {
#pragma unroll
    for (int i = 1; i < DEEP; ++i) s += part[i][tx];
    *to = s;
  }
}

// blockIdx.y: a scale's or bias's gradient
template <typename T>
__global__ void __launch_bounds__(1024) column_finish_kernel(Backward<T> p, const T* parts, int blocks) {
  const long long c = (long long)blockIdx.x * 32 + (threadIdx.x & 31);
  const int k = blockIdx.y;
  T* to = k == SUM_BEFORE_W ? p.before_w_g : (k == SUM_BEFORE_B ? p.before_b_g : (k == SUM_AFTER_W ? p.after_w_g : p.after_b_g));
  if (to) add_rows<T, 32, 1024>(parts + (long long)k * p.cols + c, (long long)SUMS * p.cols, blocks, to + c, c < p.cols);
}

// The gate groups that more than one row block has a part of: the first part may be in the second slot of its block, the
// others are in first slots.  As many threads to a column as there are parts to add (64 groups of 2500 columns over 296 row
// blocks, five parts each: with 32 threads to a column, most of them idle, this took 25 us of 33 for the column sums).
template <typename T, int COLUMNS>
__global__ void __launch_bounds__(256) gate_finish_kernel(Backward<T> p, const T* gate_parts, int blocks) {
  const long long c = (long long)blockIdx.x * COLUMNS + threadIdx.x % COLUMNS, groups = p.rows / p.rows_per_gate;
  for (long long g = blockIdx.y; g < groups; g += gridDim.y) {
    const long long first = g * p.rows_per_gate, last = first + p.rows_per_gate - 1;
    const int b0 = block_of(p.rows, blocks, first), b1 = block_of(p.rows, blocks, last);
    if (b0 == b1) continue;
    T* to = p.gate_g + g * p.cols + c;
    add_rows<T, COLUMNS, 256>(gate_parts + 2LL * (b0 + 1) * p.cols + c, 2 * p.cols, b1 - b0, to, c < p.cols);
    if (threadIdx.x < COLUMNS && c < p.cols) *to += gate_parts[(2LL * b0 + (first != block_begin(p.rows, blocks, b0))) * p.cols + c];
  }
}

// ---- rows that fit a CTA's registers: every operand is read once --------------------------------------------------
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T e[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> ld_pack(const T* p) { return *reinterpret_cast<const Pack<T, VEC>*>(p); }
template <typename T, int VEC> __device__ __forceinline__ void st_pack(T* p, const Pack<T, VEC>& v) { *reinterpret_cast<Pack<T, VEC>*>(p) = v; }

// Sums of N values over the threads of a row; every thread gets them.  The values are folded together (each step of the
// butterfly halves their number: 2^M - 1 + 5 - M shuffles for 2^M values instead of 5 each), the warps' sums go through `part`
// (2^M x 32), each warp adds those up for itself: one barrier; consecutive calls must use different halves of the buffer.
template <int N> struct Log2Up { static constexpr int value = N <= 1 ? 0 : 1 + Log2Up<(N + 1) / 2>::value; };
template <> struct Log2Up<1> { static constexpr int value = 0; };
template <typename T, int N>
__device__ __forceinline__ void row_sums(T (&v)[N], T* part, int warps) {
  constexpr int M = Log2Up<N>::value, G = 32 >> M;         // G lanes end up with the sum of one value
  const int lane = threadIdx.x & 31;
  T w[1 << M];
#pragma unroll
  for (int k = 0; k < (1 << M); ++k) w[k] = k < N ? v[k < N ? k : 0] : (T)0;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const int half = (1 << M) >> (m + 1), d = 16 >> m;
    const bool up = (lane & d) != 0;
#pragma unroll
    for (int k = 0; k < half; ++k) {
      const T give = up ? w[k] : w[k + half], keep = up ? w[k + half] : w[k];
      w[k] = keep + __shfl_xor_sync(0xffffffffu, give, d);
    }
  }
#pragma unroll
  for (int d = G >> 1; d > 0; d >>= 1) w[0] += __shfl_xor_sync(0xffffffffu, w[0], d);
  if (warps > 1) {
    if ((lane & (G - 1)) == 0) part[(lane / G) * 32 + (threadIdx.x >> 5)] = w[0];
    __syncthreads();
    const T* mine = part + (lane / G) * 32;
    T s = (lane & (G - 1)) < warps ? mine[lane & (G - 1)] : (T)0;
    if (warps > G)
      for (int i = (lane & (G - 1)) + G; i < warps; i += G) s += mine[i];
#pragma unroll
    for (int d = G >> 1; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    w[0] = s;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = __shfl_sync(0xffffffffu, w[0], k * G);
}

// blockDim.x threads per row, ITEMS packs of VEC values each; blockDim.y rows per CTA where a warp holds a row
template <typename T, int VEC, int ITEMS>
__global__ void __launch_bounds__(1024) forward_rows_kernel(Forward<T> p) {
  __shared__ T part[2][32];
  const long long r = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (r >= p.rows) return;                                 // whole warps: blockDim.y > 1 only with a warp per row
  const int n = (int)p.cols, warps = blockDim.x >> 5, step = blockDim.x * VEC, c0 = threadIdx.x * VEC;
  const T inv_n = (T)1 / (T)n;
  const T* res = p.residual + r * p.ld_residual;
  const T* x = p.block ? p.block + r * p.ld_block : nullptr;
  const T* gate = p.gate ? p.gate + (r / p.rows_per_gate) * n : nullptr;
  Pack<T, VEC> h[ITEMS], u[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = c0 + i * step;
#pragma unroll
    for (int e = 0; e < VEC; ++e) { h[i].e[e] = (T)0; u[i].e[e] = (T)0; }
    if (c < n) {
      h[i] = ld_pack<T, VEC>(res + c);
      if (x) u[i] = ld_pack<T, VEC>(x + c);
    }
  }
  int turn = 0;
  // mean and 1 / std of values held in registers (positions behind the row hold zeros)
  auto stats = [&](const Pack<T, VEC> (&v)[ITEMS], T& mean, T& rstd) {
    mean = (T)0;
    if (p.layer) {
      T s[1] = {(T)0};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0] += v[i].e[e];
      row_sums<T, 1>(s, part[turn], warps);
      turn ^= 1;
      mean = s[0] * inv_n;
    }
    T q[1] = {(T)0};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (c0 + i * step < n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const T d = v[i].e[e] - mean; q[0] += d * d; }
    row_sums<T, 1>(q, part[turn], warps);
    turn ^= 1;
    rstd = rsqrt_of(q[0] * inv_n + p.eps);
  };
  if (x) {
    if (p.after_w) {
      T mean, rstd;
      stats(u, mean, rstd);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = c0 + i * step;
        if (c < n) {
          const Pack<T, VEC> w = ld_pack<T, VEC>(p.after_w + c);
          Pack<T, VEC> b;
          if (p.after_b) b = ld_pack<T, VEC>(p.after_b + c);
#pragma unroll
          for (int e = 0; e < VEC; ++e) u[i].e[e] = (u[i].e[e] - mean) * rstd * w.e[e] + (p.after_b ? b.e[e] : (T)0);
        }
      }
    }
    T* total = p.total + r * p.ld_total;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * step;
      if (c < n) {
        Pack<T, VEC> g;
        if (gate) g = ld_pack<T, VEC>(gate + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] += p.scale * (gate ? g.e[e] * u[i].e[e] : u[i].e[e]);
        st_pack<T, VEC>(total + c, h[i]);
      }
    }
  } else if (p.total) {
    T* total = p.total + r * p.ld_total;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (c0 + i * step < n) st_pack<T, VEC>(total + c0 + i * step, h[i]);
  }
  if (!p.out) return;
  T mean, rstd;
  stats(h, mean, rstd);
  T* out = p.out + r * p.ld_out;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = c0 + i * step;
    if (c < n) {
      const Pack<T, VEC> w = ld_pack<T, VEC>(p.before_w + c);
      Pack<T, VEC> b, y;
      if (p.before_b) b = ld_pack<T, VEC>(p.before_b + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) y.e[e] = (h[i].e[e] - mean) * rstd * w.e[e] + (p.before_b ? b.e[e] : (T)0);
      st_pack<T, VEC>(out + c, y);
    }
  }
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <int BYTES> __device__ __forceinline__ void copy_async(void* smem, const void* g) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(smem);
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(g) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(g), "n"(BYTES) : "memory");
}

// The gradients in one pass: a CTA takes a block of consecutive rows; the next row's operands are on their way into shared
// memory (cp.async; every thread copies what it will read itself, so there is no barrier for data) while a row is worked
// on, and the column sums of its rows stay in registers.  What bounds it is the issue rate: a row's reductions (three for
// rms, four for layer) cost a warp as much as 60 of its values, so a thread takes 8 values (with 4, and the reduction for
// the block's normalisation folded into the other one by linearity -- ten sums at once -- 8192 rows of 2500 took 290 us).
template <typename T, int VEC, int ITEMS, bool LAYER, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT <= 320 ? 2 : 1) backward_rows_kernel(Backward<T> p, T* parts, T* gate_parts, int blocks) {
  constexpr int STAGES = 2;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ T part[2][2 * 32];
  T* const data = reinterpret_cast<T*>(smem_raw);
  const int n = (int)p.cols, warps = blockDim.x >> 5, step = blockDim.x * VEC, c0 = threadIdx.x * VEC;
  const int slot = step * ITEMS;                           // elements of one operand's row in shared memory
  const T inv_n = (T)1 / (T)n;
  const int b = blockIdx.x, per_gate = (int)p.rows_per_gate;
  const int r0 = (int)block_begin(p.rows, blocks, b), r1 = (int)block_begin(p.rows, blocks, b + 1);
  const bool has_y = p.out_g != nullptr, has_t = p.total_g != nullptr, has_x = p.block != nullptr, has_a = p.after_w != nullptr;
  const bool has_g = p.gate != nullptr, gates = p.gate_g && per_gate > 1, gate_rows = p.gate_g && per_gate == 1;

  auto request = [&](int r) {
    if (r < r1) {
      T* to = data + ((r - r0) & 1) * 4 * slot;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = c0 + i * step;
        if (c < n) {
          if (has_y) {
            copy_async<VEC * (int)sizeof(T)>(to + c, p.total + (long long)r * p.ld_total + c);
            copy_async<VEC * (int)sizeof(T)>(to + slot + c, p.out_g + (long long)r * p.ld_out_g + c);
          }
          if (has_t) copy_async<VEC * (int)sizeof(T)>(to + 2 * slot + c, p.total_g + (long long)r * p.ld_total_g + c);
          if (has_x) copy_async<VEC * (int)sizeof(T)>(to + 3 * slot + c, p.block + (long long)r * p.ld_block + c);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  request(r0);

  Pack<T, VEC> sw[ITEMS], sb[ITEMS], aw[ITEMS], ab[ITEMS], gs[ITEMS];      // column sums of this block's rows
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) sw[i].e[e] = sb[i].e[e] = aw[i].e[e] = ab[i].e[e] = gs[i].e[e] = (T)0;
  int g = r0 / per_gate, g_left = (g + 1) * per_gate - r0;                 // gate row, rows it still serves
  bool g_whole = g * per_gate == r0;                       // this block has had the group's rows from its first one on
  int turn = 0, slot_b = 0;                                // slot_b: 1 once the block's first group is over

  for (int r = r0; r < r1; ++r) {
    request(r + 1);                                        // into the stage that the row before this one was read from
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const T* from = data + ((r - r0) & 1) * 4 * slot;
    Pack<T, VEC> h[ITEMS], y[ITEMS], x[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * step;
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i].e[e] = y[i].e[e] = x[i].e[e] = (T)0;
      if (c < n) {
        if (has_y) { h[i] = ld_pack<T, VEC>(from + c); y[i] = ld_pack<T, VEC>(from + slot + c); }
        if (has_x) x[i] = ld_pack<T, VEC>(from + 3 * slot + c);
      }
    }
    // ---- statistics of both rows
    T m[2] = {(T)0, (T)0};
    if (LAYER) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) { m[0] += h[i].e[e]; m[1] += x[i].e[e]; }
      row_sums<T, 2>(m, part[turn ^= 1], warps);
      m[0] *= inv_n;
      m[1] = has_a ? m[1] * inv_n : (T)0;
    }
    T q[2] = {(T)0, (T)0};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (c0 + i * step < n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          h[i].e[e] -= m[0];
          x[i].e[e] -= m[1];
          q[0] += h[i].e[e] * h[i].e[e];
          q[1] += x[i].e[e] * x[i].e[e];
        }
    row_sums<T, 2>(q, part[turn ^= 1], warps);
    const T rstd = has_y ? rsqrt_of(q[0] * inv_n + p.eps) : (T)0, rstd_a = has_a ? rsqrt_of(q[1] * inv_n + p.eps) : (T)1;
    // ---- through the normalisation before the next block: h becomes h_hat, then r
    T s[2] = {(T)0, (T)0};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * step;
      if (c < n) {
        Pack<T, VEC> w;
        if (has_y) w = ld_pack<T, VEC>(p.before_w + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          h[i].e[e] *= rstd;
          x[i].e[e] *= rstd_a;
          sw[i].e[e] += y[i].e[e] * h[i].e[e];
          sb[i].e[e] += y[i].e[e];
          if (has_y) y[i].e[e] *= w.e[e];
          s[0] += y[i].e[e] * h[i].e[e];
          if (LAYER) s[1] += y[i].e[e];
        }
      }
    }
    if (LAYER) row_sums<T, 2>(s, part[turn ^= 1], warps);
    else row_sums<T, 1>(reinterpret_cast<T(&)[1]>(s), part[turn ^= 1], warps);
    const T m1 = s[0] * inv_n, m2 = s[1] * inv_n;
    // ---- through the gate and the normalisation after the block
    --g_left;
    const bool flush = gates && (g_left == 0 || r + 1 == r1);
    T a[2] = {(T)0, (T)0};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * step;
      if (c >= n) continue;
      if (has_t) {
        const Pack<T, VEC> t = ld_pack<T, VEC>(from + 2 * slot + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] = t.e[e] + (y[i].e[e] - h[i].e[e] * m1 - m2) * rstd;
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] = (y[i].e[e] - h[i].e[e] * m1 - m2) * rstd;
      }
      st_pack<T, VEC>(p.residual_g + (long long)r * p.ld_residual_g + c, h[i]);
      if (!has_x) continue;
      Pack<T, VEC> w, wb, ga;
      if (has_a) w = ld_pack<T, VEC>(p.after_w + c);
      if (has_g) ga = ld_pack<T, VEC>(p.gate + (long long)g * n + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i].e[e] *= p.scale;                  // scale * r
      if (p.gate_g) {
        if (p.after_b) wb = ld_pack<T, VEC>(p.after_b + c);
        Pack<T, VEC> u;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          u.e[e] = x[i].e[e];
          if (has_a) u.e[e] = u.e[e] * w.e[e] + (p.after_b ? wb.e[e] : (T)0);
          u.e[e] *= h[i].e[e];
          gs[i].e[e] += u.e[e];
        }
        if (gate_rows) st_pack<T, VEC>(p.gate_g + (long long)g * n + c, u);
        if (flush) {
          T* to = g_whole && g_left == 0 ? p.gate_g + (long long)g * n : gate_parts + (2LL * b + slot_b) * n;
          st_pack<T, VEC>(to + c, gs[i]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) gs[i].e[e] = (T)0;
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (has_g) h[i].e[e] *= ga.e[e];                                   // du
        if (has_a) {
          aw[i].e[e] += h[i].e[e] * x[i].e[e];
          ab[i].e[e] += h[i].e[e];
          h[i].e[e] *= w.e[e];
          a[0] += h[i].e[e] * x[i].e[e];
          if (LAYER) a[1] += h[i].e[e];
        }
      }
      if (!has_a) st_pack<T, VEC>(p.block_g + (long long)r * p.ld_block_g + c, h[i]);
    }
    if (has_x && has_a) {
      if (LAYER) row_sums<T, 2>(a, part[turn ^= 1], warps);
      else row_sums<T, 1>(reinterpret_cast<T(&)[1]>(a), part[turn ^= 1], warps);
      a[0] *= inv_n;
      a[1] *= inv_n;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = c0 + i * step;
        if (c >= n) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] = (h[i].e[e] - x[i].e[e] * a[0] - a[1]) * rstd_a;
        st_pack<T, VEC>(p.block_g + (long long)r * p.ld_block_g + c, h[i]);
      }
    }
    if (g_left == 0) {
      ++g;
      g_left = per_gate;
      g_whole = true;
      slot_b = 1;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = c0 + i * step;
    if (c >= n) continue;
    T* to = parts + (long long)b * SUMS * n + c;
    if (p.before_w_g) st_pack<T, VEC>(to + (long long)SUM_BEFORE_W * n, sw[i]);
    if (p.before_b_g) st_pack<T, VEC>(to + (long long)SUM_BEFORE_B * n, sb[i]);
    if (p.after_w_g) st_pack<T, VEC>(to + (long long)SUM_AFTER_W * n, aw[i]);
    if (p.after_b_g) st_pack<T, VEC>(to + (long long)SUM_AFTER_B * n, ab[i]);
  }
}

// Rows too wide for that: the row in registers, read once; the column sums of the CTA's rows in shared memory, where every
// thread adds to its own columns only (no barrier).  The next row is asked for into L2 while a row is worked on.  4097 to 8192
// fp32 columns; 5286 rows of 6564 254 us, where a pass over the rows and one over the columns took 480 (127 at HBM's rate).
template <typename T, int VEC, int ITEMS, bool LAYER>
__global__ void __launch_bounds__(1024) backward_hold_kernel(Backward<T> p, T* parts, T* gate_parts, int blocks) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ T part[2][2 * 32];
  const int n = (int)p.cols, warps = blockDim.x >> 5, step = blockDim.x * VEC, c0 = threadIdx.x * VEC, slot = step * ITEMS;
  T* const sums = reinterpret_cast<T*>(smem_raw);          // before_w, before_b, after_w, after_b, gate: [5][slot]
  const T inv_n = (T)1 / (T)n;
  const int b = blockIdx.x, per_gate = (int)p.rows_per_gate;
  const int r0 = (int)block_begin(p.rows, blocks, b), r1 = (int)block_begin(p.rows, blocks, b + 1);
  const bool has_y = p.out_g != nullptr, has_x = p.block != nullptr, has_a = p.after_w != nullptr;
  const bool gates = p.gate_g && per_gate > 1, gate_rows = p.gate_g && per_gate == 1;
  const Pack<T, VEC> zero = {};
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int k = 0; k <= SUMS; ++k) st_pack<T, VEC>(sums + k * slot + c0 + i * step, zero);
  int g = r0 / per_gate, g_left = (g + 1) * per_gate - r0;                 // gate row, rows it still serves
  bool g_whole = g * per_gate == r0;                       // this block has had the group's rows from its first one on
  int turn = 0, slot_b = 0;                                // slot_b: 1 once the block's first group is over

#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    Pack<T, VEC> h[ITEMS], y[ITEMS], x[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * step;
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[i].e[e] = y[i].e[e] = x[i].e[e] = (T)0;
      if (c < n) {
        if (has_y) { h[i] = ld_pack<T, VEC>(p.total + (long long)r * p.ld_total + c); y[i] = ld_pack<T, VEC>(p.out_g + (long long)r * p.ld_out_g + c); }
        if (has_x) x[i] = ld_pack<T, VEC>(p.block + (long long)r * p.ld_block + c);
        if (r + 1 < r1 && (threadIdx.x * VEC * (int)sizeof(T)) % 128 == 0) {
          const long long q = r + 1;
          if (has_y) { prefetch_l2(p.total + q * p.ld_total + c); prefetch_l2(p.out_g + q * p.ld_out_g + c); }
          if (has_x) prefetch_l2(p.block + q * p.ld_block + c);
          if (p.total_g) prefetch_l2(p.total_g + q * p.ld_total_g + c);
        }
      }
    }
    T m[2] = {(T)0, (T)0}, q[2] = {(T)0, (T)0}, d[2] = {(T)0, (T)0}, a[2] = {(T)0, (T)0};
    if (LAYER) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) { m[0] += h[i].e[e]; m[1] += x[i].e[e]; }
      row_sums<T, 2>(m, part[turn ^= 1], warps);
      m[0] *= inv_n;
      m[1] = has_a ? m[1] * inv_n : (T)0;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (c0 + i * step < n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          h[i].e[e] -= m[0];
          x[i].e[e] -= m[1];
          q[0] += h[i].e[e] * h[i].e[e];
          q[1] += x[i].e[e] * x[i].e[e];
        }
    row_sums<T, 2>(q, part[turn ^= 1], warps);
    const T rstd = has_y ? rsqrt_of(q[0] * inv_n + p.eps) : (T)1, rstd_a = has_a ? rsqrt_of(q[1] * inv_n + p.eps) : (T)1;
    if (has_y) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = c0 + i * step;
        if (c >= n) continue;
        const Pack<T, VEC> w = ld_pack<T, VEC>(p.before_w + c);
        Pack<T, VEC> sw = ld_pack<T, VEC>(sums + SUM_BEFORE_W * slot + c), sb = ld_pack<T, VEC>(sums + SUM_BEFORE_B * slot + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          h[i].e[e] *= rstd;
          sw.e[e] += y[i].e[e] * h[i].e[e];
          sb.e[e] += y[i].e[e];
          y[i].e[e] *= w.e[e];
          d[0] += y[i].e[e] * h[i].e[e];
          if (LAYER) d[1] += y[i].e[e];
        }
        st_pack<T, VEC>(sums + SUM_BEFORE_W * slot + c, sw);
        st_pack<T, VEC>(sums + SUM_BEFORE_B * slot + c, sb);
      }
      row_sums<T, 2>(d, part[turn ^= 1], warps);
      d[0] *= inv_n;
      d[1] *= inv_n;
    }
    --g_left;
    const bool flush = gates && (g_left == 0 || r + 1 == r1);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = c0 + i * step;
      if (c >= n) continue;
      if (has_y)
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] = (y[i].e[e] - h[i].e[e] * d[0] - d[1]) * rstd;
      if (p.total_g) {
        const Pack<T, VEC> t = ld_pack<T, VEC>(p.total_g + (long long)r * p.ld_total_g + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] += t.e[e];
      }
      st_pack<T, VEC>(p.residual_g + (long long)r * p.ld_residual_g + c, h[i]);
      if (!has_x) continue;
      Pack<T, VEC> w, wb, ga;
      if (has_a) w = ld_pack<T, VEC>(p.after_w + c);
      if (p.gate) ga = ld_pack<T, VEC>(p.gate + (long long)g * n + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        h[i].e[e] *= p.scale;
        x[i].e[e] *= rstd_a;
      }
      if (p.gate_g) {
        if (p.after_b) wb = ld_pack<T, VEC>(p.after_b + c);
        Pack<T, VEC> u;
#pragma unroll
        for (int e = 0; e < VEC; ++e) u.e[e] = (has_a ? x[i].e[e] * w.e[e] + (p.after_b ? wb.e[e] : (T)0) : x[i].e[e]) * h[i].e[e];
        if (gate_rows) {
          st_pack<T, VEC>(p.gate_g + (long long)g * n + c, u);
        } else {
          const Pack<T, VEC> before = ld_pack<T, VEC>(sums + SUMS * slot + c);
#pragma unroll
          for (int e = 0; e < VEC; ++e) u.e[e] += before.e[e];
          if (flush) {
            T* to = g_whole && g_left == 0 ? p.gate_g + (long long)g * n : gate_parts + (2LL * b + slot_b) * n;
            st_pack<T, VEC>(to + c, u);
          }
          st_pack<T, VEC>(sums + SUMS * slot + c, flush ? zero : u);
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (p.gate) h[i].e[e] *= ga.e[e];
      if (has_a) {
        Pack<T, VEC> sw = ld_pack<T, VEC>(sums + SUM_AFTER_W * slot + c), sb = ld_pack<T, VEC>(sums + SUM_AFTER_B * slot + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sw.e[e] += h[i].e[e] * x[i].e[e];
          sb.e[e] += h[i].e[e];
          h[i].e[e] *= w.e[e];
          a[0] += h[i].e[e] * x[i].e[e];
          if (LAYER) a[1] += h[i].e[e];
        }
        st_pack<T, VEC>(sums + SUM_AFTER_W * slot + c, sw);
        st_pack<T, VEC>(sums + SUM_AFTER_B * slot + c, sb);
      } else {
        st_pack<T, VEC>(p.block_g + (long long)r * p.ld_block_g + c, h[i]);
      }
    }
    if (has_x && has_a) {
      row_sums<T, 2>(a, part[turn ^= 1], warps);
      a[0] *= inv_n;
      a[1] *= inv_n;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = c0 + i * step;
        if (c >= n) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[i].e[e] = (h[i].e[e] - x[i].e[e] * a[0] - a[1]) * rstd_a;
        st_pack<T, VEC>(p.block_g + (long long)r * p.ld_block_g + c, h[i]);
      }
    }
    if (g_left == 0) {
      ++g;
      g_left = per_gate;
      g_whole = true;
      slot_b = 1;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int c = c0 + i * step;
    if (c >= n) continue;
    T* to = parts + (long long)b * SUMS * n + c;
#pragma unroll
    for (int k = 0; k < SUMS; ++k) st_pack<T, VEC>(to + (long long)k * n, ld_pack<T, VEC>(sums + k * slot + c));
  }
}

inline int round32(long long v) { return (int)((v + 31) / 32 * 32); }


template <typename T> bool packed_ok(int vec, long long cols, std::initializer_list<const void*> ps, std::initializer_list<long long> lds) {
  if (cols % vec) return false;
  uintptr_t bits = 0;
  for (const void* q : ps) bits |= (uintptr_t)q;
  for (long long ld : lds) if (ld % vec) return false;
  return (bits & (vec * sizeof(T) - 1)) == 0;
}


template <typename T, int VEC, int ITEMS> void launch_forward(cb200_stream* s, const Forward<T>& p) {
  const int threads = round32((p.cols + VEC * ITEMS - 1) / (VEC * ITEMS));
  const int side = threads == 32 ? 4 : 1;                  // a warp per row: four rows per CTA
  forward_rows_kernel<T, VEC, ITEMS><<<(unsigned)((p.rows + side - 1) / side), dim3(threads, side), 0, s->stream>>>(p);
}

template <typename T> int run_forward(cb200_stream* s, const Forward<T>& p) {
  DeviceGuard guard(s->device);
  constexpr int V = 16 / sizeof(T);
  const bool vec = packed_ok<T>(V, p.cols, {p.out, p.total, p.block, p.residual, p.gate, p.after_w, p.after_b, p.before_w, p.before_b},
                                {p.ld_out, p.ld_total, p.ld_block, p.ld_residual});
  // few rows: a row is spread over many threads (latency); many: 16 values per thread in flight
  const bool few = p.rows < 2LL * s->sm_count;
  if (vec && p.cols <= V * 1024 && (few || p.cols <= V * 32)) launch_forward<T, V, 1>(s, p);
  else if (vec && p.cols <= V * 2 * 64) launch_forward<T, V, 2>(s, p);
  else if (vec && p.cols <= V * 4 * 1024) launch_forward<T, V, 4>(s, p);
  else if (!vec && p.cols <= 1024 && (few || p.cols <= 32)) launch_forward<T, 1, 1>(s, p);
  else if (!vec && p.cols <= 4 * 1024) launch_forward<T, 1, 4>(s, p);
  else if (!vec && p.cols <= 8 * 1024) launch_forward<T, 1, 8>(s, p);
  else if (!vec && sizeof(T) == 4 && p.cols <= 16 * 1024) launch_forward<T, 1, sizeof(T) == 4 ? 16 : 4>(s, p);
  else forward_wide_kernel<T><<<(unsigned)p.rows, WIDE_THREADS, 0, s->stream>>>(p);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

template <typename T, void (*KERNEL)(Backward<T>, T*, T*, int)>
int launch_backward_kernel(cb200_stream* s, const Backward<T>& p, int threads, size_t smem, T* parts, T* gate_parts, int blocks) {
  static std::once_flag once[64];
  static cudaError_t result[64];
  const int dev = s->device & 63;
  std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 << 10); });
  if (result[dev] != cudaSuccess) return cb200_cuda_fail(result[dev], "cudaFuncSetAttribute", __FILE__, __LINE__);
  KERNEL<<<(unsigned)blocks, threads, smem, s->stream>>>(p, parts, gate_parts, blocks);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

template <typename T, int VEC, int ITEMS>
int launch_backward(cb200_stream* s, const Backward<T>& p, int threads, size_t smem, T* parts, T* gate_parts, int blocks) {
  if (threads <= 320)
    return p.layer ? launch_backward_kernel<T, backward_rows_kernel<T, VEC, ITEMS, true, 320>>(s, p, threads, smem, parts, gate_parts, blocks)
                   : launch_backward_kernel<T, backward_rows_kernel<T, VEC, ITEMS, false, 320>>(s, p, threads, smem, parts, gate_parts, blocks);
  if (threads <= 512)
    return p.layer ? launch_backward_kernel<T, backward_rows_kernel<T, VEC, ITEMS, true, 512>>(s, p, threads, smem, parts, gate_parts, blocks)
                   : launch_backward_kernel<T, backward_rows_kernel<T, VEC, ITEMS, false, 512>>(s, p, threads, smem, parts, gate_parts, blocks);
  return p.layer ? launch_backward_kernel<T, backward_hold_kernel<T, VEC, ITEMS, true>>(s, p, threads, smem, parts, gate_parts, blocks)
                 : launch_backward_kernel<T, backward_hold_kernel<T, VEC, ITEMS, false>>(s, p, threads, smem, parts, gate_parts, blocks);
}

template <typename T> int finish_columns(cb200_stream* s, const Backward<T>& p, const T* parts, const T* gate_parts, int blocks) {
  if (p.before_w_g || p.before_b_g || p.after_w_g || p.after_b_g) {
    column_finish_kernel<T><<<dim3((unsigned)((p.cols + 31) / 32), SUMS), 1024, 0, s->stream>>>(p, parts, blocks);
    CB_LAUNCH_CHECK(s);
  }
  if (p.gate_g && p.rows_per_gate > 1 && blocks > 1) {
    const long long groups = p.rows / p.rows_per_gate, each = blocks / groups;
    const unsigned y = (unsigned)(groups < 4096 ? groups : 4096);
    auto grid = [&](int columns) { return dim3((unsigned)((p.cols + columns - 1) / columns), y); };
    if (each >= 64) gate_finish_kernel<T, 8><<<grid(8), 256, 0, s->stream>>>(p, gate_parts, blocks);
    else if (each >= 16) gate_finish_kernel<T, 32><<<grid(32), 256, 0, s->stream>>>(p, gate_parts, blocks);
    else gate_finish_kernel<T, 128><<<grid(128), 256, 0, s->stream>>>(p, gate_parts, blocks);
    CB_LAUNCH_CHECK(s);
  }
  return CB200_OK;
}

template <typename T> int run_backward(cb200_stream* s, const Backward<T>& p) {
  DeviceGuard guard(s->device);
  constexpr int V = 16 / sizeof(T);
  const bool vec = packed_ok<T>(V, p.cols, {p.block_g, p.residual_g, p.gate_g, p.out_g, p.total_g, p.total, p.block, p.gate, p.after_w, p.after_b,
                                            p.before_w}, {p.ld_block_g, p.ld_residual_g, p.ld_out_g, p.ld_total_g, p.ld_total, p.ld_block});
  // values per thread: its five column sums of each stay in registers (64-bit ones: half as many values)
  constexpr int VALUES = sizeof(T) == 8 ? 4 : 8;
  // (wide rows of single values: as many threads as there may be; 12265 rows of 5081 1185 us with 640, 933 with 1024)
  const int fewest = round32((p.cols + VALUES - 1) / VALUES), threads = vec || fewest <= 512 || fewest > 1024 ? fewest : 1024;
  // two rows of four operands, or (wider rows) the five column sums
  const size_t smem = (size_t)(threads <= 512 ? 2 * 4 : SUMS + 1) * threads * VALUES * sizeof(T), room = 216 << 10;
  if (threads <= 1024) {
    long long per_sm = (long long)(room / smem), by_regs = threads <= 320 ? 65536 / (threads * 96) : 1;
    if (per_sm > by_regs) per_sm = by_regs;
    if (per_sm > 16) per_sm = 16;
    if (per_sm < 1) per_sm = 1;
    const int blocks = (int)(p.rows < s->sm_count * per_sm ? p.rows : s->sm_count * per_sm);
    void* ws = nullptr;
    const size_t parts_n = ((size_t)blocks * SUMS * p.cols + 3) / 4 * 4, gate_n = (size_t)blocks * 2 * p.cols;
    int rc = cb200_scratch(s, (parts_n + gate_n) * sizeof(T), &ws);
    if (rc) return rc;
    T* parts = (T*)ws;
    T* gate_parts = parts + parts_n;
    rc = vec ? launch_backward<T, V, VALUES / V>(s, p, threads, smem, parts, gate_parts, blocks)
             : launch_backward<T, 1, VALUES>(s, p, threads, smem, parts, gate_parts, blocks);
    if (rc) return rc;
    return finish_columns<T>(s, p, parts, gate_parts, blocks);
  }
  const long long col_tiles = (p.cols + 127) / 128;
  long long blocks = (2LL * s->sm_count * 8 + col_tiles - 1) / col_tiles;
  if (blocks > p.rows) blocks = p.rows;
  if (blocks > 1024) blocks = 1024;
  void* ws = nullptr;
  const size_t stats_n = (size_t)p.rows * 4, parts_n = (size_t)blocks * SUMS * p.cols, gate_n = (size_t)blocks * 2 * p.cols;
  int rc = cb200_scratch(s, (stats_n + parts_n + gate_n) * sizeof(T), &ws);
  if (rc) return rc;
  T* stats = (T*)ws;
  T* parts = stats + stats_n;
  T* gate_parts = parts + parts_n;
  backward_wide_kernel<T><<<(unsigned)p.rows, WIDE_THREADS, 0, s->stream>>>(p, stats);
  CB_LAUNCH_CHECK(s);
  if (p.before_w_g || p.before_b_g || p.after_w_g || p.after_b_g || (p.gate_g && p.rows_per_gate > 1)) {
    column_sums_kernel<T><<<dim3((unsigned)col_tiles, (unsigned)blocks), 128, 0, s->stream>>>(p, stats, parts, gate_parts,
                                                                                              (int)blocks);
    CB_LAUNCH_CHECK(s);
  }
  return finish_columns<T>(s, p, parts, gate_parts, (int)blocks);
}

int check_desc(const char* what, int dtype, const cb200_block_desc* d) {
  CB_REQUIRE(dtype == CB200_FLOAT || dtype == CB200_DOUBLE, "%s: only float and double tensors", what);
  CB_REQUIRE(d, "%s: null descriptor", what);
  CB_REQUIRE(d->kind == KIND_RMS || d->kind == KIND_LAYER, "%s: unknown normalisation %d", what, d->kind);
  const double epsilon = dtype == CB200_FLOAT ? (double)(float)d->epsilon : d->epsilon;      // (as the kernels have it)
  CB_REQUIRE(epsilon > 0.0 && isfinite(epsilon), "%s: epsilon must be positive in the element type", what);
  CB_REQUIRE(d->rows >= 0 && d->cols >= 1 && d->rows <= 2147483647LL && d->cols <= 2147483647LL, "%s: bad extents", what);
  CB_REQUIRE(d->gate_rows >= 1 && (d->rows == 0 || (d->gate_rows <= d->rows && d->rows % d->gate_rows == 0)),
             "%s: %lld gate rows do not divide %lld rows", what, (long long)d->gate_rows, (long long)d->rows);
  return CB200_OK;
}

// a matrix operand: its pitch covers its row; null is fine
int check_matrix(const char* what, const char* name, const void* p, int64_t ld, int dtype, const cb200_block_desc* d) {
  if (!p) return CB200_OK;
  CB_REQUIRE(ld >= d->cols, "%s: pitch of %s smaller than its row", what, name);
  CB_REQUIRE(((uintptr_t)p % cb200_dtype_size(dtype)) == 0, "%s: %s is not aligned to its element type", what, name);
  return CB200_OK;
}

// dense vectors and gates; null is fine
int check_aligned(const char* what, std::initializer_list<const void*> ps, int dtype) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= (uintptr_t)p;
  CB_REQUIRE(bits % cb200_dtype_size(dtype) == 0, "%s: a gate, scale, bias or gradient of one is not aligned to its element type", what);
  return CB200_OK;
}

// a result and another operand either are one and the same matrix (where `same_ok`) or share no memory
int check_apart(const char* what, const char* names, const void* a, int64_t lda, const void* b, int64_t ldb, bool same_ok,
                int dtype, int64_t b_rows, const cb200_block_desc* d, int64_t a_rows = -1) {
  if (!a || !b || d->rows == 0) return CB200_OK;
  if (same_ok && a == b && lda == ldb) return CB200_OK;
  if (a_rows < 0) a_rows = d->rows;
  const size_t size = cb200_dtype_size(dtype);
  const char* a0 = (const char*)a;
  const char* b0 = (const char*)b;
  const char* a1 = a0 + ((size_t)(a_rows - 1) * lda + d->cols) * size;
  const char* b1 = b0 + ((size_t)(b_rows - 1) * ldb + d->cols) * size;
  CB_REQUIRE(a1 <= b0 || b1 <= a0, "%s: %s overlap", what, names);
  return CB200_OK;
}

// a vector of cols elements shares none with a matrix (which may have gaps between its rows)
int check_vector_apart(const char* what, const char* matrix, const void* m, int64_t ld, int64_t rows, const char* vector, const void* v, int dtype,
                       const cb200_block_desc* d) {
  if (!m || !v || rows == 0) return CB200_OK;
  const int64_t size = (int64_t)cb200_dtype_size(dtype), n = d->cols * size, pitch = ld * size;
  const int64_t at = (int64_t)((intptr_t)v - (intptr_t)m);              // bytes from the matrix's first element
  const int64_t r = at < n ? 0 : (at - n) / pitch + 1;                  // the first row that ends behind the vector's start
  CB_REQUIRE(r >= rows || r * pitch >= at + n, "%s: %s overlaps %s", what, matrix, vector);
  return CB200_OK;
}

template <typename T>
int forward(cb200_stream* s, void* output, int64_t ld_output, void* total, int64_t ld_total, const void* block,
            int64_t ld_block, const void* residual, int64_t ld_residual, const void* gate, const void* after_scale,
            const void* after_bias, const void* before_scale, const void* before_bias, const cb200_block_desc* d) {
  Forward<T> p;
  p.out = (T*)output; p.ld_out = ld_output;
  p.total = (T*)total; p.ld_total = ld_total;
  p.block = (const T*)block; p.ld_block = ld_block;
  p.residual = (const T*)residual; p.ld_residual = ld_residual;
  p.gate = (const T*)gate;
  p.after_w = (const T*)after_scale; p.after_b = (const T*)after_bias;
  p.before_w = (const T*)before_scale; p.before_b = (const T*)before_bias;
  p.layer = d->kind == KIND_LAYER;
  p.eps = (T)d->epsilon; p.scale = (T)d->residual_scale;
  p.rows = d->rows; p.cols = d->cols; p.rows_per_gate = d->rows / d->gate_rows;
  return run_forward<T>(s, p);
}

}  // namespace

extern "C" {

int cb200_block_normalize(cb200_stream* s, int dtype, void* output, int64_t ld_output, void* total, int64_t ld_total,
                          const void* block, int64_t ld_block, const void* residual, int64_t ld_residual,
                          const void* gate, const void* after_scale, const void* after_bias, const void* before_scale,
                          const void* before_bias, const cb200_block_desc* d) {
  const char* what = "block_normalize";
  CB_REQUIRE(s, "block_normalize: null stream");
  int rc = check_desc(what, dtype, d);
  if (rc) return rc;
  CB_REQUIRE(residual, "block_normalize: null residual");
  CB_REQUIRE(output || total, "block_normalize: neither output nor total is wanted");
  CB_REQUIRE(!block || total, "block_normalize: a block needs a total to be added into");
  CB_REQUIRE(block || (!gate && !after_scale), "block_normalize: gate and after-normalisation belong to a block");
  CB_REQUIRE((output != nullptr) == (before_scale != nullptr), "block_normalize: output and the normalisation before the next block go together");
  CB_REQUIRE((!after_bias || after_scale) && (!before_bias || before_scale), "block_normalize: a bias without a scale");
  if ((rc = check_aligned(what, {gate, after_scale, after_bias, before_scale, before_bias}, dtype)) ||
      (rc = check_matrix(what, "output", output, ld_output, dtype, d)) || (rc = check_matrix(what, "total", total, ld_total, dtype, d)) ||
      (rc = check_matrix(what, "block", block, ld_block, dtype, d)) ||
      (rc = check_matrix(what, "residual", residual, ld_residual, dtype, d)) ||
      (rc = check_apart(what, "output and total", output, ld_output, total, ld_total, false, dtype, d->rows, d)) ||
      (rc = check_apart(what, "output and block", output, ld_output, block, ld_block, true, dtype, d->rows, d)) ||
      (rc = check_apart(what, "output and residual", output, ld_output, residual, ld_residual, true, dtype, d->rows, d)) ||
      (rc = check_apart(what, "total and block", total, ld_total, block, ld_block, true, dtype, d->rows, d)) ||
      (rc = check_apart(what, "total and residual", total, ld_total, residual, ld_residual, true, dtype, d->rows, d)) ||
      (rc = check_apart(what, "output and gate", output, ld_output, gate, d->cols, false, dtype, d->gate_rows, d)) ||
      (rc = check_apart(what, "total and gate", total, ld_total, gate, d->cols, false, dtype, d->gate_rows, d)))
    return rc;
  struct { const char* name; const void* p; } vectors[4] = {{"a scale", after_scale}, {"a bias", after_bias}, {"a scale", before_scale}, {"a bias", before_bias}};
  for (auto& v : vectors)
    if ((rc = check_vector_apart(what, "output", output, ld_output, d->rows, v.name, v.p, dtype, d)) ||
        (rc = check_vector_apart(what, "total", total, ld_total, d->rows, v.name, v.p, dtype, d)))
      return rc;
  if (d->rows == 0) return CB200_OK;
  return dtype == CB200_FLOAT
             ? forward<float>(s, output, ld_output, total, ld_total, block, ld_block, residual, ld_residual, gate, after_scale,
                              after_bias, before_scale, before_bias, d)
             : forward<double>(s, output, ld_output, total, ld_total, block, ld_block, residual, ld_residual, gate, after_scale,
                               after_bias, before_scale, before_bias, d);
}

}  // extern "C"

namespace {

template <typename T>
int backward(cb200_stream* s, void* block_gradient, int64_t ld_block_gradient, void* residual_gradient,
             int64_t ld_residual_gradient, void* gate_gradient, void* after_scale_gradient, void* after_bias_gradient,
             void* before_scale_gradient, void* before_bias_gradient, const void* output_gradient,
             int64_t ld_output_gradient, const void* total_gradient, int64_t ld_total_gradient, const void* total,
             int64_t ld_total, const void* block, int64_t ld_block, const void* gate, const void* after_scale,
             const void* after_bias, const void* before_scale, const cb200_block_desc* d) {
  Backward<T> p;
  p.block_g = (T*)block_gradient; p.ld_block_g = ld_block_gradient;
  p.residual_g = (T*)residual_gradient; p.ld_residual_g = ld_residual_gradient;
  p.gate_g = (T*)gate_gradient;
  p.after_w_g = (T*)after_scale_gradient; p.after_b_g = (T*)after_bias_gradient;
  p.before_w_g = (T*)before_scale_gradient; p.before_b_g = (T*)before_bias_gradient;
  p.out_g = (const T*)output_gradient; p.ld_out_g = ld_output_gradient;
  p.total_g = (const T*)total_gradient; p.ld_total_g = ld_total_gradient;
  p.total = (const T*)total; p.ld_total = ld_total;
  p.block = (const T*)block; p.ld_block = ld_block;
  p.gate = (const T*)gate; p.after_w = (const T*)after_scale; p.after_b = (const T*)after_bias;
  p.before_w = (const T*)before_scale;
  p.layer = d->kind == KIND_LAYER;
  p.eps = (T)d->epsilon; p.scale = (T)d->residual_scale;
  p.rows = d->rows; p.cols = d->cols; p.rows_per_gate = d->rows / d->gate_rows;
  return run_backward<T>(s, p);
}

}  // namespace

extern "C" {

int cb200_block_normalize_gradients(cb200_stream* s, int dtype, void* block_gradient, int64_t ld_block_gradient,
                                    void* residual_gradient, int64_t ld_residual_gradient, void* gate_gradient,
                                    void* after_scale_gradient, void* after_bias_gradient, void* before_scale_gradient,
                                    void* before_bias_gradient, const void* output_gradient, int64_t ld_output_gradient,
                                    const void* total_gradient, int64_t ld_total_gradient, const void* total,
                                    int64_t ld_total, const void* block, int64_t ld_block, const void* gate,
                                    const void* after_scale, const void* after_bias, const void* before_scale,
                                    const cb200_block_desc* d) {
  const char* what = "block_normalize_gradients";
  CB_REQUIRE(s, "block_normalize_gradients: null stream");
  int rc = check_desc(what, dtype, d);
  if (rc) return rc;
  CB_REQUIRE(residual_gradient, "block_normalize_gradients: null residual_gradient");
  CB_REQUIRE(output_gradient || total_gradient, "block_normalize_gradients: no gradient arrives");
  CB_REQUIRE((output_gradient != nullptr) == (before_scale != nullptr), "block_normalize_gradients: output_gradient and the normalisation before the next block go together");
  CB_REQUIRE(!before_scale || total, "block_normalize_gradients: the normalisation before the next block needs the total");
  CB_REQUIRE((block != nullptr) == (block_gradient != nullptr), "block_normalize_gradients: block and block_gradient go together");
  CB_REQUIRE(block || (!gate && !after_scale), "block_normalize_gradients: gate and after-normalisation belong to a block");
  CB_REQUIRE((!gate_gradient || gate) && (!after_scale_gradient || after_scale) && (!after_bias_gradient || after_scale) &&
                 (!before_scale_gradient || before_scale) && (!before_bias_gradient || before_scale) && (!after_bias || after_scale),
             "block_normalize_gradients: a gradient of something that is not there");
  struct { const char* name; const void* p; int64_t ld; } in[4] = {{"output_gradient", output_gradient, ld_output_gradient},
      {"total_gradient", total_gradient, ld_total_gradient}, {"total", total, ld_total}, {"block", block, ld_block}};
  struct { const char* name; const void* p; int64_t ld; } out[2] = {{"block_gradient", block_gradient, ld_block_gradient},
      {"residual_gradient", residual_gradient, ld_residual_gradient}};
  if ((rc = check_aligned(what, {gate_gradient, after_scale_gradient, after_bias_gradient, before_scale_gradient, before_bias_gradient, gate, after_scale,
                                 after_bias, before_scale}, dtype)))
    return rc;
  for (auto& m : in) if ((rc = check_matrix(what, m.name, m.p, m.ld, dtype, d))) return rc;
  for (auto& m : out) if ((rc = check_matrix(what, m.name, m.p, m.ld, dtype, d))) return rc;
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < 4; ++i)
      // the residual gradient may be written over the gradient that reached the sum
      if ((rc = check_apart(what, "a gradient and an operand", out[o].p, out[o].ld, in[i].p, in[i].ld, o == 1 && i == 1, dtype, d->rows, d)))
        return rc;
  for (int i = 0; i < 4; ++i)
    if ((rc = check_apart(what, "gate_gradient and an operand", gate_gradient, d->cols, in[i].p, in[i].ld, false, dtype, d->rows, d, d->gate_rows)))
      return rc;
  if ((rc = check_apart(what, "gate_gradient and gate", gate_gradient, d->cols, gate, d->cols, false, dtype, d->gate_rows, d, d->gate_rows)))
    return rc;
  if ((rc = check_apart(what, "block_gradient and residual_gradient", block_gradient, ld_block_gradient, residual_gradient,
                        ld_residual_gradient, false, dtype, d->rows, d)) ||
      (rc = check_apart(what, "block_gradient and gate", block_gradient, ld_block_gradient, gate, d->cols, false, dtype, d->gate_rows, d)) ||
      (rc = check_apart(what, "residual_gradient and gate", residual_gradient, ld_residual_gradient, gate, d->cols, false, dtype, d->gate_rows, d)) ||
      (rc = check_apart(what, "block_gradient and gate_gradient", block_gradient, ld_block_gradient, gate_gradient, d->cols, false, dtype, d->gate_rows, d)) ||
      (rc = check_apart(what, "residual_gradient and gate_gradient", residual_gradient, ld_residual_gradient, gate_gradient, d->cols, false, dtype, d->gate_rows, d)))
    return rc;
  // the vectors, read and written
  const void* read_vectors[3] = {after_scale, after_bias, before_scale};
  const void* sums[4] = {after_scale_gradient, after_bias_gradient, before_scale_gradient, before_bias_gradient};
  for (const void* v : read_vectors)
    if ((rc = check_vector_apart(what, "block_gradient", block_gradient, ld_block_gradient, d->rows, "a scale or bias", v, dtype, d)) ||
        (rc = check_vector_apart(what, "residual_gradient", residual_gradient, ld_residual_gradient, d->rows, "a scale or bias", v, dtype, d)) ||
        (rc = check_vector_apart(what, "gate_gradient", gate_gradient, d->cols, d->gate_rows, "a scale or bias", v, dtype, d)))
      return rc;
  for (int i = 0; i < 4; ++i) {
    const char* name = "the gradient of a scale or bias";
    for (auto& m : in) if ((rc = check_vector_apart(what, m.name, m.p, m.ld, d->rows, name, sums[i], dtype, d))) return rc;
    for (auto& m : out) if ((rc = check_vector_apart(what, m.name, m.p, m.ld, d->rows, name, sums[i], dtype, d))) return rc;
    if ((rc = check_vector_apart(what, "gate", gate, d->cols, d->gate_rows, name, sums[i], dtype, d)) ||
        (rc = check_vector_apart(what, "gate_gradient", gate_gradient, d->cols, d->gate_rows, name, sums[i], dtype, d)))
      return rc;
    for (const void* v : read_vectors) if ((rc = check_vector_apart(what, "a scale or bias", v, d->cols, 1, name, sums[i], dtype, d))) return rc;
    for (int j = 0; j < i; ++j) if ((rc = check_vector_apart(what, name, sums[j], d->cols, 1, name, sums[i], dtype, d))) return rc;
  }
  if (d->rows == 0) {
    // sums over no rows
    const size_t bytes = (size_t)d->cols * cb200_dtype_size(dtype);
    DeviceGuard guard(s->device);
    for (const void* v : sums) if (v) CB_CUDA(cudaMemsetAsync(const_cast<void*>(v), 0, bytes, s->stream));
    if (gate_gradient) CB_CUDA(cudaMemsetAsync(gate_gradient, 0, bytes * d->gate_rows, s->stream));
    return CB200_OK;
  }
  return dtype == CB200_FLOAT
             ? backward<float>(s, block_gradient, ld_block_gradient, residual_gradient, ld_residual_gradient, gate_gradient,
                               after_scale_gradient, after_bias_gradient, before_scale_gradient, before_bias_gradient,
                               output_gradient, ld_output_gradient, total_gradient, ld_total_gradient, total, ld_total, block,
                               ld_block, gate, after_scale, after_bias, before_scale, d)
             : backward<double>(s, block_gradient, ld_block_gradient, residual_gradient, ld_residual_gradient, gate_gradient,
                                after_scale_gradient, after_bias_gradient, before_scale_gradient, before_bias_gradient,
                                output_gradient, ld_output_gradient, total_gradient, ld_total_gradient, total, ld_total, block,
                                ld_block, gate, after_scale, after_bias, before_scale, d);
}

}  // extern "C"
