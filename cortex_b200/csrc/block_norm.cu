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
  long long seg = r0;                                      // first row of the current gate group inside this block
  for (long long r = r0; r < r1; ++r) {
    if (p.out_g) {
      const T dy = p.out_g[r * p.ld_out_g + c];
      s[SUM_BEFORE_W] += dy * ((p.total[r * p.ld_total + c] - stats[4 * r]) * stats[4 * r + 1]);
      s[SUM_BEFORE_B] += dy;
    }
    if (p.block) {
      const T d = p.scale * p.residual_g[r * p.ld_residual_g + c];
      const T x = p.block[r * p.ld_block + c];
      const T hat = (x - stats[4 * r + 2]) * stats[4 * r + 3];
      const long long g = r / p.rows_per_gate;
      const T du = p.gate ? d * p.gate[g * p.cols + c] : d;
      if (p.after_w) {
        s[SUM_AFTER_W] += du * hat;
        s[SUM_AFTER_B] += du;
      }
      if (gates) {
        gs += d * (p.after_w ? hat * aw + ab : x);
        const long long end = (g + 1) * p.rows_per_gate;
        if (r + 1 == end || r + 1 == r1) {
          const bool whole = seg == g * p.rows_per_gate && r + 1 == end;
          T* to = whole ? p.gate_g + g * p.cols : gate_parts + (2LL * b + (seg != r0)) * p.cols;
          to[c] = gs;
          gs = (T)0;
          seg = r + 1;
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < SUMS; ++k) parts[((long long)b * SUMS + k) * p.cols + c] = s[k];
}

template <typename T>
__global__ void __launch_bounds__(128) column_finish_kernel(Backward<T> p, const T* parts, int blocks) {
  const long long c = (long long)blockIdx.x * 128 + threadIdx.x;
  if (c >= p.cols) return;
  const int k = blockIdx.y;
  T* to = k == SUM_BEFORE_W ? p.before_w_g : (k == SUM_BEFORE_B ? p.before_b_g : (k == SUM_AFTER_W ? p.after_w_g : p.after_b_g));
  if (!to) return;
  T s = (T)0;
  for (int b = 0; b < blocks; ++b) s += parts[((long long)b * SUMS + k) * p.cols + c];
  to[c] = s;
}

// gate groups that more than one row block has a part of; group g = blockIdx.y (strided)
template <typename T>
__global__ void __launch_bounds__(128) gate_finish_kernel(Backward<T> p, const T* gate_parts, int blocks) {
  const long long c = (long long)blockIdx.x * 128 + threadIdx.x;
  if (c >= p.cols) return;
  const long long groups = p.rows / p.rows_per_gate;
  for (long long g = blockIdx.y; g < groups; g += gridDim.y) {
    const long long first = g * p.rows_per_gate, last = first + p.rows_per_gate - 1;
    const int b0 = block_of(p.rows, blocks, first), b1 = block_of(p.rows, blocks, last);
    if (b0 == b1) continue;
    T s = gate_parts[(2LL * b0 + (first != block_begin(p.rows, blocks, b0))) * p.cols + c];
    for (int b = b0 + 1; b <= b1; ++b) s += gate_parts[2LL * b * p.cols + c];
    p.gate_g[g * p.cols + c] = s;
  }
}

template <typename T> int run_forward(cb200_stream* s, const Forward<T>& p) {
  DeviceGuard guard(s->device);
  forward_wide_kernel<T><<<(unsigned)p.rows, WIDE_THREADS, 0, s->stream>>>(p);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

template <typename T> int run_backward(cb200_stream* s, const Backward<T>& p) {
  DeviceGuard guard(s->device);
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
  const bool gates = p.gate_g && p.rows_per_gate > 1;
  if (p.before_w_g || p.before_b_g || p.after_w_g || p.after_b_g || gates) {
    column_sums_kernel<T><<<dim3((unsigned)col_tiles, (unsigned)blocks), 128, 0, s->stream>>>(p, stats, parts, gate_parts,
                                                                                              (int)blocks);
    CB_LAUNCH_CHECK(s);
    column_finish_kernel<T><<<dim3((unsigned)col_tiles, SUMS), 128, 0, s->stream>>>(p, parts, (int)blocks);
    CB_LAUNCH_CHECK(s);
  }
  if (gates) {
    const long long groups = p.rows / p.rows_per_gate;
    gate_finish_kernel<T><<<dim3((unsigned)col_tiles, (unsigned)(groups < 1024 ? groups : 1024)), 128, 0, s->stream>>>(
        p, gate_parts, (int)blocks);
    CB_LAUNCH_CHECK(s);
  }
  return CB200_OK;
}

int check_desc(const char* what, int dtype, const cb200_block_desc* d) {
  CB_REQUIRE(dtype == CB200_FLOAT || dtype == CB200_DOUBLE, "%s: only float and double tensors", what);
  CB_REQUIRE(d, "%s: null descriptor", what);
  CB_REQUIRE(d->kind == KIND_RMS || d->kind == KIND_LAYER, "%s: unknown normalisation %d", what, d->kind);
  CB_REQUIRE(d->epsilon > 0.0 && isfinite(d->epsilon), "%s: epsilon must be positive", what);
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
  if ((rc = check_matrix(what, "output", output, ld_output, dtype, d)) || (rc = check_matrix(what, "total", total, ld_total, dtype, d)) ||
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
  if (d->rows == 0) {
    // sums over no rows
    const size_t bytes = (size_t)d->cols * cb200_dtype_size(dtype);
    DeviceGuard guard(s->device);
    void* sums[5] = {after_scale_gradient, after_bias_gradient, before_scale_gradient, before_bias_gradient, nullptr};
    for (void* v : sums) if (v) CB_CUDA(cudaMemsetAsync(v, 0, bytes, s->stream));
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
