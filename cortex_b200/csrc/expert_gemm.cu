// Products grouped by expert: rows of A are grouped by offsets in device memory and every group has a matrix of its own.
//
//   expert_gemm           C[r, :]  = act(alpha * A[r, :] . op(B_e) + beta * C[r, :] + bias_e)       r in group e
//   expert_gemm_weights   C_e      = alpha * sum_{r in group e} A[r, :]^T B[r, :] + beta * C_e
//                         bias_gradient_e = alpha * sum_{r in group e} A[r, :] + beta * bias_gradient_e
//
// Rows outside every group are neither read into a result nor written.
//
// Here: the entries, the rules that choose a kernel by sizes, type and alignment, the kernels for few rows per expert (bound by
// one pass over the matrices or results), the tiles for doubles and for fp32 operands of any alignment, and the bias gradient.
// fp32 products on the tensor cores are in the files ending in _tc (3xTF32) and _f16 (scaled halves, large products).
#include "common.cuh"
#include "expert_groups.cuh"
#include <math.h>

bool cb200_expert_tc_ok(const void* A, long long lda, const void* B, long long ldb, long long b_stride);
int cb200_expert_rows_tc(cb200_stream* s, float* C, long long ldc, int trans_b, float alpha, const float* A, int rows, int K,
                         long long lda, const float* B, int experts, int N, long long b_stride, long long ldb, float beta,
                         const int* offsets, const float* bias, int act, const int* only_if);
int cb200_expert_weights_tc(cb200_stream* s, float* C, long long c_stride, long long ldc, float alpha, const float* A, int rows,
                            int M, long long lda, const float* B, int N, long long ldb, int experts, float beta,
                            const int* offsets, const int* only_if);
bool cb200_expert_f16_ok(cb200_stream* s, long long rows, long long K, long long N, long long experts);
bool cb200_expert_weights_f16_ok(cb200_stream* s, long long rows, long long M, long long N, long long experts);
int cb200_expert_rows_f16(cb200_stream* s, float* C, long long ldc, int trans_b, float alpha, const float* A, int rows, int K,
                          long long lda, const float* B, int experts, int N, long long b_stride, long long ldb, float beta,
                          const int* offsets, const float* bias, int act, const int** guard);
int cb200_expert_weights_f16(cb200_stream* s, float* C, long long c_stride, long long ldc, float alpha, const float* A, int rows, int M,
                             long long lda, const float* B, int N, long long ldb, int experts, float beta, const int* offsets,
                             float* bias_gradient, const int** guard);

namespace {

static __device__ __noinline__ double act_transcendental(double v, int act) {
  return act == CB200_ACT_TANH ? tanh(v) : 1.0 / (1.0 + exp(-v));
}
template <typename T> __device__ __forceinline__ T act_apply(T v, int act) {
  if (act == CB200_ACT_NONE) return v;
  if (act == CB200_ACT_RELU) return groups::relu(v);
  return (T)act_transcendental((double)v, act);
}

template <typename T> struct Product {
  T* C; long long c_stride, ldc;
  const T* A; long long lda;
  const T* B; long long b_stride, ldb;
  int trans_b, act;
  int rows, M, N, K, experts;      // expert_gemm: K, N of op(B); expert_gemm_weights: C_e is M x N
  T alpha, beta;
  const T* bias;
  T* bias_g;
  const int* offsets;
  const int* only_if;              // null, or a device word: do nothing while it is zero
  int* status;
};

// A 64 x 64 tile by 256 threads, operands of any pitch and alignment.  Element (m, k) of the left operand at
// a[m * sam + k * sak], (k, n) of the right one at b[k * sbk + n * sbn].  float: 4 x 4 plain FMAs per thread.
template <typename T> struct Tile64;

template <typename T>
__device__ __forceinline__ void finish(T* to, T sum, int n, T alpha, T beta, const T* bias, int act) {
  T o = alpha * sum;
  if (beta != (T)0) o += beta * (*to);
  if (bias) o += bias[n];
  *to = act_apply<T>(o, act);
}

template <> struct Tile64<float> {
  float acc[4][4];
  __device__ __forceinline__ void run(const float* a, long long sam, long long sak, const float* b, long long sbk, long long sbn, int m_left,
                                      int n_left, int K) {
    __shared__ float As[16][64 + 1];
    __shared__ float Bs[16][64 + 1];
    const int t = threadIdx.x, tx = t % 16, ty = t / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    for (int k0 = 0; k0 < K; k0 += 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int k, m;
        if (sak == 1) { k = t % 16; m = t / 16 + 16 * i; } else { m = t % 64; k = t / 64 + 4 * i; }
        As[k][m] = (m < m_left && k0 + k < K) ? a[(long long)m * sam + (long long)(k0 + k) * sak] : 0.f;
        int kb, n;
        if (sbn == 1) { n = t % 64; kb = t / 64 + 4 * i; } else { kb = t % 16; n = t / 16 + 16 * i; }
        Bs[kb][n] = (n < n_left && k0 + kb < K) ? b[(long long)(k0 + kb) * sbk + (long long)n * sbn] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = As[k][ty + 16 * i];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = Bs[k][tx + 16 * j];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += x[i] * y[j];
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ void store(float* c, long long ldc, int m_left, int n_left, float alpha, float beta, const float* bias, int act) {
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = ty + 16 * i, n = tx + 16 * j;
        if (m < m_left && n < n_left) finish<float>(c + (long long)m * ldc + n, acc[i][j], n, alpha, beta, bias, act);
      }
  }
};

// double: the fp64 matrix instruction (m16n8k8), 8 warps as 2 x 4 of 32 x 16, the next 16 values of k on their way into
// registers meanwhile, two buffers in turn.  Row pitch 68 (4 mod 16): the 16 fragment elements of a half-warp lie in 16
// different banks.  Bound by the matrix pipe where there are tiles enough: 8192 x 2048 x 2048 over 2 experts 2.44 to 2.61 ms,
// 26 to 28 TFLOP/s of the 35.5 that a library product reaches (m8n8k4 and two barriers a step: 2.8 ms).
template <> struct Tile64<double> {
  double acc[2][2][4];
  __device__ __forceinline__ void run(const double* a, long long sam, long long sak, const double* b, long long sbk, long long sbn, int m_left,
                                      int n_left, int K) {
    constexpr int LD = 68;
    __shared__ double As2[2][16][LD];
    __shared__ double Bs2[2][16][LD];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, wm = (warp >> 2) * 32, wn = (warp & 3) * 16, fr = lane >> 2, fk = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.0;
    double ra[4], rb[4];
    auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int k, m;
        if (sak == 1) { k = t % 16; m = t / 16 + 16 * i; } else { m = t % 64; k = t / 64 + 4 * i; }
        ra[i] = (m < m_left && k0 + k < K) ? a[(long long)m * sam + (long long)(k0 + k) * sak] : 0.0;
        int kb, n;
        if (sbn == 1) { n = t % 64; kb = t / 64 + 4 * i; } else { kb = t % 16; n = t / 16 + 16 * i; }
        rb[i] = (n < n_left && k0 + kb < K) ? b[(long long)(k0 + kb) * sbk + (long long)n * sbn] : 0.0;
      }
    };
    if (K > 0) load(0);
    __syncthreads();                                         // (the tile before has been read)
    for (int k0 = 0; k0 < K; k0 += 16) {
      // two buffers in turn: one barrier per step
      double (&As)[16][LD] = As2[(k0 >> 4) & 1];
      double (&Bs)[16][LD] = Bs2[(k0 >> 4) & 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (sak == 1) As[t % 16][t / 16 + 16 * i] = ra[i]; else As[t / 64 + 4 * i][t % 64] = ra[i];
        if (sbn == 1) Bs[t / 64 + 4 * i][t % 64] = rb[i]; else Bs[t % 16][t / 16 + 16 * i] = rb[i];
      }
      __syncthreads();
      if (k0 + 16 < K) load(k0 + 16);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        double x[2][4], y[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = wm + i * 16 + fr, k = kk * 8 + fk;
          x[i][0] = As[k][m];
          x[i][1] = As[k][m + 8];
          x[i][2] = As[k + 4][m];
          x[i][3] = As[k + 4][m + 8];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          y[j][0] = Bs[kk * 8 + fk][wn + j * 8 + fr];
          y[j][1] = Bs[kk * 8 + fk + 4][wn + j * 8 + fr];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            asm volatile("mma.sync.aligned.m16n8k8.row.col.f64.f64.f64.f64 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                         : "+d"(acc[i][j][0]), "+d"(acc[i][j][1]), "+d"(acc[i][j][2]), "+d"(acc[i][j][3])
                         : "d"(x[i][0]), "d"(x[i][1]), "d"(x[i][2]), "d"(x[i][3]), "d"(y[j][0]), "d"(y[j][1]));
      }
    }
  }
  __device__ __forceinline__ void store(double* c, long long ldc, int m_left, int n_left, double alpha, double beta, const double* bias, int act) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = (warp >> 2) * 32, wn = (warp & 3) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {                            // 16-row tile i / 2, its upper or lower 8 rows
      const int m = wm + i * 8 + (lane >> 2);
      if (m >= m_left) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = wn + j * 8 + (lane & 3) * 2 + e;
          if (n < n_left) finish<double>(c + (long long)m * ldc + n, acc[i >> 1][j][(i & 1) * 2 + e], n, alpha, beta, bias, act);
        }
    }
  }
};

// K slices where the tiles leave SMs free: every slice parks its 64 x 64 sums in L2, and the CTA of a tile that arrives last
// adds them in slice order; nobody waits.  False for the CTAs that are done.
struct Slices {
  void* park;
  int* arrived;                // per tile, zero between launches
  int count;
};

template <typename T> __device__ __forceinline__ bool join_slices(Tile64<T>& c, const Slices& s, int slice, long long unit, int* last) {
  T* acc = reinterpret_cast<T*>(c.acc);
  T* park = (T*)s.park + unit * s.count * 4096 + threadIdx.x;
#pragma unroll
  for (int i = 0; i < 16; ++i) __stcg(park + slice * 4096 + i * 256, acc[i]);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *last = atomicAdd(s.arrived + unit, 1) == s.count - 1;
  __syncthreads();
  if (!*last) return false;
  __threadfence();
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = __ldcg(park + i * 256);
  for (int k = 1; k < s.count; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] += __ldcg(park + k * 4096 + i * 256);
  if (threadIdx.x == 0) s.arrived[unit] = 0;
  return true;
}

// the part of 0 .. K - 1 that slice `slice` of `count` adds up, whole steps of 16
__device__ __forceinline__ void slice_bounds(int K, int slice, int count, int& begin, int& end) {
  const long long steps = ((long long)K + 15) / 16;
  begin = (int)(steps * slice / count * 16);
  end = (int)min((long long)K, steps * (slice + 1) / count * 16);
}

// workspace for `units` results of `values` each in `slices` parts
template <typename T> int get_slices(cb200_stream* s, long long units, long long values, int slices, Slices& out) {
  out.park = nullptr; out.arrived = nullptr; out.count = slices;
  if (slices == 1) return CB200_OK;
  const int rc = cb200_partials(s, (size_t)(units * values) * slices * sizeof(T), &out.park);
  return rc ? rc : cb200_tile_flags(s, (size_t)units, &out.arrived);
}

// blockIdx.x: column tile and slice, blockIdx.y: row tile
template <typename T>
__global__ void __launch_bounds__(256, 3) expert_rows_tile_kernel(Product<T> p, Slices s) {
  __shared__ groups::Tile tile;
  __shared__ int found;
  if (p.only_if && *p.only_if == 0) return;
  const int tn = (int)blockIdx.x / s.count, slice = (int)blockIdx.x - tn * s.count;
  for (int t = (int)blockIdx.y;; t += (int)gridDim.y) {
    __syncthreads();
    if (threadIdx.x < 32) {
      groups::Tile own;
      const bool f = groups::find_tile(p.offsets, p.experts, p.rows, 64, t, p.status, own);
      if (threadIdx.x == 0) { tile = own; found = f; }
    }
    __syncthreads();
    if (!found) return;
    const int m0 = tile.lo + tile.index * 64, n0 = tn * 64;
    int k0, k1;
    slice_bounds(p.K, slice, s.count, k0, k1);
    const T* b = p.B + tile.expert * p.b_stride + (p.trans_b ? (long long)n0 * p.ldb + k0 : (long long)k0 * p.ldb + n0);
    Tile64<T> c;
    c.run(p.A + (long long)m0 * p.lda + k0, p.lda, 1, b, p.trans_b ? 1 : p.ldb, p.trans_b ? p.ldb : 1, tile.hi - m0, p.N - n0, k1 - k0);
    if (s.count > 1 && !join_slices<T>(c, s, slice, (long long)t * (gridDim.x / s.count) + tn, &found)) continue;
    c.store(p.C + (long long)m0 * p.ldc + n0, p.ldc, tile.hi - m0, p.N - n0, p.alpha, p.beta,
            p.bias ? p.bias + (long long)tile.expert * p.N + n0 : nullptr, p.act);
  }
}

// blockIdx.x: column tile and slice, blockIdx.y: row tile of the result, blockIdx.z: expert
template <typename T>
__global__ void __launch_bounds__(256, 3) expert_weights_tile_kernel(Product<T> p, int tiles_m, Slices s) {
  __shared__ int lo, hi, last;
  if (p.only_if && *p.only_if == 0) return;
  const int e = (int)blockIdx.z, tn = (int)blockIdx.x / s.count, slice = (int)blockIdx.x - tn * s.count;
  if (threadIdx.x < 32) {
    int a, b;
    groups::group_rows(p.offsets, p.rows, e, p.status, a, b);
    if (threadIdx.x == 0) { lo = a; hi = b; }
  }
  __syncthreads();
  const int n0 = tn * 64;
  int k0, k1;
  slice_bounds(hi - lo, slice, s.count, k0, k1);
  const T* a = p.A + (long long)(lo + k0) * p.lda;
  const T* b = p.B + (long long)(lo + k0) * p.ldb + n0;
  for (int tm = (int)blockIdx.y; tm < tiles_m; tm += (int)gridDim.y) {
    const int m0 = tm * 64;
    Tile64<T> c;
    c.run(a + m0, 1, p.lda, b, p.ldb, 1, p.M - m0, p.N - n0, k1 - k0);
    if (s.count > 1 && !join_slices<T>(c, s, slice, ((long long)e * tiles_m + tm) * (gridDim.x / s.count) + tn, &last)) continue;
    c.store(p.C + e * p.c_stride + (long long)m0 * p.ldc + n0, p.ldc, p.M - m0, p.N - n0, p.alpha, p.beta, nullptr, CB200_ACT_NONE);
  }
}

// ---- few rows per expert: the matrices are read once, as fast as memory delivers them ---------------------------------
// A tile is up to 8 rows of one group; a warp takes 4 rows of its expert's matrix ([out, in]: contiguous along the reduction)
// and strides over the reduction with 16-byte loads, the rows of A coming from L1.  The 4 x R sums of a lane are folded over
// the warp (31 shuffles for 32 of them) so that each ends in one lane, which finishes and stores it.
constexpr int FEW = 8, FEW_OUT = 4, FEW_WARPS = 8;

template <typename T, int V, int R>
__device__ __forceinline__ void few_rows(const Product<T>& p, const groups::Tile& tile, int t0, int left, int n0) {
  struct alignas(sizeof(T) * V) Pack { T e[V]; };
  constexpr int VALUES = FEW_OUT * R;
  const int lane = threadIdx.x & 31;
  const T* w = p.B + tile.expert * p.b_stride;
  const T* a = p.A + (long long)t0 * p.lda;
  T acc[VALUES];
#pragma unroll
  for (int i = 0; i < VALUES; ++i) acc[i] = (T)0;
  const T* wr[FEW_OUT];
#pragma unroll
  for (int j = 0; j < FEW_OUT; ++j) wr[j] = w + (long long)min(n0 + j, p.N - 1) * p.ldb;      // (stores are bounded below)
#pragma unroll ((R == 8 ? 1 : 2) * (V == 1 && sizeof(T) == 4 ? 2 : 1))
  for (int k = lane * V; k < p.K; k += 32 * V) {           // V > 1: K is a multiple of V
    Pack m[FEW_OUT], x[R];
#pragma unroll
    for (int j = 0; j < FEW_OUT; ++j) m[j] = *reinterpret_cast<const Pack*>(wr[j] + k);
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = *reinterpret_cast<const Pack*>(a + (long long)min(r, left - 1) * p.lda + k);
#pragma unroll
    for (int j = 0; j < FEW_OUT; ++j)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[j * R + r] += m[j].e[e] * x[r].e[e];
  }
  // fold: after step d a lane keeps the half of the values that its bit selects
  int which = 0;
#pragma unroll
  for (int half = VALUES / 2, d = 16; d > 0; d >>= 1) {
    if (half > 0) {
      const bool up = (lane & d) != 0;
#pragma unroll
      for (int i = 0; i < VALUES / 2; ++i)
        if (i < half) {
          const T give = up ? acc[i] : acc[i + half], keep = up ? acc[i + half] : acc[i];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
        }
      which = which * 2 + (up ? 1 : 0);
      half >>= 1;
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], d);
    }
  }
  const int n = n0 + which / R, r = which % R;
  constexpr int SAME = 32 / VALUES;                        // lanes that end with the same value
  if ((lane & (SAME - 1)) == 0 && n < p.N && r < left) {
    T* c = p.C + (long long)(t0 + r) * p.ldc + n;
    T o = p.alpha * acc[0];
    if (p.beta != (T)0) o += p.beta * (*c);
    if (p.bias) o += p.bias[(long long)tile.expert * p.N + n];
    *c = act_apply<T>(o, p.act);
  }
}

// The same for matrices [in, out], contiguous along the result: a lane has 16 bytes of columns (V values adjacent, or single
// ones 32 apart), the warps take V rows of the matrix in turn, and their sums meet in shared memory in the order of the warps,
// those of K slices in L2 as in the tile kernels.
template <typename T, int V, int R>
__device__ __forceinline__ void few_rows_mn(const Product<T>& p, const groups::Tile& tile, int t0, int left, int block, T* part,
                                            const Slices& s, int slice, int* last) {
  struct alignas(sizeof(T) * V) Pack { T e[V]; };
  constexpr int L = 16 / sizeof(T), PACKS = L / V, COLS = 32 * L;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long n0 = (long long)block * COLS;
  const long long steps = ((long long)p.K + V - 1) / V;
  const int k0 = (int)(steps * slice / s.count * V), k1 = (int)min((long long)p.K, steps * (slice + 1) / s.count * V);
  const T* a = p.A + (long long)t0 * p.lda;
  const T* w[PACKS];
#pragma unroll
  for (int j = 0; j < PACKS; ++j)                            // (stores are bounded below)
    w[j] = p.B + tile.expert * p.b_stride + min(n0 + lane * V + j * 32 * V, (long long)p.N - V);
  T acc[R][L];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < L; ++j) acc[r][j] = (T)0;
#pragma unroll ((R == 8 ? 1 : 2) * (V == 1 ? 2 : 1))
  for (int k = k0 + warp * V; k < k1; k += FEW_WARPS * V) {  // V > 1: K is a multiple of V
    Pack m[V][PACKS], x[R];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < PACKS; ++j) m[v][j] = *reinterpret_cast<const Pack*>(w[j] + (long long)(k + v) * p.ldb);
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = *reinterpret_cast<const Pack*>(a + (long long)min(r, left - 1) * p.lda + k);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < L; ++j) acc[r][j] += x[r].e[v] * m[v][j / V].e[j % V];
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < L; ++j) part[(warp * R + r) * COLS + (j / V) * 32 * V + lane * V + j % V] = acc[r][j];
  __syncthreads();
  const T* bias = p.bias ? p.bias + (long long)tile.expert * p.N : nullptr;
  const long long unit = (long long)blockIdx.x / s.count;
  T* park = (T*)s.park + unit * s.count * (FEW * COLS);
#pragma unroll 1
  for (int i = (int)threadIdx.x; i < R * COLS; i += FEW_WARPS * 32) {
    const int r = i / COLS;
    const long long n = n0 + i % COLS;
    if (n >= p.N || r >= left) continue;
    T sum = part[i];
#pragma unroll
    for (int k = 1; k < FEW_WARPS; ++k) sum += part[k * R * COLS + i];
    if (s.count > 1) __stcg(park + slice * (FEW * COLS) + i, sum);
    else finish<T>(p.C + (long long)(t0 + r) * p.ldc + n, sum, (int)n, p.alpha, p.beta, bias, p.act);
  }
  if (s.count == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *last = atomicAdd(s.arrived + unit, 1) == s.count - 1;
  __syncthreads();
  if (!*last) return;
  __threadfence();
  if (threadIdx.x == 0) s.arrived[unit] = 0;
#pragma unroll 1
  for (int i = (int)threadIdx.x; i < R * COLS; i += FEW_WARPS * 32) {
    const int r = i / COLS;
    const long long n = n0 + i % COLS;
    if (n >= p.N || r >= left) continue;
    T sum = __ldcg(park + i);
    for (int k = 1; k < s.count; ++k) sum += __ldcg(park + k * (FEW * COLS) + i);
    finish<T>(p.C + (long long)(t0 + r) * p.ldc + n, sum, (int)n, p.alpha, p.beta, bias, p.act);
  }
}

template <typename T, int V, bool MN>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) expert_few_rows_kernel(Product<T> p, int n_blocks, Slices s) {
  if (groups::all_may_be_found(p.rows, p.experts, FEW) && blockIdx.x == gridDim.x - 1) {
    groups::check_offsets(p.offsets, p.experts, p.rows, p.status);         // a CTA behind those of the tiles
    return;
  }
  const int unit = (int)blockIdx.x / s.count, slice = (int)blockIdx.x - unit * s.count, t = unit / n_blocks, block = unit - t * n_blocks;
  const int n0 = (block * FEW_WARPS + ((int)threadIdx.x >> 5)) * FEW_OUT;
  groups::Tile tile;
  if (!groups::find_tile(p.offsets, p.experts, p.rows, FEW, t, p.status, tile)) return;
  const int t0 = tile.lo + tile.index * FEW, left = min(FEW, tile.hi - t0);
  if (MN) {
    __shared__ T part[FEW_WARPS * FEW * 32 * 16 / sizeof(T)];
    __shared__ int last;
    if (left == 1) few_rows_mn<T, V, 1>(p, tile, t0, left, block, part, s, slice, &last);
    else if (left == 2) few_rows_mn<T, V, 2>(p, tile, t0, left, block, part, s, slice, &last);
    else if (left <= 4) few_rows_mn<T, V, 4>(p, tile, t0, left, block, part, s, slice, &last);
    else few_rows_mn<T, V, 8>(p, tile, t0, left, block, part, s, slice, &last);
    return;
  }
  if (n0 >= p.N) return;
  if (left == 1) few_rows<T, V, 1>(p, tile, t0, left, n0);
  else if (left == 2) few_rows<T, V, 2>(p, tile, t0, left, n0);
  else if (left <= 4) few_rows<T, V, 4>(p, tile, t0, left, n0);
  else few_rows<T, V, 8>(p, tile, t0, left, n0);
}

// By the rows alone (which expert gets how many is not known here).  This kernel / the tile kernels, us, 8 experts of 4096 x
// 1024 (fp32 134 MB, 20 us) with 1, 4, 8, 12 rows each: products 13, 29, 41, 53 / 43, 44, 45, 47; input gradients 18, 42, 50, 71 /
// 43, 46, 46, 66; doubles 35, 59, 90, 116 / 149, 196, 197, 197 and 54, 100, 137, 194 / 197, 197, 198, 199; 41 experts of
// 3676 x 611, which TMA cannot address, 74, 121, 188, 247 / 214, 224, 248, 250 and 90, 181, 193, 313 / 240, 258, 265, 268.  Every
// tile of 8 rows reads its expert's matrix again: the limit on all rows is for routings that send everything to one expert.
bool few_rows_ok(const Product<float>& p) { return p.rows <= (p.trans_b ? 8LL : 6LL) * p.experts && p.rows <= 1024; }
bool few_rows_ok(const Product<double>& p) { return p.rows <= 12LL * p.experts && p.rows <= 1024; }

template <typename T> int run_few_rows(cb200_stream* s, const Product<T>& p) {
  DeviceGuard guard(s->device);
  constexpr int V = 16 / sizeof(T);
  const long long tiles = (p.rows + FEW - 1) / FEW + (p.experts < p.rows ? p.experts : p.rows) - 1;
  const long long per = p.trans_b ? FEW_WARPS * FEW_OUT : 32 * V, n_blocks = (p.N + per - 1) / per, ctas = tiles * n_blocks;
  CB_REQUIRE(ctas < 2147483647LL, "expert_gemm: too many tiles");
  const bool wide = (((uintptr_t)p.A | (uintptr_t)p.B) & 15) == 0 && p.lda % V == 0 && p.ldb % V == 0 && p.b_stride % V == 0 && p.K % V == 0 &&
                    (p.trans_b || p.N % V == 0);
  const unsigned threads = FEW_WARPS * 32;
  // K slices until every SM has a CTA (128 values of K each at least), then up to four to an SM where they stay long: joining
  // costs 4 us (8 experts, one row each: K = 4096 into 1024 columns 41 us uncut, 18 in slices; K = 1024 into 4096 12 and 16)
  int slices = 1;
  while (!p.trans_b && slices < 16 && ctas * slices * 2 <= 4LL * s->sm_count && p.K / (slices * 2) >= (ctas * slices < s->sm_count ? 128 : 1024))
    slices *= 2;
  Slices sl;
  const int rc = get_slices<T>(s, ctas, FEW * 32 * V, slices, sl);
  if (rc) return rc;
  const unsigned grid = (unsigned)(ctas * slices + (groups::all_may_be_found(p.rows, p.experts, FEW) ? 1 : 0));
  if (p.trans_b && wide) expert_few_rows_kernel<T, V, false><<<grid, threads, 0, s->stream>>>(p, (int)n_blocks, sl);
  else if (p.trans_b) expert_few_rows_kernel<T, 1, false><<<grid, threads, 0, s->stream>>>(p, (int)n_blocks, sl);
  else if (wide) expert_few_rows_kernel<T, V, true><<<grid, threads, 0, s->stream>>>(p, (int)n_blocks, sl);
  else expert_few_rows_kernel<T, 1, true><<<grid, threads, 0, s->stream>>>(p, (int)n_blocks, sl);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

// bias_gradient[e, m] = alpha * sum of the group's rows + beta * bias_gradient[e, m]: a warp reads 32 * V columns of a row,
// the CTA's 32 warps take every 32nd row with four rows in flight each; where columns and experts are too few for the SMs the
// rows are cut into slices (blockIdx.z) joined as above; fixed order throughout (7169 x 328 over 2 experts: 13 us, one CTA
// for all rows of 128 columns 78 us)
template <typename T, int V>
__global__ void __launch_bounds__(1024) expert_bias_gradient_kernel(Product<T> p, Slices sl) {
  struct alignas(sizeof(T) * V) Pack { T e[V]; };
  __shared__ int lo, hi, last;
  __shared__ T part[32][32 * V];
  const int e = (int)blockIdx.y;
  if (threadIdx.x < 32) {
    int a, b;
    groups::group_rows(p.offsets, p.rows, e, p.status, a, b);
    if (threadIdx.x == 0) {
      lo = a + (int)((long long)(b - a) * blockIdx.z / sl.count);
      hi = a + (int)((long long)(b - a) * (blockIdx.z + 1) / sl.count);
    }
  }
  __syncthreads();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, m = ((int)blockIdx.x * 32 + tx) * V;
  T s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = (T)0;
  if (m < p.M) {
    const T* a = p.A + m;
    int r = lo + ty;
    for (; r + 96 < hi; r += 128) {
      Pack v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const Pack*>(a + (long long)(r + 32 * i) * p.lda);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] += v[i].e[j];
    }
    for (; r < hi; r += 32) {
      const Pack v = *reinterpret_cast<const Pack*>(a + (long long)r * p.lda);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] += v.e[j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) part[ty][tx * V + j] = s[j];
  __syncthreads();
  const long long at = (long long)blockIdx.x * 32 * V + threadIdx.x;
  const bool mine = threadIdx.x < 32 * V && at < p.M;
  T sum = (T)0;
  if (mine) {
    sum = part[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < 32; ++w) sum += part[w][threadIdx.x];
  }
  if (sl.count > 1) {
    T* park = (T*)sl.park + (long long)e * p.M + at;
    const long long apart = (long long)p.experts * p.M;
    if (mine) __stcg(park + blockIdx.z * apart, sum);
    __threadfence();
    __syncthreads();
    int* arrived = sl.arrived + ((long long)e * gridDim.x + blockIdx.x);
    if (threadIdx.x == 0) last = atomicAdd(arrived, 1) == sl.count - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    if (threadIdx.x == 0) *arrived = 0;
    if (mine) {
      sum = __ldcg(park);
      for (int i = 1; i < sl.count; ++i) sum += __ldcg(park + i * apart);
    }
  }
  if (!mine) return;
  T* to = p.bias_g + (long long)e * p.M + at;
  T o = p.alpha * sum;
  if (p.beta != (T)0) o += p.beta * (*to);
  *to = o;
}

// ---- weight gradients of few rows per expert: the results are written once, as fast as memory takes them --------------
// A warp has 8 rows of C_e (columns of A) and 128 columns, four to a lane: V of them adjacent where B and C take 16-byte
// accesses, else 32 apart, so that a warp's stores are whole lines whatever the pitch.  The group's rows are added in order with
// FMAs; A's values are the same for all lanes.  The CTAs of the first columns add up the bias gradient beside.
constexpr int FEW_M = 8;

template <typename T, int V>
__global__ void __launch_bounds__(256, sizeof(T) == 8 ? 2 : (V == 1 ? 3 : 4)) expert_few_weights_kernel(Product<T> p, int tiles_m) {
  constexpr int PACKS = 4 / V;
  struct alignas(sizeof(T) * V) Pack { T e[V]; };
  __shared__ int bounds[2];
  const int e = (int)blockIdx.z, lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  if (warp == 0) {
    int a, b;
    groups::group_rows(p.offsets, p.rows, e, p.status, a, b);
    if (lane == 0) { bounds[0] = a; bounds[1] = b; }
  }
  __syncthreads();
  const int lo = bounds[0], hi = bounds[1];
  const long long n0 = (long long)blockIdx.x * 128 + lane * V;
  for (int tm = (int)blockIdx.y; tm < tiles_m; tm += (int)gridDim.y) {
    const int m0 = tm * (8 * FEW_M) + warp * FEW_M, m_left = p.M - m0;
    if (m_left <= 0) return;
    T acc[FEW_M][PACKS * V], sum[FEW_M];
#pragma unroll
    for (int i = 0; i < FEW_M; ++i) {
      sum[i] = (T)0;
#pragma unroll
      for (int j = 0; j < PACKS * V; ++j) acc[i][j] = (T)0;
    }
    const T* a = p.A + m0;
#pragma unroll 2
    for (int r = lo; r < hi; ++r) {
      Pack b[PACKS];
      T x[FEW_M];
#pragma unroll
      for (int j = 0; j < PACKS; ++j) {
        const long long n = n0 + j * 32 * V;
        if (n < p.N) b[j] = *reinterpret_cast<const Pack*>(p.B + (long long)r * p.ldb + n);      // V > 1: N is a multiple of V
        else
#pragma unroll
          for (int v = 0; v < V; ++v) b[j].e[v] = (T)0;
      }
#pragma unroll
      for (int i = 0; i < FEW_M; i += V) {                   // (V > 1: M is a multiple of V; stores are bounded below)
        const Pack from = *reinterpret_cast<const Pack*>(a + (long long)r * p.lda + (i < m_left ? i : 0));
#pragma unroll
        for (int v = 0; v < V; ++v) x[i + v] = from.e[v];
      }
#pragma unroll
      for (int i = 0; i < FEW_M; ++i) {
        sum[i] += x[i];
#pragma unroll
        for (int j = 0; j < PACKS; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) acc[i][j * V + v] += x[i] * b[j].e[v];
      }
    }
    T* c = p.C + e * p.c_stride + (long long)m0 * p.ldc;
#pragma unroll
    for (int i = 0; i < FEW_M; ++i) {
      if (i >= m_left) break;
#pragma unroll
      for (int j = 0; j < PACKS; ++j) {
        const long long n = n0 + j * 32 * V;
        if (n >= p.N) continue;
        Pack* to = reinterpret_cast<Pack*>(c + (long long)i * p.ldc + n);
        Pack o;
        if (p.beta != (T)0) o = *to;
#pragma unroll
        for (int v = 0; v < V; ++v) o.e[v] = p.beta != (T)0 ? p.alpha * acc[i][j * V + v] + p.beta * o.e[v] : p.alpha * acc[i][j * V + v];
        *to = o;
      }
      if (p.bias_g && blockIdx.x == 0 && lane == 0) {
        T* to = p.bias_g + (long long)e * p.M + m0 + i;
        *to = p.beta != (T)0 ? p.alpha * sum[i] + p.beta * *to : p.alpha * sum[i];
      }
    }
  }
}

// Measured, this kernel / the tile kernels: 8 experts of 1024 x 4096 (134 MB, 20 us) with 1, 8, 16, 24 rows each 27, 53, 84,
// 115 / 111, 113, 115, 119 us; 3 of 1506 x 1291 (operands that TMA cannot address) 10, 19, 31, 43 / 41, 41, 42, 43 us;
// doubles, 8 of 1024 x 4096 with 1, 8, 16 rows 49, 101, 159 / 106, 118, 135 us.  The limit on all rows is for routings that
// send everything to one expert, whose few CTAs then walk all of them one after another.
template <typename T> bool few_weights_ok(const Product<T>& p) {
  return p.rows <= (sizeof(T) == 4 ? 16LL : 8LL) * p.experts && p.rows <= 512;
}

template <typename T> int run_few_weights(cb200_stream* s, const Product<T>& p) {
  DeviceGuard guard(s->device);
  constexpr int V = 16 / sizeof(T);
  const int tiles_m = (p.M + 8 * FEW_M - 1) / (8 * FEW_M);
  const dim3 grid((unsigned)((p.N + 127) / 128), (unsigned)(tiles_m < 65535 ? tiles_m : 65535), (unsigned)p.experts);
  const bool wide = (((uintptr_t)p.A | (uintptr_t)p.B | (uintptr_t)p.C) & 15) == 0 && p.M % V == 0 && p.N % V == 0 && p.lda % V == 0 &&
                    p.ldb % V == 0 && p.ldc % V == 0 && p.c_stride % V == 0;
  if (wide) expert_few_weights_kernel<T, V><<<grid, 256, 0, s->stream>>>(p, tiles_m);
  else expert_few_weights_kernel<T, 1><<<grid, 256, 0, s->stream>>>(p, tiles_m);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

template <typename T> int run_bias_gradient(cb200_stream* s, const Product<T>& p) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = ((uintptr_t)p.A & 15) == 0 && p.lda % V == 0 && p.M % V == 0;
  const long long blocks = ((long long)p.M + (wide ? 32 * V : 32) - 1) / (wide ? 32 * V : 32), units = blocks * p.experts;
  // at least 256 rows (two turns of the CTA) to a slice, and no more CTAs than two to an SM
  int slices = 1;
  while (slices < 16 && units * slices * 2 <= 2LL * s->sm_count && p.rows / p.experts / (slices * 2) >= 256) slices *= 2;
  Slices sl;
  const int rc = get_slices<T>(s, units, wide ? 32 * V : 32, slices, sl);
  if (rc) return rc;
  const dim3 grid((unsigned)blocks, (unsigned)p.experts, (unsigned)slices);
  if (wide) expert_bias_gradient_kernel<T, V><<<grid, 1024, 0, s->stream>>>(p, sl);
  else expert_bias_gradient_kernel<T, 1><<<grid, 1024, 0, s->stream>>>(p, sl);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

// Slices of the reduction for `tiles` tiles: as many as three CTAs to an SM take, at least 128 values of `K` each
int tile_slices(const cb200_stream* s, long long tiles, long long K) {
  int slices = 1;
  while (slices < 16 && tiles * slices * 2 <= 3LL * s->sm_count && K / (slices * 2) >= 128) slices *= 2;
  return slices;
}

template <typename T> int run_rows(cb200_stream* s, const Product<T>& p) {
  if (!p.only_if && few_rows_ok(p)) return run_few_rows<T>(s, p);
  DeviceGuard guard(s->device);
  const long long tiles = (p.rows + 63) / 64 + (p.experts < p.rows ? p.experts : p.rows), tiles_n = (p.N + 63) / 64;
  Slices sl;
  const int slices = p.only_if ? 1 : tile_slices(s, tiles * tiles_n, p.K), rc = get_slices<T>(s, tiles * tiles_n, 4096, slices, sl);
  if (rc) return rc;
  expert_rows_tile_kernel<T><<<dim3((unsigned)(tiles_n * slices), (unsigned)(tiles < 65535 ? tiles : 65535)), 256, 0, s->stream>>>(p, sl);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

template <typename T> int run_weights(cb200_stream* s, const Product<T>& p) {
  DeviceGuard guard(s->device);
  const int tiles_m = (p.M + 63) / 64;
  const long long tiles_n = (p.N + 63) / 64, tiles = tiles_n * tiles_m * p.experts;
  Slices sl;
  const int slices = p.only_if ? 1 : tile_slices(s, tiles, p.rows / p.experts), rc = get_slices<T>(s, tiles, 4096, slices, sl);
  if (rc) return rc;
  expert_weights_tile_kernel<T><<<dim3((unsigned)(tiles_n * slices), (unsigned)(tiles_m < 65535 ? tiles_m : 65535), (unsigned)p.experts),
                                  256, 0, s->stream>>>(p, tiles_m, sl);
  CB_LAUNCH_CHECK(s);
  return p.bias_g ? run_bias_gradient<T>(s, p) : CB200_OK;
}

// ---- fp32: the tensor-core kernels, behind a copy of operands that TMA cannot address -----------------------------------
// A warp (eight lanes where rows are short) takes a row at a time; blockIdx.y is the matrix.
template <int LANES>
__global__ void __launch_bounds__(256) pack_rows_kernel(float* __restrict__ dst, long long ld_dst, const float* __restrict__ src,
                                                        long long ld, long long stride, long long rows, int cols) {
  const int sub = (int)threadIdx.x % LANES;
  src += (long long)blockIdx.y * stride;
  dst += (long long)blockIdx.y * rows * ld_dst;
  for (long long r = (long long)blockIdx.x * (256 / LANES) + (int)threadIdx.x / LANES; r < rows; r += (long long)gridDim.x * (256 / LANES)) {
    const float* from = src + r * ld;
    float* to = dst + r * ld_dst;
    for (int c = sub; c < cols; c += 8 * LANES) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j * LANES < cols) v[j] = from[c + j * LANES];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j * LANES < cols) to[c + j * LANES] = v[j];
    }
  }
}

// `matrices` of rows x cols, `stride` apart, into dense rows of a multiple of 4 (32 x 2894 x 226, 168 MB read
// and written: 24 us, all eight loads of a lane's turn in flight)
int pack(cb200_stream* s, float* dst, const float* src, long long ld, long long stride, int matrices, long long rows, int cols) {
  const int lanes = cols <= 64 ? 8 : 32;
  const long long need = (rows + 256 / lanes - 1) / (256 / lanes), cap = ((long long)s->sm_count * 32 + matrices - 1) / matrices;
  const dim3 grid((unsigned)(need < cap ? need : cap), (unsigned)matrices);
  const long long ld_dst = (cols + 3) / 4 * 4;
  if (lanes == 8) pack_rows_kernel<8><<<grid, 256, 0, s->stream>>>(dst, ld_dst, src, ld, stride, rows, cols);
  else pack_rows_kernel<32><<<grid, 256, 0, s->stream>>>(dst, ld_dst, src, ld, stride, rows, cols);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

// No memory left for the halves (up to 2 GB)?  The call goes on without them.
bool no_room(int rc, const int* only_if) {
  if (rc != CB200_ERR_NOMEM || only_if) return false;
  cudaGetLastError();                                            // (or the next launch would report it)
  return true;
}

int rows_tc(cb200_stream* s, Product<float> p) {
  if (few_rows_ok(p) && s->opt_gemm_auto_presplit != 2 && s->opt_gemm_tile_n == 0) return run_few_rows<float>(s, p);
  const long long b_rows = p.trans_b ? p.N : p.K;
  const int b_cols = p.trans_b ? p.K : p.N;
  if (p.experts == 1) p.b_stride = b_rows * p.ldb;
  const bool pack_a = !cb200_expert_tc_ok(p.A, p.lda, p.A, 4, 4), pack_b = !cb200_expert_tc_ok(p.B, p.ldb, p.B, 4, p.b_stride);
  bool halves = cb200_expert_f16_ok(s, p.rows, p.K, p.N, p.experts);
  if (halves) {
    // products at twice the rate; what follows runs only where the data do not fit scaled halves
    const int rc = cb200_expert_rows_f16(s, p.C, p.ldc, p.trans_b, p.alpha, p.A, p.rows, p.K, p.lda, p.B, p.experts, p.N, p.b_stride, p.ldb,
                                   p.beta, p.offsets, p.bias, p.act, &p.only_if);
    if (!no_room(rc, p.only_if)) {
      if (rc) return rc;
      if (pack_a || pack_b) return run_rows<float>(s, p);       // (the workspace holds the halves)
    } else {
      halves = false;
    }
  }
  if (!halves && (pack_a || pack_b)) {
    DeviceGuard guard(s->device);
    const long long lda = (p.K + 3) / 4 * 4, ldb = (b_cols + 3) / 4 * 4;
    const size_t a_n = pack_a ? (size_t)p.rows * lda : 0, b_n = pack_b ? (size_t)p.experts * b_rows * ldb : 0;
    void* ws = nullptr;
    int rc = cb200_scratch(s, (a_n + b_n) * sizeof(float), &ws);
    if (rc) return rc;
    float* a = (float*)ws;
    float* b = a + a_n;
    if (pack_a) {
      if ((rc = pack(s, a, p.A, p.lda, 0, 1, p.rows, p.K))) return rc;
      p.A = a; p.lda = lda;
    }
    if (pack_b) {
      if ((rc = pack(s, b, p.B, p.ldb, p.b_stride, p.experts, b_rows, b_cols))) return rc;
      p.B = b; p.ldb = ldb; p.b_stride = b_rows * ldb;
    }
  }
  return cb200_expert_rows_tc(s, p.C, p.ldc, p.trans_b, p.alpha, p.A, p.rows, p.K, p.lda, p.B, p.experts, p.N, p.b_stride, p.ldb,
                              p.beta, p.offsets, p.bias, p.act, p.only_if);
}

int weights_tc(cb200_stream* s, Product<float> p) {
  if (p.rows == 0) return run_few_weights<float>(s, p);
  if (few_weights_ok(p) && s->opt_gemm_auto_presplit != 2 && s->opt_gemm_tile_n == 0) return run_few_weights<float>(s, p);
  const bool pack_a = !cb200_expert_tc_ok(p.A, p.lda, p.A, 4, 4), pack_b = !cb200_expert_tc_ok(p.B, p.ldb, p.B, 4, 4);
  bool halves = cb200_expert_weights_f16_ok(s, p.rows, p.M, p.N, p.experts);
  if (halves) {
    const int rc = cb200_expert_weights_f16(s, p.C, p.c_stride, p.ldc, p.alpha, p.A, p.rows, p.M, p.lda, p.B, p.N, p.ldb, p.experts, p.beta,
                                      p.offsets, p.bias_g, &p.only_if);
    if (!no_room(rc, p.only_if)) {
      if (rc) return rc;
      p.bias_g = nullptr;                                        // done with the column pass
      if (pack_a || pack_b) return run_weights<float>(s, p);
    } else {
      halves = false;
    }
  }
  if (!halves && p.bias_g) {
    DeviceGuard guard(s->device);
    int rc = run_bias_gradient<float>(s, p);
    if (rc) return rc;
  }
  if (!halves && (pack_a || pack_b)) {
    DeviceGuard guard(s->device);
    const long long lda = (p.M + 3) / 4 * 4, ldb = (p.N + 3) / 4 * 4;
    const size_t a_n = pack_a ? (size_t)p.rows * lda : 0, b_n = pack_b ? (size_t)p.rows * ldb : 0;
    void* ws = nullptr;
    int rc = cb200_scratch(s, (a_n + b_n) * sizeof(float), &ws);
    if (rc) return rc;
    float* a = (float*)ws;
    float* b = a + a_n;
    if (pack_a) {
      if ((rc = pack(s, a, p.A, p.lda, 0, 1, p.rows, p.M))) return rc;
      p.A = a; p.lda = lda;
    }
    if (pack_b) {
      if ((rc = pack(s, b, p.B, p.ldb, 0, 1, p.rows, p.N))) return rc;
      p.B = b; p.ldb = ldb;
    }
  }
  return cb200_expert_weights_tc(s, p.C, p.c_stride, p.ldc, p.alpha, p.A, p.rows, p.M, p.lda, p.B, p.N, p.ldb, p.experts, p.beta, p.offsets, p.only_if);
}

// kernels step 32-bit indexes past the last row and column, by a tile or a warp's stride at most
constexpr int64_t MAX_EXTENT = 2147483647LL - 65535;

int check_common(const char* what, cb200_stream* s, int dtype, const void* C, const void* A, const void* B, const void* bias, int64_t rows,
                 int64_t experts, const int32_t* offsets) {
  CB_REQUIRE(s && C && A && B && offsets, "%s: null argument", what);
  CB_REQUIRE(dtype == CB200_FLOAT || dtype == CB200_DOUBLE, "%s: only defined for float and double tensors", what);
  CB_REQUIRE(rows >= 0 && rows <= MAX_EXTENT, "%s: bad row count", what);
  CB_REQUIRE(experts >= 1 && experts <= groups::MAX_EXPERTS, "%s: %lld experts outside [1, %d]", what, (long long)experts,
             (int)groups::MAX_EXPERTS);
  const uintptr_t size = cb200_dtype_size(dtype);
  CB_REQUIRE((((uintptr_t)C | (uintptr_t)A | (uintptr_t)B | (uintptr_t)bias) % size) == 0 && ((uintptr_t)offsets & 3) == 0,
             "%s: an operand is not aligned to its element type", what);
  return CB200_OK;
}

template <typename T>
Product<T> product(cb200_stream* s, void* C, int64_t c_stride, int64_t ldc, int trans_b, double alpha, const void* A,
                   int64_t rows, int64_t M, int64_t K, int64_t lda, const void* B, int64_t experts, int64_t N, int64_t b_stride,
                   int64_t ldb, double beta, const int32_t* offsets, const void* bias, void* bias_g, int act) {
  Product<T> p;
  p.C = (T*)C; p.c_stride = c_stride; p.ldc = ldc;
  p.A = (const T*)A; p.lda = lda;
  p.B = (const T*)B; p.b_stride = b_stride; p.ldb = ldb;
  p.trans_b = trans_b != 0; p.act = act;
  p.rows = (int)rows; p.M = (int)M; p.N = (int)N; p.K = (int)K; p.experts = (int)experts;
  p.alpha = (T)alpha; p.beta = (T)beta;
  p.bias = (const T*)bias; p.bias_g = (T*)bias_g;
  p.offsets = offsets; p.only_if = nullptr; p.status = s->status_dev;
  return p;
}

}  // namespace

extern "C" {

int cb200_expert_gemm(cb200_stream* s, int dtype, void* C, int64_t ldc, int trans_b, double alpha, const void* A, int64_t rows,
                      int64_t a_cols, int64_t lda, const void* B, int64_t experts, int64_t b_cols, int64_t b_stride, int64_t ldb,
                      double beta, const int32_t* offsets, const void* bias, int act) {
  int rc = check_common("expert_gemm", s, dtype, C, A, B, bias, rows, experts, offsets);
  if (rc) return rc;
  CB_REQUIRE(a_cols >= 1 && b_cols >= 1 && a_cols <= MAX_EXTENT && b_cols <= MAX_EXTENT, "expert_gemm: bad extents");
  CB_REQUIRE(ldc >= b_cols && lda >= a_cols && ldb >= (trans_b ? a_cols : b_cols), "expert_gemm: pitch smaller than the row");
  CB_REQUIRE(b_stride >= (trans_b ? b_cols : a_cols) * ldb || experts == 1, "expert_gemm: the experts' matrices overlap");
  CB_REQUIRE(act >= CB200_ACT_NONE && act <= CB200_ACT_LOGISTIC, "expert_gemm: unknown activation %d", act);
  if (rows == 0) return CB200_OK;
  if (dtype == CB200_FLOAT)
    return rows_tc(s, product<float>(s, C, 0, ldc, trans_b, alpha, A, rows, 0, a_cols, lda, B, experts, b_cols, b_stride,
                                     ldb, beta, offsets, bias, nullptr, act));
  return run_rows<double>(s, product<double>(s, C, 0, ldc, trans_b, alpha, A, rows, 0, a_cols, lda, B, experts, b_cols, b_stride,
                                             ldb, beta, offsets, bias, nullptr, act));
}

int cb200_expert_gemm_weights(cb200_stream* s, int dtype, void* C, int64_t c_stride, int64_t ldc, double alpha, const void* A,
                              int64_t rows, int64_t a_cols, int64_t lda, const void* B, int64_t b_cols, int64_t ldb,
                              int64_t experts, double beta, const int32_t* offsets, void* bias_gradient) {
  int rc = check_common("expert_gemm_weights", s, dtype, C, A, B, bias_gradient, rows, experts, offsets);
  if (rc) return rc;
  CB_REQUIRE(a_cols >= 1 && b_cols >= 1 && a_cols <= MAX_EXTENT && b_cols <= MAX_EXTENT, "expert_gemm_weights: bad extents");
  CB_REQUIRE(ldc >= b_cols && lda >= a_cols && ldb >= b_cols, "expert_gemm_weights: pitch smaller than the row");
  CB_REQUIRE(c_stride >= a_cols * ldc || experts == 1, "expert_gemm_weights: the experts' matrices overlap");
  if (dtype == CB200_FLOAT) {
    const Product<float> p = product<float>(s, C, c_stride, ldc, 0, alpha, A, rows, a_cols, 0, lda, B, experts, b_cols, 0, ldb, beta,
                                            offsets, nullptr, bias_gradient, CB200_ACT_NONE);
    return weights_tc(s, p);
  }
  const Product<double> p = product<double>(s, C, c_stride, ldc, 0, alpha, A, rows, a_cols, 0, lda, B, experts, b_cols, 0, ldb, beta,
                                            offsets, nullptr, bias_gradient, CB200_ACT_NONE);
  return few_weights_ok(p) ? run_few_weights<double>(s, p) : run_weights<double>(s, p);
}

}  // extern "C"
