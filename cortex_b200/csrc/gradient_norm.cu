// The global norm over a list of gradient buffers, and the gradients scaled down to a bound on it.
//
//   norm  = sqrt(sum over every element of every buffer of g^2)
//   scale = max_norm / norm   where norm > max_norm and norm is finite, else 1
//   clipped = scale * g
//
// The buffers of one launch travel as a table in the kernel's parameters (no upload, nothing to keep alive, captured
// into a graph as it is).  Each buffer is cut into chunks that start on a 16-byte boundary, CTAs take chunks in turn,
// squares are summed in double (products of floats are exact there and cannot overflow; doubles whose squares could leave the
// range are summed apart, scaled by a power of two), one partial sum per CTA goes to a fixed slot, and the CTA that finishes
// last adds the slots in order: the result has the same bits on every run.
#include "common.cuh"
#include <math.h>
#include <algorithm>
#include <new>

namespace {

// Buffers per launch: 28 bytes each in the kernel's parameters.  Two tables, because parameters cost time to pass: a
// small network's call is bound by its two launches.
constexpr int SMALL_TABLE = 32, TABLE = 512;
constexpr int THREADS = 256;
constexpr int CHUNK = 4096;        // elements

template <typename T, int MOST> struct Pieces {
  const T* g[MOST];
  T* out[MOST];
  long long count[MOST];
  int first[MOST + 1];             // the buffer's first chunk; first[n] = all chunks
  int n;
};

// Where the norm and the scale of a call live between its kernels: words of the stream's partial-sum block.
// Gradients are multiplied by scale, then by tail (1, but where the product of the two is below the normal range).
struct NormResult { double norm, scale, tail; };

// Sums of squares.  Of doubles: those between 2^-480 and 2^480 as they are (2^43 of them stay in range), the others
// times 2^-600 and 2^600, so that a norm is finite wherever it is a double, and no value is lost below it.
template <typename T> struct Squares;
template <> struct Squares<float> {
  static constexpr int N = 1;
  double s[1];
  __device__ __forceinline__ void zero() { s[0] = 0.0; }
  template <int M> __device__ __forceinline__ void add(const float (&x)[M]) {
    double two[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < M; ++i) two[i & 1] += (double)x[i] * (double)x[i];
    s[0] += two[0] + two[1];
  }
  __device__ __forceinline__ double norm() const { return sqrt(s[0]); }
};
template <> struct Squares<double> {
  static constexpr int N = 3;
  static constexpr double BIG = 0x1p480, SMALL = 0x1p-480, DOWN = 0x1p-600, UP = 0x1p600;
  double s[3];                     // as they are, big, small
  __device__ __forceinline__ void zero() { s[0] = s[1] = s[2] = 0.0; }
  template <int M> __device__ __forceinline__ void add(const double (&x)[M]) {
    double two[2] = {0.0, 0.0};
    int least = 0x7fffffff, most = 0;                  // the words with the exponents
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int a = __double2hiint(x[i]) & 0x7fffffff;
      least = min(least, a);
      most = max(most, a);
      two[i & 1] += x[i] * x[i];
    }
    if (least >= (1023 - 480) << 20 && most < (1023 + 480) << 20) {
      s[0] += two[0] + two[1];
      return;
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const double a = fabs(x[i]);
      if (a > BIG) s[1] += a * DOWN * (a * DOWN);
      else if (a < SMALL) s[2] += a * UP * (a * UP);
      else s[0] += a * a;                              // (a NaN too)
    }
  }
  __device__ __forceinline__ double norm() const {
    if (s[1] != 0.0) return sqrt(s[1] + s[0] * DOWN * DOWN) * UP;
    if (s[0] != 0.0) return sqrt(s[0] + s[2] * DOWN * DOWN);
    return sqrt(s[2]) * DOWN;
  }
};

template <typename T> struct Vec;
template <> struct Vec<float> { struct alignas(16) type { float e[4]; }; static constexpr int N = 4; };
template <> struct Vec<double> { struct alignas(16) type { double e[2]; }; static constexpr int N = 2; };

// Elements [lo, hi) of buffer `p` that chunk `c` covers: chunks are cut at 16-byte boundaries of the buffer.
template <typename T, int MOST>
__device__ __forceinline__ void chunk_range(const Pieces<T, MOST>& t, int c, int& p, long long& lo, long long& hi) {
  int a = 0, b = t.n;
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if (t.first[m] <= c) a = m; else b = m;
  }
  p = a;
  const long long off = (long long)(((uintptr_t)t.g[p] & 15) / sizeof(T));
  const long long k = c - t.first[p];
  lo = k * CHUNK - off;
  hi = lo + CHUNK;
  if (lo < 0) lo = 0;
  if (hi > t.count[p]) hi = t.count[p];
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[THREADS / 32];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) v += part[w];
  __syncthreads();
  return v;
}

// partials: one slot per CTA of every launch of the call; `slot0` this launch's first, `slots` all of them.
// `last` : the call's last launch; its last CTA to finish writes the result.
template <typename T, int MOST>
__global__ void __launch_bounds__(THREADS)
square_sum_kernel(const __grid_constant__ Pieces<T, MOST> t, double* partials, int slot0, int slots, int last, int* counter,
                  NormResult* result, T* norm_out, double max_norm) {
  typedef typename Vec<T>::type V;
  constexpr int N = Vec<T>::N, WHOLE = CHUNK / N / THREADS;           // 16-byte loads of a whole chunk per thread
  Squares<T> sum;
  sum.zero();
  const int chunks = t.first[t.n];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    int p;
    long long lo, hi;
    chunk_range(t, c, p, lo, hi);
    const T* g = t.g[p];
    if (hi - lo == CHUNK) {                                // starts on a 16-byte boundary
      const V* v = reinterpret_cast<const V*>(g + lo);
      V x[WHOLE];
#pragma unroll
      for (int i = 0; i < WHOLE; ++i) x[i] = v[threadIdx.x + i * THREADS];
      T all[WHOLE * N];
#pragma unroll
      for (int i = 0; i < WHOLE; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) all[i * N + e] = x[i].e[e];
      sum.add(all);
    } else {
#pragma unroll 4
      for (long long i = lo + threadIdx.x; i < hi; i += THREADS) {
        const T one[1] = {g[i]};
        sum.add(one);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < Squares<T>::N; ++k) sum.s[k] = block_sum(sum.s[k]);
  __shared__ bool finish;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < Squares<T>::N; ++k) partials[(slot0 + blockIdx.x) * Squares<T>::N + k] = sum.s[k];
    __threadfence();
    finish = last && atomicAdd(counter, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!finish) return;
  __threadfence();
  sum.zero();
  for (int i = threadIdx.x; i < slots; i += THREADS)
#pragma unroll
    for (int k = 0; k < Squares<T>::N; ++k) sum.s[k] += __ldcg(partials + (long long)i * Squares<T>::N + k);
#pragma unroll
  for (int k = 0; k < Squares<T>::N; ++k) sum.s[k] = block_sum(sum.s[k]);
  if (threadIdx.x == 0) {
    const double norm = sum.norm();
    result->norm = norm;
    result->scale = result->tail = 1.0;
    if (norm > max_norm && isfinite(norm)) {
      result->scale = max_norm / norm;
      if (result->scale < 0x1p-900) {                  // (then norm is above 2^-173: times 2^-600 it keeps its bits)
        result->scale = max_norm / (norm * 0x1p-600);
        result->tail = 0x1p-600;
      }
    }
    if (norm_out) *norm_out = (T)norm;
    *counter = 0;                                    // left zero for the next launch
  }
}

// A CTA per chunk (2^28 floats: 497 us for the whole call, against 553 with 16 CTAs per SM that take chunks in turn), from the
// last chunk to the first: what the norm's pass read last is still in L2.  Stores are streaming, so they do not push it out.
template <typename T, int MOST>
__global__ void __launch_bounds__(THREADS) scale_kernel(const __grid_constant__ Pieces<T, MOST> t, const NormResult* result) {
  typedef typename Vec<T>::type V;
  constexpr int N = Vec<T>::N, WHOLE = CHUNK / N / THREADS;
  const T scale = (T)(result->scale * result->tail);
  const int chunks = t.first[t.n];
  const int c = chunks - 1 - (int)blockIdx.x;
  int p;
  long long lo, hi;
  chunk_range(t, c, p, lo, hi);
  const T* g = t.g[p];
  T* o = t.out[p];
  if (scale == (T)1 && g == o) return;               // within the bound, in place: nothing changes
  if (!(scale >= (T)1e-30)) {                      // a scale down here would have lost its low bits
    for (long long i = lo + threadIdx.x; i < hi; i += THREADS) o[i] = (T)((double)g[i] * result->scale * result->tail);
  } else if (hi - lo == CHUNK && ((uintptr_t)(o + lo) & 15) == 0) {
    const V* v = reinterpret_cast<const V*>(g + lo);
    V x[WHOLE];
#pragma unroll
    for (int i = 0; i < WHOLE; ++i) x[i] = v[threadIdx.x + i * THREADS];
#pragma unroll
    for (int i = 0; i < WHOLE; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[i].e[e] *= scale;
      __stcs(reinterpret_cast<float4*>(o + lo) + threadIdx.x + i * THREADS, *reinterpret_cast<const float4*>(&x[i]));
    }
  } else {
#pragma unroll 4
    for (long long i = lo + threadIdx.x; i < hi; i += THREADS) o[i] = g[i] * scale;
  }
}

template <typename T, int MOST>
int fill(Pieces<T, MOST>& t, int n, const void* const* g, void* const* out, const int64_t* counts) {
  t.n = 0;
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    const long long off = (long long)(((uintptr_t)g[i] & 15) / sizeof(T));
    t.g[t.n] = (const T*)g[i];
    t.out[t.n] = out ? (T*)out[i] : nullptr;
    t.count[t.n] = counts[i];
    t.first[t.n] = (int)chunks;
    chunks += (counts[i] + off + CHUNK - 1) / CHUNK;
    if (chunks > 2000000000LL) { cb200_set_error("global_norm: more than 8e12 elements"); return CB200_ERR_INVALID; }
    ++t.n;
  }
  t.first[t.n] = (int)chunks;
  return CB200_OK;
}

template <typename T, int MOST>
int norm_and_clip_table(cb200_stream* s, int n, const void* const* g, const int64_t* counts, void* const* out, double max_norm,
                        void* norm) {
  DeviceGuard guard(s->device);
  const int launches = n > MOST ? (n + MOST - 1) / MOST : 1;
  const int most = s->sm_count * 16;                  // CTAs of one launch
  void* block = nullptr;
  int* counter = nullptr;
  int rc = cb200_partials(s, sizeof(NormResult) + (size_t)launches * most * Squares<T>::N * sizeof(double), &block);
  if (rc) return rc;
  if ((rc = cb200_tile_flags(s, 1, &counter))) return rc;
  NormResult* result = (NormResult*)block;
  double* partials = (double*)(result + 1);
  static thread_local Pieces<T, MOST> t;             // up to 14 KB: off the caller's stack
  int slots = 0;
  for (int l = 0; l < launches; ++l) {
    const int at = l * MOST, m = n - at < MOST ? n - at : MOST;
    if ((rc = fill(t, m, g + at, out ? out + at : nullptr, counts + at))) return rc;
    int grid = t.first[t.n] < most ? t.first[t.n] : most;
    if (grid < 1) grid = 1;
    square_sum_kernel<T, MOST><<<grid, THREADS, 0, s->stream>>>(t, partials, slots, slots + grid, l == launches - 1, counter, result,
                                                                (T*)norm, out ? max_norm : INFINITY);
    CB_LAUNCH_CHECK(s);
    slots += grid;
  }
  if (!out) return CB200_OK;
  for (int l = launches - 1; l >= 0; --l) {          // the last launch's table is still filled
    const int at = l * MOST, m = n - at < MOST ? n - at : MOST;
    if (l != launches - 1 && (rc = fill(t, m, g + at, out + at, counts + at))) return rc;
    const int grid = t.first[t.n];
    if (grid < 1) continue;
    scale_kernel<T, MOST><<<grid, THREADS, 0, s->stream>>>(t, result);
    CB_LAUNCH_CHECK(s);
  }
  return CB200_OK;
}

template <typename T>
int norm_and_clip(cb200_stream* s, int n, const void* const* g, const int64_t* counts, void* const* out, double max_norm,
                  void* norm) {
  return n <= SMALL_TABLE ? norm_and_clip_table<T, SMALL_TABLE>(s, n, g, counts, out, max_norm, norm)
                          : norm_and_clip_table<T, TABLE>(s, n, g, counts, out, max_norm, norm);
}

int check_list(const char* what, cb200_stream* s, int dtype, int n, const void* const* g, const int64_t* counts) {
  CB_REQUIRE(s, "%s: null stream", what);
  CB_REQUIRE(dtype == CB200_FLOAT || dtype == CB200_DOUBLE, "%s: only float and double buffers", what);
  CB_REQUIRE(n >= 0 && n <= (1 << 20), "%s: %d buffers outside [0, 2^20]", what, n);
  CB_REQUIRE(n == 0 || (g && counts), "%s: null list", what);
  const uintptr_t size = cb200_dtype_size(dtype);
  for (int i = 0; i < n; ++i) {
    CB_REQUIRE(counts[i] >= 0, "%s: buffer %d has a negative element count", what, i);
    CB_REQUIRE(counts[i] == 0 || g[i], "%s: buffer %d is null", what, i);
    CB_REQUIRE(((uintptr_t)g[i] % size) == 0, "%s: buffer %d is not aligned to its element type", what, i);
  }
  return CB200_OK;
}

// Writing one result must not change what another one is computed from: destinations share no memory with one another,
// with the norm, or with any gradient but their own (in place).
struct Span { uintptr_t lo, hi; int index; };

int check_destinations(int n, const void* const* g, const int64_t* counts, void* const* out, const void* norm, size_t size) {
  std::unique_ptr<Span[]> spans(new (std::nothrow) Span[(size_t)2 * n + 1]);
  if (!spans) { cb200_set_error("clip_gradients: out of host memory"); return CB200_ERR_NOMEM; }
  Span* d = spans.get();
  int m = 0, k = 0;
  for (int i = 0; i < n; ++i)
    if (counts[i] > 0) d[m++] = {(uintptr_t)out[i], (uintptr_t)out[i] + (uintptr_t)counts[i] * size, i};
  Span* src = d + m;
  for (int i = 0; i < n; ++i)
    if (counts[i] > 0) src[k++] = {(uintptr_t)g[i], (uintptr_t)g[i] + (uintptr_t)counts[i] * size, i};
  if (norm) src[k++] = {(uintptr_t)norm, (uintptr_t)norm + size, -1};
  auto before = [](const Span& a, const Span& b) { return a.lo < b.lo; };
  std::sort(d, d + m, before);
  std::sort(src, src + k, before);
  for (int i = 1; i < m; ++i)
    CB_REQUIRE(d[i - 1].hi <= d[i].lo, "clip_gradients: destinations %d and %d overlap", d[i - 1].index, d[i].index);
  // destinations are disjoint and sorted: each source can only meet the ones from the first that ends behind its start
  for (int j = 0; j < k; ++j) {
    int a = 0, b = m;
    while (a < b) {
      const int c = (a + b) / 2;
      if (d[c].hi <= src[j].lo) a = c + 1; else b = c;
    }
    for (; a < m && d[a].lo < src[j].hi; ++a)
      CB_REQUIRE(src[j].index == d[a].index && src[j].lo == d[a].lo,
                 src[j].index < 0 ? "clip_gradients: destination %d overlaps the norm" : "clip_gradients: destination %d overlaps another gradient",
                 d[a].index);
  }
  // the same gradient twice, in place: the sources overlap, and each is its own destination -- caught above, since its
  // destinations overlap; a norm inside a gradient would change it before it is scaled
  if (norm)
    for (int j = 0; j < k; ++j)
      CB_REQUIRE(src[j].index < 0 || src[j].hi <= (uintptr_t)norm || (uintptr_t)norm + size <= src[j].lo,
                 "clip_gradients: gradient %d overlaps the norm", src[j].index);
  return CB200_OK;
}

}  // namespace

extern "C" {

int cb200_global_norm(cb200_stream* s, int dtype, int n, const void* const* gradients, const int64_t* counts, void* norm) {
  int rc = check_list("global_norm", s, dtype, n, gradients, counts);
  if (rc) return rc;
  CB_REQUIRE(norm, "global_norm: null norm");
  CB_REQUIRE(((uintptr_t)norm % cb200_dtype_size(dtype)) == 0, "global_norm: the norm is not aligned to its element type");
  return dtype == CB200_FLOAT ? norm_and_clip<float>(s, n, gradients, counts, nullptr, 0.0, norm)
                              : norm_and_clip<double>(s, n, gradients, counts, nullptr, 0.0, norm);
}

int cb200_clip_gradients(cb200_stream* s, int dtype, int n, const void* const* gradients, const int64_t* counts,
                         void* const* clipped, double max_norm, void* norm) {
  int rc = check_list("clip_gradients", s, dtype, n, gradients, counts);
  if (rc) return rc;
  CB_REQUIRE(max_norm > 0.0 && isfinite(max_norm), "clip_gradients: the bound must be positive and finite");
  CB_REQUIRE(n == 0 || clipped, "clip_gradients: null list of destinations");
  const uintptr_t size = cb200_dtype_size(dtype);
  for (int i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    CB_REQUIRE(clipped[i], "clip_gradients: destination %d is null", i);
    CB_REQUIRE(((uintptr_t)clipped[i] % size) == 0, "clip_gradients: destination %d is not aligned to its element type", i);
  }
  CB_REQUIRE(((uintptr_t)norm % size) == 0, "clip_gradients: the norm is not aligned to its element type");
  if ((rc = check_destinations(n, gradients, counts, clipped, norm, size))) return rc;
  return dtype == CB200_FLOAT ? norm_and_clip<float>(s, n, gradients, counts, clipped, max_norm, norm)
                              : norm_and_clip<double>(s, n, gradients, counts, clipped, max_norm, norm);
}

}  // extern "C"
