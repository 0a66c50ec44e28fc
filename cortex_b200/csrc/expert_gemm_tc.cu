// fp32 products grouped by expert on the 5th-generation tensor cores: the 3xTF32 scheme of gemm! (hi = the fp32 word, of
// which the tensor core reads the top 19 bits, lo = x - trunc(x); main and cross terms in two TMEM accumulators) over
// ragged groups whose bounds are read from device memory.
//
//   WEIGHTS = 0   128 x BN tile of C[rows, N]: rows of one group, that group's matrix as the B operand.  A tile that ends
//                 behind its group loads rows of the next one (rows of an accumulator are independent) and does not store
//                 them.  B is a 3-d tensor map, so a tile that ends behind its expert's matrix reads zeros.
//   WEIGHTS = 1   128 x BN tile of C_e [M, N] = A_e^T B_e: the reduction runs over the group's rows.  Both operands are
//                 MN-major; rows of the last k-block that belong to the next group are zeroed, hi tile included, by the
//                 warps that compute the lo tiles (so an infinity or a NaN there does not matter).
//
// Every CTA finds its tile itself (groups::find_tile, ~1 us, while TMEM and barriers are set up); the grid is the most
// tiles that the sizes allow, and CTAs without a tile leave at once.
// Reductions longer than `chunk` k-blocks are cut: the tensor core adds with truncation, so every chunk's sum is rounded
// to nearest onto C (or onto the slice's parked tile) and the accumulators restart from zero.
//
// Warp roles as in gemm_tf32x3_kernel: 0-7 lo tiles and epilogue, 8 TMA producer, 9 TMEM and MMA issue.
#include "gemm3x_common.cuh"
#include "expert_groups.cuh"
#include <mutex>
#include <type_traits>

using namespace sm100;
using namespace gemm3x;

namespace {

constexpr int BM = 128, BK = 16;
constexpr int CONV_WARPS = 8;
constexpr int THREADS = (CONV_WARPS + 2) * 32;
constexpr int BOX = BK * 128;                             // bytes of one 32 x BK MN-major TMA box

template <int BN> struct Cfg {
  static constexpr int A_TILE = BM * BK * 4, B_TILE = BN * BK * 4, RAW = A_TILE + B_TILE, STAGE = 2 * RAW;
  static constexpr int STAGES = (196608 / STAGE) > 8 ? 8 : (196608 / STAGE);
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
};

struct Grouped {
  GemmParams g;
  const int* offsets;
  int experts, rows;
  int chunk;               // k-blocks between roundings of the accumulators
  long long c_stride;      // WEIGHTS: distance of the experts' results
  int tiles_m;             // WEIGHTS: row tiles of one result
};

template <int BN, int WEIGHTS>
__global__ void __launch_bounds__(THREADS, 1)
expert_tf32x3_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ Grouped args) {
  typedef Cfg<BN> C;
  constexpr int STAGES = C::STAGES, A_TILE = C::A_TILE;
  constexpr bool MMA_WHOLE = BN < 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = (uint64_t*)(smem + STAGES * C::STAGE);
  // bars[0..S) full, [S..2S) conv, [2S..3S) empty, [3S] accumulators ready, [3S+1] accumulators read out
  uint32_t* tmem_slot = (uint32_t*)(bars + 3 * STAGES + 2);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  int* where = (int*)(tmem_slot + 3);                      // {found, expert, lo, hi, index}

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  GemmParams p = args.g;
  const int tiles_n = (p.N + BN - 1) / BN;
  const int unit = (int)blockIdx.x / p.ksplit_n, k_slice = (int)blockIdx.x - unit * p.ksplit_n;
  const int n0 = (unit % tiles_n) * BN;

  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_full = smem_u32(bars), bar_conv = smem_u32(bars + STAGES), bar_empty = smem_u32(bars + 2 * STAGES),
                 bar_acc = smem_u32(bars + 3 * STAGES), bar_read = bar_acc + 8;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_conv + 8 * s, CONV_WARPS);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_acc, 1);
    mbar_init(bar_read, CONV_WARPS);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == CONV_WARPS + 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == CONV_WARPS && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    groups::Tile t = {0, 0, 0, 0};
    bool found = true;
    if (WEIGHTS) {
      const int m_tile = unit / tiles_n;
      t.expert = m_tile / args.tiles_m;
      t.index = m_tile - t.expert * args.tiles_m;
      groups::group_rows(args.offsets, args.rows, t.expert, p.status, t.lo, t.hi);
    } else {
      found = groups::find_tile(args.offsets, args.experts, args.rows, BM, unit / tiles_n, p.status, t);
    }
    if (lane == 0) { where[0] = found; where[1] = t.expert; where[2] = t.lo; where[3] = t.hi; where[4] = t.index; }
  }
  int inject = 0;
  if (warp == CONV_WARPS) inject = p.status[3];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int expert = where[1], lo = where[2], hi = where[3];
  if (!where[0]) {
    // no such tile: with K slices every CTA of the tile's cluster leaves here
    if (warp == CONV_WARPS + 1) tmem_dealloc(tmem_base, C::TMEM_COLS);
    return;
  }
  int m0, nkb_all;
  if (WEIGHTS) {
    m0 = where[4] * BM;
    p.C += expert * args.c_stride;
    nkb_all = (hi - lo + BK - 1) / BK;
  } else {
    m0 = lo + where[4] * BM;
    p.M = hi;
    if (p.bias) p.bias += (long long)expert * p.N;
    nkb_all = (p.K + BK - 1) / BK;
  }
  const int kb_begin = (int)((long long)nkb_all * k_slice / p.ksplit_n);
  int nkb = (int)((long long)nkb_all * (k_slice + 1) / p.ksplit_n) - kb_begin;
  // an empty reduction (a group without rows, a slice without k-blocks): one k-block of zeros
  const bool empty = WEIGHTS && nkb == 0;
  if (empty) nkb = 1;
  const int n_chunks = (nkb + args.chunk - 1) / args.chunk, per = (nkb + n_chunks - 1) / n_chunks;

  if (warp == CONV_WARPS) {
    // ------------------------------ TMA producer ------------------------------
    auto producer = [&](auto whole_tag) {
      constexpr bool PROD_WHOLE = decltype(whole_tag)::value;
      if (!PROD_WHOLE && lane != 0) return;
      int issued = 0, s = 0;
      uint32_t ph = 0;
      const bool withhold = (inject & 1) != 0;              // host-injected fault: arm nothing, load nothing
      for (int i = 0; i < nkb; ++i) {
        if (!mbar_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 100 + s)) break;
        const uint32_t full = bar_full + 8 * s;
        const uint32_t a_dst = smem_base + s * C::STAGE, b_dst = a_dst + A_TILE;
        const int k0 = (kb_begin + i) * BK;
        if (withhold) {
          if (++s == STAGES) { s = 0; ph ^= 1; }
          continue;
        }
        if (!PROD_WHOLE || elect_one()) {
          mbar_arrive_expect_tx(full, C::RAW);
          if (WEIGHTS) {
#pragma unroll
            for (int j = 0; j < BM / 32; ++j) tma_load_2d(a_dst + j * BOX, &tmA, m0 + 32 * j, lo + k0, full);
#pragma unroll
            for (int j = 0; j < BN / 32; ++j) tma_load_2d(b_dst + j * BOX, &tmB, n0 + 32 * j, lo + k0, full);
          } else {
            tma_load_2d(a_dst, &tmA, k0, m0, full);
            if (!p.b_mn_major) {
              tma_load_3d(b_dst, &tmB, k0, n0, expert, full);
            } else {
#pragma unroll
              for (int j = 0; j < BN / 32; ++j) tma_load_3d(b_dst + j * BOX, &tmB, n0 + 32 * j, k0, expert, full);
            }
          }
        }
        issued = i + 1;
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (*abort_flag) {
        for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
          for (int it = 0; it < (1 << 16); ++it)
            if (mbar_try_wait(bar_full + 8 * (i % STAGES), (i / STAGES) & 1)) break;
      }
    };
    if (BN < 256 || WEIGHTS || p.b_mn_major) producer(std::true_type{});
    else producer(std::false_type{});
  } else if (warp == CONV_WARPS + 1) {
    // ------------------------------ MMA issuer --------------------------------
    if (MMA_WHOLE || lane == 0) {
      const int b_mn = WEIGHTS ? 1 : p.b_mn_major;
      const uint32_t idesc = make_idesc_tf32(BM, BN, WEIGHTS, b_mn);
      constexpr uint32_t K_SBO = 8 * BK * 4;
      const uint32_t a_lbo = WEIGHTS ? (uint32_t)BOX : 16u, b_lbo = b_mn ? (uint32_t)BOX : 16u;
      const uint32_t a_sbo = WEIGHTS ? 512u : K_SBO, b_sbo = b_mn ? 512u : K_SBO;
      const uint32_t a_sw = WEIGHTS ? SWZ_128B_BASE32B : SWZ_64B, b_sw = b_mn ? SWZ_128B_BASE32B : SWZ_64B;
      const uint32_t a_step = (WEIGHTS ? 1024u : 32u) >> 4, b_step = (b_mn ? 1024u : 32u) >> 4;
      const uint32_t tmem_main = tmem_base, tmem_cross = tmem_base + BN;
      const uint64_t d_a = make_smem_desc(smem_base, a_lbo, a_sbo, a_sw);
      const uint64_t d_b = make_smem_desc(smem_base + A_TILE, b_lbo, b_sbo, b_sw);
      const uint32_t a_hiw = (uint32_t)(d_a >> 32), b_hiw = (uint32_t)(d_b >> 32);
      const uint32_t a_low0 = (uint32_t)d_a, b_low0 = (uint32_t)d_b;
      constexpr uint32_t LO_TILE = C::RAW >> 4, STAGE_STEP = C::STAGE >> 4;
      uint32_t accumulate = 0, ph = 0, stage_off = 0, rph = 0;
      int s = 0, in_chunk = 0;
      int commits = 0;
      for (int i = 0; i < nkb; ++i) {
        if (in_chunk == per) {
          // the chunk's sums go out before its accumulators are overwritten
          if (!MMA_WHOLE || elect_one()) mma_commit(bar_acc);
          if (MMA_WHOLE) __syncwarp();
          ++commits;
          if (!mbar_wait(bar_read, rph, abort_flag, p.status, 250)) break;
          rph ^= 1;
          tc_fence_after();
          in_chunk = 0;
          accumulate = 0;
        }
        ++in_chunk;
        if (!mbar_wait(bar_conv + 8 * s, ph, abort_flag, p.status, 200 + s)) break;
        tc_fence_after();
        if (!MMA_WHOLE || elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BK / 8; ++kk) {
            const uint32_t al = a_low0 + stage_off + kk * a_step, bl = b_low0 + stage_off + kk * b_step;
            mma_tf32_ss_words(tmem_cross, al + LO_TILE, a_hiw, bl, b_hiw, idesc, kk ? 1u : accumulate);
            mma_tf32_ss_words(tmem_cross, al, a_hiw, bl + LO_TILE, b_hiw, idesc, 1);
            mma_tf32_ss_words(tmem_main, al, a_hiw, bl, b_hiw, idesc, kk ? 1u : accumulate);
          }
          mma_commit(bar_empty + 8 * s);
        }
        accumulate = 1;
        if (MMA_WHOLE) __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1; stage_off = 0; } else { stage_off += STAGE_STEP; }
      }
      if (!MMA_WHOLE || elect_one()) mma_commit(bar_acc);
      if (MMA_WHOLE) __syncwarp();
      if (*abort_flag) {
        // every MMA issued must have retired before TMEM is freed: the phase of the commit above
        for (int it = 0; it < (1 << 16); ++it)
          if (mbar_try_wait(bar_acc, (uint32_t)(commits & 1))) break;
      }
    }
  } else {
    // ------------------- hi / lo split, then epilogue (warps 0-7) ---------------
    const int tid = threadIdx.x;
    bool ok = true;
    int i = 0;
    for (int c = 0; ok && c < n_chunks; ++c) {
      const int end = min(nkb, (c + 1) * per);
      for (; i < end; ++i) {
        const int s = i % STAGES, ph = (i / STAGES) & 1;
        if (!mbar_wait(bar_full + 8 * s, ph, abort_flag, p.status, 300 + s)) { ok = false; break; }
        uint8_t* raw = smem + s * C::STAGE;
        uint8_t* low = raw + C::RAW;
        const int valid = empty ? 0 : (WEIGHTS ? hi - lo - (kb_begin + i) * BK : BK);      // rows of this k-block inside the group
        if (WEIGHTS && valid < BK) {
#pragma unroll 1
          for (int off = tid * 16; off < C::RAW; off += CONV_WARPS * 32 * 16)
            if (((off & (BOX - 1)) >> 7) >= valid) *reinterpret_cast<float4*>(raw + off) = make_float4(0.f, 0.f, 0.f, 0.f);
          // every thread zeroed 16-byte pieces that it reads itself below
        }
#pragma unroll
        for (int k = 0; k < C::RAW / 16 / (CONV_WARPS * 32); ++k) {
          const int off = (tid + k * CONV_WARPS * 32) * 16;
          const float4 v = *reinterpret_cast<const float4*>(raw + off);
          float4 l;
          l.x = lo_part(v.x); l.y = lo_part(v.y); l.z = lo_part(v.z); l.w = lo_part(v.w);
          *reinterpret_cast<float4*>(low + off) = l;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_conv + 8 * s);
      }
      if (ok) ok = mbar_wait(bar_acc, (uint32_t)(c & 1), abort_flag, p.status, 400);
      ok = __all_sync(0xffffffffu, ok);                      // tcgen05.ld below is warp-collective
      if (!ok) break;
      tc_fence_after();
      const bool last = c + 1 == n_chunks;
      if (p.ksplit_n > 1) {
        if (p.ksplit_cluster) {
          dump_tile_smem<BN>(p, tmem_base, reinterpret_cast<float*>(smem), warp, lane);      // one chunk only
        } else {
          float* park = p.ksplit_ws + ((long long)unit * p.ksplit_n + k_slice) * (BM * BN);
          if (c == 0) dump_tile<BN>(p, tmem_base, park, warp, lane);
          else add_tile<BN>(tmem_base, park, warp, lane);
        }
      } else {
        // staging lies in the pipeline stages, which are free only behind the last k-block
        epilogue_tile<BN>(p, tmem_base, m0, n0, warp, lane, last ? reinterpret_cast<float*>(smem) : nullptr,
                          c == 0 ? p.beta : 1.f, last, c > 0);
      }
      if (!last) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_read);
      }
    }
    if (p.ksplit_n > 1 && !p.ksplit_cluster) {
      // slices parked in L2: the CTA that arrives last sums them in slice order and stores; nobody waits
      if (ok) __threadfence();
      asm volatile("bar.sync 1, %0;" ::"n"(CONV_WARPS * 32) : "memory");
      int* arrived = reinterpret_cast<int*>(tmem_slot + 2);
      if (threadIdx.x == 0) *arrived = *abort_flag ? -1 : atomicAdd(p.tile_flags + unit, 1);
      asm volatile("bar.sync 1, %0;" ::"n"(CONV_WARPS * 32) : "memory");
      if (*arrived == p.ksplit_n - 1) {
        __threadfence();
        epilogue_tile<BN>(p, tmem_base, m0, n0, warp, lane, reinterpret_cast<float*>(smem), p.beta, true, false, nullptr,
                          p.ksplit_ws + (long long)unit * p.ksplit_n * (BM * BN), p.ksplit_n);
        if (threadIdx.x == 0) p.tile_flags[unit] = 0;        // left zero for the next launch
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (p.ksplit_n > 1 && p.ksplit_cluster) {
    cluster_sync_all();
    if (warp < CONV_WARPS && !*abort_flag) {
      const int n = p.ksplit_n, rank = (int)cluster_ctarank();
      constexpr int ITEMS = 8 * (BN / 64);
      float* staging = reinterpret_cast<float*>(smem + 128 * BN * 4);       // behind the parked tile
      for (int it = rank + n * warp; it < ITEMS; it += n * CONV_WARPS)
        epilogue_tile<BN>(p, tmem_base, m0, n0, warp, lane, staging, p.beta, true, false, nullptr, nullptr, n, smem_u32(smem), it);
    }
    cluster_sync_all();
  }
  if (warp == CONV_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ------------------------------ host side -------------------------------------

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

int tmap(CUtensorMap* tm, const float* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
         CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) { cb200_set_error("cuTensorMapEncodeTiled is not available from this driver"); return CB200_ERR_CUDA; }
  const cuuint32_t ones[3] = {1, 1, 1};
  CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, (cuuint32_t)rank, (void*)base, dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { cb200_set_error("cuTensorMapEncodeTiled failed with %d", (int)r); return CB200_ERR_CUDA; }
  return CB200_OK;
}

int tmap_2d(CUtensorMap* tm, const float* base, long long rows, long long cols, long long ld, int box_cols, int box_rows,
            CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 4};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  return tmap(tm, base, 2, dims, strides, box, swizzle);
}

int tmap_3d(CUtensorMap* tm, const float* base, long long count, long long rows, long long cols, long long ld, long long stride,
            int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 4, (cuuint64_t)stride * 4};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  return tmap(tm, base, 3, dims, strides, box, swizzle);
}

template <int BN, int WEIGHTS> cudaError_t attributes(int dev) {
  static std::once_flag once[64];
  static cudaError_t result[64];
  std::call_once(once[dev & 63], [&] {
    result[dev & 63] = cudaFuncSetAttribute(expert_tf32x3_kernel<BN, WEIGHTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::SMEM);
  });
  return result[dev & 63];
}

template <int BN, int WEIGHTS>
int launch(cb200_stream* s, const CUtensorMap& tmA, const CUtensorMap& tmB, const Grouped& a, long long ctas) {
  cudaError_t e = attributes<BN, WEIGHTS>(s->device);
  if (e != cudaSuccess) return cb200_cuda_fail(e, "cudaFuncSetAttribute", __FILE__, __LINE__);
  CB_REQUIRE(ctas <= 2147483647LL, "expert_gemm: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg<BN>::SMEM;
  cfg.stream = s->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.g.ksplit_cluster ? (unsigned)a.g.ksplit_n : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.g.ksplit_cluster ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, expert_tf32x3_kernel<BN, WEIGHTS>, tmA, tmB, a);
  if (e != cudaSuccess) return cb200_cuda_fail(e, "cudaLaunchKernelEx(expert_tf32x3_kernel)", __FILE__, __LINE__);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

// Tile width and K slices for `tiles_m` row tiles (an estimate for ragged groups) of N columns reduced over `nkb`
// k-blocks: the timing model of gemm!, t = waves x (5 us + k-blocks per slice x c[BN]) + hand-over.
void choose(const cb200_stream* s, long long tiles_m, int N, int nkb, int max_slices, int& bn_out, int& slices_out) {
  const int bn_max = N > 128 ? 256 : (N > 64 ? 128 : 64);
  double best = 1e30;
  bn_out = bn_max;
  slices_out = 1;
  for (int bn = 256; bn >= 64; bn >>= 1) {
    if (bn > bn_max) continue;
    if (s->opt_gemm_tile_n > 0 && bn != s->opt_gemm_tile_n && s->opt_gemm_tile_n <= bn_max) continue;
    const double c = bn == 256 ? 0.56 : (bn == 128 ? 0.455 : 0.39);
    const long long tiles = tiles_m * ((N + bn - 1) / bn);
    for (int sl = 1; sl <= max_slices; ++sl) {
      if (sl > 1 && (tiles * sl > s->sm_count || nkb / sl < 4)) break;
      if (s->opt_gemm_k_slices > 0 && sl != s->opt_gemm_k_slices && s->opt_gemm_k_slices <= max_slices && nkb / s->opt_gemm_k_slices >= 4) continue;
      const long long waves = (tiles * sl + s->sm_count - 1) / s->sm_count;
      const double t = (double)waves * (5.0 + (double)((nkb + sl - 1) / sl) * c) + (sl > 1 ? (bn / 64) * (1.3 + 0.45 * sl) : 0.0);
      if (t < best - 1e-9) { best = t; bn_out = bn; slices_out = sl; }
    }
  }
}

void common(GemmParams& g, cb200_stream* s, float* C, long long ldc, int M, int N, int K, float alpha, float beta, const float* bias,
            int act) {
  g.C = C; g.ldc = ldc; g.M = M; g.N = N; g.K = K; g.alpha = alpha; g.beta = beta; g.bias = bias; g.act = act;
  g.a_mn_major = g.b_mn_major = 0;
  g.store_mode = STORE_ROW_MAJOR; g.hw = 1; g.flags = 0; g.group_n = 1; g.drain_every = 0; g.C_lo = nullptr;
  g.k_split = 1; g.split_from = 0; g.partials = nullptr; g.split_block = 1;
  g.ksplit_n = 1; g.ksplit_cluster = 0; g.ksplit_ws = nullptr; g.tile_flags = nullptr; g.status = s->status_dev;
  g.n_peers = 0;
  for (int d = 0; d < MAX_PEERS; ++d) g.peers[d] = nullptr;
}

// k-blocks between roundings: 2048 values of k, where the truncating additions have shrunk a sum by 1.4e-5 at most
constexpr int CHUNK = 2048 / BK;

}  // namespace

// Operands that TMA can address: 16-byte bases, pitches and distances that are multiples of 4 elements.
bool cb200_expert_tc_ok(const void* A, long long lda, const void* B, long long ldb, long long b_stride) {
  return ((((uintptr_t)A | (uintptr_t)B) & 15) == 0) && lda % 4 == 0 && ldb % 4 == 0 && b_stride % 4 == 0;
}

int cb200_expert_rows_tc(cb200_stream* s, float* C, long long ldc, int trans_b, float alpha, const float* A, int rows, int K,
                         long long lda, const float* B, int experts, int N, long long b_stride, long long ldb, float beta,
                         const int* offsets, const float* bias, int act) {
  DeviceGuard guard(s->device);
  Grouped a;
  common(a.g, s, C, ldc, 0, N, K, alpha, beta, bias, act);
  a.g.b_mn_major = trans_b ? 0 : 1;
  a.offsets = offsets; a.experts = experts; a.rows = rows; a.chunk = CHUNK; a.c_stride = 0; a.tiles_m = 0;
  const long long most = (rows + BM - 1) / BM + (experts < rows ? experts : rows) - (experts > 0 ? 1 : 0);
  const long long tiles_m = most < 1 ? 1 : most;
  const int nkb = (K + BK - 1) / BK;
  int BN, slices;
  // a slice is one chunk: its parked tile is in shared memory, which the next chunk's stages would need
  choose(s, tiles_m, N, nkb, K <= 8 * 2048 ? 8 : 1, BN, slices);
  if (slices > 1 && (nkb + slices - 1) / slices > CHUNK) slices = 1;
  a.g.ksplit_n = slices;
  a.g.ksplit_cluster = slices > 1;
  CUtensorMap tmA, tmB;
  int rc = tmap_2d(&tmA, A, rows, K, lda, BK, BM, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc) return rc;
  if (trans_b) rc = tmap_3d(&tmB, B, experts, N, K, ldb, b_stride, BK, BN, CU_TENSOR_MAP_SWIZZLE_64B);
  else rc = tmap_3d(&tmB, B, experts, K, N, ldb, b_stride, 32, BK, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B);
  if (rc) return rc;
  const long long ctas = tiles_m * ((N + BN - 1) / BN) * slices;
  if (BN == 256) return launch<256, 0>(s, tmA, tmB, a, ctas);
  if (BN == 128) return launch<128, 0>(s, tmA, tmB, a, ctas);
  return launch<64, 0>(s, tmA, tmB, a, ctas);
}

int cb200_expert_weights_tc(cb200_stream* s, float* C, long long c_stride, long long ldc, float alpha, const float* A, int rows,
                            int M, long long lda, const float* B, int N, long long ldb, int experts, float beta,
                            const int* offsets) {
  DeviceGuard guard(s->device);
  Grouped a;
  common(a.g, s, C, ldc, M, N, 0, alpha, beta, nullptr, CB200_ACT_NONE);
  a.g.a_mn_major = a.g.b_mn_major = 1;
  a.offsets = offsets; a.experts = experts; a.rows = rows; a.chunk = CHUNK; a.c_stride = c_stride;
  a.tiles_m = (M + BM - 1) / BM;
  const long long tiles_m = (long long)a.tiles_m * experts;
  int BN, slices;
  choose(s, tiles_m, N, (rows / experts + BK) / BK, 16, BN, slices);
  a.g.ksplit_n = slices;
  int rc;
  const long long units = tiles_m * ((N + BN - 1) / BN);
  if (slices > 1) {
    // slices meet in L2: how long a slice is depends on the groups, so it may take several chunks
    void* ws = nullptr;
    if ((rc = cb200_partials(s, (size_t)units * slices * BM * BN * sizeof(float), &ws))) return rc;
    if ((rc = cb200_tile_flags(s, (size_t)units, &a.g.tile_flags))) return rc;
    a.g.ksplit_ws = (float*)ws;
  }
  CUtensorMap tmA, tmB;
  if ((rc = tmap_2d(&tmA, A, rows, M, lda, 32, BK, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B))) return rc;
  if ((rc = tmap_2d(&tmB, B, rows, N, ldb, 32, BK, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B))) return rc;
  if (BN == 256) return launch<256, 1>(s, tmA, tmB, a, units * slices);
  if (BN == 128) return launch<128, 1>(s, tmA, tmB, a, units * slices);
  return launch<64, 1>(s, tmA, tmB, a, units * slices);
}
