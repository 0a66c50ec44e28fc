// fp32 products grouped by expert on the 5th-generation tensor cores: the 3xTF32 scheme of gemm! (hi = the fp32 word, of
// which the tensor core reads the top 19 bits, lo = x - trunc(x); main and cross terms in two TMEM accumulators) over
// ragged groups whose bounds are read from device memory.
//
// One kernel: C[r, :] for the rows r of a group, the group's matrix as the other operand (a 3-d tensor map, so a tile that ends
// behind its expert's matrix reads zeros); and C_e = A_e^T B_e, reduced over the group's rows.
//
// Every CTA finds its tile itself (groups::find_tile, ~1 us, while TMEM and barriers are set up); the grid is the most
// tiles that the sizes allow, and CTAs without a tile leave at once.
// The tensor core adds with truncation, which shrinks a sum by about 2e-9 of itself for every value of k it runs over: an
// accumulator takes RUN of them at most (512: 1.5e-6 of error against 64 bits, 256: 0.9e-6), several take turns, and what is
// longer is cut into chunks whose sums are rounded to nearest onto C (or onto the slice's parked tile).
//
// Warp roles as in gemm_tf32x3_kernel: 0-7 lo tiles and epilogue, 8 TMA producer, 9 TMEM and MMA issue.
#include "gemm3x_common.cuh"
#include "expert_groups.cuh"
#include <mutex>

using namespace sm100;
using namespace gemm3x;

namespace {

constexpr int BM = 128;
constexpr int RUN = 256;                                  // values of k that one main accumulator adds up at most
constexpr int CONV_WARPS = 8;
constexpr int THREADS = (CONV_WARPS + 2) * 32;

// The whole warp waits, and agrees: lanes that gave up never leave others behind in a warp-wide operation.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, site));
}

// ---- C[r, :] for the rows of every group ------------------------------------------------------------------------
// The expert's matrix is the operand with 128 rows (its N output features, whole tiles but the last) and the ragged
// rows of the group are the other one, up to BN of them: the tensor core takes any multiple of 16 there, so a group of
// 30 rows costs 32 columns of accumulator, not 128 lanes.  A tile's columns that belong to the next group are computed
// (columns of an accumulator are independent) and not stored.  Lane = output feature in TMEM, so the 32 lanes of a warp
// store 128 consecutive bytes of a row of C whatever its pitch and alignment.
//
// ---- C_e = A_e^T B_e over the rows of every group (WEIGHTS) -------------------------------------------------------
// The same kernel with the columns of B in the lanes (128 consecutive values of a row of C_e) and the columns of A, up
// to BN of them, in the accumulator's columns: both operands reduce down their columns (MN-major), over the group's
// rows; rows of the last k-block that belong to the next group are zeroed by the warps that compute the lo tiles.
// K slices meet in L2 (how long a slice is depends on the group; products whose slices are longer than a chunk do it too):
// the CTA that arrives last adds them in order and stores; nobody waits.
struct RowsArgs {
  float* C;
  long long ldc;
  long long c_stride;          // WEIGHTS: distance of the experts' results
  int cols, tiles_r;           // WEIGHTS: rows of a result (columns of A), tiles of BN of them
  float* park;                 // K slices that meet in L2: parked tiles
  int* arrived;                // and arrival counts, zero between launches
  const float* bias;           // [experts, N] or null
  const int* offsets;
  int* status;
  int N, K, experts, rows;
  int units;                   // most tiles there can be
  int w_mn;                    // the matrices are [K, N]: N is their contiguous axis
  int act;
  float alpha, beta;
  const int* only_if;          // null, or a device word: do nothing while it is zero
  int slices;                  // CTAs of a cluster that share a tile, each over a slice of K
};

template <int BN, int BK> struct RowsCfg {
  static constexpr int A_TILE = BM * BK * 4, B_TILE = BN * BK * 4, RAW = A_TILE + B_TILE, STAGE = 2 * RAW;
  // narrow tiles: two CTAs per SM, one streaming while the other sets up or stores
  static constexpr int CTAS = BN <= 64 ? 2 : 1;
  static constexpr int STAGES = (196608 / CTAS / STAGE) > 8 ? 8 : (196608 / CTAS / STAGE);
  // main accumulators that take turns, joined in the epilogue; a reduction longer than a chunk goes out to C in between
  static constexpr int MAINS = BN == 32 ? 4 : 3;
  static constexpr int CHUNK = MAINS * RUN / BK;                               // k-blocks
  static constexpr int TMEM_COLS = BN == 32 ? 256 : (MAINS + 1) * BN;          // mains, then the cross terms
  static constexpr int BOX_ROWS = BN < 64 ? BN : 64;          // rows of one TMA box of the ragged operand
  static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
  static_assert(BM * BN * 4 <= STAGES * STAGE, "a parked tile must fit the pipeline stages");
};

// A guarded launch is set up while its predecessors end, and waits for them here.
__device__ __forceinline__ bool nothing_to_do(const int* only_if) {
  if (!only_if) return false;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  return *only_if == 0;
}

// 32 accumulator columns (rows first .. first + 31 of C) of one output feature per lane.  No branch between the values: one
// per value (the activation's) keeps a warp from having more than one in flight (42 cycles a store; a weight gradient of 8
// experts of 1024 x 4096 with 32 rows each 121 us, 68 without).
__device__ __forceinline__ void store_columns(const RowsArgs& p, float* C, uint32_t (&r)[32], int first, int hi, int n,
                                              const float* bias, float beta, bool last) {
  if (n >= p.N) return;
  float* c = C + (long long)first * p.ldc + n;
  const float b = (bias && last) ? bias[n] : 0.f;
  const int left = hi - first;
  if (beta != 0.f) {
    float old[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) old[j] = j < left ? c[(long long)j * p.ldc] : 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(p.alpha * __uint_as_float(r[j]) + beta * old[j] + b);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(p.alpha * __uint_as_float(r[j]) + b);
  }
  if (last && p.act == CB200_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(groups::relu(__uint_as_float(r[j])));
  } else if (last && p.act != CB200_ACT_NONE) {
#pragma unroll
    for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(apply_act(__uint_as_float(r[j]), p.act));
  }
  if (left >= 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j) c[(long long)j * p.ldc] = __uint_as_float(r[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) c[(long long)j * p.ldc] = __uint_as_float(r[j]);
  }
}

template <int BN, int BK, bool WEIGHTS>
__global__ void __launch_bounds__(THREADS, RowsCfg<BN, BK>::CTAS)
expert_tf32x3_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ RowsArgs p) {
  typedef RowsCfg<BN, BK> C;
  constexpr int STAGES = C::STAGES, A_TILE = C::A_TILE;
  constexpr int W_BOX = BK * 128;                            // bytes of one 32 x BK box of an MN-major matrix
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = (uint64_t*)(smem + STAGES * C::STAGE);
  // bars[0..S) full, [S..2S) conv, [2S..3S) empty, [3S] accumulators ready, [3S+1] accumulators read out
  uint32_t* tmem_slot = (uint32_t*)(bars + 3 * STAGES + 2);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  int* where = (int*)(tmem_slot + 2);                        // {found, expert, lo, hi, index}, then a word for arrivals

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (nothing_to_do(p.only_if)) return;
  const int tiles_n = (p.N + BM - 1) / BM;
  const int first_unit = (int)blockIdx.x / p.slices, slice = (int)blockIdx.x - first_unit * p.slices;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_full = smem_u32(bars), bar_conv = smem_u32(bars + STAGES), bar_empty = smem_u32(bars + 2 * STAGES),
                 bar_acc = smem_u32(bars + 3 * STAGES), bar_read = bar_acc + 8;
  if (warp == CONV_WARPS + 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == CONV_WARPS && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  int inject = 0;
  if (warp == CONV_WARPS) inject = p.status[3];
  // One tile per CTA; a guarded launch (only_if) has a small grid whose CTAs take tiles in turn.
#pragma unroll 1
  for (int unit = first_unit; unit < p.units; unit += (int)gridDim.x / p.slices) {
  const int n0 = (unit % tiles_n) * BM;
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
  if (warp == 1) {
    groups::Tile t = {0, 0, 0, 0};
    bool found = true;
    if (WEIGHTS) {
      const int rest = unit / tiles_n;
      t.expert = rest / p.tiles_r;
      t.index = rest - t.expert * p.tiles_r;
      groups::group_rows(p.offsets, p.rows, t.expert, p.status, t.lo, t.hi);
    } else {
      found = groups::find_tile(p.offsets, p.experts, p.rows, BN, unit / tiles_n, p.status, t);
    }
    if (lane == 0) { where[0] = found; where[1] = t.expert; where[2] = t.lo; where[3] = t.hi; where[4] = t.index; }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (!where[0]) {
    // no such tile (and none behind it): with K slices every CTA of the tile's cluster leaves here
    if (warp == CONV_WARPS + 1) tmem_dealloc(tmem_base, C::TMEM_COLS);
    return;
  }
  // rows t0 .. hi - 1 of C (of C_e) belong to this tile, as far as its columns go
  const int expert = where[1], g_lo = where[2], g_hi = where[3];
  const int t0 = WEIGHTS ? where[4] * BN : g_lo + where[4] * BN, hi = WEIGHTS ? p.cols : g_hi;
  const int cols = min(BN, hi - t0);                         // accumulator columns
  const int boxes = WEIGHTS ? (cols + 31) / 32 : (cols + C::BOX_ROWS - 1) / C::BOX_ROWS;
  const int raw_bytes = A_TILE + boxes * (WEIGHTS ? W_BOX : C::BOX_ROWS * BK * 4);
  float* const out = WEIGHTS ? p.C + expert * p.c_stride : p.C;
  const int nkb_all = ((WEIGHTS ? g_hi - g_lo : p.K) + BK - 1) / BK;
  const int kb_begin = (int)((long long)nkb_all * slice / p.slices);
  int nkb = (int)((long long)nkb_all * (slice + 1) / p.slices) - kb_begin;
  // an empty reduction (a group without rows, a slice without k-blocks): one k-block of zeros
  const bool empty = WEIGHTS && nkb == 0;
  if (empty) nkb = 1;
  const int n_chunks = (nkb + C::CHUNK - 1) / C::CHUNK, per = (nkb + n_chunks - 1) / n_chunks;
  const int run = max((per + C::MAINS - 1) / C::MAINS, RUN / BK);              // k-blocks into one main accumulator
  const float* bias = p.bias ? p.bias + (long long)expert * p.N : nullptr;

  if (warp == CONV_WARPS) {
    // ------------------------------ TMA producer ------------------------------
    int issued = 0, s = 0;
    uint32_t ph = 0;
    const bool withhold = (inject & 1) != 0;                 // host-injected fault: arm nothing, load nothing
    for (int i = 0; i < nkb; ++i) {
      if (!warp_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 100 + s)) break;
      const uint32_t full = bar_full + 8 * s;
      const uint32_t w_dst = smem_base + s * C::STAGE, x_dst = w_dst + A_TILE;
      const int k0 = (kb_begin + i) * BK;
      if (!withhold && elect_one()) {
        mbar_arrive_expect_tx(full, (uint32_t)raw_bytes);
        if (WEIGHTS) {
#pragma unroll
          for (int j = 0; j < BM / 32; ++j) tma_load_2d(w_dst + j * W_BOX, &tmW, n0 + 32 * j, g_lo + k0, full);
          for (int j = 0; j < boxes; ++j) tma_load_2d(x_dst + j * W_BOX, &tmX, t0 + 32 * j, g_lo + k0, full);
        } else if (!p.w_mn) {
          tma_load_3d(w_dst, &tmW, k0, n0, expert, full);
        } else {
#pragma unroll
          for (int j = 0; j < BM / 32; ++j) tma_load_3d(w_dst + j * W_BOX, &tmW, n0 + 32 * j, k0, expert, full);
        }
        if (!WEIGHTS)
          for (int j = 0; j < boxes; ++j) tma_load_2d(x_dst + j * C::BOX_ROWS * BK * 4, &tmX, k0, t0 + j * C::BOX_ROWS, full);
      }
      if (!withhold) issued = i + 1;
      if (++s == STAGES) { s = 0; ph ^= 1; }
    }
    if (*abort_flag) {
      // copies already issued land before this CTA gives its shared memory back
      for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
        for (int it = 0; it < (1 << 16); ++it)
          if (mbar_try_wait(bar_full + 8 * (i % STAGES), (i / STAGES) & 1)) break;
    }
  } else if (warp == CONV_WARPS + 1) {
    // ------------------------------ MMA issuer --------------------------------
    {
      const bool a_mn = WEIGHTS || p.w_mn;
      const uint32_t idesc = make_idesc_tf32(BM, (cols + 15) / 16 * 16, a_mn, WEIGHTS);
      constexpr uint32_t K_SWZ = BK == 32 ? SWZ_128B : SWZ_64B, K_SBO = 8 * BK * 4;
      const uint32_t a_step = (a_mn ? 1024u : 32u) >> 4;
      constexpr uint32_t b_step = (WEIGHTS ? 1024u : 32u) >> 4;
      const uint32_t tmem_cross = tmem_base + C::MAINS * BN;
      const uint64_t d_a = a_mn ? make_smem_desc(smem_base, W_BOX, 512, SWZ_128B_BASE32B) : make_smem_desc(smem_base, 16, K_SBO, K_SWZ);
      const uint64_t d_b = WEIGHTS ? make_smem_desc(smem_base + A_TILE, W_BOX, 512, SWZ_128B_BASE32B)
                                   : make_smem_desc(smem_base + A_TILE, 16, K_SBO, K_SWZ);
      const uint32_t a_hiw = (uint32_t)(d_a >> 32), b_hiw = (uint32_t)(d_b >> 32);
      const uint32_t a_low0 = (uint32_t)d_a, b_low0 = (uint32_t)d_b;
      constexpr uint32_t LO_TILE = C::RAW >> 4, STAGE_STEP = C::STAGE >> 4;
      uint32_t accumulate = 0, cross = 0, ph = 0, stage_off = 0, rph = 0, tmem_main = tmem_base;
      int s = 0, in_chunk = 0, in_run = 0, commits = 0;
      for (int i = 0; i < nkb; ++i) {
        if (in_chunk == per) {
          // the chunk's sums go out before its accumulators are overwritten
          if (elect_one()) mma_commit(bar_acc);
          __syncwarp();
          ++commits;
          if (!warp_wait(bar_read, rph, abort_flag, p.status, 250)) break;
          rph ^= 1;
          tc_fence_after();
          in_chunk = in_run = 0;
          accumulate = cross = 0;
          tmem_main = tmem_base;
        }
        if (C::MAINS > 1 && in_run == run) {
          in_run = 0;
          accumulate = 0;
          tmem_main += BN;
        }
        ++in_chunk;
        ++in_run;
        if (!warp_wait(bar_conv + 8 * s, ph, abort_flag, p.status, 200 + s)) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BK / 8; ++kk) {
            const uint32_t al = a_low0 + stage_off + kk * a_step, bl = b_low0 + stage_off + kk * b_step;
            mma_tf32_ss_words(tmem_cross, al + LO_TILE, a_hiw, bl, b_hiw, idesc, kk ? 1u : cross);
            mma_tf32_ss_words(tmem_cross, al, a_hiw, bl + LO_TILE, b_hiw, idesc, 1);
            mma_tf32_ss_words(tmem_main, al, a_hiw, bl, b_hiw, idesc, kk ? 1u : accumulate);
          }
          mma_commit(bar_empty + 8 * s);
        }
        accumulate = cross = 1;
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1; stage_off = 0; } else { stage_off += STAGE_STEP; }
      }
      if (elect_one()) mma_commit(bar_acc);
      __syncwarp();
      if (*abort_flag) {
        // every MMA issued must have retired before TMEM is freed: the phase of the commit above
        for (int it = 0; it < (1 << 16); ++it)
          if (mbar_try_wait(bar_acc, (uint32_t)(commits & 1))) break;
      }
    }
  } else {
    // ------------------- hi / lo split, then epilogue (warps 0-7) ---------------
    const int tid = threadIdx.x, q = warp & 3, half = warp >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16);
    bool ok = true;
    int i = 0;
    for (int c = 0; ok && c < n_chunks; ++c) {
      const int end = min(nkb, (c + 1) * per);
      for (; i < end; ++i) {
        const int s = i % STAGES, ph = (i / STAGES) & 1;
        if (!warp_wait(bar_full + 8 * s, ph, abort_flag, p.status, 300 + s)) { ok = false; break; }
        uint8_t* raw = smem + s * C::STAGE;
        uint8_t* low = raw + C::RAW;
        auto split = [&](int off) {
          const float4 v = *reinterpret_cast<const float4*>(raw + off);
          float4 l;
          l.x = lo_part(v.x); l.y = lo_part(v.y); l.z = lo_part(v.z); l.w = lo_part(v.w);
          *reinterpret_cast<float4*>(low + off) = l;
        };
        constexpr int PASS = CONV_WARPS * 32 * 16;
        if (WEIGHTS) {
          const int valid = empty ? 0 : g_hi - g_lo - (kb_begin + i) * BK;       // rows of this k-block inside the group
          if (valid < BK) {
            // (the 16-byte pieces that this thread reads itself below; a k row is 128 bytes of every box)
#pragma unroll 1
            for (int off = tid * 16; off < raw_bytes; off += PASS)
              if (((off & (W_BOX - 1)) >> 7) >= valid) *reinterpret_cast<float4*>(raw + off) = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
        if (raw_bytes == C::RAW) {
#pragma unroll
          for (int k = 0; k < C::RAW / PASS; ++k) split(tid * 16 + k * PASS);
        } else {
#pragma unroll
          for (int k = 0; k < A_TILE / PASS; ++k) split(tid * 16 + k * PASS);
          for (int off = A_TILE + tid * 16; off < raw_bytes; off += PASS) split(off);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_conv + 8 * s);
      }
      if (ok) ok = warp_wait(bar_acc, (uint32_t)(c & 1), abort_flag, p.status, 400);
      if (!ok) break;
      tc_fence_after();
      const bool last = c + 1 == n_chunks;
      const int mains = (end - c * per + run - 1) / run;     // main accumulators in use
#pragma unroll 1
      for (int cc = half; cc * 32 < cols; cc += 2) {
        uint32_t r[32], rc[32];
        tmem_ld_32x32(lane_base + (uint32_t)(cc * 32), r);
        tmem_ld_32x32(lane_base + (uint32_t)(C::MAINS * BN + cc * 32), rc);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(rc[j]));
#pragma unroll 1
        for (int m = 1; m < mains; ++m) {
          tmem_ld_32x32(lane_base + (uint32_t)(m * BN + cc * 32), rc);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(rc[j]));
        }
        if (p.park) {
          float4* slot = reinterpret_cast<float4*>(p.park + ((long long)unit * p.slices + slice) * (BM * BN)) + (q * 32 + lane);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            float4* to = slot + (cc * 8 + (j >> 2)) * 128;
            float4 v = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
            if (c > 0) {                                     // the slice's earlier chunks: this thread's own values
              const float4 o = __ldcg(to);
              v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
            }
            __stcg(to, v);
          }
        } else if (p.slices > 1) {
          // parked in this CTA's own shared memory ([columns / 4][128 lanes] float4); one chunk only, so the stages are free
          float4* slot = reinterpret_cast<float4*>(smem) + (q * 32 + lane);
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            slot[(cc * 8 + (j >> 2)) * 128] = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                                                          __uint_as_float(r[j + 3]));
        } else {
          store_columns(p, out, r, t0 + cc * 32, hi, n0 + q * 32 + lane, bias, c == 0 ? p.beta : 1.f, last);
        }
      }
      if (!last) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_read);
      }
    }
    if (p.park) {
      if (ok) __threadfence();
      asm volatile("bar.sync 1, %0;" ::"n"(CONV_WARPS * 32) : "memory");
      if (threadIdx.x == 0) where[5] = *abort_flag ? -1 : atomicAdd(p.arrived + unit, 1);
      asm volatile("bar.sync 1, %0;" ::"n"(CONV_WARPS * 32) : "memory");
      if (where[5] == p.slices - 1) {
        __threadfence();
#pragma unroll 1
        for (int cc = half; cc * 32 < cols; cc += 2) {
          const float4* from = reinterpret_cast<const float4*>(p.park + (long long)unit * p.slices * (BM * BN)) + (cc * 8 * 128 + q * 32 + lane);
          float4 a[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] = __ldcg(from + j * 128);
          for (int sl = 1; sl < p.slices; ++sl) {
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __ldcg(from + (long long)sl * (BM * BN / 4) + j * 128);
#pragma unroll
            for (int j = 0; j < 8; ++j) { a[j].x += v[j].x; a[j].y += v[j].y; a[j].z += v[j].z; a[j].w += v[j].w; }
          }
          uint32_t r[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            r[4 * j] = __float_as_uint(a[j].x); r[4 * j + 1] = __float_as_uint(a[j].y);
            r[4 * j + 2] = __float_as_uint(a[j].z); r[4 * j + 3] = __float_as_uint(a[j].w);
          }
          store_columns(p, out, r, t0 + cc * 32, hi, n0 + q * 32 + lane, bias, p.beta, true);
        }
        if (threadIdx.x == 0) p.arrived[unit] = 0;           // left zero for the next launch
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (!WEIGHTS && p.slices > 1 && !p.park) {
    // Every thread of every CTA takes both barriers.  Between them the tile's 32 x 32 pieces are dealt round the cluster's
    // CTAs and warps, each summed in slice order whoever does it.
    cluster_sync_all();
    if (warp < CONV_WARPS && !*abort_flag) {
      const int n = p.slices, items = 4 * ((cols + 31) / 32);
      for (int it = (int)cluster_ctarank() + n * warp; it < items; it += n * CONV_WARPS) {
        const int q = it & 3, cc = it >> 2;
        const uint32_t off = smem_base + (uint32_t)((cc * 8 * 128 + q * 32 + lane) * 16);
        float4 a[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int sl = 0; sl < n; ++sl) {
          const uint32_t from = mapa(off, (uint32_t)sl);
          float4 v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = ld_dsmem_v4(from + j * 2048);
#pragma unroll
          for (int j = 0; j < 8; ++j) { a[j].x += v[j].x; a[j].y += v[j].y; a[j].z += v[j].z; a[j].w += v[j].w; }
        }
        uint32_t r[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          r[4 * j] = __float_as_uint(a[j].x); r[4 * j + 1] = __float_as_uint(a[j].y);
          r[4 * j + 2] = __float_as_uint(a[j].z); r[4 * j + 3] = __float_as_uint(a[j].w);
        }
        store_columns(p, out, r, t0 + cc * 32, hi, n0 + q * 32 + lane, bias, p.beta, true);
      }
    }
    cluster_sync_all();
  }
  const bool more = unit + (int)gridDim.x / p.slices < p.units && !*abort_flag;
  __syncthreads();
  if (!more) {
    if (warp == CONV_WARPS + 1) {
      tc_fence_after();
      tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    return;
  }
  if (threadIdx.x == 0)
    for (int s = 0; s < 3 * STAGES + 2; ++s) mbar_inval(bar_full + 8 * s);
  }
}

// ---- many tiles of short reductions -------------------------------------------------------------------------------
// Where a tile is a few k-blocks, setting up a CTA, filling its pipeline and storing its sums take longer than the products.
// Here a CTA stays (one to an SM) and takes tiles in turn: the producer finds the next tile, says in a ring which it is and
// loads on; four more warps store a tile's sums from one set of accumulators while the next tile's go into the other.
// The arithmetic is that of the kernel above; a chunk of a long reduction is an entry of the ring like a tile.
constexpr int EPI_WARPS = 4, STREAM_THREADS = (CONV_WARPS + 2 + EPI_WARPS) * 32, RING = 8;

template <int BN, int BK> struct StreamCfg {
  static constexpr int A_TILE = BM * BK * 4, B_TILE = BN * BK * 4, RAW = A_TILE + B_TILE, STAGE = 2 * RAW;
  static constexpr int STAGES = (196608 / STAGE) > 8 ? 8 : (196608 / STAGE);
  static constexpr int MAINS = BN == 128 ? 1 : 3, SET = (MAINS + 1) * BN;      // TMEM columns of a set of accumulators
  static constexpr int CHUNK = MAINS * RUN / BK;      // k-blocks
  static constexpr int SMEM = STAGES * STAGE + 1024 + 1024;
  static_assert(2 * SET == 512, "two sets of accumulators");
};

struct Entry { int more, expert, g_lo, g_hi, t0, n0, kb_begin, nkb, chunk, last; };

template <int BN, int BK, bool WEIGHTS>
__global__ void __launch_bounds__(STREAM_THREADS, 1)
expert_stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ RowsArgs p) {
  typedef StreamCfg<BN, BK> C;
  constexpr int STAGES = C::STAGES, A_TILE = C::A_TILE;
  constexpr int W_BOX = BK * 128;                            // bytes of one 32 x BK box of an MN-major matrix
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = (uint64_t*)(smem + STAGES * C::STAGE);
  // bars: full, conv, empty [STAGES each]; sums ready, sums read [2 each]; entry written, entry done [RING each]; MMAs retired
  uint32_t* tmem_slot = (uint32_t*)(bars + 3 * STAGES + 5 + 2 * RING);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  Entry* ring = (Entry*)(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (nothing_to_do(p.only_if)) return;
  const int tiles_n = (p.N + BM - 1) / BM;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_full = smem_u32(bars), bar_conv = smem_u32(bars + STAGES), bar_empty = smem_u32(bars + 2 * STAGES),
                 bar_acc = smem_u32(bars + 3 * STAGES), bar_read = bar_acc + 16, bar_entry = bar_read + 16, bar_done = bar_entry + 8 * RING,
                 bar_retired = bar_done + 8 * RING;
  if (warp == CONV_WARPS + 1) {
    tmem_alloc(smem_u32(tmem_slot), 2 * C::SET);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_conv + 8 * s, CONV_WARPS);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc + 8 * b, 1);
      mbar_init(bar_read + 8 * b, EPI_WARPS);
    }
    for (int e = 0; e < RING; ++e) {
      mbar_init(bar_entry + 8 * e, 1);
      mbar_init(bar_done + 8 * e, EPI_WARPS);
    }
    mbar_init(bar_retired, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == CONV_WARPS && lane == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // columns of the accumulator and bytes of a stage for an entry
  auto columns = [&](const Entry& e) { return min(BN, (WEIGHTS ? p.cols : e.g_hi) - e.t0); };
  auto boxes_of = [&](int cols) { return WEIGHTS ? (cols + 31) / 32 : (cols + 63) / 64; };
  auto bytes_of = [&](int cols) { return A_TILE + boxes_of(cols) * (WEIGHTS ? W_BOX : 64 * BK * 4); };

  if (warp == CONV_WARPS) {
    // ------------------------------ tiles and TMA -----------------------------
    const bool withhold = (p.status[3] & 1) != 0;            // host-injected fault: arm nothing, load nothing
    int issued = 0, s = 0, it = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int unit = (int)blockIdx.x; ok; unit += (int)gridDim.x) {
      Entry e;
      e.more = unit < p.units;
      int chunks = 1, per = 0, nkb = 0;
      if (e.more) {
        groups::Tile t = {0, 0, 0, 0};
        e.n0 = (unit % tiles_n) * BM;
        if (WEIGHTS) {
          const int rest = unit / tiles_n;
          t.expert = rest / p.tiles_r;
          t.index = rest - t.expert * p.tiles_r;
          groups::group_rows(p.offsets, p.rows, t.expert, p.status, t.lo, t.hi);
        } else {
          e.more = groups::find_tile(p.offsets, p.experts, p.rows, BN, unit / tiles_n, p.status, t);
        }
        e.expert = t.expert; e.g_lo = t.lo; e.g_hi = t.hi;
        e.t0 = WEIGHTS ? t.index * BN : t.lo + t.index * BN;
        nkb = max(((WEIGHTS ? t.hi - t.lo : p.K) + BK - 1) / BK, 1);           // (a group without rows: a k-block of zeros)
        chunks = (nkb + C::CHUNK - 1) / C::CHUNK;
        per = (nkb + chunks - 1) / chunks;
      }
      for (int c = 0; c < chunks; ++c, ++it) {
        const int slot = it % RING;
        if (!warp_wait(bar_done + 8 * slot, ((it / RING) & 1) ^ 1, abort_flag, p.status, 500 + slot)) { ok = false; break; }
        e.kb_begin = c * per;
        e.nkb = min(per, nkb - c * per);
        e.chunk = c;
        e.last = c + 1 == chunks;
        if (lane == 0) {
          ring[slot] = e;
          mbar_arrive(bar_entry + 8 * slot);
        }
        __syncwarp();
        if (!e.more) { ok = false; break; }
        const int boxes = boxes_of(columns(e)), raw_bytes = bytes_of(columns(e));
        for (int i = 0; i < e.nkb; ++i) {
          if (!warp_wait(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 100 + s)) { ok = false; break; }
          const uint32_t full = bar_full + 8 * s;
          const uint32_t w_dst = smem_base + s * C::STAGE, x_dst = w_dst + A_TILE;
          const int k0 = (e.kb_begin + i) * BK;
          if (!withhold && elect_one()) {
            mbar_arrive_expect_tx(full, (uint32_t)raw_bytes);
            if (WEIGHTS) {
#pragma unroll
              for (int j = 0; j < BM / 32; ++j) tma_load_2d(w_dst + j * W_BOX, &tmW, e.n0 + 32 * j, e.g_lo + k0, full);
              for (int j = 0; j < boxes; ++j) tma_load_2d(x_dst + j * W_BOX, &tmX, e.t0 + 32 * j, e.g_lo + k0, full);
            } else {
              if (!p.w_mn) {
                tma_load_3d(w_dst, &tmW, k0, e.n0, e.expert, full);
              } else {
#pragma unroll
                for (int j = 0; j < BM / 32; ++j) tma_load_3d(w_dst + j * W_BOX, &tmW, e.n0 + 32 * j, k0, e.expert, full);
              }
              for (int j = 0; j < boxes; ++j) tma_load_2d(x_dst + j * 64 * BK * 4, &tmX, k0, e.t0 + j * 64, full);
            }
          }
          if (!withhold) ++issued;
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
      }
    }
    if (*abort_flag) {
      // copies already issued land before this CTA gives its shared memory back
      for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
        for (int n = 0; n < (1 << 16); ++n)
          if (mbar_try_wait(bar_full + 8 * (i % STAGES), (i / STAGES) & 1)) break;
    }
  } else if (warp == CONV_WARPS + 1) {
    // ------------------------------ MMA issuer --------------------------------
    const bool a_mn = WEIGHTS || p.w_mn;
    constexpr uint32_t K_SWZ = BK == 32 ? SWZ_128B : SWZ_64B, K_SBO = 8 * BK * 4;
    const uint32_t a_step = (a_mn ? 1024u : 32u) >> 4;
    constexpr uint32_t b_step = (WEIGHTS ? 1024u : 32u) >> 4;
    const uint64_t d_a = a_mn ? make_smem_desc(smem_base, W_BOX, 512, SWZ_128B_BASE32B) : make_smem_desc(smem_base, 16, K_SBO, K_SWZ);
    const uint64_t d_b = WEIGHTS ? make_smem_desc(smem_base + A_TILE, W_BOX, 512, SWZ_128B_BASE32B)
                                 : make_smem_desc(smem_base + A_TILE, 16, K_SBO, K_SWZ);
    const uint32_t a_hiw = (uint32_t)(d_a >> 32), b_hiw = (uint32_t)(d_b >> 32);
    const uint32_t a_low0 = (uint32_t)d_a, b_low0 = (uint32_t)d_b;
    constexpr uint32_t LO_TILE = C::RAW >> 4, STAGE_STEP = C::STAGE >> 4;
    uint32_t ph = 0, stage_off = 0;
    int s = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int slot = it % RING, set = it & 1;
      if (!warp_wait(bar_entry + 8 * slot, (it / RING) & 1, abort_flag, p.status, 520 + slot)) break;
      const Entry e = ring[slot];
      if (!e.more) break;
      if (!warp_wait(bar_read + 8 * set, ((it >> 1) & 1) ^ 1, abort_flag, p.status, 250 + set)) break;
      tc_fence_after();
      const uint32_t idesc = make_idesc_tf32(BM, (columns(e) + 15) / 16 * 16, a_mn, WEIGHTS);
      const int run = max((e.nkb + C::MAINS - 1) / C::MAINS, RUN / BK);        // k-blocks into one main accumulator
      uint32_t tmem_main = tmem_base + set * C::SET, accumulate = 0, cross = 0;
      const uint32_t tmem_cross = tmem_main + C::MAINS * BN;
      int in_run = 0;
      for (int i = 0; i < e.nkb; ++i) {
        if (C::MAINS > 1 && in_run == run) {
          in_run = 0;
          accumulate = 0;
          tmem_main += BN;
        }
        ++in_run;
        if (!warp_wait(bar_conv + 8 * s, ph, abort_flag, p.status, 200 + s)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BK / 8; ++kk) {
            const uint32_t al = a_low0 + stage_off + kk * a_step, bl = b_low0 + stage_off + kk * b_step;
            mma_tf32_ss_words(tmem_cross, al + LO_TILE, a_hiw, bl, b_hiw, idesc, kk ? 1u : cross);
            mma_tf32_ss_words(tmem_cross, al, a_hiw, bl + LO_TILE, b_hiw, idesc, 1);
            mma_tf32_ss_words(tmem_main, al, a_hiw, bl, b_hiw, idesc, kk ? 1u : accumulate);
          }
          mma_commit(bar_empty + 8 * s);
        }
        accumulate = cross = 1;
        __syncwarp();
        if (++s == STAGES) { s = 0; ph ^= 1; stage_off = 0; } else { stage_off += STAGE_STEP; }
      }
      if (ok && elect_one()) mma_commit(bar_acc + 8 * set);
      __syncwarp();
    }
    if (*abort_flag) {
      // every MMA issued must have retired before TMEM is freed
      if (elect_one()) mma_commit(bar_retired);
      __syncwarp();
      for (int n = 0; n < (1 << 16); ++n)
        if (mbar_try_wait(bar_retired, 0)) break;
    }
  } else if (warp < CONV_WARPS) {
    // ------------------------------ hi / lo split ------------------------------
    constexpr int PASS = CONV_WARPS * 32 * 16;
    const int tid = threadIdx.x;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int slot = it % RING;
      if (!warp_wait(bar_entry + 8 * slot, (it / RING) & 1, abort_flag, p.status, 540 + slot)) break;
      const Entry e = ring[slot];
      if (!e.more) break;
      const int raw_bytes = bytes_of(columns(e));
      for (int i = 0; i < e.nkb; ++i) {
        if (!warp_wait(bar_full + 8 * s, ph, abort_flag, p.status, 300 + s)) { ok = false; break; }
        uint8_t* raw = smem + s * C::STAGE;
        uint8_t* low = raw + C::RAW;
        auto split = [&](int off) {
          const float4 v = *reinterpret_cast<const float4*>(raw + off);
          float4 l;
          l.x = lo_part(v.x); l.y = lo_part(v.y); l.z = lo_part(v.z); l.w = lo_part(v.w);
          *reinterpret_cast<float4*>(low + off) = l;
        };
        if (WEIGHTS) {
          const int valid = e.g_hi - e.g_lo - (e.kb_begin + i) * BK;             // rows of this k-block inside the group
          if (valid < BK) {
            // (the 16-byte pieces that this thread reads itself below; a k row is 128 bytes of every box)
#pragma unroll 1
            for (int off = tid * 16; off < raw_bytes; off += PASS)
              if (((off & (W_BOX - 1)) >> 7) >= valid) *reinterpret_cast<float4*>(raw + off) = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
        if (raw_bytes == C::RAW) {
#pragma unroll
          for (int k = 0; k < C::RAW / PASS; ++k) split(tid * 16 + k * PASS);
        } else {
#pragma unroll
          for (int k = 0; k < A_TILE / PASS; ++k) split(tid * 16 + k * PASS);
          for (int off = A_TILE + tid * 16; off < raw_bytes; off += PASS) split(off);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_conv + 8 * s);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    }
  } else {
    // ------------------------------ epilogue -----------------------------------
    const int q = warp & 3;                                  // the TMEM lanes of this warp
    for (int it = 0;; ++it) {
      const int slot = it % RING, set = it & 1;
      if (!warp_wait(bar_entry + 8 * slot, (it / RING) & 1, abort_flag, p.status, 560 + slot)) break;
      const Entry e = ring[slot];
      if (!e.more) break;
      if (!warp_wait(bar_acc + 8 * set, (uint32_t)((it >> 1) & 1), abort_flag, p.status, 400 + set)) break;
      tc_fence_after();
      const int cols = columns(e), run = max((e.nkb + C::MAINS - 1) / C::MAINS, RUN / BK), mains = (e.nkb + run - 1) / run;
      const uint32_t lane_base = tmem_base + set * C::SET + ((uint32_t)(q * 32) << 16);
      float* const out = WEIGHTS ? p.C + e.expert * p.c_stride : p.C;
      const float* bias = p.bias ? p.bias + (long long)e.expert * p.N : nullptr;
#pragma unroll 1
      for (int cc = 0; cc * 32 < cols; ++cc) {
        uint32_t r[32], rc[32];
        tmem_ld_32x32(lane_base + (uint32_t)(cc * 32), r);
        tmem_ld_32x32(lane_base + (uint32_t)(C::MAINS * BN + cc * 32), rc);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(rc[j]));
#pragma unroll 1
        for (int m = 1; m < mains; ++m) {
          tmem_ld_32x32(lane_base + (uint32_t)(m * BN + cc * 32), rc);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(rc[j]));
        }
        store_columns(p, out, r, e.t0 + cc * 32, WEIGHTS ? p.cols : e.g_hi, e.n0 + q * 32 + lane, bias, e.chunk == 0 ? p.beta : 1.f, e.last);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_read + 8 * set);
        mbar_arrive(bar_done + 8 * slot);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == CONV_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * C::SET);
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

template <typename A, void (*KERNEL)(CUtensorMap, CUtensorMap, A)>
int launch(cb200_stream* s, int smem, const CUtensorMap& tmA, const CUtensorMap& tmB, const A& a, long long ctas, int cluster,
           int threads = THREADS) {
  static std::once_flag once[64];
  static cudaError_t result[64];
  const int dev = s->device & 63;
  std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (result[dev] != cudaSuccess) return cb200_cuda_fail(result[dev], "cudaFuncSetAttribute", __FILE__, __LINE__);
  CB_REQUIRE(ctas <= 2147483647LL, "expert_gemm: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s->stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (a.only_if) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, tmA, tmB, a);
  if (e != cudaSuccess) return cb200_cuda_fail(e, "cudaLaunchKernelEx(expert kernel)", __FILE__, __LINE__);
  CB_LAUNCH_CHECK(s);
  return CB200_OK;
}

// room for the slices of `units` tiles that meet in L2
int get_park(cb200_stream* s, RowsArgs& a, long long units, int BN) {
  void* ws = nullptr;
  const int rc = cb200_partials(s, (size_t)units * a.slices * BM * BN * sizeof(float), &ws);
  a.park = (float*)ws;
  return rc ? rc : cb200_tile_flags(s, (size_t)units, &a.arrived);
}

// Tile width and K slices for `tiles_m` row tiles (an estimate for ragged groups) of N columns reduced over `nkb`
// k-blocks: the timing model of gemm!, t = waves x (5 us + k-blocks per slice x c[BN]) + hand-over.
void choose(const cb200_stream* s, long long tiles_m, int N, int nkb, int max_slices, int& bn_out, int& slices_out) {
  const int bn_max = N > 64 ? 128 : 64;
  double best = 1e30;
  bn_out = bn_max;
  slices_out = 1;
  for (int bn = 128; bn >= 64; bn >>= 1) {
    if (bn > bn_max) continue;
    if (s->opt_gemm_tile_n > 0 && bn != s->opt_gemm_tile_n && s->opt_gemm_tile_n <= bn_max) continue;
    const double c = bn == 128 ? 0.455 : 0.39;
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

}  // namespace

// Operands that TMA can address: 16-byte bases, pitches and distances that are multiples of 4 elements.
bool cb200_expert_tc_ok(const void* A, long long lda, const void* B, long long ldb, long long b_stride) {
  return ((((uintptr_t)A | (uintptr_t)B) & 15) == 0) && lda % 4 == 0 && ldb % 4 == 0 && b_stride % 4 == 0;
}

int cb200_expert_rows_tc(cb200_stream* s, float* C, long long ldc, int trans_b, float alpha, const float* A, int rows, int K,
                         long long lda, const float* B, int experts, int N, long long b_stride, long long ldb, float beta,
                         const int* offsets, const float* bias, int act, const int* only_if) {
  DeviceGuard guard(s->device);
  // how many rows a tile may take: what an even split of the rows over the experts fills
  const long long even = (rows + experts - 1) / experts;
  int BN = even <= 32 ? 32 : (even <= 64 ? 64 : 128);
  if (s->opt_gemm_tile_n > 0) BN = s->opt_gemm_tile_n < 128 ? s->opt_gemm_tile_n : 128;
  const bool forced = s->opt_gemm_tile_n > 0 || s->opt_gemm_k_slices > 0;
  int bk = 0;
  long long units = 0;
  auto cut = [&] {
    bk = BN <= 64 ? 32 : 16;
    units = ((rows + BN - 1) / BN + (experts < rows ? experts : rows) - 1) * ((N + BM - 1) / BM);
  };
  cut();
  // K slices where the tiles leave SMs free: the CTAs of a cluster if a slice is one chunk (its parked tile lies in shared
  // memory that the next chunk's stages would need), else CTAs that meet in L2 (3 experts of 600 x 4000 with 300 rows each
  // 155 us uncut)
  const int chunk = BN == 128 ? RowsCfg<128, 16>::CHUNK : (BN == 64 ? RowsCfg<64, 32>::CHUNK : RowsCfg<32, 32>::CHUNK);
  const int nkb = (K + bk - 1) / bk, wanted = s->opt_gemm_k_slices;
  const long long room = s->sm_count * (BN <= 64 ? 2 : 1);
  int slices = 1;
  bool meet = false;
  for (int sl = 2; sl <= 8; sl *= 2)
    if ((wanted > 0 ? sl <= wanted : units * sl <= room) && nkb / sl >= 4) slices = sl;
  if ((nkb + slices - 1) / slices > chunk) {
    meet = slices > 1;
    if (meet && wanted == 0) slices = (int)(room / units < 16 ? room / units : 16);
  }
  if (only_if) { slices = 1; meet = false; }
  // Tiles that follow one another where nothing is sliced (this / the kernel of one tile a CTA, us): 16 experts of 2048 x 128
  // with 64, 256 rows each 18, 33 / 22, 39; 32 of 1024 x 1024 with 32, 64, 128 rows 53, 76, 109 / 77, 89, 121; but two narrow
  // tiles to an SM are faster at long reductions: 64 of 1024 x 4096 with 20, 64 rows 417, 559 / 285, 467.
  const bool stream = !forced && slices == 1 && (K <= 1024 || even > 64);
  if (stream) {
    BN = even <= 64 ? 64 : 128;
    cut();
  }
  RowsArgs a;
  a.C = C; a.ldc = ldc; a.c_stride = 0; a.cols = a.tiles_r = 0; a.park = nullptr; a.arrived = nullptr;
  a.bias = bias; a.offsets = offsets; a.status = s->status_dev;
  a.N = N; a.K = K; a.experts = experts; a.rows = rows; a.w_mn = trans_b ? 0 : 1; a.act = act;
  a.alpha = alpha; a.beta = beta; a.slices = slices; a.only_if = only_if;
  const CUtensorMapSwizzle swz = bk == 32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap tmW, tmX;
  int rc;
  if (groups::all_may_be_found(rows, experts, BN)) ++units;
  CB_REQUIRE(units * slices <= 2147483647LL, "expert_gemm: too many tiles");
  if (meet && (rc = get_park(s, a, units, BN))) return rc;
  if ((rc = tmap_2d(&tmX, A, rows, K, lda, bk, BN < 64 ? BN : 64, swz))) return rc;
  if (trans_b) rc = tmap_3d(&tmW, B, experts, N, K, ldb, b_stride, bk, BM, swz);
  else rc = tmap_3d(&tmW, B, experts, K, N, ldb, b_stride, 32, bk, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B);
  if (rc) return rc;
  a.units = (int)units;
  const int cluster = meet ? 1 : slices;
  if (stream) {
    const long long ctas = units < s->sm_count ? units : s->sm_count;
    if (BN == 128) return launch<RowsArgs, expert_stream_kernel<128, 16, false>>(s, StreamCfg<128, 16>::SMEM, tmW, tmX, a, ctas, 1, STREAM_THREADS);
    return launch<RowsArgs, expert_stream_kernel<64, 32, false>>(s, StreamCfg<64, 32>::SMEM, tmW, tmX, a, ctas, 1, STREAM_THREADS);
  }
  const long long ctas = only_if && units > s->sm_count ? s->sm_count : units * slices;
  if (BN == 128) return launch<RowsArgs, expert_tf32x3_kernel<128, 16, false>>(s, RowsCfg<128, 16>::SMEM, tmW, tmX, a, ctas, cluster);
  if (BN == 64) return launch<RowsArgs, expert_tf32x3_kernel<64, 32, false>>(s, RowsCfg<64, 32>::SMEM, tmW, tmX, a, ctas, cluster);
  return launch<RowsArgs, expert_tf32x3_kernel<32, 32, false>>(s, RowsCfg<32, 32>::SMEM, tmW, tmX, a, ctas, cluster);
}

int cb200_expert_weights_tc(cb200_stream* s, float* C, long long c_stride, long long ldc, float alpha, const float* A, int rows,
                            int M, long long lda, const float* B, int N, long long ldb, int experts, float beta,
                            const int* offsets, const int* only_if) {
  DeviceGuard guard(s->device);
  const long long tiles_l = (N + BM - 1) / BM;
  int BN, slices;
  choose(s, tiles_l * experts, M, (rows / experts + 16) / 16, only_if ? 1 : 16, BN, slices);
  // short reductions in tiles that follow one another (this / the kernel of one tile a CTA, us): 8 experts of 1024 x 4096 with
  // 20, 64, 96, 160 rows each 43, 65, 81, 114 / 64, 80, 92, 113; 32 of 512 x 512 with 64, 96 rows 37, 47 / 35, 39
  const bool stream = s->opt_gemm_tile_n == 0 && s->opt_gemm_k_slices == 0 && slices == 1 && rows <= 96LL * experts;
  if (stream) BN = M > 64 ? 128 : 64;
  RowsArgs a;
  a.C = C; a.ldc = ldc; a.c_stride = c_stride; a.cols = M; a.tiles_r = (M + BN - 1) / BN; a.park = nullptr; a.arrived = nullptr;
  a.bias = nullptr; a.offsets = offsets; a.status = s->status_dev;
  a.N = N; a.K = 0; a.experts = experts; a.rows = rows; a.w_mn = 1; a.act = CB200_ACT_NONE;
  a.alpha = alpha; a.beta = beta; a.slices = slices; a.only_if = only_if;
  const long long units = tiles_l * a.tiles_r * experts;
  CB_REQUIRE(units * slices <= 2147483647LL, "expert_gemm_weights: too many tiles");
  a.units = (int)units;
  const long long ctas = only_if && units > s->sm_count ? s->sm_count : units * slices;
  int rc;
  if (slices > 1 && (rc = get_park(s, a, units, BN))) return rc;
  CUtensorMap tmW, tmX;
  if ((rc = tmap_2d(&tmW, B, rows, N, ldb, 32, 16, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B))) return rc;
  if ((rc = tmap_2d(&tmX, A, rows, M, lda, 32, 16, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B))) return rc;
  if (stream) {
    const long long ctas = units < s->sm_count ? units : s->sm_count;
    if (BN == 128) return launch<RowsArgs, expert_stream_kernel<128, 16, true>>(s, StreamCfg<128, 16>::SMEM, tmW, tmX, a, ctas, 1, STREAM_THREADS);
    return launch<RowsArgs, expert_stream_kernel<64, 16, true>>(s, StreamCfg<64, 16>::SMEM, tmW, tmX, a, ctas, 1, STREAM_THREADS);
  }
  if (BN == 128) return launch<RowsArgs, expert_tf32x3_kernel<128, 16, true>>(s, RowsCfg<128, 16>::SMEM, tmW, tmX, a, ctas, 1);
  return launch<RowsArgs, expert_tf32x3_kernel<64, 16, true>>(s, RowsCfg<64, 16>::SMEM, tmW, tmX, a, ctas, 1);
}
