// Grouped product of NVFP4 rows with NVFP4 weights on tcgen05 (sm_100a): four-bit codes go to the tensor cores as they are.
//   C[t, n] = xs[t] ws[n] sum_b sx[t, b] sw[n, b] sum_{k in block b} x[t, k] w[g][n, k]        blocks of 16 values
//
// The 128 weight rows of a tile are the M side of the MMA, its tokens the N side.  A TMA thread streams boxes of 256 values: 128
// bytes of codes a row (128-byte swizzle) and 16 bytes of scales.  Two warps turn the scales of a stage into the cells that the
// instruction reads (weights and activations keep the layout of their rows in memory, which the decode chain reads too), the
// issuing warp copies them to tensor memory (tcgen05.cp) and issues four kind::mxf4nvf4 MMAs a stage, K = 64 each, which multiply codes,
// apply both blocks' scales and add in fp32.  Four epilogue warps apply the two fp32 scales.
//   * "dual" mode runs gate and up in one main loop; the epilogue writes silu(gate) * up;
//   * the epilogue scatters and scales like the other GEMMs (dst_row / row_scale / resid).
// Every wait is bounded; on expiry the CTA raises status word 1, leaves its loops, frees its TMEM and returns.
#include "fp4_common.cuh"

namespace bl {

constexpr int F4_THREADS = 256;             // warp 0 TMA, 1 MMA + TMEM, 2..5 epilogue, 6 and 7 scales
constexpr int F4_MAX_STAGES = 8;

struct F4Tile { int group, row0, row_end, pad; };

struct F4Args {
  int N, K, tiles_w;
  const F4Tile* tiles;
  const int* n_tiles;
  int max_tiles;
  const uint8_t* x;         // the rows, for their fp32 scales
  const uint8_t* w;
  const uint8_t* w2;
  long row_bytes, group_bytes;
  float* c_f32;
  __nv_bfloat16* c_bf16;
  long ldc;
  const int* dst_row;
  const float* row_scale;
  const float* resid;
  long ldr;
  unsigned* status;
};

// What a stage holds, in bytes from its start, and what it has in tensor memory, in columns
template <bool DUAL, int BN>
struct F4Shape {
  static constexpr int MATS = DUAL ? 2 : 1;
  static constexpr int BOX = BN < 64 ? BN : 64;                    // token rows of a box
  static constexpr int B = MATS * 16384, RA = B + BN * 128, RB = RA + MATS * 2048, TA = RB + BN * 16, TB = TA + MATS * 2048;
  static constexpr int B_CELLS = BN > 128 ? 8 : 4;                 // columns of an instruction's token scales
  static constexpr int STAGE = (TB + 4 * 128 * B_CELLS + 1023) / 1024 * 1024;
  static constexpr int STAGES = 222 * 1024 / STAGE > F4_MAX_STAGES ? F4_MAX_STAGES : 222 * 1024 / STAGE;
  static constexpr int SCALE_COLS = 16 * MATS + 4 * B_CELLS;
  static constexpr int ACCS = 2 * MATS * BN + STAGES * SCALE_COLS <= 512 ? 2 : 1;
  static constexpr int SCALE0 = ACCS * MATS * BN;                  // first column of the scales
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024;
  static_assert(STAGES >= 2 && SCALE0 + STAGES * SCALE_COLS <= 512, "tensor memory");
};

template <bool DUAL, int BN>
__global__ void __launch_bounds__(F4_THREADS, 1)
fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs,
                const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws,
                const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_ws2, const F4Args a) {
  using S = F4Shape<DUAL, BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[S::STAGES], cells_bar[S::STAGES], empty_bar[S::STAGES], acc_full[S::ACCS], acc_empty[S::ACCS];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&cells_bar[s], 2); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < S::ACCS; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 4); }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch();
  const uint32_t tmem = s_tmem_base;
  volatile int* abort_flag = &s_abort;
  const int total = min(*a.n_tiles, a.max_tiles) * a.tiles_w, kblocks = (a.K + 255) / 256;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0; uint32_t phase = 0;
      for (int t = blockIdx.x; t < total && !*abort_flag; t += gridDim.x) {
        const F4Tile mt = a.tiles[t / a.tiles_w];
        const int n0 = (t % a.tiles_w) * 128, boxes = (min(BN, mt.row_end - mt.row0) + S::BOX - 1) / S::BOX;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) break;
          uint8_t* s = smem + (size_t)stage * S::STAGE;
          mbar_expect_tx(&full_bar[stage], S::MATS * (16384 + 2048) + boxes * S::BOX * (128 + 16));
          // rows past a matrix and values past a row arrive as zeros
          tma_load_3d(s, &map_w, kb * 128, n0, mt.group, &full_bar[stage]);
          tma_load_3d(s + S::RA, &map_ws, kb * 16, n0, mt.group, &full_bar[stage]);
          if (DUAL) {
            tma_load_3d(s + 16384, &map_w2, kb * 128, n0, mt.group, &full_bar[stage]);
            tma_load_3d(s + S::RA + 2048, &map_ws2, kb * 16, n0, mt.group, &full_bar[stage]);
          }
          for (int b = 0; b < boxes; ++b) {
            tma_load_3d(s + S::B + b * S::BOX * 128, &map_x, kb * 128, mt.row0 + b * S::BOX, 0, &full_bar[stage]);
            tma_load_3d(s + S::RB + b * S::BOX * 16, &map_xs, kb * 16, mt.row0 + b * S::BOX, 0, &full_bar[stage]);
          }
          ++issued;
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (*abort_flag) {
        // copies of this thread may still be landing in shared memory: the CTA must not exit under them
        unsigned long long t0 = globaltimer();
        while (issued > 0 && globaltimer() - t0 < 2000000ull) {}
      }
    }
  } else if (warp == 1) {
    int stage = 0; uint32_t phase = 0;
    uint32_t ab = 0, aphase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const F4Tile mt = a.tiles[t / a.tiles_w];
      const uint32_t idesc = fp4_idesc((min(BN, mt.row_end - mt.row0) + 31) / 32 * 32);
      if (!mbar_wait_warp(&acc_empty[ab], aphase ^ 1, abort_flag)) break;
      const uint32_t d0 = tmem + ab * (S::MATS * BN);
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait_warp(&full_bar[stage], phase, abort_flag) || !mbar_wait_warp(&cells_bar[stage], phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t sm = smem_u32(smem + (size_t)stage * S::STAGE), sc = tmem + S::SCALE0 + stage * S::SCALE_COLS;
        const uint32_t sb = sc + 16 * S::MATS;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int m = 0; m < S::MATS; ++m) fp4_scales_to_tmem(sc + 16 * m + 4 * k, sm + S::TA + 2048 * m + 512 * k);
#pragma unroll
          for (int h = 0; h < S::B_CELLS / 4; ++h) fp4_scales_to_tmem(sb + S::B_CELLS * k + 4 * h, sm + S::TB + 2048 * h + 512 * k);
        }
        const uint64_t da = umma_desc(sm), db = umma_desc(sm + S::B);
#pragma unroll
        for (int k = 0; k < 4; ++k) {                              // 64 values are 32 bytes
#pragma unroll
          for (int m = 0; m < S::MATS; ++m)
            umma_fp4(d0 + m * BN, da + (uint64_t)(m * 16384 / 16 + 2 * k), db + (uint64_t)(2 * k), idesc, sc + 16 * m + 4 * k,
                     sb + S::B_CELLS * k, kb > 0 || k > 0 ? 1u : 0u);
        }
        umma_commit(&empty_bar[stage]);
        if (kb == kblocks - 1) umma_commit(&acc_full[ab]);
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
      }
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
    }
  } else if (warp >= 6) {
    int stage = 0; uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const F4Tile mt = a.tiles[t / a.tiles_w];
      const int groups = (min(BN, mt.row_end - mt.row0) + 31) / 32;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait_warp(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
        uint8_t* s = smem + (size_t)stage * S::STAGE;
        if (warp == 6) {
#pragma unroll
          for (int m = 0; m < S::MATS; ++m)
            fp4_turn_scales(reinterpret_cast<const uint4*>(s + S::RA + 2048 * m), reinterpret_cast<uint4*>(s + S::TA + 2048 * m), lane, 4);
        } else {
#pragma unroll
          for (int h = 0; h < S::B_CELLS / 4; ++h)
            fp4_turn_scales(reinterpret_cast<const uint4*>(s + S::RB + 2048 * h), reinterpret_cast<uint4*>(s + S::TB + 2048 * h), lane, groups - 4 * h);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&cells_bar[stage]);
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else {
    const int q = warp & 3;                                        // TMEM lane quarter of this warp
    uint32_t ab = 0, aphase = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const F4Tile mt = a.tiles[t / a.tiles_w];
      const int n = (t % a.tiles_w) * 128 + q * 32 + lane, nt = min(BN, mt.row_end - mt.row0);   // weight row = output column
      const long scale_at = a.K / 2 + a.K / 16, wrow = (long)mt.group * a.group_bytes + (long)min(n, a.N - 1) * a.row_bytes + scale_at;
      const float ws = *reinterpret_cast<const float*>(a.w + wrow), ws2 = DUAL ? *reinterpret_cast<const float*>(a.w2 + wrow) : 0.0f;
      // a row's scale is a factor of every value: store_tokens applies it where there is a factor at all
      const TokenOut out{a.c_f32, a.c_bf16, (unsigned)a.ldc, DUAL ? a.row_scale : reinterpret_cast<const float*>(a.x), a.resid, (unsigned)a.ldr, a.N};
      if (!mbar_wait_warp(&acc_full[ab], aphase, abort_flag)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + ((uint32_t)(q * 32) << 16) + ab * (S::MATS * BN);
#pragma unroll 1
      for (int b = 0; b < nt; b += 32) {
        const int r = mt.row0 + b + lane;
        int orow = -1;
        float xs = 0.0f, factor = 1.0f;
        if (b + lane < nt) {
          orow = a.dst_row ? a.dst_row[r] : r;
          xs = *reinterpret_cast<const float*>(a.x + (long)r * a.row_bytes + scale_at);
          if (a.row_scale) factor = a.row_scale[r];
        }
#pragma unroll 1
        for (int h = 0; h < 32 && b + h < nt; h += 16) {
          uint32_t v[16], u[DUAL ? 16 : 1];
          tmem_ld16(tbase + b + h, v);
          if constexpr (DUAL) tmem_ld16(tbase + BN + b + h, u);
          tmem_ld_wait();
          float f[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            f[i] = __uint_as_float(v[i]) * ws;
            if constexpr (DUAL) {
              const float x = __shfl_sync(0xFFFFFFFFu, xs, h + i);
              f[i] *= x;
              f[i] = (f[i] / (1.0f + __expf(-f[i]))) * (__uint_as_float(u[i]) * ws2 * x);
            }
          }
          store_tokens<16>(out, f, orow, DUAL ? factor : xs * factor, h, n);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[ab]);
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (threadIdx.x == 0 && s_abort && a.status) atomicMax(a.status, 1u);
}

}  // namespace bl

using namespace bl;

struct Fp4GemmCall {
  const void* x; const void* w; const void* w2; const void* tiles; const int* n_tiles; float* c_f32; void* c_bf16;
  const int* dst_row; const float* row_scale; const float* resid; unsigned* status; cudaStream_t stream;
  long rows_x, ldc, ldr;
  int n_groups, N, K, max_tiles, tile_rows, sms;
};

namespace bl {

template <bool DUAL, int BN>
static int fp4_gemm_go(const Fp4GemmCall& c, const F4Args& a) {
  using S = F4Shape<DUAL, BN>;
  CUtensorMap mx, mxs, mw, mws, mw2, mws2;
  int rc = fp4_maps(&mx, &mxs, c.x, c.K, c.rows_x, 1, S::BOX);
  if (!rc) rc = fp4_maps(&mw, &mws, c.w, c.K, c.N, c.n_groups, 128);
  mw2 = mw; mws2 = mws;
  if (!rc && DUAL) rc = fp4_maps(&mw2, &mws2, c.w2, c.K, c.N, c.n_groups, 128);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) {
    cudaFuncSetAttribute(fp4_gemm_kernel<DUAL, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    limit.mark();
  }
  const long total = (long)c.max_tiles * a.tiles_w;
  return (int)launch(fp4_gemm_kernel<DUAL, BN>, dim3((unsigned)(total < c.sms ? total : c.sms)), dim3(F4_THREADS), S::SMEM, c.stream, mx, mxs,
                     mw, mws, mw2, mws2, a);
}

}  // namespace bl

extern "C" {

// C[dst_row[t] or t, n] = row_scale[t] * sum_k X[t, k] W[g][n, k] (+ resid) per token tile of the table, of at most tile_rows (32, 64,
// 128, with one matrix 256) rows.  X [rows_x], W and W2 [n_groups, N] NVFP4 rows of K values; exactly one of c_f32 / c_bf16;
// W2 != null: output = row_scale[t] * silu(X W^T) * (X W2^T).
int bl_fp4_gemm(const Fp4GemmCall* c) {
  const bool dual = c->w2 != nullptr;
  BL_REQUIRE(c->K >= 64 && c->K % 64 == 0 && c->N >= 1 && c->rows_x >= 1 && c->n_groups >= 1 && c->max_tiles >= 1 && c->sms >= 1, BL_ERR_SHAPE);
  BL_REQUIRE(c->tile_rows == 32 || c->tile_rows == 64 || c->tile_rows == 128 || (c->tile_rows == 256 && !dual), BL_ERR_SHAPE);
  BL_REQUIRE(((uintptr_t)c->x & 15) == 0 && ((uintptr_t)c->w & 15) == 0 && ((uintptr_t)c->w2 & 15) == 0, BL_ERR_ALIGN);
  BL_REQUIRE((c->c_f32 != nullptr) != (c->c_bf16 != nullptr) && c->ldc < 1L << 30 && c->ldr < 1L << 30, BL_ERR_SHAPE);
  F4Args a{};
  a.N = c->N; a.K = c->K; a.tiles_w = (c->N + 127) / 128;
  a.tiles = (const F4Tile*)c->tiles; a.n_tiles = c->n_tiles; a.max_tiles = c->max_tiles;
  BL_REQUIRE((long)a.max_tiles * a.tiles_w < 1L << 31, BL_ERR_LIMIT);
  a.x = (const uint8_t*)c->x; a.w = (const uint8_t*)c->w; a.w2 = (const uint8_t*)c->w2;
  a.row_bytes = fp4_row_bytes(c->K); a.group_bytes = a.row_bytes * c->N;
  a.c_f32 = c->c_f32; a.c_bf16 = (__nv_bfloat16*)c->c_bf16; a.ldc = c->ldc;
  a.dst_row = c->dst_row; a.row_scale = c->row_scale; a.resid = c->resid; a.ldr = c->ldr; a.status = c->status;
  if (dual) {
    if (c->tile_rows == 32) return fp4_gemm_go<true, 32>(*c, a);
    if (c->tile_rows == 64) return fp4_gemm_go<true, 64>(*c, a);
    return fp4_gemm_go<true, 128>(*c, a);
  }
  if (c->tile_rows == 32) return fp4_gemm_go<false, 32>(*c, a);
  if (c->tile_rows == 64) return fp4_gemm_go<false, 64>(*c, a);
  if (c->tile_rows == 128) return fp4_gemm_go<false, 128>(*c, a);
  return fp4_gemm_go<false, 256>(*c, a);
}

}  // extern "C"
