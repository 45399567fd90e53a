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
#include "fp4_pipe.cuh"

namespace bl {

struct F4Tile { int group, row0, row_end, pad; };

struct F4Args {
  int N, K, tiles_w, tile_rows;
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

struct F4GemmTiles {
  const F4Args& a;
  int total, kblocks;
  __device__ __forceinline__ int count() const { return total > (int)blockIdx.x ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0; }
  __device__ __forceinline__ F4Work at(int i) const {
    const int t = (int)blockIdx.x + i * (int)gridDim.x;
    const F4Tile mt = a.tiles[t / a.tiles_w];
    return F4Work{mt.group, t % a.tiles_w * 128, mt.row0, min(a.tile_rows, mt.row_end - mt.row0), 0, kblocks};
  }
};

template <bool DUAL, int BN>
__global__ void __launch_bounds__(F4_THREADS, 1)
fp4_gemm_kernel(const __grid_constant__ F4Maps map, const F4Args a) {
  using S = F4Shape<DUAL, BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) F4Bars<S> bar;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  f4_open<S>(bar);
  pdl_wait();
  pdl_launch();
  F4GemmTiles tiles{a, min(*a.n_tiles, a.max_tiles) * a.tiles_w, (a.K + 255) / 256};

  if (warp == 0) {
    if (lane == 0) f4_produce<DUAL, S>(smem, bar, map, tiles, [] { return true; });
  } else if (warp == 1) {
    f4_issue<DUAL, S>(smem, bar, tiles);
  } else if (warp >= 6) {
    f4_turn<DUAL, S>(smem, bar, tiles);
  } else {
    const int q = warp & 3;                                        // TMEM lane quarter of this warp
    uint32_t ab = 0, aphase = 0;
    for (int i = 0; i < tiles.count(); ++i) {
      const F4Work mt = tiles.at(i);
      const int n = mt.n0 + q * 32 + lane, nt = mt.rows;             // weight row = output column
      const long scale_at = a.K / 2 + a.K / 16, wrow = (long)mt.group * a.group_bytes + (long)min(n, a.N - 1) * a.row_bytes + scale_at;
      const float ws = *reinterpret_cast<const float*>(a.w + wrow), ws2 = DUAL ? *reinterpret_cast<const float*>(a.w2 + wrow) : 0.0f;
      // a row's scale is a factor of every value: store_tokens applies it where there is a factor at all
      const TokenOut out{a.c_f32, a.c_bf16, (unsigned)a.ldc, DUAL ? a.row_scale : reinterpret_cast<const float*>(a.x), a.resid, (unsigned)a.ldr, a.N};
      if (!mbar_wait_warp(&bar.acc_full[ab], aphase, &bar.abort)) break;
      tc_fence_after();
      const uint32_t tbase = bar.tmem + ((uint32_t)(q * 32) << 16) + ab * (S::MATS * BN);
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
      if (lane == 0) mbar_arrive(&bar.acc_empty[ab]);
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
    }
  }

  f4_close<S>(bar, a.status);
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
  F4Maps m;
  const int rc = f4_maps<DUAL, S>(&m, c.x, c.rows_x, c.w, c.w2, c.K, c.N, c.n_groups);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) {
    cudaFuncSetAttribute(fp4_gemm_kernel<DUAL, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    limit.mark();
  }
  const long total = (long)c.max_tiles * a.tiles_w;
  return (int)launch(fp4_gemm_kernel<DUAL, BN>, dim3((unsigned)(total < c.sms ? total : c.sms)), dim3(F4_THREADS), S::SMEM, c.stream, m, a);
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
  a.N = c->N; a.K = c->K; a.tiles_w = (c->N + 127) / 128; a.tile_rows = c->tile_rows;
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
