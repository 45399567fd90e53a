// Grouped product of NVFP4 rows with NVFP4 weights on tcgen05 (sm_100a): four-bit codes go to the tensor cores as they are.
//   C[t, n] = xs[t] ws[n] sum_b sx[t, b] sw[n, b] sum_{k in block b} x[t, k] w[g][n, k]        blocks of 16 values
//
// The weight rows of a tile are the M side of the MMA, its tokens the N side.  TMA threads stream boxes of 256 values: 128 bytes of
// codes a row (128-byte swizzle) and, for several boxes at once, 16 bytes of scales.  Weights and activations keep the layout of their rows in
// memory, which the decode chain reads too: four warps bring a stage's scales into the cells of tensor memory that the instruction reads
// (tcgen05.st).  The issuing warp issues four kind::mxf4nvf4 MMAs a stage, K = 64 each, which multiply codes, apply both blocks' scales and
// add in fp32.  Eight epilogue warps apply the two fp32 scales.
//   * "dual" mode runs gate and up in one main loop; the epilogue writes silu(gate) * up;
//   * the epilogue scatters and scales like the other GEMMs (dst_row / row_scale / resid).
// 4,096 tokens x 8,192 x 4,096: 100 us (2.75 PFLOP/s), of which the main loop 85, waiting for TMA (1.04 GB to the processors, 1.6 sectors a
// request of L2, which is at 54 % of its throughput); gate and up of 2,000 ids on 128
// experts of 768 x 2,048: 63 us (249 MB, 4.0 TB/s; 54 without an epilogue, which one accumulator of each matrix leaves no room to
// overlap); down of 4,096 ids: 96 us, of which the stores of 268 MB are 20.
// Every wait is bounded; on expiry the CTA raises status word 1, leaves its loops, frees its TMEM and returns.
#include "fp4_pipe.cuh"

namespace bl {

constexpr int F4_GEMM_ROOM = 200 * 1024, F4_GEMM_WARPS = 8;

struct F4Tile { int group, row0, row_end, pad; };

struct F4Args {
  int N, K, tiles_w, tile_rows;
  const F4Tile* tiles;
  const int* n_tiles;
  int max_tiles, fixed;
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
  int rows_out;             // of the output: others are none
  int wide;                 // rows of the output (and of resid) start at 16 bytes and hold whole 16 bytes
};

template <int AR>
struct F4GemmTiles {
  const F4Args& a;
  int total, kblocks;
  __device__ __forceinline__ int count() const { return total > (int)blockIdx.x ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0; }
  __device__ __forceinline__ F4Work work(const F4Tile& mt, int column) const {
    return F4Work{mt.group, column * AR, mt.row0, min(a.tile_rows, mt.row_end - mt.row0), 0, kblocks};
  }
  __device__ __forceinline__ F4Work at(int i) const {
    const int t = (int)blockIdx.x + i * (int)gridDim.x;
    return work(a.tiles[t / a.tiles_w], t % a.tiles_w);
  }
};

// 16 tokens of the 32 columns from n0 on (below `end`), `f` this lane's column of them (lane = column); rows below zero are none.
// Wide: they are turned in shared memory, so that a lane stores 16 bytes of a token: a store of four bytes, or two, costs its warp some 19
// clocks with the address of its token, 16 bytes cost them for four tokens, or eight.
__device__ __forceinline__ void f4_store16(const F4Args& a, const float (&f)[16], const int* rows, int n0, int end, uint8_t* stage, int lane) {
  if (a.wide && a.c_bf16 && !a.resid) {
    __nv_bfloat16* s = reinterpret_cast<__nv_bfloat16*>(stage);
#pragma unroll
    for (int j = 0; j < 16; ++j) s[32 * j + lane] = __float2bfloat16_rn(f[j]);
    __syncwarp();
    const int n = n0 + 8 * (lane & 3), none = n < end ? 0 : -1;
    int row[2];
    uint4 v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      row[j] = rows[8 * j + (lane >> 2)] | none;
      v[j] = *reinterpret_cast<const uint4*>(s + 32 * (8 * j + (lane >> 2)) + 8 * (lane & 3));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (row[j] >= 0) *reinterpret_cast<uint4*>(a.c_bf16 + (unsigned long long)(unsigned)row[j] * (unsigned)a.ldc + n) = v[j];
    __syncwarp();
    return;
  }
  float* s = reinterpret_cast<float*>(stage);
#pragma unroll
  for (int j = 0; j < 16; ++j) s[32 * j + lane] = f[j];
  __syncwarp();
  if (a.wide) {
    const int n = n0 + 4 * (lane & 7), none = n < end ? 0 : -1;
    int row[4];
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      row[j] = rows[4 * j + (lane >> 3)] | none;
      v[j] = *reinterpret_cast<const float4*>(s + 32 * (4 * j + (lane >> 3)) + 4 * (lane & 7));
    }
    if (a.resid) {
      float4 r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] = row[j] >= 0 ? *reinterpret_cast<const float4*>(a.resid + (unsigned long long)(unsigned)row[j] * (unsigned)a.ldr + n)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j].x += r[j].x; v[j].y += r[j].y; v[j].z += r[j].z; v[j].w += r[j].w; }
    }
    if (a.c_f32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row[j] >= 0) *reinterpret_cast<float4*>(a.c_f32 + (unsigned long long)(unsigned)row[j] * (unsigned)a.ldc + n) = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[j].x, v[j].y), hi = __floats2bfloat162_rn(v[j].z, v[j].w);
        if (row[j] >= 0)
          *reinterpret_cast<uint2*>(a.c_bf16 + (unsigned long long)(unsigned)row[j] * (unsigned)a.ldc + n) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      }
    }
  } else {
    const int n = n0 + lane;
#pragma unroll 8
    for (int j = 0; j < 16; ++j) {
      const int row = rows[j];
      float v = s[32 * j + lane];
      if (row < 0 || n >= end) continue;
      if (a.resid) v += a.resid[(unsigned long long)(unsigned)row * (unsigned)a.ldr + n];
      if (a.c_f32) a.c_f32[(unsigned long long)(unsigned)row * (unsigned)a.ldc + n] = v;
      else a.c_bf16[(unsigned long long)(unsigned)row * (unsigned)a.ldc + n] = __float2bfloat16_rn(v);
    }
  }
  __syncwarp();
}

template <bool DUAL, int BN, int AR>
__global__ void __launch_bounds__(F4_EPILOGUE + 32 * F4_GEMM_WARPS, 1)
fp4_gemm_kernel(const __grid_constant__ F4Maps map, const F4Args a) {
  using S = F4Shape<DUAL, BN, F4_GEMM_ROOM, F4_GEMM_WARPS, AR>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) F4Bars<S> bar;
  __shared__ __align__(16) int s_row[2][BN];
  __shared__ __align__(16) float s_xs[2][BN], s_factor[2][DUAL ? BN : 1];
  __shared__ __align__(16) uint8_t s_stage[F4_GEMM_WARPS][2048];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  f4_open<S>(bar, map);
  // A table that the host wrote and the weights are there before the launch in front of this one ends; the rows are not.
  if (!a.fixed || warp >= 6) {
    pdl_wait();
    pdl_launch();
  }
  F4GemmTiles<AR> tiles{a, (a.fixed ? a.max_tiles : min(*a.n_tiles, a.max_tiles)) * a.tiles_w, (a.K + 255) / 256};

  if (warp == 0) {
    if (lane == 0) f4_weights<S>(smem, bar, map, tiles);
  } else if (warp == 6) {
    if (lane == 0) f4_tokens<S>(smem, bar, map, tiles);
  } else if (warp == 1) {
    f4_issue<S>(smem, bar, tiles);
  } else if (warp < 6) {
    f4_cells<S>(smem, bar, tiles);
  } else {
    const int q = warp & 3, half = (warp - 7) >> 2, et = threadIdx.x - F4_EPILOGUE;          // TMEM lane quarter of this warp; 0 .. 255
    const int n_tiles = tiles.count();
    const long scale_at = a.K / 2 + a.K / 16;
    // What a tile needs beside its products is asked for while the tile before is worked on, a token a thread, and laid down in shared
    // memory behind it; the entry of the table a tile earlier.  Where K is short these warps are what a tile waits for: the entry is not looked
    // into before it is used, and the places of the tiles are walked without divisions (down of 4,096 ids 98.8 -> 96.2 us).
    struct Beside { int row; float xs, factor, ws, ws2; } nxt{};
    auto open = [&](const F4Work& w) {
      const int r = w.row0 + et;
      nxt.row = -1;
      if (et < w.rows) {
        nxt.row = a.dst_row ? a.dst_row[r] : r;
        nxt.xs = *reinterpret_cast<const float*>(a.x + (long)r * a.row_bytes + scale_at);
        nxt.factor = a.row_scale ? a.row_scale[r] : 1.0f;
      }
      const long at = (long)w.group * a.group_bytes + (long)min(w.n0 + q * 32 + lane, a.N - 1) * a.row_bytes + scale_at;
      nxt.ws = *reinterpret_cast<const float*>(a.w + at);
      if (DUAL) nxt.ws2 = *reinterpret_cast<const float*>(a.w2 + at);
    };
    uint32_t ab = 0, aphase = 0;
    F4Work w{}, w1{};                                              // this tile and the next one, behind it an entry and its column
    F4Tile t2{};
    int c2 = 0;
    if (n_tiles > 0) { w1 = tiles.at(0); open(w1); }
    const int m_step = (int)gridDim.x / a.tiles_w, c_step = (int)gridDim.x % a.tiles_w;
    int m = (int)blockIdx.x / a.tiles_w, c = (int)blockIdx.x % a.tiles_w;
    auto ask = [&]() {                                             // the entry of the tile one further
      m += m_step;
      c += c_step;
      if (c >= a.tiles_w) { c -= a.tiles_w; ++m; }
      t2 = a.tiles[m];
      c2 = c;
    };
    if (n_tiles > 1) ask();
    for (int i = 0; i < n_tiles; ++i) {
      w = w1;
      if (i + 1 < n_tiles) w1 = tiles.work(t2, c2);
      const float ws = nxt.ws, ws2 = nxt.ws2;
      if (et < BN) {
        s_row[i & 1][et] = nxt.row < a.rows_out ? nxt.row : -1;           // here, where it has arrived
        s_xs[i & 1][et] = DUAL ? nxt.xs : nxt.xs * nxt.factor;
        if (DUAL) s_factor[i & 1][et] = nxt.factor;
      }
      if (i + 1 < n_tiles) open(w1);
      if (i + 2 < n_tiles) ask();
      if (!f4_all<F4_GEMM_WARPS>(mbar_wait_warp(&bar.acc_full[ab], aphase, &bar.abort))) break;
      tc_fence_after();
      const uint32_t tbase = bar.tmem + ((uint32_t)(q * 32) << 16) + ab * (S::MATS * BN);
#pragma unroll 1
      for (int b = 16 * half; b < w.rows && q * 32 < AR; b += 32) {               // the two warps of a quarter take 16 tokens each in turn
        uint32_t v[16], u[DUAL ? 16 : 1];
        tmem_ld16(tbase + b, v);
        if constexpr (DUAL) tmem_ld16(tbase + BN + b, u);
        tmem_ld_wait();
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 x4 = *reinterpret_cast<const float4*>(&s_xs[i & 1][b + j]);
          const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            f[j + c] = __uint_as_float(v[j + c]) * ws * x[c];
            if constexpr (DUAL) {
              f[j + c] = fp4_silu(f[j + c]) * (__uint_as_float(u[j + c]) * ws2 * x[c]);
              if (a.row_scale) f[j + c] *= s_factor[i & 1][b + j + c];
            }
          }
        }
        f4_store16(a, f, &s_row[i & 1][b], w.n0 + q * 32, min(a.N, w.n0 + AR), s_stage[warp - 7], lane);
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
  int n_groups, N, K, max_tiles, tile_rows, sms, fixed, rows_out;
};

namespace bl {

template <bool DUAL, int BN, int AR>
static int fp4_gemm_go(const Fp4GemmCall& c, F4Args& a) {
  a.tiles_w = (c.N + AR - 1) / AR;
  using S = F4Shape<DUAL, BN, F4_GEMM_ROOM, F4_GEMM_WARPS, AR>;
  F4Maps m;
  const int rc = f4_maps<S>(&m, c.x, c.rows_x, c.w, c.w2, c.K, c.N, c.n_groups);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) {
    cudaFuncSetAttribute(fp4_gemm_kernel<DUAL, BN, AR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    limit.mark();
  }
  const long total = (long)c.max_tiles * a.tiles_w;
  return (int)launch(fp4_gemm_kernel<DUAL, BN, AR>, dim3((unsigned)(total < c.sms ? total : c.sms)), dim3(S::THREADS), S::SMEM, c.stream, m, a);
}

}  // namespace bl

extern "C" {

// Rows of C from 0 to rows_out - 1, others nowhere:
// C[dst_row[t] or t, n] = row_scale[t] * sum_k X[t, k] W[g][n, k] (+ resid) per token tile of the table, of at most tile_rows (32, 64,
// 128, with one matrix 256) rows.  X [rows_x], W and W2 [n_groups, N] NVFP4 rows of K values; exactly one of c_f32 / c_bf16;
// fixed: the table has exactly max_tiles tiles, and no launch in flight writes it or the weights.
// W2 != null: output = row_scale[t] * silu(X W^T) * (X W2^T).
int bl_fp4_gemm(const Fp4GemmCall* c) {
  const bool dual = c->w2 != nullptr;
  BL_REQUIRE(c->K >= 64 && c->K % 64 == 0 && c->N >= 1 && c->rows_x >= 1 && c->n_groups >= 1 && c->max_tiles >= 1 && c->sms >= 1, BL_ERR_SHAPE);
  BL_REQUIRE(c->tile_rows == 32 || c->tile_rows == 64 || c->tile_rows == 128 || (c->tile_rows == 256 && !dual), BL_ERR_SHAPE);
  BL_REQUIRE(((uintptr_t)c->x & 15) == 0 && ((uintptr_t)c->w & 15) == 0 && ((uintptr_t)c->w2 & 15) == 0, BL_ERR_ALIGN);
  BL_REQUIRE((c->c_f32 != nullptr) != (c->c_bf16 != nullptr) && c->ldc < 1L << 30 && c->ldr < 1L << 30, BL_ERR_SHAPE);
  F4Args a{};
  a.N = c->N; a.K = c->K; a.tile_rows = c->tile_rows;
  a.tiles = (const F4Tile*)c->tiles; a.n_tiles = c->n_tiles; a.max_tiles = c->max_tiles; a.fixed = c->fixed;
  BL_REQUIRE((long)a.max_tiles * ((c->N + 15) / 16) < 1L << 31, BL_ERR_LIMIT);
  a.x = (const uint8_t*)c->x; a.w = (const uint8_t*)c->w; a.w2 = (const uint8_t*)c->w2;
  a.row_bytes = fp4_row_bytes(c->K); a.group_bytes = a.row_bytes * c->N;
  a.c_f32 = c->c_f32; a.c_bf16 = (__nv_bfloat16*)c->c_bf16; a.ldc = c->ldc;
  a.dst_row = c->dst_row; a.row_scale = c->row_scale; a.resid = c->resid; a.ldr = c->ldr; a.status = c->status; a.rows_out = c->rows_out;
  const int es = c->c_f32 ? 4 : 2;
  a.wide = (((uintptr_t)c->c_f32 | (uintptr_t)c->c_bf16 | (uintptr_t)c->resid) & 15) == 0 && c->ldc * es % 16 == 0 && (!c->resid || c->ldr % 4 == 0) &&
           c->N % (c->c_f32 || c->resid ? 4 : 8) == 0;
  // Weight rows of a tile: as few as still find a processor for each tile at once.
  auto one_wave = [&](int ar) { return (long)c->max_tiles * ((c->N + ar - 1) / ar) <= c->sms; };
  const int rows = c->tile_rows, ar = one_wave(16) ? 16 : one_wave(32) ? 32 : one_wave(64) ? 64 : 128;
  if (dual) {
    if (rows == 32) return ar <= 32 ? fp4_gemm_go<true, 32, 32>(*c, a) : ar == 64 ? fp4_gemm_go<true, 32, 64>(*c, a) : fp4_gemm_go<true, 32, 128>(*c, a);
    if (rows == 64) return ar <= 64 ? fp4_gemm_go<true, 64, 64>(*c, a) : fp4_gemm_go<true, 64, 128>(*c, a);
    return fp4_gemm_go<true, 128, 128>(*c, a);
  }
  if (rows == 32)
    return ar == 16 ? fp4_gemm_go<false, 32, 16>(*c, a) : ar == 32 ? fp4_gemm_go<false, 32, 32>(*c, a) : ar == 64 ? fp4_gemm_go<false, 32, 64>(*c, a)
                                                                                                                  : fp4_gemm_go<false, 32, 128>(*c, a);
  if (rows == 64)
    return ar <= 32 ? fp4_gemm_go<false, 64, 32>(*c, a) : ar == 64 ? fp4_gemm_go<false, 64, 64>(*c, a) : fp4_gemm_go<false, 64, 128>(*c, a);
  if (rows == 128) return ar <= 64 ? fp4_gemm_go<false, 128, 64>(*c, a) : fp4_gemm_go<false, 128, 128>(*c, a);
  return fp4_gemm_go<false, 256, 128>(*c, a);
}

}  // extern "C"
