// Rows of activations in NVFP4 (sm_100a): E2M1 codes, an E4M3 scale for every 16 of them and one fp32 scale for the row,
//   g = max(amax(row) / 2688, 2^-100),  s = E4M3(amax(block) / (6 g)),  code = E2M1(x / (s g)),
// optionally behind an RMSNorm and scattered to the places of a routed pass (a token's row once for each of its experts).
// A thread has 16 values, or up to four times that, and keeps them: a row is read once.  Rows of up to 1,024 values are a warp's, wider ones
// a block's.  The 16 values are a block of their own for 16-bit rows.  Of fp32 rows they are four quarters of four blocks, whose other
// quarters lie in the lanes next to it: a block to a thread made every load of 16 bytes touch 16 lines, which took 5 of 27 us for the gain
// alone (4,096 x 4,096 values behind a norm).
#include "fp4_common.cuh"

namespace bl {

struct Fp4RowsArgs {
  const void* x; long ldx; int type;      // 0 bf16, 1 f16, 2 fp32
  const float* gain; double eps;
  const float* tensor_scale;              // one scale for all rows instead of their own
  int M, K;
  uint8_t* out; long ld_out; long rows_out;
  const int* pos_of; int copies;          // row m goes to rows pos_of[m * copies + j]; null: to row m
};

// NB: times 16 values of a thread; WARP: a warp has a row, else a block of threads has; F32: fp32 rows
template <int NB, bool WARP, bool F32>
__global__ void __launch_bounds__(WARP ? 256 : 512, NB == 1 ? (!F32 ? (WARP ? 8 : 4) : WARP ? 5 : 2) : NB == 2 && !WARP ? 2 : 1) fp4_rows_kernel(const Fp4RowsArgs a) {
  __shared__ double s_sum[16];
  __shared__ unsigned s_max[16];
  pdl_wait();
  pdl_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int m = WARP ? blockIdx.x * 8 + warp : blockIdx.x, w0 = WARP ? 0 : warp, wn = WARP ? 1 : warps;
  if (m >= a.M) return;
  // first value of 16-bit rows' block b, or of quarter j of fp32 rows' block b
  auto first = [&](int b, int j) { return F32 ? 512 * (w0 + b * wn) + 128 * j + 4 * lane : 16 * (32 * (w0 + b * wn) + lane); };
  auto load4 = [&](const float* row, int at, float* v) {
    const float4 f = at < a.K ? *reinterpret_cast<const float4*>(row + at) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  };
  float v[F32 ? NB : 1][16];
  uint32_t half[F32 ? 1 : NB][8];                     // 16-bit rows stay as they are until they are rounded
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) load4(reinterpret_cast<const float*>(a.x) + (long)m * a.ldx, first(b, j), v[b] + 4 * j);
    } else {
      uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
      if (first(b, 0) < a.K) {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.x) + (long)m * a.ldx + first(b, 0));
        lo = p[0]; hi = p[1];
      }
      half[b][0] = lo.x; half[b][1] = lo.y; half[b][2] = lo.z; half[b][3] = lo.w;
      half[b][4] = hi.x; half[b][5] = hi.y; half[b][6] = hi.z; half[b][7] = hi.w;
    }
  }
  if constexpr (F32) {
    if (a.gain) {
      auto whole = [&](double ss) {
        ss = warp_sum_d(ss);
        if (!WARP) {
          if (lane == 0) s_sum[warp] = ss;
          __syncthreads();
          ss = 0.0;
          for (int w = 0; w < warps; ++w) ss += s_sum[w];
        }
        return ss;
      };
      double ss = 0.0;
#pragma unroll
      for (int b = 0; b < NB; ++b) ss += fp4_squares16(v[b]);
      ss = whole(ss);
      if (!fp4_sum_holds(ss)) {                       // the same for all threads of the row
        if (!WARP) __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int b = 0; b < NB; ++b) ss += fp4_squares16_wide(v[b]);
        ss = whole(ss);
      }
      const float r = fp4_rsqrt(ss / (double)a.K + a.eps);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float g[4];
          load4(a.gain, first(b, j), g);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[b][4 * j + i] = first(b, j) < a.K ? v[b][4 * j + i] * r * g[i] : 0.0f;
        }
    }
  }
  unsigned own[NB][4], top = 0;                       // the largest of a block, or of each block that a quarter is of
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned t = fp4_top<4>(v[b] + 4 * j);
        t = max(t, __shfl_xor_sync(0xFFFFFFFFu, t, 1));
        own[b][j] = max(t, __shfl_xor_sync(0xFFFFFFFFu, t, 2));
        top = max(top, own[b][j]);
      }
    } else {
      unsigned t = half[b][0] & 0x7fff7fffu;          // magnitudes of either type grow with their bits, and NaN is above everything
#pragma unroll
      for (int j = 1; j < 8; ++j) t = __vmaxu2(t, half[b][j] & 0x7fff7fffu);
      t = max(t >> 16, t & 0xffffu);
      own[b][0] = a.type == 0 ? t << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)t)));
      top = max(top, own[b][0]);
    }
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (!WARP) {
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? s_max[lane] : 0u);
  }
  float g = fp4_row_scale(top);
  if (a.tensor_scale && top < FP4_INF) {
    g = *a.tensor_scale;
    g = g < __uint_as_float(FP4_INF) ? fmaxf(g, FP4_LEAST) : __uint_as_float(0x7fc00000u);        // NaN where it is no finite number
  }
  const float inv6g = fp4_inv6(g);
  auto places = [&](auto&& store) {
    for (int j = 0; j < a.copies; ++j) {
      const long p = a.pos_of ? a.pos_of[(long)m * a.copies + j] : m;
      if (p >= 0 && p < a.rows_out) store(a.out + p * a.ld_out);
    }
  };
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if constexpr (F32) {
      // lane i of four finds the scale of the block that quarters i are of
      const int i = lane & 3;
      unsigned scale = 0;
      float s = 0.0f;
      if (g > 0.0f) scale = fp4_block_scale(__uint_as_float(i == 0 ? own[b][0] : i == 1 ? own[b][1] : i == 2 ? own[b][2] : own[b][3]), g, inv6g, s);
      const float d = s * g, inv = scale ? __fdividef(1.0f, d) : 0.0f;
      unsigned codes[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float dj = __shfl_sync(0xFFFFFFFFu, d, (lane & ~3) | j), ij = __shfl_sync(0xFFFFFFFFu, inv, (lane & ~3) | j);
        codes[j] = ij > 0.0f ? fp4_codes<4>(v[b] + 4 * j, dj, ij * FP4_BELOW, ij * FP4_ABOVE) : 0u;
      }
      // the four quarters of a block to the lane that has its scale: blocks 0, 1 and 2, 3 change lanes two apart, then those next to each other
      const unsigned c01 = codes[0] | codes[1] << 16, c23 = codes[2] | codes[3] << 16, h = i >> 1, odd = i & 1;
      const unsigned mine = h ? c23 : c01, theirs = __shfl_xor_sync(0xFFFFFFFFu, h ? c01 : c23, 2);
      const unsigned kept = odd ? (mine >> 16) | (theirs & 0xffff0000u) : (mine & 0xffffu) | theirs << 16;          // quarters i and i ^ 2 of block i
      const unsigned other = __shfl_xor_sync(0xFFFFFFFFu, odd ? (mine & 0xffffu) | theirs << 16 : (mine >> 16) | (theirs & 0xffff0000u), 1);
      const unsigned lo = odd ? other : kept, hi = odd ? kept : other, near = (lo & 0xffffu) | hi << 16, far = (lo >> 16) | (hi & 0xffff0000u);
      const int at = (512 * (w0 + b * wn) + 128 * i + 4 * (lane & ~3)) / 16;
      if (16 * at >= a.K) continue;
      places([&](uint8_t* row) {
        *reinterpret_cast<uint2*>(row + 8 * at) = h ? make_uint2(far, near) : make_uint2(near, far);
        row[a.K / 2 + at] = (uint8_t)scale;
        if (at == 0) *reinterpret_cast<float*>(row + a.K / 2 + a.K / 16) = g;
      });
    } else {
      const int at = first(b, 0) / 16;
      if (first(b, 0) >= a.K) break;
      unsigned scale;
      float f[16];
      fp4_open16(half[b], a.type, f);
      const uint2 codes = fp4_block(f, own[b][0], g, inv6g, scale);
      places([&](uint8_t* row) {
        *reinterpret_cast<uint2*>(row + 8 * at) = codes;
        row[a.K / 2 + at] = (uint8_t)scale;
        if (at == 0) *reinterpret_cast<float*>(row + a.K / 2 + a.K / 16) = g;
      });
    }
  }
}

template <bool F32>
static int fp4_rows_go(const Fp4RowsArgs& a, cudaStream_t st) {
  const int blocks = a.K / 16;
  if (blocks <= 32) return (int)launch(fp4_rows_kernel<1, true, F32>, dim3((a.M + 7) / 8), dim3(256), 0, st, a);
  if (blocks <= 64) return (int)launch(fp4_rows_kernel<2, true, F32>, dim3((a.M + 7) / 8), dim3(256), 0, st, a);
  // (fp32 rows of 4,096 behind a norm: 23.5 us with 32 values a thread, 26 with 16; 16-bit ones are the same)
  const int nb = blocks <= (F32 ? 128 : 256) ? 1 : blocks <= 512 ? 2 : 4, thr = ((blocks + nb - 1) / nb + 31) / 32 * 32;
  if (nb == 1) return (int)launch(fp4_rows_kernel<1, false, F32>, dim3(a.M), dim3(thr), 0, st, a);
  if (nb == 2) return (int)launch(fp4_rows_kernel<2, false, F32>, dim3(a.M), dim3(thr), 0, st, a);
  return (int)launch(fp4_rows_kernel<4, false, F32>, dim3(a.M), dim3(thr), 0, st, a);
}

}  // namespace bl

using namespace bl;

struct Fp4RowsCall {
  const void* x; const float* gain; const float* tensor_scale; const int* pos_of; void* out; cudaStream_t stream;
  long ldx, rows_out;
  double eps;
  int type, M, K, copies;
};

extern "C" {

// NVFP4 rows of M rows of x (type 0 bf16, 1 f16, 2 fp32; ldx elements); gain != null: RMSNorm with that gain first (fp32 rows);
// tensor_scale != null: that scale for every row (2^-100 at least; NaN where it is not finite); pos_of != null: row m goes to rows pos_of[m * copies + j] < rows_out (others
// nowhere).
int bl_fp4_rows(const Fp4RowsCall* c) {
  BL_REQUIRE(c->M >= 1 && c->K >= 64 && c->K % 64 == 0 && c->copies >= 1 && c->rows_out >= 1, BL_ERR_SHAPE);
  BL_REQUIRE(c->K <= 32768, BL_ERR_LIMIT);
  BL_REQUIRE(c->type >= 0 && c->type <= 2 && (!c->gain || c->type == 2), BL_ERR_TYPE);
  BL_REQUIRE(c->ldx >= c->K && c->ldx % (c->type == 2 ? 4 : 8) == 0 && ((uintptr_t)c->x & 15) == 0 && ((uintptr_t)c->out & 15) == 0 &&
                 ((uintptr_t)c->gain & 15) == 0, BL_ERR_ALIGN);
  BL_REQUIRE(c->pos_of || (c->copies == 1 && c->rows_out >= c->M), BL_ERR_SHAPE);
  Fp4RowsArgs a{c->x, c->ldx, c->type, c->gain, c->eps, c->tensor_scale, c->M, c->K, (uint8_t*)c->out, fp4_row_bytes(c->K), c->rows_out,
                c->pos_of, c->copies};
  return c->type == 2 ? fp4_rows_go<true>(a, c->stream) : fp4_rows_go<false>(a, c->stream);
}

}  // extern "C"
