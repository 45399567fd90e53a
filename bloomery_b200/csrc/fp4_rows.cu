// Rows of activations in NVFP4 (sm_100a): E2M1 codes, an E4M3 scale for every 16 of them and one fp32 scale for the row,
//   g = max(amax(row) / 2688, 2^-100),  s = E4M3(amax(block) / (6 g)),  code = E2M1(x / (s g)),
// optionally behind an RMSNorm and scattered to the places of a routed pass (a token's row once for each of its experts).
// One block a row, 16 values a thread and up to four times that: the row is read once and stays in registers.
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

template <int NB>
__global__ void __launch_bounds__(512) fp4_rows_kernel(const Fp4RowsArgs a) {
  __shared__ double s_sum[16];
  __shared__ unsigned s_max[16];
  pdl_wait();
  pdl_launch();
  const int m = blockIdx.x, tid = threadIdx.x, nthr = blockDim.x, warp = tid >> 5, lane = tid & 31, warps = nthr >> 5;
  const int blocks = a.K / 16;
  float v[NB][16];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (tid + b * nthr < blocks) fp4_load16(a.x, a.type, (long)m * a.ldx + 16 * (tid + b * nthr), v[b]);
  if (a.gain) {
    double ss = 0.0;
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (tid + b * nthr < blocks) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fma((double)v[b][i], (double)v[b][i], ss);
      }
    ss = warp_sum_d(ss);
    if (lane == 0) s_sum[warp] = ss;
    __syncthreads();
    double all = 0.0;
    for (int w = 0; w < warps; ++w) all += s_sum[w];
    const float r = fp4_rsqrt(all / (double)a.K + a.eps);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (tid + b * nthr < blocks) fp4_scale16(v[b], r, a.gain + 16 * (tid + b * nthr));
  }
  unsigned top = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (tid + b * nthr < blocks) top = max(top, fp4_top16(v[b]));
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (lane == 0) s_max[warp] = top;
  __syncthreads();
  for (int w = 0; w < warps; ++w) top = max(top, s_max[w]);
  float g = fp4_row_scale(top);
  if (a.tensor_scale && top < FP4_INF) g = fmaxf(*a.tensor_scale, FP4_LEAST);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int at = tid + b * nthr;
    if (at >= blocks) break;
    unsigned scale;
    const uint2 codes = fp4_block(v[b], g, scale);
    for (int j = 0; j < a.copies; ++j) {
      const long p = a.pos_of ? a.pos_of[(long)m * a.copies + j] : m;
      if (p < 0 || p >= a.rows_out) continue;
      uint8_t* row = a.out + p * a.ld_out;
      *reinterpret_cast<uint2*>(row + 8 * at) = codes;
      row[a.K / 2 + at] = (uint8_t)scale;
      if (at == 0) *reinterpret_cast<float*>(row + a.K / 2 + a.K / 16) = g;
    }
  }
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
// tensor_scale != null: that scale for every row; pos_of != null: row m goes to rows pos_of[m * copies + j] < rows_out (others
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
  const int blocks = c->K / 16, nb = blocks <= 256 ? 1 : blocks <= 512 ? 2 : 4;
  const int thr = ((blocks + nb - 1) / nb + 31) / 32 * 32;
  if (nb == 1) return (int)launch(fp4_rows_kernel<1>, dim3(c->M), dim3(thr), 0, c->stream, a);
  if (nb == 2) return (int)launch(fp4_rows_kernel<2>, dim3(c->M), dim3(thr), 0, c->stream, a);
  return (int)launch(fp4_rows_kernel<4>, dim3(c->M), dim3(thr), 0, c->stream, a);
}

}  // extern "C"
