// What the NVFP4 kernels share: the quantiser of a block of 16 values and the tcgen05 instructions of block-scaled four-bit
// operands.
//
// A row of K values is K / 2 bytes of E2M1 codes (the even value in the low half), K / 16 E4M3 scales and one fp32 scale, padded
// to 16 bytes: value = code * scale * row scale.  Weights of a checkpoint and quantised activations have the same layout.
//
// Quantising is exact: the scale of a block is the E4M3 value nearest to amax / (6 g), a code the E2M1 value nearest to x / d
// with d = scale * g in fp32, ties to the even code, in the reals.  Quotients in fp32 decide all but the values next to a midpoint
// m; there the sign of fma(-m, d, x) decides, which has one rounding and so the right sign.
#pragma once
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include "tc_common.cuh"

namespace bl {

constexpr float FP4_ROW = 2688.0f;                    // 6 * 448: what a row's largest value becomes
constexpr float FP4_LEAST = 7.888609052210118e-31f;   // 2^-100, the least row scale: keeps a row of zeros, and 1 / d, in range
constexpr unsigned FP4_INF = 0x7f800000u;

__host__ __device__ constexpr long fp4_row_bytes(int K) { return (K / 2 + K / 16 + 4 + 15) / 16 * 16; }

// The scale of a row whose largest magnitude has these bits; NaN where that is none.
__device__ __forceinline__ float fp4_row_scale(unsigned amax_bits) {
  return amax_bits < FP4_INF ? fmaxf(__fdiv_rn(__uint_as_float(amax_bits), FP4_ROW), FP4_LEAST) : __uint_as_float(0x7fc00000u);
}

// E4M3 code nearest to amax / (6 g), inv6g next to 1 / (6 g); its value in `s`
__device__ __forceinline__ unsigned fp4_block_scale(float amax, float g, float inv6g, float& s) {
  unsigned c = __nv_cvt_float_to_fp8(fminf(amax * inv6g, 448.0f), __NV_SATFINITE, __NV_E4M3);
  // its neighbours: there is none (NaN, which decides nothing) below 0 and above 448
  const __half2_raw around = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((c - 1 & 0xff) | (c + 1) << 8), __NV_E4M3);
  const float2 n = __half22float2(*reinterpret_cast<const __half2*>(&around));
  const __half_raw mid = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3);
  s = __half2float(*reinterpret_cast<const __half*>(&mid));
  const float lo = fmaf(-3.0f * (s + n.x), g, amax), hi = fmaf(-3.0f * (s + n.y), g, amax);       // 6 times the midpoints: seven bits
  if (hi > 0.0f || (hi == 0.0f && (c & 1))) { ++c; s = n.y; }
  else if (lo < 0.0f || (lo == 0.0f && (c & 1))) { --c; s = n.x; }
  return c;
}

// Two fp32 values in one register pair, and the instruction that works on both
__device__ __forceinline__ uint64_t f2_pack(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 f2_open(uint64_t v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// Codes of eight values times `f` (value i in bits 4i ..), or of four
template <int N>
__device__ __forceinline__ uint32_t fp4_round(const float* x, float f) {
  const uint64_t ff = f2_pack(f, f);
  float2 y[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) y[i] = f2_open(f2_mul(f2_pack(x[2 * i], x[2 * i + 1]), ff));
  uint32_t r;
  if constexpr (N == 8)
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(y[0].x), "f"(y[0].y), "f"(y[1].x), "f"(y[1].y), "f"(y[2].x), "f"(y[2].y), "f"(y[3].x), "f"(y[3].y));
  else
    asm("{\n\t.reg .b8 a, b;\n\t.reg .b16 w;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "mov.b16 w, {a, b};\n\tcvt.u32.u16 %0, w;\n\t}"
        : "=r"(r) : "f"(y[0].x), "f"(y[0].y), "f"(y[1].x), "f"(y[1].y));
  return r;
}
// Codes of N values, steps of d.  The quotients are off by less than 2^-21; where 2^-20 to either side gives another code the midpoint
// is looked at itself.
template <int N>
__device__ __forceinline__ uint32_t fp4_codes(const float* x, float d, float lo, float hi) {
  uint32_t a = fp4_round<N>(x, lo);
  const uint32_t b = fp4_round<N>(x, hi);
  // 16-bit values meet midpoints often (their quotients are ratios of small numbers): one value at a time, and only those
  for (uint32_t m = a ^ b; m;) {
    const int i = (__ffs(m) - 1) >> 2;
    m &= ~(0xfu << (4 * i));
    const unsigned c = a >> (4 * i) & 7u;             // b's is one step above: c < 7
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = x[j];
#pragma unroll
    for (int n = N / 2; n > 0; n /= 2)
#pragma unroll
      for (int j = 0; j < n; ++j) v[j] = i & n ? v[j + n] : v[j];
    const float mid = c < 4 ? 0.5f * (float)c + 0.25f : c == 4 ? 2.5f : c == 5 ? 3.5f : 5.0f, r = fmaf(-mid, d, fabsf(v[0]));
    if (r > 0.0f || (r == 0.0f && (c & 1))) a += 1u << (4 * i);
  }
  return a;
}
constexpr float FP4_BELOW = 1.0f - 9.5367431640625e-7f, FP4_ABOVE = 1.0f + 9.5367431640625e-7f;      // 2^-20 to either side

// A block of 16 values of a row with scale g, the largest of them with the bits `top`: its codes and the byte of its scale.  A row with
// anything that is not finite has NaN for g and gets zeros: its products are NaN by the row scale alone.
__device__ __forceinline__ uint2 fp4_block(const float* x, unsigned top, float g, float inv6g, unsigned& scale) {
  scale = 0;
  if (!(g > 0.0f)) return make_uint2(0u, 0u);
  float s;
  scale = fp4_block_scale(__uint_as_float(top), g, inv6g, s);
  if (scale == 0u) return make_uint2(0u, 0u);
  const float d = s * g, inv = __fdividef(1.0f, d), lo = inv * FP4_BELOW, hi = inv * FP4_ABOVE;
  return make_uint2(fp4_codes<8>(x, d, lo, hi), fp4_codes<8>(x + 8, d, lo, hi));
}

// ---- pieces of a row --------------------------------------------------------------------------------------
__device__ __forceinline__ void fp4_open16(const uint32_t (&w)[8], int type, float* v) {       // 16 values of type 0 bf16, 1 f16
  if (type == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u); }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void fp4_load16(const void* x, int type, long at, float* v) {       // 2: fp32
  if (type == 2) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float4 f = p[i]; v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w; }
  } else {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + at);
    const uint4 lo = p[0], hi = p[1];
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    fp4_open16(w, type, v);
  }
}
// 1 / sqrt(x) in fp32: two of Newton's steps in 64 bits behind rsqrtf, which leave 2^-52 or so in front of the rounding, are a few
// instructions where the library's root and quotient are a hundred that have to be fetched.
__device__ __forceinline__ float fp4_rsqrt(double x) {
  if (!(x > 1e-30 && x < 1e30)) return (float)(1.0 / sqrt(x));
  double y = (double)rsqrtf((float)x);
  const double h = 0.5 * x;
  y = y * fma(-h * y, y, 1.5);
  y = y * fma(-h * y, y, 1.5);
  return (float)y;
}
// v * r * gain
__device__ __forceinline__ void fp4_scale16(float* v, float r, const float* gain) {
  const float4* g4 = reinterpret_cast<const float4*>(gain);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 g = g4[i];
    v[4 * i] = v[4 * i] * r * g.x; v[4 * i + 1] = v[4 * i + 1] * r * g.y;
    v[4 * i + 2] = v[4 * i + 2] * r * g.z; v[4 * i + 3] = v[4 * i + 3] * r * g.w;
  }
}
// Sum of squares of 16 values: 16 roundings to 24 bits of a part, of which hundreds are added in 64 bits behind this (two fp32 parts
// with what each rounding left cost 136 clocks a warp, this 16; the root of the whole then moves by one unit of its last place
// in one row of twenty or so).
__device__ __forceinline__ double fp4_squares16(const float* v) {
  float s = v[0] * v[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) s = fmaf(v[i], v[i], s);
  return (double)s;
}
// Whether a row's sum of those can stand: a part past fp32's largest is infinite, and squares below its normal numbers lose bits that count
// where there is little else.  Else it is made again in 64 bits throughout.
__device__ __forceinline__ bool fp4_sum_holds(double ss) { return ss > 0x1p-100 && ss < 0x1p200; }
__device__ __forceinline__ double fp4_squares16_wide(const float* v) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = fma((double)v[i], (double)v[i], s);
  return s;
}
// The largest magnitude as bits: a NaN is above everything.
template <int N>
__device__ __forceinline__ unsigned fp4_top(const float* v) {
  float top = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[i])));
  return __float_as_uint(top) & 0x7fffffffu;
}
// 1 / (6 g), near enough for a first guess at a block's scale (6 g itself may be past fp32's largest)
__device__ __forceinline__ float fp4_inv6(float g) { return __frcp_rn(g) * (1.0f / 6.0f); }
// Block `at` of a row of K values with scale g
__device__ __forceinline__ void fp4_store_block(uint8_t* row, int K, int at, const float* v, unsigned top, float g, float inv6g) {
  unsigned scale;
  const uint2 codes = fp4_block(v, top, g, inv6g, scale);
  *reinterpret_cast<uint2*>(row + 8 * at) = codes;
  row[K / 2 + at] = (uint8_t)scale;
  if (at == 0) *reinterpret_cast<float*>(row + K / 2 + K / 16) = g;
}

// x / (1 + exp(-x)), a few units of 2^-23 off (a quotient whose denominator is past 2^126 is zero, where the value is below 2^-119)
__device__ __forceinline__ float fp4_silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// ---- instructions ---------------------------------------------------------------------------------------
// kind::mxf4nvf4 instruction descriptor: D = f32, A = B = E2M1 (K-major), scales E4M3 without sign, M 128 x N, K 64
__host__ __device__ constexpr uint32_t fp4_idesc(int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_fp4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "elect.sync _|e, 0xFFFFFFFF;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}

// The scales of 64 values of a row are one 32-bit cell of tensor memory: row r of an operand has its cell in lane r % 32, the same in all four
// quarters, column r / 32.  Four warps, one for each quarter, take the 16 bytes of 256 values of each row out of its box in shared memory (SPAN
// pieces of 16 bytes a row, swizzled so that eight rows lie in different banks) and store the cells of four instructions: word k of
// row 32 j + lane goes to column k * COLUMNS + j.
__device__ __forceinline__ void fp4_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
template <int SPAN>
__device__ __forceinline__ uint4 fp4_raw(const uint8_t* box, int row, int at) {
  const int turn = SPAN == 4 ? row >> 1 & 3 : row >> 2 & 1;
  return *reinterpret_cast<const uint4*>(box + row * (16 * SPAN) + ((at ^ turn) << 4));
}
template <int SPAN, int COLUMNS>
__device__ __forceinline__ void fp4_cells(uint32_t (&c)[4 * COLUMNS], const uint8_t* box, int at, int lane, int groups) {
#pragma unroll
  for (int j = 0; j < COLUMNS; ++j) {
    const uint4 r = j < groups ? fp4_raw<SPAN>(box, 32 * j + lane, at) : make_uint4(0u, 0u, 0u, 0u);
    c[j] = r.x; c[COLUMNS + j] = r.y; c[2 * COLUMNS + j] = r.z; c[3 * COLUMNS + j] = r.w;
  }
}

// Maps of NVFP4 rows [groups][rows][row bytes]: codes in boxes of 256 values (zeros past the row's end), scales in boxes of
// 256 * span.
inline int fp4_maps(CUtensorMap* codes, CUtensorMap* scales, const void* base, int K, long rows, long groups, int box_rows, int span) {
  const cuuint64_t rb = (cuuint64_t)fp4_row_bytes(K);
  cuuint64_t dims[3] = {(cuuint64_t)K / 2, (cuuint64_t)rows, (cuuint64_t)groups};
  cuuint64_t str[2] = {rb, rb * (cuuint64_t)rows};
  cuuint32_t box[3] = {128, (cuuint32_t)box_rows, 1};
  int rc = make_map_any(codes, base, 3, dims, str, box, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  dims[0] = (cuuint64_t)K / 16;
  box[0] = 16 * span;
  return make_map_any(scales, (const uint8_t*)base + K / 2, 3, dims, str, box, CU_TENSOR_MAP_DATA_TYPE_UINT8,
                      span == 4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
}

}  // namespace bl
