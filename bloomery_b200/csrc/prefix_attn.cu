// Decode attention of rows that share a prefix.
//
// Row r of group g attends to keys 0 .. n_r - 1 of its sequence; the first P_g of them lie in pages that the whole group shares:
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = q . k_j,   m = max_j s_j
// A running maximum and sum make it one pass over the keys.
#include "common.cuh"

namespace bl {

constexpr int kPxPage = 64;

struct PrefixArgs {
  const float* q;                 // [M][n_q][HEAD], scaled
  const uint8_t* k; const uint8_t* v;
  const int* row_pos; const int* row_seq; const int* table;
  int n_slots, max_pages, n_pages, n_q, n_kv, M;
  const int* meta;                // [M][first row, rows, shared positions] of the row's group
  __nv_bfloat16* out;
  unsigned* fault; int layer;
};

template <int HEAD, bool Q8>
__device__ __forceinline__ float px_value(const uint8_t* row, int d) {
  if constexpr (Q8) {
    const float s = __half2float(reinterpret_cast<const __half*>(row)[d >> 5]);
    return s * (float)reinterpret_cast<const int8_t*>(row + HEAD / 16)[d];
  } else {
    return __half2float(reinterpret_cast<const __half*>(row)[d]);
  }
}

// grid (n_q, M), HEAD threads: a thread per value, a key after the other
template <int HEAD, bool Q8>
__global__ void __launch_bounds__(HEAD) prefix_rows_kernel(const PrefixArgs a) {
  constexpr int ROW = Q8 ? HEAD / 32 * 34 : HEAD * 2;
  __shared__ float s_part[2][HEAD / 32];
  const int h = blockIdx.x, m = blockIdx.y, d = threadIdx.x, kvh = h / (a.n_q / a.n_kv);
  pdl_wait();
  pdl_launch();
  __nv_bfloat16* out = a.out + ((long)m * a.n_q + h) * HEAD + d;
  const int seq = a.row_seq[m];
  if (seq < 0) { *out = __float2bfloat16_rn(0.f); return; }
  const int n = a.row_pos[m] + 1;
    int lead = a.meta[3 * m];
  while (a.row_seq[lead] < 0) ++lead;              // this row is live, so there is one
  bool bad = n <= 0 || n > a.max_pages * kPxPage || seq >= a.n_slots || a.row_seq[lead] >= a.n_slots;
  if (bad && d == 0) raise_fault(a.fault, a.layer, FS_KEY_COUNT);
  const int* shared_pages = a.table + (long)a.row_seq[lead] * a.max_pages;
  const int* own_pages = a.table + (long)seq * a.max_pages;
  const int shared = a.meta[3 * m + 2];
  const float q = a.q[((long)m * a.n_q + h) * HEAD + d];
  float mx = -INFINITY, l = 0.f, acc = 0.f;
  for (int j = 0; !bad && j < n; ++j) {
    const int page = (j < shared ? shared_pages : own_pages)[j / kPxPage];
    if (page < 0 || page >= a.n_pages) {
      bad = true;
      if (d == 0) raise_fault(a.fault, a.layer, FS_PAGE);
      break;
    }
    const long row = (((long)page * a.n_kv + kvh) * kPxPage + j % kPxPage) * ROW;
    float s = warp_sum(q * px_value<HEAD, Q8>(a.k + row, d));
    if ((d & 31) == 0) s_part[j & 1][d >> 5] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < HEAD / 32; ++w) s += s_part[j & 1][w];
    const float top = fmaxf(mx, s), corr = __expf(mx - top), p = __expf(s - top);
    l = l * corr + p;
    acc = acc * corr + p * px_value<HEAD, Q8>(a.v + row, d);
    mx = top;
  }
  *out = __float2bfloat16_rn(bad ? __int_as_float(0x7fc00000) : acc / l);
}

}  // namespace bl

using namespace bl;

extern "C" int bl_prefix_attention(const float* q, const void* k_cache, const void* v_cache, const int* row_pos, const int* row_seq,
                                   const int* block_table, int n_slots, int max_pages, int n_pages, int head, int n_q, int n_kv, int M,
                                   const int* meta, int n_units, void* work, int kv_q8, void* out, int sms, unsigned* fault, int layer,
                                   cudaStream_t st) {
  BL_REQUIRE(head == 128 || head == 64, BL_ERR_SHAPE);
  BL_REQUIRE(n_kv >= 1 && n_q >= 1 && n_q % n_kv == 0 && n_q / n_kv <= 16, BL_ERR_SHAPE);
  BL_REQUIRE(M >= 1 && M <= 1024 && n_slots >= 1 && max_pages >= 1 && n_pages >= 1, BL_ERR_SHAPE);
  BL_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) == 0, BL_ERR_ALIGN);
  PrefixArgs a{q, (const uint8_t*)k_cache, (const uint8_t*)v_cache, row_pos, row_seq, block_table, n_slots, max_pages, n_pages, n_q, n_kv, M,
               meta, (__nv_bfloat16*)out, fault, layer};
  const dim3 grid(n_q, M);
  if (head == 128) {
    if (kv_q8) return (int)launch(prefix_rows_kernel<128, true>, grid, dim3(128), 0, st, a);
    return (int)launch(prefix_rows_kernel<128, false>, grid, dim3(128), 0, st, a);
  }
  if (kv_q8) return (int)launch(prefix_rows_kernel<64, true>, grid, dim3(64), 0, st, a);
  return (int)launch(prefix_rows_kernel<64, false>, grid, dim3(64), 0, st, a);
}
