// Decode attention of rows that share a prefix.
//
// Row r of group g attends to keys 0 .. n_r - 1 of its sequence; the first P_g of them lie in pages that the whole group shares:
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = q . k_j,   m = max_j s_j
// The keys are cut into fragments; each leaves its maximum, its sum and its unnormalised output, and a second launch joins them.
//
// f16 caches run on the 5th-generation tensor cores.  The query rows of a tile are what reads one stretch of keys: for the shared
// keys of a group the stacked (row, head) pairs of one KV head, 128 a tile and up to two tiles a fragment, so that a key / value
// tile is fetched once for 256 query rows; for a row's own keys its heads alone.  Per 128 keys (two pages) and tile:
//   S = Q K^T     tcgen05.mma kind::f16, M = N = 128, into tensor memory
//   softmax       one thread per query row; the probabilities go back as f16 into the score columns they came from
//   O += P V      P from tensor memory, V as it lies in the cache: rows of keys, the MN-major form of a B operand
// The work of a call is one line of (unit, key tile) pairs, shared keys first; every CTA takes an equal stretch of it, whatever
// the lengths, and goes through the fragments that its stretch cuts.
// Roles: warps 0..3 softmax of the first tile, 4..7 of the second (warp id modulo 4 = TMEM lane quarter), warp 8 the TMA producer
// (two-stage rings for keys and values, 128 KB in flight), warp 9 the MMA issuer and TMEM owner.
// Queries and probabilities are rounded to f16 (11 bits; queries scaled by a power of two a row): less than the output's 8 bits.
// Every wait is bounded (1 s); on expiry the CTA raises the fault word, frees its TMEM and returns.
#include "tc_common.cuh"

namespace bl {

constexpr int kPxPage = 64;
constexpr int kPxMaxRows = 1024;
constexpr float kPxLog2e = 1.4426950408889634f;
constexpr float kPxLazy = 8.0f;                         // the maximum may lag by 2^8 before the output is rescaled

struct PrefixArgs {
  const float* q;                 // [M][n_q][HEAD], scaled
  const uint8_t* k; const uint8_t* v;
  const int* row_pos; const int* row_seq; const int* table;
  int n_slots, max_pages, n_pages, n_q, n_kv, M;
  const int* meta;                // [M][first row, rows, shared positions of the row's group; unit, place in the unit's tiles]
  __nv_bfloat16* out;
  unsigned* fault; int layer;
  // units: up to two tiles of rows of one group that read its shared keys together
  const int* units;               // [n_units][first row, rows, shared positions, first row of the group, rows of the group]
  int n_units, n_cta;
  int* sched;                     // {T, SP, SS}, then SP's running sums [n_units + 1], then SS's [M + 1]
  float4* part_p; float2* ml_p;   // shared keys: [fragment][tile][HEAD / 4][128], [fragment][tile][128]
  float4* part_s; float2* ml_s;   // own keys: [fragment][HEAD / 4][G], [fragment][G]
};
constexpr int kPxMeta = 5, kPxUnit = 5;

template <int HEAD>
__device__ __forceinline__ float px_value(const uint8_t* row, int d) {
  const float s = __half2float(reinterpret_cast<const __half*>(row)[d >> 5]);
  return s * (float)reinterpret_cast<const int8_t*>(row + HEAD / 16)[d];
}

// q8_0 caches.  grid (n_q, M), HEAD threads: a thread per value, a key after the other
template <int HEAD>
__global__ void __launch_bounds__(HEAD) prefix_rows_kernel(const PrefixArgs a) {
  constexpr int ROW = HEAD / 32 * 34;
  __shared__ float s_part[2][HEAD / 32];
  const int h = blockIdx.x, m = blockIdx.y, d = threadIdx.x, kvh = h / (a.n_q / a.n_kv);
  pdl_wait();
  pdl_launch();
  __nv_bfloat16* out = a.out + ((long)m * a.n_q + h) * HEAD + d;
  const int seq = a.row_seq[m];
  if (seq < 0) { *out = __float2bfloat16_rn(0.f); return; }
  const int n = a.row_pos[m] + 1;
    int lead = a.meta[kPxMeta * m];
  while (a.row_seq[lead] < 0) ++lead;              // this row is live, so there is one
  bool bad = n <= 0 || n > a.max_pages * kPxPage || seq >= a.n_slots || a.row_seq[lead] >= a.n_slots;
  if (bad && d == 0) raise_fault(a.fault, a.layer, FS_KEY_COUNT);
  const int* shared_pages = a.table + (long)a.row_seq[lead] * a.max_pages;
  const int* own_pages = a.table + (long)seq * a.max_pages;
  const int shared = a.meta[kPxMeta * m + 2];
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
    float s = warp_sum(q * px_value<HEAD>(a.k + row, d));
    if ((d & 31) == 0) s_part[j & 1][d >> 5] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < HEAD / 32; ++w) s += s_part[j & 1][w];
    const float top = fmaxf(mx, s), corr = __expf(mx - top), p = __expf(s - top);
    l = l * corr + p;
    acc = acc * corr + p * px_value<HEAD>(a.v + row, d);
    mx = top;
  }
  *out = __float2bfloat16_rn(bad ? __int_as_float(0x7fc00000) : acc / l);
}


// Keys of row m: 0 for a dead row and for one that cannot be served.
__device__ __forceinline__ int px_keys(const PrefixArgs& a, int m, bool& bad) {
  const int seq = a.row_seq[m], n = a.row_pos[m] + 1;
  bad = seq >= 0 && (n <= 0 || n > a.max_pages * kPxPage || seq >= a.n_slots);
  return seq < 0 || bad ? 0 : n;
}

// The line of work: T tiles, CTA c takes c T / C .. (c + 1) T / C - 1.  Per KV head the units' tiles (SP), all heads' first, then per
// KV head the rows' own tiles (SS).  A fragment is what a stretch shares with a (KV head, unit) or (KV head, row); their numbers
// (index + CTA) grow by one at least from each to the next, so they name a place in the scratch.
struct PxFrag { bool own; int unit, kvh, t_lo, n_t, id; };

struct PxLine {
  const int* cum_p; const int* cum_s;
  int n_units, M, n_kv, SP, SS, cta;
  int g, end;
  __device__ __forceinline__ static int find(const int* cum, int n, int at) {      // the last i with cum[i] <= at
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (cum[mid] <= at) lo = mid; else hi = mid; }
    return lo;
  }
  __device__ __forceinline__ bool next(PxFrag& f) {
    if (g >= end) return false;
    const int TP = n_kv * SP;
    f.own = g >= TP;
    const int per = f.own ? SS : SP, at = f.own ? g - TP : g, n = f.own ? M : n_units;
    const int* cum = f.own ? cum_s : cum_p;
    f.kvh = at / per;
    const int rem = at - f.kvh * per;
    f.unit = find(cum, n, rem);
    f.t_lo = rem - cum[f.unit];
    f.n_t = min(cum[f.unit + 1] - rem, end - g);
    f.id = f.kvh * n + f.unit + cta;
    g += f.n_t;
    return true;
  }
};

// K-major tiles use umma_desc(); V as B operand in MN-major form: atoms of 64 values x 8 keys (1,024 bytes), 8-key groups one atom
// apart, blocks of 64 values a page's 8 KB apart.
__device__ __forceinline__ uint64_t px_desc_v(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
  d |= (uint64_t)(8192 >> 4) << 16;                     // leading: between blocks of 64 values
  d |= (uint64_t)(1024 >> 4) << 32;                     // stride: between groups of 8 keys
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16, D = f32, A = B = f16; B K-major or MN-major
__host__ __device__ constexpr uint32_t px_idesc(int m, int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ float px_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t px_pack(float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ void px_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
               "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

constexpr int kPxThreads = 320;
constexpr int kPxHalf = 128 * 128;                      // 16 KB: 128 rows of 64 f16 values, one swizzle atom wide
constexpr int px_tile(int head) { return head / 64 * kPxHalf; }
constexpr int px_smem(int head, int n_units, int M) { return 6 * px_tile(head) + 1024 + (n_units + M + 2) * 4; }

template <int HEAD>
__global__ void __launch_bounds__(kPxThreads, 1)
prefix_attn_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const PrefixArgs a) {
  constexpr int NH = HEAD / 64, TILE = px_tile(HEAD), PAGE_BYTES = kPxPage * 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_bad[8];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;                // [2 tiles][NH][128 rows][128 bytes]
  uint8_t* sK = sQ + 2 * TILE;       // [2 stages][NH][128 keys][128 bytes]
  uint8_t* sV = sK + 2 * TILE;       // [2 stages][2 pages][NH][64 keys][128 bytes]
  int* s_cum_p = reinterpret_cast<int*>(sV + 2 * TILE);         // [n_units + 1]
  int* s_cum_s = s_cum_p + a.n_units + 1;                       // [M + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.n_q / a.n_kv, rows_tile = 128 / G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4); mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_done[i], 1);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch();
  // ---- the line of work: tiles of every unit and row, then their running sums
  for (int m = threadIdx.x; m < a.M; m += kPxThreads) {
    bool bad;
    const int n = px_keys(a, m, bad), shared = a.meta[m * kPxMeta + 2];
    if (bad && blockIdx.x == 0) raise_fault(a.fault, a.layer, FS_KEY_COUNT);
    s_cum_s[m + 1] = max(0, n - shared + 127) / 128;
  }
  for (int u = threadIdx.x; u < a.n_units; u += kPxThreads) {
    const int* unit = a.units + u * kPxUnit;
    int live = 0;                                               // a unit without a live row reads nothing
    for (int m = unit[0]; !live && m < unit[0] + unit[1]; ++m) { bool bad; live = px_keys(a, m, bad); }
    s_cum_p[u + 1] = live ? (unit[2] + 127) / 128 : 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp < 2) {
    int* cum = warp ? s_cum_s : s_cum_p;
    const int n = warp ? a.M : a.n_units;
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      int v = i0 + lane < n ? cum[i0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += up; }
      if (i0 + lane < n) cum[i0 + lane + 1] = base + v;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) cum[0] = 0;
  }
  __syncthreads();
  PxLine line;
  line.cum_p = s_cum_p; line.cum_s = s_cum_s; line.n_units = a.n_units; line.M = a.M; line.n_kv = a.n_kv;
  line.SP = s_cum_p[a.n_units]; line.SS = s_cum_s[a.M]; line.cta = blockIdx.x;
  const int T = a.n_kv * (line.SP + line.SS);
  const int n_cta = min(a.n_cta, T);                            // a tile each at least, so that fragments' CTAs follow each other
  line.g = (int)blockIdx.x < n_cta ? (int)((long)blockIdx.x * T / n_cta) : 0;
  line.end = (int)blockIdx.x < n_cta ? (int)((long)(blockIdx.x + 1) * T / n_cta) : 0;
  if (blockIdx.x == 0) {                                        // for the launch that joins the fragments
    if (threadIdx.x == 0) { a.sched[0] = T; a.sched[1] = line.SP; a.sched[2] = line.SS; }
    for (int i = threadIdx.x; i < a.n_units + a.M + 2; i += kPxThreads) a.sched[3 + i] = s_cum_p[i];
  }
  const uint32_t tmem_base = s_tmem_base;
  volatile int* abort_flag = &s_abort;
  const uint32_t tS0 = tmem_base, tO0 = tmem_base + 256;        // scores of tile x at column 128 x, its output at 256 + HEAD x
  // keys of a fragment: from, end (absolute positions), and the tiles of rows
  auto shape = [&](const PxFrag& f, int& key0, int& key_end, int& n_x) {
    if (f.own) {
      bool bad;
      key0 = a.meta[f.unit * kPxMeta + 2] + 128 * f.t_lo;
      key_end = px_keys(a, f.unit, bad);
      n_x = 1;
    } else {
      key0 = 128 * f.t_lo;
      key_end = a.units[f.unit * kPxUnit + 2];
      n_x = a.units[f.unit * kPxUnit + 1] > rows_tile ? 2 : 1;
    }
    key_end = min(key_end, key0 + 128 * f.n_t);
  };
  PxFrag f;

  if (warp == 8) {
    // ---- producer: the warp looks pages up 32 at a time, lane 0 waits and copies
    int tile = 0;
    bool ok = true;
    for (int nf = 0; ok && line.next(f); ++nf) {
      int key0, key_end, n_x;
      shape(f, key0, key_end, n_x);
      int seq = -1;
      if (f.own) {
        seq = a.row_seq[f.unit];
      } else {                                                  // the first row of the group that has a table
        const int r0 = a.units[f.unit * kPxUnit + 3], rows = a.units[f.unit * kPxUnit + 4];
        for (int i = 0; seq < 0 && i < rows; i += 32) {
          const int mine = i + lane < rows ? a.row_seq[r0 + i + lane] : -1;
          const unsigned live = __ballot_sync(0xffffffffu, mine >= 0 && mine < a.n_slots);
          if (live) seq = __shfl_sync(0xffffffffu, mine, __ffs(live) - 1);
        }
      }
      const int* pages = a.table + (long)max(seq, 0) * a.max_pages;
      const int col0 = key0 / kPxPage, n_cols = (key_end - key0 + kPxPage - 1) / kPxPage;
      int chunk = 0;
      bool bad = false;
      for (int c = 0; ok && c < n_cols; c += 2, ++tile) {
        if ((c & 31) == 0) {
          chunk = c + lane < n_cols ? pages[col0 + c + lane] : 0;
          const bool off = chunk < 0 || chunk >= a.n_pages || seq < 0;
          if (off) { chunk = 0; raise_fault(a.fault, a.layer, FS_PAGE); }
          bad = bad || __any_sync(0xffffffffu, off);
        }
        const int p0 = __shfl_sync(0xffffffffu, chunk, c & 31), p1 = __shfl_sync(0xffffffffu, chunk, (c + 1) & 31);
        const int n_p = min(2, n_cols - c);
        const int st = tile & 1;
        const uint32_t par = (uint32_t)((tile >> 1) & 1);
        if (lane == 0) {
          ok = mbar_wait(&k_empty[st], par ^ 1, abort_flag);
          if (ok) {
            // behind this wait the softmax of four fragments ago is over: the flag may be used again
            if (c == 0 || bad) s_bad[nf & 7] = bad;
            mbar_expect_tx(&k_full[st], n_p * NH * PAGE_BYTES);
            for (int p = 0; p < n_p; ++p)
              for (int h = 0; h < NH; ++h)
                tma_load_2d(sK + st * TILE + h * kPxHalf + p * PAGE_BYTES, &tma_k, h * 64, ((p ? p1 : p0) * a.n_kv + f.kvh) * kPxPage, &k_full[st]);
            ok = mbar_wait(&v_empty[st], par ^ 1, abort_flag);
          }
          if (ok) {
            mbar_expect_tx(&v_full[st], n_p * NH * PAGE_BYTES);
            for (int p = 0; p < n_p; ++p)
              for (int h = 0; h < NH; ++h)
                tma_load_2d(sV + st * TILE + (p * NH + h) * PAGE_BYTES, &tma_v, h * 64, ((p ? p1 : p0) * a.n_kv + f.kvh) * kPxPage, &v_full[st]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
    }
    if (*abort_flag) {
      // copies of ours may still be landing: give them a bounded moment before the block's memory goes away
      const unsigned long long t0 = globaltimer();
      while (globaltimer() - t0 < 2000000ull) { }
    }
  } else if (warp == 9) {
    // ---- issuer
    constexpr uint32_t idesc_s = px_idesc(128, 128, false), idesc_o = px_idesc(128, HEAD, true);
    auto qk = [&](int x, int st) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint64_t dq = umma_desc(smem_u32(sQ + x * TILE + h * kPxHalf)), dk = umma_desc(smem_u32(sK + st * TILE + h * kPxHalf));
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16(tS0 + x * 128, dq + (uint64_t)(k * 2), dk + (uint64_t)(k * 2), idesc_s, h + k > 0 ? 1u : 0u);
      }
      umma_commit(&s_full[x]);
    };
    int tile = 0, n_s[2] = {0, 0}, n_f[2] = {0, 0};             // tiles through the rings; tiles and fragments of each tile of rows
    bool ok = true;
    while (ok && line.next(f)) {
      int key0, key_end, n_x;
      shape(f, key0, key_end, n_x);
      for (int x = 0; ok && x < n_x; ++x) ok = mbar_wait_warp(&q_full[x], (uint32_t)(n_f[x] & 1), abort_flag);
      ok = ok && mbar_wait_warp(&k_full[tile & 1], (uint32_t)((tile >> 1) & 1), abort_flag);
      if (!ok) break;
      tc_fence_after();
      for (int x = 0; x < n_x; ++x) qk(x, tile & 1);
      umma_commit(&k_empty[tile & 1]);
      for (int t = 0; ok && t < f.n_t; ++t, ++tile) {
        const int st = tile & 1, nx = st ^ 1;
        const bool more = t + 1 < f.n_t, two = key_end - (key0 + 128 * t) > kPxPage;
        ok = mbar_wait_warp(&v_full[st], (uint32_t)((tile >> 1) & 1), abort_flag);
        for (int x = 0; ok && x < n_x; ++x) {
          ok = mbar_wait_warp(&p_full[x], (uint32_t)(n_s[x]++ & 1), abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tP = tS0 + x * 128, tO = tO0 + x * HEAD;
          const uint64_t dv = px_desc_v(smem_u32(sV + st * TILE)), dw = px_desc_v(smem_u32(sV + st * TILE + NH * PAGE_BYTES));
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16_ta(tO, tP + k * 8, dv + (uint64_t)(k * 128), idesc_o, t + k > 0 ? 1u : 0u);
          if (two) {
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16_ta(tO, tP + 32 + k * 8, dw + (uint64_t)(k * 128), idesc_o, 1u);
          }
          if (x == n_x - 1) umma_commit(&v_empty[st]);
          if (more) {
            if (x == 0) {
              ok = mbar_wait_warp(&k_full[nx], (uint32_t)(((tile + 1) >> 1) & 1), abort_flag);
              if (!ok) break;
              tc_fence_after();
            }
            qk(x, nx);
            if (x == n_x - 1) umma_commit(&k_empty[nx]);
          } else {
            umma_commit(&o_done[x]);
          }
        }
      }
      for (int x = 0; x < n_x; ++x) ++n_f[x];
    }
  } else {
    // ---- softmax: a thread per query row ------------------------------------------------------------------
    const int x = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;                          // row of the tile
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tS0 + x * 128 + lane_base, tO = tO0 + x * HEAD + lane_base;
    int tile = 0, n_s = 0, n_f = 0;
    bool ok = true;
    for (int nf = 0; ok && line.next(f); ++nf) {
      int key0, key_end, n_x;
      shape(f, key0, key_end, n_x);
      if (x >= n_x) { tile += f.n_t; continue; }
      // rows of this tile, and how far this thread's row reaches into the fragment
      const int row0 = f.own ? f.unit : a.units[f.unit * kPxUnit] + x * rows_tile;
      const int n_rows = f.own ? 1 : min(rows_tile, a.units[f.unit * kPxUnit + 1] - x * rows_tile);
      const int live = n_rows * G;                              // query rows of this tile
      int limit = 0;
      if (r < live) {
        bool bad;
        limit = min(px_keys(a, row0 + r / G, bad), key_end);
      }
      float to_log2 = 0.f;
      if (quarter * 32 < live) {
        // queries to f16: four lanes a row, scaled by a power of two to a largest element in [512, 1024)
#pragma unroll 1
        for (int p = 0; p < 4; ++p) {
          const int i = quarter * 32 + p * 8 + (lane >> 2);
          float4 v[HEAD / 16];
          float top = 0.f;
          const float* src = a.q + ((long)(row0 + i / G) * a.n_q + f.kvh * G + i % G) * HEAD + (lane & 3) * 4;
#pragma unroll
          for (int c = 0; c < HEAD / 16; ++c) {
            v[c] = i < live ? __ldg(reinterpret_cast<const float4*>(src + c * 16)) : make_float4(0.f, 0.f, 0.f, 0.f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v[c].x), fabsf(v[c].y)), fmaxf(fabsf(v[c].z), fabsf(v[c].w))));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = (int)(__float_as_uint(top) >> 23);      // top >= 0
          const int se = e == 0 ? 127 : min(254, 263 - e);
          const float scale = __uint_as_float((unsigned)se << 23);
          const float back = kPxLog2e / scale;
          const float mine = __shfl_sync(0xffffffffu, back, (lane & 7) * 4);
          if ((lane >> 3) == p) to_log2 = mine;
          const int row = i, sw = row & 7;
#pragma unroll
          for (int c = 0; c < HEAD / 16; ++c) {
            const int col = (lane & 3) * 4 + c * 16;            // value: 8 bytes of 16-byte chunk (col % 64) / 8
            uint8_t* dst = sQ + x * TILE + (col >> 6) * kPxHalf + row * 128 + ((((col & 63) >> 3) ^ sw) << 4) + ((col & 4) << 1);
            *reinterpret_cast<uint2*>(dst) = make_uint2(px_pack(v[c].x * scale, v[c].y * scale), px_pack(v[c].z * scale, v[c].w * scale));
          }
        }
        fence_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[x]);
      float m = -INFINITY, l = 0.f;
      for (int t = 0; t < f.n_t; ++t, ++tile, ++n_s) {
        ok = mbar_wait_warp(&s_full[x], (uint32_t)(n_s & 1), abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int k0 = key0 + 128 * t, part = (key_end - k0) % kPxPage;
        if (quarter * 32 < live) {
          uint32_t v[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(tS + 32 * c, v[c]);
          tmem_ld_wait();
          if (__any_sync(0xffffffffu, k0 + 128 > limit)) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (k0 + 32 * c + i >= limit) v[c][i] = 0xff800000u;      // -inf
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 2)
#pragma unroll
            for (int c = 0; c < 4; ++c) mx4[c] = fmaxf(fmaxf(mx4[c], __uint_as_float(v[c][i])), __uint_as_float(v[c][i + 1]));
          float m_new = fmaxf(m, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
          if (m != -INFINITY && (m_new - m) * to_log2 <= kPxLazy) m_new = m;
          const float mb = (m_new == -INFINITY) ? 0.f : m_new * to_log2;      // a row with no key yet keeps zeros
          const float corr = (m == -INFINITY) ? 0.f : px_ex2(m * to_log2 - mb);
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              uint32_t e0, e1;
              asm("{\n\t.reg .b64 rs, rk, rm, rr;\n\t"
                  "mov.b64 rs, {%2, %3};\n\tmov.b64 rk, {%4, %4};\n\tmov.b64 rm, {%5, %5};\n\t"
                  "fma.rn.f32x2 rr, rs, rk, rm;\n\tmov.b64 {%0, %1}, rr;\n\t}"
                  : "=r"(e0), "=r"(e1) : "r"(v[c][i]), "r"(v[c][i + 1]), "f"(to_log2), "f"(-mb));
              const float p0 = px_ex2(__uint_as_float(e0)), p1 = px_ex2(__uint_as_float(e1));
              sum[i & 2] += p0; sum[(i & 2) + 1] += p1;
              pk[i >> 1] = px_pack(p0, p1);
            }
            px_st16(tS + 16 * c, pk);
          }
          if (t > 0 && __any_sync(0xffffffffu, corr != 1.0f)) {   // the product of the last tile is complete: its commit lies in front of these scores'
#pragma unroll 1
            for (int c = 0; c < HEAD / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st32(tO + c * 32, o);
            }
          }
          l = l * corr + ((sum[0] + sum[2]) + (sum[1] + sum[3]));
          m = m_new;
          tmem_st_wait();
        }
        if (key_end - k0 < 128 && part) {
          // the last page ends inside the tile: what lies behind the keys may be anything, and zero times that must be zero
          const int st = tile & 1;
          ok = mbar_wait_warp(&v_full[st], (uint32_t)((tile >> 1) & 1), abort_flag);
          if (!ok) break;
          uint8_t* page = sV + st * TILE + (key_end - k0) / kPxPage * NH * PAGE_BYTES;
#pragma unroll
          for (int h = 0; h < NH; ++h)
            for (int i = part * 8 + r; i < kPxPage * 8; i += 128) *reinterpret_cast<uint4*>(page + h * PAGE_BYTES + i * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[x]);
      }
      ok = ok && mbar_wait_warp(&o_done[x], (uint32_t)(n_f++ & 1), abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (quarter * 32 < live) {
        const int pitch = f.own ? G : 128;
        float4* part = f.own ? a.part_s + (long)f.id * (HEAD / 4) * G : a.part_p + ((long)f.id * 2 + x) * (HEAD / 4) * 128;
        float2* ml = f.own ? a.ml_s + (long)f.id * G : a.ml_p + ((long)f.id * 2 + x) * 128;
#pragma unroll 1
        for (int c = 0; c < HEAD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_ld_wait();
          if (r < live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              __stcg(part + (c * 8 + i) * pitch + r, make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                                 __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])));
          }
        }
        if (r < live) __stcg(ml + r, make_float2(m == -INFINITY ? m : m * to_log2, *(volatile int*)&s_bad[nf & 7] ? __int_as_float(0x7fc00000) : l));
        tc_fence_before();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
  if (threadIdx.x == 0 && s_abort) raise_fault(a.fault, a.layer, FS_WAIT_TIMEOUT);
}

// Joins the fragments of a row's heads: grid (n_kv, M), a thread for four values of a head (heads next to each other).
template <int HEAD>
__global__ void __launch_bounds__(256) prefix_join_kernel(const PrefixArgs a) {
  const int kvh = blockIdx.x, m = blockIdx.y, G = a.n_q / a.n_kv;
  pdl_wait();
  pdl_launch();
  bool bad;
  const int n = px_keys(a, m, bad);
  const int* meta = a.meta + m * kPxMeta;
  const int T = a.sched[0], SP = a.sched[1], SS = a.sched[2], unit = meta[3];
  // fragments of the unit's shared keys and of the row's own: consecutive CTAs each
  const int n_cta = min(a.n_cta, T);
  auto cta_of = [&](int g) { return (int)(((long)(g + 1) * n_cta - 1) / T); };
  int p0 = 0, np = 0, s0 = 0, ns = 0;
  if (n > 0 && unit >= 0) {
    const int lo = kvh * SP + a.sched[3 + unit], hi = kvh * SP + a.sched[3 + unit + 1];
    p0 = cta_of(lo); np = cta_of(hi - 1) - p0 + 1;
    p0 += kvh * a.n_units + unit;
  }
  const int* cum_s = a.sched + 3 + a.n_units + 1;
  if (n > 0 && cum_s[m + 1] > cum_s[m]) {
    const int base = a.n_kv * SP + kvh * SS;
    s0 = cta_of(base + cum_s[m]); ns = cta_of(base + cum_s[m + 1] - 1) - s0 + 1;
    s0 += kvh * a.M + m;
  }
  const int tile = meta[4] / 128, lane0 = meta[4] % 128;
  for (int i = threadIdx.x; i < G * (HEAD / 4); i += blockDim.x) {
    const int h = i % G, c = i / G;
    const float2* ml_p = a.ml_p + ((long)p0 * 2 + tile) * 128 + lane0 + h;      // 256 a fragment
    const float2* ml_s = a.ml_s + (long)s0 * G + h;                             // G a fragment
    const float4* part_p = a.part_p + (((long)p0 * 2 + tile) * (HEAD / 4) + c) * 128 + lane0 + h;
    const float4* part_s = a.part_s + ((long)s0 * (HEAD / 4) + c) * G + h;
    float top = -INFINITY;
#pragma unroll 4
    for (int f = 0; f < np; ++f) top = fmaxf(top, __ldcg(ml_p + (long)f * 256).x);
#pragma unroll 4
    for (int f = 0; f < ns; ++f) top = fmaxf(top, __ldcg(ml_s + (long)f * G).x);
    float den = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 v) {                                       // ascending order, fixed
      const float w = ml.x == -INFINITY ? 0.f : px_ex2(ml.x - top);
      den = fmaf(w, ml.y, den);
      if (w != 0.f) { o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w); }
    };
#pragma unroll 4
    for (int f = 0; f < np; ++f) add(__ldcg(ml_p + (long)f * 256), __ldcg(part_p + (long)f * 2 * (HEAD / 4) * 128));
#pragma unroll 4
    for (int f = 0; f < ns; ++f) add(__ldcg(ml_s + (long)f * G), __ldcg(part_s + (long)f * (HEAD / 4) * G));
    const float inv = bad ? __int_as_float(0x7fc00000) : n > 0 ? 1.f / den : 0.f;
    const __nv_bfloat162 b0 = __floats2bfloat162_rn(o.x * inv, o.y * inv), b1 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(a.out + ((long)m * a.n_q + kvh * G + h) * HEAD + c * 4) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
  }
}

}  // namespace bl

using namespace bl;

template <int HEAD>
static int prefix_go(const PrefixArgs& a, cudaStream_t st) {
  CUtensorMap mk, mv;
  const cuuint64_t dims[2] = {(cuuint64_t)HEAD, (cuuint64_t)a.n_pages * a.n_kv * kPxPage};
  const cuuint64_t strides[1] = {(cuuint64_t)HEAD * 2};
  const cuuint32_t box[2] = {64, kPxPage};
  int rc = make_map_any(&mk, a.k, 2, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = make_map_any(&mv, a.v, 2, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) {
    const cudaError_t e = cudaFuncSetAttribute(prefix_attn_kernel<HEAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, px_smem(HEAD, kPxMaxRows, kPxMaxRows));
    if (e != cudaSuccess) return (int)e;
    limit.mark();
  }
  const cudaError_t e = launch(prefix_attn_kernel<HEAD>, dim3(a.n_cta), dim3(kPxThreads), (size_t)px_smem(HEAD, a.n_units, a.M), st, mk, mv, a);
  if (e != cudaSuccess) return (int)e;
  return (int)launch(prefix_join_kernel<HEAD>, dim3(a.n_kv, a.M), dim3(256), 0, st, a);
}

extern "C" {

// Bytes of scratch that bl_prefix_attention takes for these sizes (n_units units, n_cta processors).
long bl_prefix_work_bytes(int head, int n_q, int n_kv, int M, int n_units, int n_cta) {
  const long G = n_q / n_kv, fp = n_units ? (long)n_kv * n_units + n_cta : 0, fs = (long)n_kv * M + n_cta;
  return ((3 + n_units + M + 2) * 4L + 255) / 256 * 256 + fp * 256 * (head * 4 + 8) + fs * G * (head * 4 + 8);
}

int bl_prefix_attention(const float* q, const void* k_cache, const void* v_cache, const int* row_pos, const int* row_seq,
                        const int* block_table, int n_slots, int max_pages, int n_pages, int head, int n_q, int n_kv, int M,
                        const int* meta, int n_units, void* work, int kv_q8, void* out, int n_cta, unsigned* fault, int layer,
                        cudaStream_t st) {
  BL_REQUIRE(head == 128 || head == 64, BL_ERR_SHAPE);
  BL_REQUIRE(n_kv >= 1 && n_q >= 1 && n_q % n_kv == 0 && n_q / n_kv <= 16, BL_ERR_SHAPE);
  BL_REQUIRE(M >= 1 && M <= kPxMaxRows && n_units >= 0 && n_units <= M && n_cta >= 1 && n_slots >= 1 && max_pages >= 1 && n_pages >= 1, BL_ERR_SHAPE);
  BL_REQUIRE((long)n_pages * n_kv * kPxPage <= 0x7fffffffL && (long)(max_pages + 2) * M * n_kv <= 0x7fffffffL, BL_ERR_LIMIT);
  BL_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)work) & 15) == 0, BL_ERR_ALIGN);
  PrefixArgs a{q, (const uint8_t*)k_cache, (const uint8_t*)v_cache, row_pos, row_seq, block_table, n_slots, max_pages, n_pages, n_q, n_kv, M,
               meta, (__nv_bfloat16*)out, fault, layer, meta + (long)M * kPxMeta, n_units, n_cta};
  const long G = n_q / n_kv, fp = n_units ? (long)n_kv * n_units + n_cta : 0, fs = (long)n_kv * M + n_cta;
  uint8_t* w = (uint8_t*)work;
  a.sched = (int*)w; w += ((3 + n_units + M + 2) * 4L + 255) / 256 * 256;
  a.part_p = (float4*)w; w += fp * 256 * head * 4;
  a.ml_p = (float2*)w; w += fp * 256 * 8;
  a.part_s = (float4*)w; w += fs * G * head * 4;
  a.ml_s = (float2*)w;
  const dim3 grid(n_q, M);
  if (kv_q8) {
    if (head == 128) return (int)launch(prefix_rows_kernel<128>, grid, dim3(128), 0, st, a);
    return (int)launch(prefix_rows_kernel<64>, grid, dim3(64), 0, st, a);
  }
  return head == 128 ? prefix_go<128>(a, st) : prefix_go<64>(a, st);
}

}  // extern "C"
