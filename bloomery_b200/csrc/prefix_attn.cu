// Decode attention of rows that share a prefix.
//
// Row r of group g attends to keys 0 .. n_r - 1 of its sequence; the first P_g of them lie in pages that the whole group shares:
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = q . k_j,   m = max_j s_j
// The keys are cut into fragments; each leaves its maximum, its sum and its unnormalised output, and a second launch joins them.
//
// Both kinds of cache run on the 5th-generation tensor cores.  A unit is up to 256 stacked (row, head) pairs of one KV head, rows
// of one group, in two tiles of 128: it reads the pages that its rows share and then the pages of each of its rows, all of them
// against all of its query rows; for a page of one row the others' scores are masked.  (A page of one row costs a whole job, of
// whose 128 rows at most 16 count.  Where own pages are most of the line they bound the call: 21 rows with up to 1,100 own positions
// behind 4,096 have 190 own pages a KV head beside 64 shared ones.  A fragment for each row's own keys cost more in the form
// that was tried, as much as eight pages on top for a short one: 64 rows with 1 to 256 keys of their own behind 32,768, 102 us.)
// Per page of 64 keys and tile of rows, a job:
//   S = Q K^T     tcgen05.mma kind::f16, M = 128, N = 64, into one of the tile's two score buffers in tensor memory
//   softmax       one thread per query row; the probabilities go back as f16 into the score columns they came from
//   O += P V      P from tensor memory, V as it lies in the cache: rows of keys, the MN-major form of a B operand
// Behind a job's second product the scores of the job after the next are multiplied, so that the softmax of a tile has scores to
// go on with while the products of the last ones run.
// The work of a call is one line of pages, unit after unit; every CTA takes an equal stretch of it, whatever the lengths, and
// goes through the fragments that its stretch cuts.
// Roles: warps 0..3 softmax of the first tile of rows, 4..7 of the second (warp id modulo 4 = TMEM lane quarter), warp 8 the TMA
// producer (four pages of keys and of values in flight), warps 9 and 10 the MMA issuers of either tile; 9 owns the TMEM.  q8_0 rows
// are fetched as they are and expanded to f16 by four warps more.
// Three roundings to the 11 bits of f16: queries (scaled by a power of two a row), probabilities (scaled by 2^7, see kPxShift) and the
// expanded keys and values of q8_0 caches.  A probability's or a value's own rounding is less than the output's 8 bits.  A query's,
// or a q8_0 key's, moves a score by some 2^-12 of the root of the sum of its terms' squares, and the probability by that much of
// itself: the output's 0.2 % where that root is 8 nats, 1 % at 40, several percent in the hundreds; the ordinary batched pass keeps
// 22 bits of queries and probabilities (flash_mma.cuh).  At scores of 1.4 standard deviations the error against 64 bits is 0.2 to 1.9 %
// above that of sums in 32 bits, both 1.65e-3 to 1.69e-3, the output's rounding.
// A value that is not finite would reach the masked rows of its tile as 0 x inf; rows whose output is not finite are summed again
// key by key, over their own keys alone.
// Device time of both launches in a graph, inputs not in L2 (32 heads over 4 of 128 values): 4 rows behind 512 shared positions 10.3 us,
// 8 behind 2,048 13.6, 21 behind 4,096 23.2, 24 rows of q8_0 behind three prefixes 30.4, 64 behind 32,768 62.1.  A short call is a
// chain of latencies: launch, lengths and schedule, queries, a page, its softmax, the join.  A long one is bound by the softmax of a
// job, one row a thread, and by the turns of the two tiles: about 1,200 clocks a job, the tensor pipe 33 % busy; its joining launch
// reads 19 MB of fragments in 8 us.
// Every wait is bounded (1 s); on expiry the CTA raises the fault word, frees its TMEM and returns.
#include <type_traits>

#include "tc_common.cuh"

namespace bl {

constexpr int kPxPage = 64;
constexpr int kPxMaxRows = 512;
constexpr float kPxLog2e = 1.4426950408889634f;
constexpr float kPxLazy = 8.0f;                         // the maximum may lag by 2^8 before the output is rescaled
// Probabilities are 2^7 times e^(s - m), at most 2^15: f16 keeps its 11 bits of all down to 2^-21 of the maximum, and something of
// them down to 2^-32 (a key that draws most of a head's attention may lie 10 to 15 nats above the others, whose sum is the output
// where its value is small).  The factor is in the sums and the outputs alike.  With 2^4 and 2^11 in place of 2^8 and 2^7 the
// output is rescaled more often: 64 rows behind 32,768 positions 64.4 us, 61.2 so; 21 behind 4,096 22.7 and 21.0.
constexpr float kPxShift = 7.0f;

struct PrefixArgs {
  const float* q;                 // [M][n_q][HEAD], scaled
  const uint8_t* k; const uint8_t* v;
  const int* row_pos; const int* row_seq; const int* table;
  int n_slots, max_pages, n_pages, n_q, n_kv, M;
  const int* meta;                // [M][first row, rows, shared positions of the row's group; unit, place in the unit's tiles]
  __nv_bfloat16* out;
  unsigned* fault; int layer;
  const int* units;               // [n_units][first row, rows, shared positions, first row of the group, rows of the group]
  int n_units, n_cta;
  int4* sched;                    // [M][pages of a KV head, of the units before, shared, keys; first own page, own pages, unit, place]: of this
                                  // call, for the joining launch
  // [fragment][tiles of rows][outputs [HEAD / 4][pitch], then maxima and sums [pitch] of 8 bytes]: `slot` float4 a tile.  What lies
  // close together needs few address translations.
  float4* part;
  int slot, slot_tiles, pitch;
  long part_bytes;
  int cols, items, sets, inv_items, inv_G;              // of the joining launch: see there
};
constexpr int kPxMeta = 5, kPxUnit = 5;

// Shared pages of a unit or a row, out of their positions: of a prefix longer than a table row, as far as the row goes.  (A plan's
// lengths are written on the card behind the call that a graph replays; a row has no keys behind its table row.)
__device__ __forceinline__ int px_shared(const PrefixArgs& a, int positions) { return min(positions / kPxPage, a.max_pages); }

// Keys of row m: 0 for a dead row and for one that cannot be served.
__device__ __forceinline__ int px_keys(const PrefixArgs& a, int m, bool& bad) {
  const int seq = a.row_seq[m], n = a.row_pos[m] + 1;
  bad = seq >= 0 && (n <= 0 || n > a.max_pages * kPxPage || seq >= a.n_slots);
  return seq < 0 || bad ? 0 : n;
}

// One head of row m, key by key: a warp, HEAD / 32 values a lane.
template <int HEAD, bool Q8>
__device__ __forceinline__ void px_row(const PrefixArgs& a, int m, int h, int n, float (&o)[HEAD / 32]) {
  constexpr int N = HEAD / 32, ROW = Q8 ? HEAD / 32 * 34 : HEAD * 2;
  const int lane = threadIdx.x & 31, kvh = h / (a.n_q / a.n_kv), seq = a.row_seq[m], shared = a.meta[m * kPxMeta + 2];
  int lead = a.meta[m * kPxMeta];
  while (a.row_seq[lead] < 0 || a.row_seq[lead] >= a.n_slots) ++lead;           // this row has a table, so there is one
  float q[N], mx = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) { q[i] = a.q[((long)m * a.n_q + h) * HEAD + lane * N + i]; o[i] = 0.f; }
  auto value = [&](const uint8_t* row, int d) {
    if constexpr (Q8) return __half2float(reinterpret_cast<const __half*>(row)[d >> 5]) * (float)reinterpret_cast<const int8_t*>(row + HEAD / 16)[d];
    else return __half2float(reinterpret_cast<const __half*>(row)[d]);
  };
  for (int j = 0; j < n; ++j) {
    const int page = a.table[(long)(j < shared ? a.row_seq[lead] : seq) * a.max_pages + j / kPxPage];
    if (page < 0 || page >= a.n_pages) {
      raise_fault(a.fault, a.layer, FS_PAGE);
      l = __int_as_float(0x7fc00000);
      break;
    }
    const long row = (((long)page * a.n_kv + kvh) * kPxPage + j % kPxPage) * ROW;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], value(a.k + row, lane * N + i), s);
    s = warp_sum(s);
    const float top = fmaxf(mx, s);
    if (s == -INFINITY && top == -INFINITY) continue;
    const float corr = __expf(mx - top), p = __expf(s - top);
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * corr + p * value(a.v + row, lane * N + i);
    mx = top;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] /= l;
}

// ---- the line of work ---------------------------------------------------------------------------------------
// Per KV head the pages of all units (S), CTA c of n takes pages c T / n .. (c + 1) T / n - 1 of the T = n_kv S.  A fragment is what
// a stretch shares with a (KV head, unit); fragments' numbers (index + CTA) grow by one from each to the next within a unit and
// by one at least between units, so they name places in the scratch.
// CTAs that a line of T pages is cut for: a page each at least, so that a unit's CTAs follow each other
__host__ __device__ __forceinline__ unsigned px_ctas(const PrefixArgs& a, unsigned T) { return T < (unsigned)a.n_cta ? T : (unsigned)a.n_cta; }

struct PxFrag {
  int unit, kvh, lo, end, id;     // pages lo .. end - 1 of the unit
  int row0, rows, shared;         // rows of the unit; its shared pages
  int row;                        // whose own pages it starts in
  int pad[3];
};

struct PxLine {
  int* keys;                      // [M] keys of a row
  int* pages;                     // [M + 1] running sum of the rows' own pages
  int* cum;                       // [n_units + 1] running sum of the units' pages
  int* seq;                       // [M]
  int* units;                     // [n_units][kPxUnit], shared pages in place of positions
  int n_units, S, g, end, cta;

  __device__ __forceinline__ static int find(const int* cum, int n, int at) {      // the last i with cum[i] <= at
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (cum[mid] <= at) lo = mid; else hi = mid; }
    return lo;
  }
  __device__ __forceinline__ static void running(int* cum, int n) {                // one warp: cum[i + 1] -> sum of cum[1 .. i + 1]
    const int lane = threadIdx.x & 31;
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
  __host__ __device__ static constexpr int words(int M, int n_units) { return 3 * M + 1 + n_units + 1 + n_units * kPxUnit; }
  // Whole block; `mem` holds words(M, n_units).  The first fragment is worked out once for all warps: a look-up costs each of them
  // some hundred instructions that are met for the first time, at a dozen clocks each.
  __device__ __forceinline__ void build(const PrefixArgs& a, int* mem, int4* s_first) {
    keys = mem; pages = keys + a.M; cum = pages + a.M + 1; seq = cum + a.n_units + 1; units = seq + a.M;
    n_units = a.n_units;
    cta = blockIdx.x;
    for (int i = threadIdx.x; i < n_units * kPxUnit; i += blockDim.x) units[i] = i % kPxUnit == 2 ? px_shared(a, a.units[i]) : a.units[i];
    // One warp has up to 32 rows in its registers (4 rows behind 512 positions 10.3 us a call, 10.9 by way of shared memory; 24 q8_0
    // rows 30.4 and 30.9).
    const bool small = a.M <= 32;
    int unit[3] = {0, 0, 0}, own = 0, n_keys = 0;
    if (small && (int)threadIdx.x < n_units) {
#pragma unroll
      for (int i = 0; i < 3; ++i) unit[i] = a.units[threadIdx.x * kPxUnit + i];
      unit[2] = px_shared(a, unit[2]);
    }
    for (int m = threadIdx.x; m < a.M; m += blockDim.x) {
      const int shared = px_shared(a, a.meta[m * kPxMeta + 2]), sq = a.row_seq[m];
      bool bad;
      const int n = px_keys(a, m, bad);
      if (bad && blockIdx.x == 0) raise_fault(a.fault, a.layer, FS_KEY_COUNT);
      keys[m] = n;
      seq[m] = sq;
      n_keys = n;
      own = max(0, n - shared * kPxPage + kPxPage - 1) / kPxPage;
      pages[m + 1] = own;
    }
    if (small) {
      if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        auto scan = [&](int v) {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v += up; }
          return v;
        };
        const int sum = scan(own);
        const unsigned live = __ballot_sync(0xffffffffu, n_keys > 0);
        const int upto = __shfl_sync(0xffffffffu, sum, (unit[0] + unit[1] - 1) & 31), prev = __shfl_sync(0xffffffffu, sum, (unit[0] - 1) & 31);
        const int before = unit[0] ? prev : 0;
        const unsigned mine = unit[1] >= 32 ? 0xffffffffu : (1u << unit[1]) - 1;
        const int total = scan((live >> unit[0] & mine) != 0 ? unit[2] + upto - before : 0);
        S = __shfl_sync(0xffffffffu, total, 31);
        const unsigned T = (unsigned)(a.n_kv * S), n = px_ctas(a, T);
        g = (unsigned)cta < n ? (int)((unsigned)cta * T / n) : 0;
        end = (unsigned)cta < n ? (int)((unsigned)(cta + 1) * T / n) : 0;
        PxFrag f = {};
        const bool some = g < end;
        if (some) {
          f.kvh = (int)((unsigned)g / (unsigned)S);
          const int rem = g - f.kvh * S;
          f.unit = __popc(__ballot_sync(0xffffffffu, total <= rem));            // units that end before
          const int last = __shfl_sync(0xffffffffu, total, f.unit);
          f.lo = rem - (f.unit ? __shfl_sync(0xffffffffu, total, f.unit - 1) : 0);
          f.end = f.lo + min(last - rem, end - g);
          f.id = f.kvh * n_units + f.unit + cta;
          f.row0 = __shfl_sync(0xffffffffu, unit[0], f.unit);
          f.rows = __shfl_sync(0xffffffffu, unit[1], f.unit);
          f.shared = __shfl_sync(0xffffffffu, unit[2], f.unit);
          const int skip = f.lo - f.shared + __shfl_sync(0xffffffffu, before, f.unit);
          f.row = f.lo > f.shared ? __popc(__ballot_sync(0xffffffffu, sum <= skip)) : f.row0;
          g += f.end - f.lo;
        }
        if (lane < a.M) pages[lane + 1] = sum;
        if (lane < n_units) cum[lane + 1] = total;
        if (lane == 0) {
          pages[0] = 0;
          cum[0] = 0;
          const int4* from = reinterpret_cast<const int4*>(&f);
          s_first[0] = make_int4(S, g, end, some);
          s_first[1] = from[0]; s_first[2] = from[1]; s_first[3] = from[2];
        }
      }
    } else {
      __syncthreads();
      if (threadIdx.x < 32) {
        running(pages, a.M);
        __syncwarp();
        for (int u = threadIdx.x; u < n_units; u += 32) {
          const int* unit = units + u * kPxUnit;
          int live = 0;                                           // a unit without a live row reads nothing
          for (int m = unit[0]; !live && m < unit[0] + unit[1]; ++m) live = keys[m];
          cum[u + 1] = live ? unit[2] + pages[unit[0] + unit[1]] - pages[unit[0]] : 0;
        }
        __syncwarp();
        running(cum, n_units);
        __syncwarp();
        if (threadIdx.x == 0) {
          S = cum[n_units];
          const unsigned T = (unsigned)(a.n_kv * S), n = px_ctas(a, T);
          g = (unsigned)cta < n ? (int)((unsigned)cta * T / n) : 0;
          end = (unsigned)cta < n ? (int)((unsigned)(cta + 1) * T / n) : 0;
          PxFrag f = {};
          const int some = next(f);
          const int4* from = reinterpret_cast<const int4*>(&f);
          s_first[0] = make_int4(S, g, end, some);
          s_first[1] = from[0]; s_first[2] = from[1]; s_first[3] = from[2];
        }
      }
    }
    __syncthreads();
    const int4 h = s_first[0];
    S = h.x; g = h.y; end = h.z;
    // for the launch that joins the fragments
    if (blockIdx.x == 0)
      for (int m = threadIdx.x; m < a.M; m += blockDim.x) {
        const int u = a.meta[m * kPxMeta + 3], shared = units[u * kPxUnit + 2];
        a.sched[2 * m] = make_int4(S, cum[u], shared, keys[m]);
        a.sched[2 * m + 1] = make_int4(shared + pages[m] - pages[units[u * kPxUnit]], pages[m + 1] - pages[m], u, a.meta[m * kPxMeta + 4]);
      }
  }
  __device__ __forceinline__ bool first(const int4* s_first, PxFrag& f) const {
    int4* to = reinterpret_cast<int4*>(&f);
    to[0] = s_first[1]; to[1] = s_first[2]; to[2] = s_first[3];
    return s_first[0].w != 0;
  }
  __device__ __forceinline__ bool next(PxFrag& f) {
    if (g >= end) return false;
    f.kvh = (int)((unsigned)g / (unsigned)S);
    const int rem = g - f.kvh * S;
    f.unit = find(cum, n_units, rem);
    f.lo = rem - cum[f.unit];
    const int n = min(cum[f.unit + 1] - rem, end - g);
    f.end = f.lo + n;
    f.id = f.kvh * n_units + f.unit + cta;
    g += n;
    const int* unit = units + f.unit * kPxUnit;
    f.row0 = unit[0]; f.rows = unit[1]; f.shared = unit[2];
    f.row = f.row0;
    if (f.lo > f.shared) f.row = f.row0 + find(pages + f.row0, f.rows, pages[f.row0] + f.lo - f.shared);
    return true;
  }
};

// The pages of a unit in order: the shared ones, then every row's own.
struct PxWalk {
  const int* keys; const int* pages;
  int row0, rows, shared, row;
  __device__ __forceinline__ void start(const PxLine& line, const PxFrag& f) {
    keys = line.keys; pages = line.pages;
    row0 = f.row0; rows = f.rows; shared = f.shared; row = f.row;
  }
  // owner: row of the unit, -1 all of them; col: page of the sequence; n: its keys.  Pages are asked for in order; for shared ones,
  // most of a long walk, nothing is looked up.
  __device__ __forceinline__ void page(int p, int& owner, int& col, int& n) {
    owner = -1; col = p; n = kPxPage;
    if (p < shared) return;
    const int at = pages[row0] + p - shared;
    while (pages[row + 1] <= at) ++row;
    owner = row - row0;
    col = shared + at - pages[row];
    n = min(kPxPage, keys[row] - kPxPage * col);
  }
};
// The same value in a uniform register, which is where the tensor instructions take their operands from: what comes from memory
// or a shuffle, and what is branched on it, would be moved there for each of them (the issuer took 2,300 clocks a job).
__device__ __forceinline__ int px_uniform(int v) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)v); }

// tiles of rows that a page concerns, one bit each
__device__ __forceinline__ unsigned px_tiles(int owner, int rows_tile, int n_x) {
  return owner == -1 ? (n_x == 2 ? 3u : 1u) : owner < rows_tile ? 1u : 2u;
}

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

constexpr int kPxHalf = 128 * 128;                      // 16 KB: 128 rows of 64 f16 values, one swizzle atom wide
constexpr int px_tile(int head) { return head / 64 * kPxHalf; }
constexpr int px_page(int head) { return head / 64 * kPxPage * 128; }             // a page of one head as f16: [HEAD / 64][64 keys][128 bytes]
// Pages of keys and of values in flight.  q8_0: four as they are in the cache, two expanded.
constexpr int px_stages(bool q8) { return q8 ? 2 : 4; }
constexpr int px_raw(int head) { return kPxPage * (head / 32 * 34); }             // a page of q8_0 rows of one head: a multiple of 16
constexpr int px_smem(int head, bool q8, int n_units, int M) {
  return 2 * px_tile(head) + 2 * px_stages(q8) * px_page(head) + (q8 ? 8 * px_raw(head) : 0) + 1024 + PxLine::words(M, n_units) * 4;
}
// q8_0 caches have four more warps, which expand the rows
constexpr int px_threads(bool q8) { return q8 ? 512 : 384; }

__device__ __forceinline__ void px_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// Four q8_0 codes times their scale as f16: a code is made the low byte of 1024 + 128 + code, which is exact.
__device__ __forceinline__ void px_codes(uint32_t c, __half2 d, uint32_t& lo, uint32_t& hi) {
  c ^= 0x80808080u;
  const uint32_t a = __byte_perm(c, 0x64646464u, 0x4140), b = __byte_perm(c, 0x64646464u, 0x4342);
  const __half2 bias = __float2half2_rn(1152.f);
  const __half2 x = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&a), bias), d), y = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&b), bias), d);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}
// Whether a q8_0 row may hold a value past f16's range.  It becomes NaN then, so that the query rows it concerns are summed key by
// key: as an infinity it could make a score of -inf, which nothing tells from a key without weight.
template <int HEAD>
__device__ __forceinline__ bool px_wide(const uint8_t* row) {
  bool wide = false;
#pragma unroll
  for (int c = 0; c < HEAD / 64; ++c) wide |= !__hble2(__habs2(reinterpret_cast<const __half2*>(row)[c]), __float2half2_rn(65504.f / 128));
  return wide;
}
// All values of a row at `dst` the same two: blocks of 64 values `pitch` bytes apart.
template <int HEAD>
__device__ __forceinline__ void px_fill(uint8_t* dst, int pitch, uint32_t v) {
#pragma unroll
  for (int c = 0; c < HEAD / 8; ++c) *reinterpret_cast<uint4*>(dst + (c >> 3) * pitch + ((c & 7) << 4)) = make_uint4(v, v, v, v);
}
// A q8_0 row in shared memory to f16 at `dst`: 16-byte chunks swizzled by the row, blocks of 64 values `pitch` bytes apart.
template <int HEAD>
__device__ __forceinline__ void px_expand(const uint8_t* row, uint8_t* dst, int pitch, int swizzle) {
  const __half* scales = reinterpret_cast<const __half*>(row);
  const uint8_t* codes = row + HEAD / 16;
#pragma unroll
  for (int c = 0; c < HEAD / 8; ++c) {                          // eight values
    const __half2 d = __half2half2(scales[c >> 2]);
    uint32_t w0, w1;
    if constexpr (HEAD == 128) {                                // rows of 136 bytes, of 68 otherwise
      const uint2 w = *reinterpret_cast<const uint2*>(codes + 8 * c);
      w0 = w.x; w1 = w.y;
    } else {
      w0 = *reinterpret_cast<const uint32_t*>(codes + 8 * c);
      w1 = *reinterpret_cast<const uint32_t*>(codes + 8 * c + 4);
    }
    uint4 o;
    px_codes(w0, d, o.x, o.y);
    px_codes(w1, d, o.z, o.w);
    *reinterpret_cast<uint4*>(dst + (c >> 3) * pitch + (((c & 7) ^ swizzle) << 4)) = o;
  }
}

__device__ __forceinline__ void px_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// a line of every 2 MB of the scratch
__device__ __forceinline__ void px_touch_scratch(const PrefixArgs& a) {
  for (long at = (long)threadIdx.x << 21; at < a.part_bytes; at += (long)blockDim.x << 21) px_prefetch(reinterpret_cast<const uint8_t*>(a.part) + at);
  if (threadIdx.x < 32) px_prefetch(a.sched + 2 * threadIdx.x);
}

// Bounds of 512 threads in both forms, that is 128 registers a lane: blocks of the joining launch fit beside the 384 threads of f16
// caches and are there when these end (with 138 registers four beams behind 512 positions took 14.9 us a call instead of 12.5).
template <int HEAD, bool Q8>
__global__ void __launch_bounds__(512, 1)
prefix_attn_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const PrefixArgs a) {
  constexpr int NH = HEAD / 64, TILE = px_tile(HEAD), PAGE = px_page(HEAD), ATOM = kPxPage * 128, ST = px_stages(Q8), RAW = px_raw(HEAD);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[4], p_full[4], pv_done[4], raw_full[8], raw_empty[8];
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort, s_bad[16];
  __shared__ int4 s_first[4];
  __shared__ float s_scale[2][128];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;                // [2 tiles][NH][128 rows][128 bytes]
  uint8_t* sK = sQ + 2 * TILE;       // [ST pages][NH][64 keys][128 bytes]
  uint8_t* sV = sK + ST * PAGE;      // [ST pages][NH][64 keys][128 bytes]
  uint8_t* sRaw = sV + ST * PAGE;    // q8_0: [4 pages][keys, values][64 rows]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.n_q / a.n_kv, rows_tile = 128 / G, inv_G = 65536 / G + 1;     // i * inv_G >> 16 is i / G for i < 128

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 4);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&k_full[i], Q8 ? 2 : 1); mbar_init(&k_empty[i], 2); mbar_init(&v_full[i], Q8 ? 2 : 1); mbar_init(&v_empty[i], 2);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; Q8 && i < 8; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 2); }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Ahead of the wait, for lines and address translations alone: a first touch of a page costs a processor the better part of a
  // microsecond, and these would follow each other.
  for (int i = threadIdx.x; i < a.M; i += blockDim.x) { px_prefetch(a.row_pos + i); px_prefetch(a.row_seq + i); px_prefetch(a.meta + i * kPxMeta); }
  if (threadIdx.x < 32) { px_prefetch(a.units + min((int)threadIdx.x, a.n_units - 1) * kPxUnit); px_prefetch(a.table + min((long)threadIdx.x * 32, (long)a.n_slots * a.max_pages - 1)); }
  px_touch_scratch(a);
  {
    const long at = ((long)blockIdx.x * blockDim.x + threadIdx.x) * 32;
    if (at < (long)a.M * a.n_q * HEAD) px_prefetch(a.q + at);
  }
  pdl_wait();
  pdl_launch();
  PxLine line;
  tc_fence_before();
  line.build(a, reinterpret_cast<int*>(sRaw + (Q8 ? 8 * RAW : 0)), s_first);
  tc_fence_after();
  const uint32_t tmem_base = s_tmem_base;
  volatile int* abort_flag = &s_abort;
  const uint32_t tS0 = tmem_base, tO0 = tmem_base + 256;        // score buffer b of tile x at column 128 x + 64 b, its output at 256 + HEAD x
  PxFrag f;
  PxWalk w;

  if (Q8 && warp >= 12) {
    // ---- q8_0 rows to f16: two warps the keys, two the values, a thread for a row of the page
    const int kv = (warp - 12) >> 1, row = threadIdx.x & 63;
    uint64_t* const full = kv ? v_full : k_full;
    uint64_t* const empty = kv ? v_empty : k_empty;
    int page = 0;
    bool ok = true;
    for (bool more = line.first(s_first, f); ok && more; more = line.next(f)) {
      w.start(line, f);
      for (int p = f.lo; p < f.end; ++p, ++page) {
        int owner, col, n;
        w.page(p, owner, col, n);
        const int slot = page & 3, st = page % ST;
        ok = mbar_wait_warp(&raw_full[2 * slot + kv], (uint32_t)((page >> 2) & 1), abort_flag);
        if (!ok) break;
        const uint8_t* raw = sRaw + (slot * 2 + kv) * RAW + row * (RAW / kPxPage);
        const bool wide = px_wide<HEAD>(raw);                   // while the page before is multiplied
        ok = mbar_wait_warp(&empty[st], (uint32_t)((page / ST) & 1) ^ 1, abort_flag);
        if (!ok) break;
        uint8_t* dst = (kv ? sV : sK) + st * PAGE + row * 128;
        if (row < n && !wide) px_expand<HEAD>(raw, dst, ATOM, row & 7);
        else px_fill<HEAD>(dst, ATOM, row < n ? 0x7fff7fffu : 0u);               // behind a sequence's end: zero, whatever lies there
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[st]);
          mbar_arrive(&raw_empty[2 * slot + kv]);
        }
      }
    }
  } else if (warp == 8) {
    // ---- producer: the warp looks pages up 32 at a time, lane 0 waits and copies
    int page = 0, nf = 0;
    bool ok = true;
    for (bool more = line.first(s_first, f); ok && more; more = line.next(f), ++nf) {
      w.start(line, f);
      const int* unit = line.units + f.unit * kPxUnit;
      int lead = -1;                                            // sequence of the first row of the group that has a table
      for (int i = 0; lead < 0 && i < unit[4]; i += 32) {
        const int mine = i + lane < unit[4] ? line.seq[unit[3] + i + lane] : -1;
        const unsigned live = __ballot_sync(0xffffffffu, mine >= 0 && mine < a.n_slots);
        if (live) lead = __shfl_sync(0xffffffffu, mine, __ffs(live) - 1);
      }
      int ids = 0;
      bool bad = false;
      for (int p = f.lo; ok && p < f.end; ++p, ++page) {
        const int i = (p - f.lo) & 31;
        if (i == 0) {
          const int mine = p + lane;
          int seq = -1, col = mine;
          if (mine < f.end) {
            seq = lead;
            if (mine >= w.shared) {
              const int at = w.pages[w.row0] + mine - w.shared, row = w.row0 + PxLine::find(w.pages + w.row0, w.rows, at);
              seq = line.seq[row];
              col = w.shared + at - w.pages[row];
            }
          }
          ids = seq >= 0 ? a.table[(long)seq * a.max_pages + col] : 0;
          const bool off = ids < 0 || ids >= a.n_pages;
          if (off) { ids = 0; raise_fault(a.fault, a.layer, FS_PAGE); }
          bad = bad || __any_sync(0xffffffffu, off);
        }
        const int block = __shfl_sync(0xffffffffu, ids, i) * a.n_kv + f.kvh, st = page & 3;
        const uint32_t par = (uint32_t)((page >> 2) & 1);
        if (lane == 0) {
#pragma unroll
          for (int kv = 0; ok && kv < 2; ++kv) {
            if constexpr (Q8) ok = mbar_wait(&raw_empty[2 * st + kv], par ^ 1, abort_flag);
            else ok = kv ? mbar_wait(&v_empty[st], par ^ 1, abort_flag) : mbar_wait(&k_empty[st], par ^ 1, abort_flag);
            if (!ok) break;
            // behind the first of these waits the softmax of a dozen pages ago is over: the flag may be used again
            if (kv == 0 && (i == 0)) s_bad[nf & 15] = bad;
            uint64_t* const full = Q8 ? &raw_full[2 * st + kv] : kv ? &v_full[st] : &k_full[st];
            mbar_expect_tx(full, Q8 ? RAW : PAGE);
            if constexpr (Q8) {
              px_bulk(sRaw + (st * 2 + kv) * RAW, (kv ? a.v : a.k) + (long)block * RAW, RAW, full);
            } else {
#pragma unroll
              for (int h = 0; h < NH; ++h) tma_load_2d((kv ? sV : sK) + st * PAGE + h * ATOM, kv ? &tma_v : &tma_k, h * 64, block * kPxPage, full);
            }
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
  } else if (warp == 9 || warp == 10) {
    // ---- issuers: one for each tile of rows, so that neither's waits and look-ups hold the other's products up
    const int x = px_uniform(warp - 9);
    constexpr uint32_t idesc_s = px_idesc(128, kPxPage, false), idesc_o = px_idesc(128, HEAD, true);
    const uint32_t uS = (uint32_t)px_uniform((int)tS0) + x * 128, uO = (uint32_t)px_uniform((int)tS0) + 256 + x * HEAD;
    int page0 = 0, n_q = 0, n_s = 0, n_o = 0;                   // pages through the rings; query tiles, first and second products
    bool ok = true;
    for (int more = px_uniform(line.first(s_first, f)); ok && more; more = px_uniform(line.next(f))) {
      w.start(line, f);
      const int n_x = px_uniform(w.rows > rows_tile ? 2 : 1), n_p = px_uniform(f.end - f.lo), shared = px_uniform(w.shared - f.lo);
      uint32_t own = 0;                                         // of the last 32 pages: whether this tile of rows takes part
      bool asked = false;
      uint32_t old = 0;
      int t = 0;                                                // pages whose keys are done with
      // S = Q K^T of the next pages: no further than their keys can have been fetched (the values of the pages between are still
      // to be released here), and two of this tile's own ahead of its second products
      auto first_products = [&](int at) {
        while (ok && t < n_p && t < at + ST) {
          bool part = n_x == 2 || x == 0;
          if (t >= shared) {
            PxWalk look = w;
            int owner, col, n;
            look.page(f.lo + t, owner, col, n);
            w.row = look.row;
            part = px_uniform((int)(px_tiles(owner, rows_tile, n_x) >> x & 1)) != 0;
          }
          if (part && n_s - n_o >= 2) return;
          const int st = (page0 + t) % ST;
          ok = mbar_wait_warp(&k_full[st], (uint32_t)(((page0 + t) / ST) & 1), abort_flag);
          if (ok && part && !asked) ok = mbar_wait_warp(&q_full[x], (uint32_t)(n_q++ & 1), abort_flag);
          if (!ok) return;
          own = (own & ~(1u << (t & 31))) | (uint32_t)part << (t & 31);
          ++t;
          if (!part) {
            if (lane == 0) mbar_arrive(&k_empty[st]);
            continue;
          }
          asked = true;
          tc_fence_after();
          const uint32_t tS = uS + (n_s & 1) * 64;
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const uint64_t dq = umma_desc(smem_u32(sQ + x * TILE + h * kPxHalf)), dk = umma_desc(smem_u32(sK + st * PAGE + h * ATOM));
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16(tS, dq + (uint64_t)(k * 2), dk + (uint64_t)(k * 2), idesc_s, h + k > 0 ? 1u : 0u);
          }
          // Two barriers, for every other job.  The softmax waits for its scores but not for every second product; when it comes
          // to a barrier, the job before the last is known to be complete (these scores were issued behind it), the last one is
          // not, and a wait by parity must not be two phases off.
          umma_commit(&s_full[2 * x + (n_s++ & 1)]);
          umma_commit(&k_empty[st]);
        }
      };
      for (int at = 0; ok && at < n_p; ++at) {
        first_products(at);
        const int st = (page0 + at) % ST;
        ok = ok && mbar_wait_warp(&v_full[st], (uint32_t)(((page0 + at) / ST) & 1), abort_flag);
        if (!ok) break;
        if (!(own >> (at & 31) & 1)) {
          if (lane == 0) mbar_arrive(&v_empty[st]);
          continue;
        }
        const int b = n_o & 1;
        ok = mbar_wait_warp(&p_full[2 * x + b], (uint32_t)((n_o >> 1) & 1), abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t tP = uS + b * 64;
        const uint64_t dv = px_desc_v(smem_u32(sV + st * PAGE));
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16_ta(uO, tP + k * 8, dv + (uint64_t)(k * 128), idesc_o, k > 0 ? 1u : old);
        old = 1;
        umma_commit(&pv_done[2 * x + b]);
        umma_commit(&v_empty[st]);
        ++n_o;
      }
      page0 += n_p;
    }
  } else if (warp < 8) {
    // ---- softmax: a thread per query row ------------------------------------------------------------------
    const int x = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;                          // row of the tile
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t tO = tO0 + x * HEAD + lane_base;
    int page = 0, mine = 0, nf = 0;                             // pages; jobs of this tile of rows; fragments
    bool ok = true;
    for (bool more = line.first(s_first, f); ok && more; more = line.next(f), ++nf) {
      w.start(line, f);
      const int n_x = w.rows > rows_tile ? 2 : 1;
      const int live = max(0, min(rows_tile, w.rows - x * rows_tile)) * G;      // query rows of this tile
      const int my = r < live ? x * rows_tile + (r * inv_G >> 16) : -3;     // row of the unit
      const int n_keys = r < live ? w.keys[w.row0 + my] : 0;
      const bool busy = quarter * 32 < live;
      // Queries to f16, scaled by a power of two a row to a largest element in [512, 1024).  Eight lanes have a row, so that a warp's
      // steps serve four rows: a fragment goes through this code once or a few times, and most of its time is fetching it.
      auto put_queries = [&]() {
        constexpr int N = HEAD / 32;                            // 16 bytes of a lane's, 128 bytes of its row apart
        const int l = lane & 7;
        const float* base = a.q + ((long)(w.row0 + x * rows_tile) * a.n_q + f.kvh * G) * HEAD + l * 4;
        uint8_t* dst = sQ + x * TILE + (l & 1) * 8;
        auto some_rows = [&](int i0, auto at_once) {
          constexpr int AT_ONCE = decltype(at_once)::value;
          float4 v[AT_ONCE][N];
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u) {
            const int i = i0 + 4 * u;
            const float* src = base + (long)((i * inv_G >> 16) * (a.n_q - G) + i) * HEAD;
#pragma unroll
            for (int j = 0; j < N; ++j) v[u][j] = i < live ? __ldg(reinterpret_cast<const float4*>(src + j * 32)) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          // no branches, so that the rows' chains of steps run side by side; rows behind the last are zeros
          unsigned top[AT_ONCE];
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u) {
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j)
              most = fmaxf(fmaxf(most, fmaxf(fabsf(v[u][j].x), fabsf(v[u][j].y))), fmaxf(fabsf(v[u][j].z), fabsf(v[u][j].w)));
            top[u] = __float_as_uint(most);                     // of non-negative floats: in order as integers
          }
#pragma unroll
          for (int o = 1; o < 8; o <<= 1)
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) top[u] = max(top[u], __shfl_xor_sync(0xffffffffu, top[u], o));
#pragma unroll
          for (int u = 0; u < AT_ONCE; ++u) {
            const int i = i0 + 4 * u, e = (int)(top[u] >> 23), se = e == 0 ? 127 : min(253, 263 - e);
            const float scale = __uint_as_float((unsigned)se << 23);
            uint8_t* at = dst + i * 128;
#pragma unroll
            for (int j = 0; j < N; ++j)
              *reinterpret_cast<uint2*>(at + (j >> 1) * kPxHalf + ((((j & 1) * 4 + (l >> 1)) ^ (i & 7)) << 4)) =
                  make_uint2(px_pack(v[u][j].x * scale, v[u][j].y * scale), px_pack(v[u][j].z * scale, v[u][j].w * scale));
            if (l == 0) s_scale[x][i] = kPxLog2e * __uint_as_float((unsigned)(254 - se) << 23);
          }
        };
        if (live > 16) {
          // the CTAs of a unit read the same rows: they begin at different ones
          const int n_it = (live + 31) >> 5;
          int it = (int)((unsigned)blockIdx.x % (unsigned)n_it);
#pragma unroll 1
          for (int k = 0; k < n_it; ++k) {
            some_rows(8 * quarter + 32 * it + (lane >> 3), std::integral_constant<int, 2>());
            it = it + 1 == n_it ? 0 : it + 1;
          }
        } else if (4 * quarter < live) {
          some_rows(4 * quarter + (lane >> 3), std::integral_constant<int, 1>());
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[x]);
      };
      float m = -INFINITY, l = 0.f, to_log2 = 0.f;
      bool begun = false;
      for (int p = f.lo; p < f.end; ++p, ++page) {
        int owner, col, held;
        w.page(p, owner, col, held);
        const unsigned who = px_tiles(owner, rows_tile, n_x);
        if (!(who >> x & 1)) continue;
        const int b = mine & 1;
        const uint32_t tS = tS0 + x * 128 + b * 64 + lane_base;
        // keys of the page that this thread's row attends to
        const int n = owner == my ? held : owner == -1 ? min(kPxPage, max(0, n_keys - kPxPage * col)) : 0;
        const bool some = __any_sync(0xffffffffu, n > 0), all = __all_sync(0xffffffffu, n == kPxPage);
        if (!begun) put_queries();
        ok = mbar_wait_warp(&s_full[2 * x + b], (uint32_t)((mine >> 1) & 1), abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (!begun) to_log2 = busy ? s_scale[x][r] : 0.f;       // written in front of what these scores waited for
        uint32_t v[2][32];
        float corr = 1.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
        if (some) {
          tmem_ld32(tS, v[0]);
          tmem_ld32(tS + 32, v[1]);
          tmem_ld_wait();
          if (!all) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (i >= n) v[i >> 5][i & 31] = 0xff800000u;      // -inf
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 4)
#pragma unroll
            for (int j = 0; j < 4; ++j) top[j] = fmaxf(fmaxf(top[j], __uint_as_float(v[0][i + j])), __uint_as_float(v[1][i + j]));
          float m_new = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
          if (m != -INFINITY && (m_new - m) * to_log2 <= kPxLazy) m_new = m;
          const float mb = (m_new == -INFINITY) ? 0.f : m_new * to_log2;      // a row with no key yet keeps zeros
          corr = (m == -INFINITY || m == m_new) ? 1.f : px_ex2(m * to_log2 - mb);
          m = m_new;
          if (begun && __any_sync(0xffffffffu, corr != 1.0f)) {
            // the output is scaled in tensor memory, behind the tile's last product
            ok = mbar_wait_warp(&pv_done[2 * x + (b ^ 1)], (uint32_t)(((mine - 1) >> 1) & 1), abort_flag);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HEAD / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(tO + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              px_st16(tO + c * 16, o);
            }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              uint32_t e0, e1;
              asm("{\n\t.reg .b64 rs, rk, rm, rr;\n\t"
                  "mov.b64 rs, {%2, %3};\n\tmov.b64 rk, {%4, %4};\n\tmov.b64 rm, {%5, %5};\n\t"
                  "fma.rn.f32x2 rr, rs, rk, rm;\n\tmov.b64 {%0, %1}, rr;\n\t}"
                  : "=r"(e0), "=r"(e1) : "r"(v[c][i]), "r"(v[c][i + 1]), "f"(to_log2), "f"(kPxShift - mb));
              const float p0 = px_ex2(__uint_as_float(e0)), p1 = px_ex2(__uint_as_float(e1));
              sum[i & 2] += p0; sum[(i & 2) + 1] += p1;
              pk[i >> 1] = px_pack(p0, p1);
            }
            px_st16(tS + 16 * c, pk);
          }
        } else {                                                // no row of this warp attends to this page
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = 0;
          px_st16(tS, pk);
          px_st16(tS + 16, pk);
        }
        if (!Q8 && held < kPxPage) {
          // A sequence ends inside the page: what lies behind may be anything, and zero times that must be zero.  The page is one
          // row's, so its tile of rows alone reads it.
          const int st = page & 3;
          ok = mbar_wait_warp(&v_full[st], (uint32_t)((page >> 2) & 1), abort_flag);
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < NH; ++h)
            for (int i = held * 8 + r; i < kPxPage * 8; i += 128) *reinterpret_cast<uint4*>(sV + st * PAGE + h * ATOM + i * 16) = make_uint4(0, 0, 0, 0);
          fence_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * x + b]);
        l = l * corr + ((sum[0] + sum[2]) + (sum[1] + sum[3]));
        begun = true;
        ++mine;
      }
      if (ok && begun) {
        ok = mbar_wait_warp(&pv_done[2 * x + ((mine - 1) & 1)], (uint32_t)(((mine - 1) >> 1) & 1), abort_flag);
        tc_fence_after();
      }
      if (!ok) break;
      if (busy) {
        float4* part = a.part + ((long)f.id * a.slot_tiles + x) * a.slot + r;
        if (begun && __any_sync(0xffffffffu, m != -INFINITY)) {
#pragma unroll 1
          for (int c = 0; c < HEAD / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_ld_wait();
            if (m != -INFINITY) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                __stcg(part + (c * 8 + i) * a.pitch, make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                                 __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])));
            }
          }
        }
        // a fragment that met a page the pool does not have gives NaN to all that it serves; a row whose every score is NaN
        // has no maximum, but a sum that tells
        const bool lost = l != l || (*(volatile int*)&s_bad[nf & 15] != 0 && m != -INFINITY);
        if (r < live)
          __stcg(reinterpret_cast<float2*>(part - r + HEAD / 4 * a.pitch) + r,
                 lost ? make_float2(0.f, __int_as_float(0x7fc00000)) : make_float2(m == -INFINITY ? m : m * to_log2, l));
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

// Joins the fragments of a row's heads: grid (n_kv, M, parts of the head), 256 threads.  A row has the fragments that cover its
// shared pages and those that cover its own; other rows' are left out.  One round trip brings the maxima and sums, a warp for a
// head, and the outputs, a thread for four values of a head and every `sets`-th fragment (of `cols` such columns, `items` in all).
constexpr int kPxMaxCtas = 160;

template <int HEAD, bool Q8>
__global__ void __launch_bounds__(256, 4) prefix_join_kernel(const PrefixArgs a) {
  __shared__ float s_w[kPxMaxCtas][16], s_inv[16];
  __shared__ float4 s_o[256];
  const int kvh = blockIdx.x, m = blockIdx.y, G = a.n_q / a.n_kv, tid = threadIdx.x, lane = tid & 31;
  const int set = tid * a.inv_items >> 16, item = tid - set * a.items, col = item * a.inv_G >> 16, h = item - col * G, c = blockIdx.z * a.cols + col;
  // lengths are older than the launch in front, which started behind what wrote them
  bool bad;
  px_keys(a, m, bad);
  px_touch_scratch(a);
  if (tid == 0) px_prefetch(a.out + ((long)m * a.n_q + kvh * G) * HEAD);
  pdl_wait();
  pdl_launch();
  const int4 s0 = __ldcg(a.sched + 2 * m), s1 = __ldcg(a.sched + 2 * m + 1);
  const int n = s0.w, shared = s0.z, own = s1.x, n_own = s1.y, x = s1.w >> 7, lane0 = s1.w & 127;
  int f1 = 0, n1 = 0, f2 = 0, n2 = 0;                           // first CTA and count: of the shared pages, of the row's own
  if (n > 0) {
    // four places on the line, a lane each
    const unsigned T = (unsigned)(a.n_kv * s0.x), base = (unsigned)(kvh * s0.x + s0.y);
    const unsigned at = base + (lane == 0 ? 0 : lane == 1 ? shared - 1 : lane == 2 ? own : own + n_own - 1);
    const int cta = (int)(((at + 1) * px_ctas(a, T) - 1) / T);
    const int c0 = __shfl_sync(0xffffffffu, cta, 0), c1 = __shfl_sync(0xffffffffu, cta, 1), c2 = __shfl_sync(0xffffffffu, cta, 2), c3 = __shfl_sync(0xffffffffu, cta, 3);
    f1 = c0;
    n1 = shared > 0 ? c1 - c0 + 1 : 0;
    if (n_own > 0) {
      f2 = c2 + (n1 > 0 && c2 == c1);                           // one fragment may hold both
      n2 = c3 - f2 + 1;
    }
  }
  const int n_f = n1 + n2, id0 = kvh * a.n_units + s1.z;
  const int step = a.slot * a.slot_tiles;                       // float4 from a fragment to the next
  auto at_of = [&](int f) { return (long)(id0 + (f < n1 ? f1 + f : f2 + f - n1)) * step; };
  const float4* part = a.part + x * a.slot + c * a.pitch + lane0 + h;
  const float2* ml = reinterpret_cast<const float2*>(a.part + x * a.slot + HEAD / 4 * a.pitch) + lane0;
  constexpr int AHEAD = 8;                                      // fragments of a thread in flight
  float4 v[AHEAD];
  auto fetch = [&](int f0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int f = f0 + i * a.sets;
      if (f < n_f && set < a.sets) v[i] = __ldcg(part + at_of(f));
    }
  };
  fetch(set);
  for (int g = tid >> 5; g < G; g += 8) {
    float top = -INFINITY, den = 0.f;
    auto load = [&](int i) { return i < n_f ? __ldcg(ml + at_of(i) * 2 + g) : make_float2(-INFINITY, 0.f); };
    const float2 first = load(lane);                            // most rows have no more than 32
    top = first.x;
    for (int i = lane + 32; i - lane < n_f; i += 32) top = fmaxf(top, load(i).x);
    top = warp_max(top);
    for (int i = lane; i - lane < n_f; i += 32) {
      const float2 q = i == lane ? first : load(i);
      const float w = q.x > -INFINITY ? px_ex2(q.x - top) : 0.f;
      den += w > 0.f || q.y != q.y ? w * q.y : 0.f;             // a NaN stays one, whatever its weight
      s_w[i][g] = w;
    }
    den = warp_sum(den);
    if (lane == 0) s_inv[g] = 1.f / den;
  }
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (set < a.sets)
    for (int f0 = set; f0 < n_f; f0 += AHEAD * a.sets) {        // ascending order, fixed
      if (f0 > set) fetch(f0);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int f = f0 + i * a.sets;
        const float w = f < n_f ? s_w[f][h] : 0.f;
        // a fragment without keys of this row (it ended inside the prefix) has no output: what lies there may be anything
        if (w != 0.f) { o.x = fmaf(w, v[i].x, o.x); o.y = fmaf(w, v[i].y, o.y); o.z = fmaf(w, v[i].z, o.z); o.w = fmaf(w, v[i].w, o.w); }
      }
    }
  s_o[tid] = o;
  __syncthreads();
  bool again = false;
  if (tid < a.items) {
    for (int i = 1; i < a.sets; ++i) { const float4 u = s_o[tid + i * a.items]; o.x += u.x; o.y += u.y; o.z += u.z; o.w += u.w; }
    const float inv = bad ? __int_as_float(0x7fc00000) : n > 0 ? s_inv[h] : 0.f;
    const __nv_bfloat162 b0 = __floats2bfloat162_rn(o.x * inv, o.y * inv), b1 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(a.out + ((long)m * a.n_q + kvh * G + h) * HEAD + c * 4) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
    again = !(fabsf((o.x + o.y) + (o.z + o.w)) * inv < INFINITY);
  }
  // a key or value that is not finite, maybe another row's: this row's own say what its output is
  if (__syncthreads_or(again && n > 0)) {
    for (int g = tid >> 5; g < G; g += 8) {
      float r[HEAD / 32];
      px_row<HEAD, Q8>(a, m, kvh * G + g, n, r);
#pragma unroll
      for (int i = 0; i < HEAD / 32; ++i)
        if (lane * (HEAD / 32) / (4 * a.cols) == (int)blockIdx.z) a.out[((long)m * a.n_q + kvh * G + g) * HEAD + lane * (HEAD / 32) + i] = __float2bfloat16_rn(r[i]);
    }
  }
}

}  // namespace bl

using namespace bl;

template <int HEAD, bool Q8>
static int prefix_go(PrefixArgs a, cudaStream_t st) {
  // The joining launch.  Few rows: a block for 32 values of a head, so that more of its fragments are in flight (8 rows behind 2,048
  // positions 13.6 us a call, 15.8 with whole heads; 24 q8_0 rows 30.4 and 33.1; 21 rows behind 4,096 23.2 and 22.7); many: as much
  // of it as 256 threads hold (100 rows behind 1,024 with up to 64 of their own 23.2 us, 29.1 in parts; 512 such rows 57.7 and 89.6).
  int z = HEAD / 32;
  const int G = a.n_q / a.n_kv;
  if (a.n_kv * a.M > a.n_cta) while (z > 1 && G * (HEAD / 4) / (z / 2) <= 256) z /= 2;
  a.cols = HEAD / 4 / z;
  a.items = G * a.cols;
  a.sets = 256 / a.items;
  a.inv_items = 65536 / a.items + 1;                            // exact for the 256 threads: items and G divide them by 256 at most
  a.inv_G = 65536 / G + 1;
  CUtensorMap mk = {}, mv = {};
  if (!Q8) {
    const cuuint64_t dims[2] = {(cuuint64_t)HEAD, (cuuint64_t)a.n_pages * a.n_kv * kPxPage};
    const cuuint64_t strides[1] = {(cuuint64_t)HEAD * 2};
    const cuuint32_t box[2] = {64, kPxPage};
    int rc = make_map_any(&mk, a.k, 2, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    rc = make_map_any(&mv, a.v, 2, dims, strides, box, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  static PerDevice limit;
  if (limit.due()) {
    const cudaError_t e = cudaFuncSetAttribute(prefix_attn_kernel<HEAD, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               px_smem(HEAD, Q8, kPxMaxRows, kPxMaxRows));
    if (e != cudaSuccess) return (int)e;
    limit.mark();
  }
  const cudaError_t e = launch(prefix_attn_kernel<HEAD, Q8>, dim3(a.n_cta), dim3(px_threads(Q8)), (size_t)px_smem(HEAD, Q8, a.n_units, a.M), st, mk, mv, a);
  if (e != cudaSuccess) return (int)e;
  return (int)launch(prefix_join_kernel<HEAD, Q8>, dim3(a.n_kv, a.M, z), dim3(256), 0, st, a);
}

extern "C" {

// Bytes of scratch that bl_prefix_attention takes for units of up to unit_rows rows (n_cta processors).
static long prefix_slots(int head, int G, int n_kv, int n_units, int unit_rows, int n_cta, int& slot, int& tiles, int& pitch) {
  const int per = 128 / G;
  tiles = unit_rows > per ? 2 : 1;
  pitch = ((unit_rows < per ? unit_rows : per) * G + 7) / 8 * 8;
  slot = (head / 4 * pitch + pitch / 2);
  return ((long)n_kv * n_units + n_cta) * tiles * slot * 16;
}
long bl_prefix_work_bytes(int head, int n_q, int n_kv, int n_units, int unit_rows, int n_cta) {
  int slot, tiles, pitch;
  return prefix_slots(head, n_q / n_kv, n_kv, n_units, unit_rows, n_cta, slot, tiles, pitch) + kPxMaxRows * 32;
}

// The call as one block of memory: a host that makes a call a layer hands over one pointer instead of two dozen arguments.
struct PrefixCall {
  const float* q; const void* k_cache; const void* v_cache; const int* row_pos; const int* row_seq; const int* block_table;
  const int* meta; void* work; void* out; unsigned* fault; cudaStream_t stream;
  int n_slots, max_pages, n_pages, head, n_q, n_kv, M, n_units, unit_rows, kv_q8, n_cta, layer;
};

int bl_prefix_attention(const PrefixCall* call) {
  const PrefixCall& p = *call;
  const int head = p.head, n_q = p.n_q, n_kv = p.n_kv, M = p.M, n_units = p.n_units, unit_rows = p.unit_rows, n_cta = p.n_cta;
  const int max_pages = p.max_pages, n_pages = p.n_pages;
  void* work = p.work;
  BL_REQUIRE(head == 128 || head == 64, BL_ERR_SHAPE);
  BL_REQUIRE(n_kv >= 1 && n_q >= 1 && n_q % n_kv == 0 && n_q / n_kv <= 16, BL_ERR_SHAPE);
  BL_REQUIRE(M >= 1 && M <= kPxMaxRows && n_units >= 1 && n_units <= M && unit_rows >= 1 && unit_rows <= 2 * (128 / (n_q / n_kv)), BL_ERR_SHAPE);
  BL_REQUIRE(n_cta >= 1 && n_cta <= kPxMaxCtas && p.n_slots >= 1 && max_pages >= 1 && n_pages >= 1, BL_ERR_SHAPE);
  BL_REQUIRE((long)n_pages * n_kv * kPxPage <= 0x7fffffffL && (long)(max_pages + 2) * M * n_kv <= 1L << 24, BL_ERR_LIMIT);
  BL_REQUIRE((((uintptr_t)p.q | (uintptr_t)p.k_cache | (uintptr_t)p.v_cache | (uintptr_t)p.out | (uintptr_t)work) & 15) == 0, BL_ERR_ALIGN);
  PrefixArgs a{p.q, (const uint8_t*)p.k_cache, (const uint8_t*)p.v_cache, p.row_pos, p.row_seq, p.block_table, p.n_slots, max_pages, n_pages,
               n_q, n_kv, M, p.meta, (__nv_bfloat16*)p.out, p.fault, p.layer, p.meta + (long)M * kPxMeta, n_units, n_cta};
  const cudaStream_t st = p.stream;
  a.sched = (int4*)work;
  a.part = (float4*)((uint8_t*)work + kPxMaxRows * 32);
  a.part_bytes = prefix_slots(head, n_q / n_kv, n_kv, n_units, unit_rows, n_cta, a.slot, a.slot_tiles, a.pitch);
  if (p.kv_q8) return head == 128 ? prefix_go<128, true>(a, st) : prefix_go<64, true>(a, st);
  return head == 128 ? prefix_go<128, false>(a, st) : prefix_go<64, false>(a, st);
}

}  // extern "C"
