// Beam search behind the logits: the choice of the next beams, and cached states that follow them.
//
// Choice.  Beam b of a search has a score (the log-probability of its tokens) and a row of logits; its continuation by token t has
//   cand(b, t) = score_b + logit_bt - lse_b,     lse_b = log sum_t e^logit_bt.
// A finished beam has one candidate, itself: (b, eos) with its score.  Candidates are ranked by cand / length^alpha and the B best
// of B * V become the next beams, ties to the lowest b * V + t.  Candidates are compared in 64 bits: added to a score in 32, two
// logits of one beam that differ could become equal and change places.
//
// States.  Child i of a search continues parent[i]'s history: pages that are full are shared by naming them in its table row.  In
// the page being filled (part = held % 64 positions) a parent's first child goes on; each further child takes the page of a beam
// that has no child -- there are as many of these -- and a copy of the positions held.  What is read is never written, so all
// copies run at once.  Pages behind belong to the slot.
#include <cfloat>

#include "common.cuh"

namespace bl {

constexpr int kMaxBeams = 64;
constexpr float kMaxAlpha = 16.f;                         // length^alpha, and a score times it, in range of 64 bits for any length of 32

constexpr int kBmThreads = 256;
constexpr int kBmList = 512;                              // survivors that are ranked side by side
constexpr int kBmMaxCells = kBmThreads;                   // chunks of a row x beams: merged with one a thread

struct BeamCell { float value; int id; };

struct BeamArgs {
  const float* logits; long stride; int V, G, B;
  const float* scores;                                    // [G][B], -inf: no beam
  const int* done; const int* lengths;                    // optional [G][B]
  int eos; float alpha;
  int n_chunks, chunk;                                    // of a row; values of a chunk (a multiple of 4 unless there is one)
  BeamCell* cells;                                        // [G * B][n_chunks][B], best first
  float2* sums;                                           // [G * B][n_chunks]: maximum, sum of exponentials
  BeamCell* best;                                         // [G * B][B]
  double* lse;                                            // [G * B]
  int* tickets;                                           // [G * B] chunks, then [G] rows; zero between calls
  int* parent; int* token; float* out_scores; int* out_done; int* out_lengths;
  unsigned* fault;
};

// The order of values as integers; the two zeros are one.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_of(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}

__device__ __forceinline__ float value_of(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ double value_of(unsigned long long u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }

struct BestScratch {
  __align__(16) unsigned long long key[kBmList + 1];
  int id[kBmList];
  double group[128], bound;
  int part[kBmThreads / 32];
  int n;
};

// A bound that k of the block's values reach: the k-th largest of the maxima of 32 groups of lanes, of 128 for more than 32.
// `mine`: the largest value of this thread; -inf is none.
template <typename T>
__device__ __forceinline__ T block_bound(T mine, int k, BestScratch& s) {
  const int tid = threadIdx.x, lane = tid & 31, lanes = k <= 32 ? 8 : 2;
  T* group = reinterpret_cast<T*>(s.group);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1)
    if (o < lanes) { const T u = __shfl_xor_sync(0xffffffffu, mine, o); mine = u > mine ? u : mine; }
  if ((lane & (lanes - 1)) == 0) group[tid / lanes] = mine;
  if (tid == 0) s.n = 0;
  __syncthreads();
  if (k <= 32) {
    const T bound = group[lane];
    int before = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) { const T u = group[j]; before += (int)(u > bound) + ((int)(u == bound) & (int)(j < lane)); }
    const unsigned at = __ballot_sync(0xffffffffu, before == k - 1);             // one lane's: the groups are in an order
    return __shfl_sync(0xffffffffu, bound, __ffs(at) - 1);
  }
  if (tid < 128) {
    const T bound = group[tid];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < 128; ++j) { const T u = group[j]; before += (int)(u > bound) + ((int)(u == bound) & (int)(j < tid)); }
    if (before == k - 1) s.bound = (double)bound;
  }
  __syncthreads();
  return (T)s.bound;
}

// list(bound) lists the values that reach the bound.  Where these are more than the list holds (cells of 64 beams, each row's in
// order, make a weak bound), the bound is narrowed by halving the values above it, until it leaves at least k and at most a list.
// Behind it s.n says how many reached the bound; still too many only where that many are equal.
template <typename T, typename Count, typename List>
__device__ __forceinline__ void block_list(T bound, int k, BestScratch& s, Count count, List list) {
  list(bound);
  __syncthreads();
  if (s.n <= kBmList) return;
  auto lo = order_of(bound);
  decltype(lo) hi = ~(decltype(lo))0;
#pragma unroll 1
  for (int step = 0; step < 64 && hi - lo > 1; ++step) {
    const decltype(lo) mid = lo + (hi - lo) / 2;
    const int mine = __reduce_add_sync(0xffffffffu, count(value_of(mid)));
    if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = mine;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kBmThreads / 32; ++w) all += s.part[w];
    __syncthreads();
    if (all > kBmList) lo = mid;
    else if (all < k) hi = mid;
    else {
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
      list(value_of(mid));
      __syncthreads();
      return;
    }
  }
}

// The listed candidates in order, s.n of them and no more than the list holds: store(rank, key, id) of the k best.  A candidate
// counts the ones before it; where there are few, two or four threads share a candidate's count.
template <bool IDS, typename Store>
__device__ __forceinline__ void block_rank(int k, const BestScratch& s, Store store) {
  const int tid = threadIdx.x, n = s.n, shift = n <= 64 ? 2 : n <= 128 ? 1 : 0;
  for (int at = tid; (at & ~31) < n << shift; at += kBmThreads) {                // whole warps
    const int e = at >> shift, part = at & ((1 << shift) - 1);
    const bool there = e < n;
    const unsigned long long key = there ? s.key[e] : 0;
    const int id = IDS && there ? s.id[e] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 1 << shift) {
      const unsigned long long u = s.key[j];
      rank += (int)(u > key);
      if (IDS) rank += (int)(u == key) & (int)(s.id[j] < id);
    }
    if (shift > 0) rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    if (shift > 1) rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (there && part == 0 && rank < k) store(rank, key, id);
  }
}

// The k best of the block's values by k rounds, where more than the list holds are equal: next(last, last id, best, id) gives a thread's best behind the last one taken.
template <typename T, typename Next, typename Store>
__device__ __forceinline__ void block_rounds(int k, BestScratch& s, Next next, Store store) {
  const int tid = threadIdx.x, lane = tid & 31;
  const T none = (T)-INFINITY;
  T last = (T)INFINITY;
  int last_id = -1;
  T* value = reinterpret_cast<T*>(s.group);
  for (int round = 0; round < k; ++round) {
    T best = none;
    int where = 0x7fffffff;
    next(last, last_id, best, where);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const T u = __shfl_xor_sync(0xffffffffu, best, o);
      const int w = __shfl_xor_sync(0xffffffffu, where, o);
      if (u > best || (u == best && w < where)) { best = u; where = w; }
    }
    __syncthreads();
    if (lane == 0) { value[tid >> 5] = best; s.id[tid >> 5] = where; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kBmThreads / 32; ++w)
      if (value[w] > best || (value[w] == best && s.id[w] < where)) { best = value[w]; where = s.id[w]; }
    if (best == none) break;
    if (tid == 0) store(round, best, where);
    last = best;
    last_id = where;
  }
}

// 2^x; what is less than 2^-126 counts as nothing beside a sum of 1 or more, which saves the instructions that keep it.
__device__ __forceinline__ float bm_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kBmLog2e = 1.4426950408889634f;
// sum[2] += e^(v - top) of two values, additions and products of both at once
__device__ __forceinline__ void bm_add2(float2& sum, float a, float b, float top) {
  float2 d;
  asm("{\n\t.reg .b64 x, t, c;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 t, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "add.rn.f32x2 x, x, t;\n\tmul.rn.f32x2 x, x, c;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a), "f"(b), "f"(-top), "f"(kBmLog2e));
  d.x = bm_ex2(d.x);
  d.y = bm_ex2(d.y);
  asm("{\n\t.reg .b64 s, x;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 x, {%2, %3};\n\tadd.rn.f32x2 s, s, x;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "+f"(sum.x), "+f"(sum.y) : "f"(d.x), "f"(d.y));
}

// One of a block's best by value and id: for fp32 the id is the key's low half.
__device__ __forceinline__ unsigned long long beam_key(float v, int id) { return (unsigned long long)order_of(v) << 32 | (unsigned)~id; }
__device__ __forceinline__ BeamCell beam_cell(unsigned long long key) {
  return BeamCell{value_of((uint32_t)(key >> 32)), (int)~(uint32_t)key};
}

// The k best of n cells that blocks left in memory, at most one a thread.
__device__ __forceinline__ void merge_cells(const BeamCell* cells, int n, int k, BestScratch& s, BeamCell* best) {
  const int tid = threadIdx.x;
  const float2 q = tid < n ? __ldcg(reinterpret_cast<const float2*>(cells + tid)) : make_float2(-INFINITY, 0.f);
  const float bound = block_bound(q.x, k, s);
  if (q.x >= bound && q.x > -INFINITY) s.key[atomicAdd(&s.n, 1)] = beam_key(q.x, __float_as_int(q.y));
  __syncthreads();
  block_rank<false>(k, s, [&](int rank, unsigned long long key, int) { best[rank] = beam_cell(key); });
  const int had = min(k, s.n);
  if (tid >= had && tid < k) best[tid] = BeamCell{-INFINITY, 0x7fffffff};
}

// True in the block that arrives last of `n`: what the others wrote before they arrived is visible to it.
__device__ __forceinline__ bool block_last(int* ticket, int n, int* s_last) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    *s_last = atomicAdd(ticket, 1) == n - 1;
    if (*s_last) *ticket = 0;                             // ready for the next call
  }
  __syncthreads();
  const bool last = *s_last;
  if (last) __threadfence();
  return last;
}

// A search's places [B]: the best of the B x B candidates that its rows left, EB a thread.
template <int EB, typename Rank>
__device__ __forceinline__ void pick_places(int B, BestScratch& s, int* s_pick, Rank rank_of) {
  double v[EB], mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < EB; ++i) {
    const int e = threadIdx.x + i * kBmThreads;
    v[i] = e < B * B ? rank_of(e) : (double)-INFINITY;
    mine = v[i] > mine ? v[i] : mine;
  }
  block_list(block_bound(mine, B, s), B, s, [&](double bound) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < EB; ++i) n += (int)(v[i] >= bound) & (int)(v[i] > -INFINITY);
    return n;
  }, [&](double bound) {
#pragma unroll
    for (int i = 0; i < EB; ++i)
      if (v[i] >= bound && v[i] > -INFINITY) {
        const int at = atomicAdd(&s.n, 1);
        if (at < kBmList) { s.key[at] = order_of(v[i]); s.id[at] = threadIdx.x + i * kBmThreads; }
      }
  });
  if (s.n <= kBmList) {
    block_rank<true>(B, s, [&](int rank, unsigned long long, int id) { s_pick[rank] = id; });
  } else {
    block_rounds<double>(B, s, [&](double last, int last_id, double& best, int& where) {
#pragma unroll
      for (int i = 0; i < EB; ++i) {
        const int id = threadIdx.x + i * kBmThreads;
        if ((v[i] < last || (v[i] == last && id > last_id)) && (v[i] > best || (v[i] == best && v[i] > -INFINITY && id < where))) { best = v[i]; where = id; }
      }
    }, [&](int rank, double, int id) { s_pick[rank] = id; });
  }
  __syncthreads();
}

// grid (n_chunks, G * B).  A block takes the sum of exponentials and the B best of a chunk; the last block of a row merges the
// row's; the last row of a search ranks the B x B candidates that are left.  Logits are read once; the batches of a tile whose
// values reach the bound are read again, out of L2.  Device time over 151,936 ids, logits not in L2: 4 rows 10.9 us, 64 (39 MB) 20.6,
// 208 of 16 searches (126 MB) with ranks by length 42.2: 3.0 TB/s.  Behind the last logit a call waits 10 to 12 us for what comes one after the other: bound,
// list and ranks of the last chunk, the row's merge and the search's, a few hundred clocks a barrier and a dozen for each
// instruction that is fetched for the first time.
template <int E, int NB>
__global__ void __launch_bounds__(kBmThreads, 4) beam_select_kernel(const BeamArgs a) {
  __shared__ BestScratch s;
  __shared__ double s_fac[kMaxBeams], s_lse[kMaxBeams], s_sum[8];
  __shared__ int s_pick[kMaxBeams], s_last;
  __shared__ float s_max[8], s_score[kMaxBeams];
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.B, V = a.V, g = r / B;
  pdl_wait();
  pdl_launch();
  const bool over = a.done && a.done[r];
  const float score = a.scores[r];
  const bool reads = !over && score > -INFINITY;          // a beam with candidates among its logits
  if (!reads && c > 0) return;
  if (reads) {
    const float* x = a.logits + (long)r * a.stride;
    const int lo = c * a.chunk, hi = min(V, lo + a.chunk);
    const bool vec = ((uintptr_t)x & 15) == 0;
    // values of batch b of a tile: this thread's, -inf behind the chunk's end
    auto load = [&](int from, float (&v)[E]) {
      const int n = hi - from;
      if (vec && n >= E * kBmThreads) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
          const float4 q = __ldg(reinterpret_cast<const float4*>(x + from + (tid + i / 4 * kBmThreads) * 4));
          v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
        }
      } else if (vec) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
          const int e = (tid + i / 4 * kBmThreads) * 4;
          if (e + 4 <= n) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(x + from + e));
            v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = e + j < n ? __ldg(x + from + e + j) : -INFINITY;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = tid + i * kBmThreads < n ? __ldg(x + from + tid + i * kBmThreads) : -INFINITY;
      }
    };
    auto id_of = [&](int from, int i) { return from + (vec ? (tid + (i >> 2) * kBmThreads) * 4 + (i & 3) : tid + i * kBmThreads); };
    float m = -INFINITY, sum = 0.f, carried = -INFINITY;  // of what this thread has seen; one of the best so far
    int carried_id = 0;
    for (int t0 = lo; t0 < hi; t0 += NB * E * kBmThreads) {
      float v[E], tops[NB], mine = carried;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        tops[b] = -INFINITY;
        if (NB > 1 && t0 + b * E * kBmThreads >= hi) continue;
        load(t0 + b * E * kBmThreads, v);
        float top = fmaxf(v[0], v[1]);
#pragma unroll
        for (int i = 2; i < E; i += 2) top = fmaxf(top, fmaxf(v[i], v[i + 1]));
        const float seen = fmaxf(top, m);
        if (seen > -INFINITY) {                           // NaN and +inf end up as a NaN of the sum
          float2 more = make_float2(sum * bm_ex2((m - seen) * kBmLog2e), 0.f);
#pragma unroll
          for (int i = 0; i < E; i += 2) bm_add2(more, v[i], v[i + 1], seen);
          sum = more.x + more.y;
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) sum += v[i] == -INFINITY ? 0.f : v[i];
        }
        m = seen;
        tops[b] = top;
        mine = fmaxf(mine, top);
      }
      // few pass: a batch that is no longer in registers is read again, and so are the values, so that registers need no index
      block_list(block_bound(mine, B, s), B, s, [&](float bound) {
        int n = (int)(carried >= bound) & (int)(carried > -INFINITY);
#pragma unroll 1
        for (int b = 0; b < NB; ++b) {
          load(t0 + b * E * kBmThreads, v);
#pragma unroll
          for (int i = 0; i < E; ++i) n += (int)(v[i] >= bound) & (int)(v[i] > -INFINITY);
        }
        return n;
      }, [&](float bound) {
        auto batch = [&](int from) {
          const float least = fmaxf(bound, -FLT_MAX);     // an id with a logit of -inf is none
          uint32_t pass = 0;
#pragma unroll
          for (int i = 0; i < E; ++i) pass |= v[i] >= least ? 1u << i : 0u;
          while (pass) {
            const int id = id_of(from, __ffs(pass) - 1), at = atomicAdd(&s.n, 1);
            pass &= pass - 1;
            if (at < kBmList) s.key[at] = beam_key(__ldg(x + id), id);
          }
        };
        if constexpr (NB == 1) {
          batch(t0);
        } else {
          uint32_t want = 0;
#pragma unroll
          for (int b = 0; b < NB; ++b) want |= (uint32_t)(tops[b] >= bound && tops[b] > -INFINITY) << b;
          while (want) {
            const int from = t0 + (__ffs(want) - 1) * E * kBmThreads;
            want &= want - 1;
            load(from, v);
            batch(from);
          }
        }
        if (carried >= bound && carried > -INFINITY) {
          const int at = atomicAdd(&s.n, 1);
          if (at < kBmList) s.key[at] = beam_key(carried, carried_id);
        }
      });
      BeamCell* out = a.cells + ((long)r * a.n_chunks + c) * B;
      if (s.n <= kBmList) {
        block_rank<false>(B, s, [&](int rank, unsigned long long key, int) { out[rank] = beam_cell(key); });
      } else {
        block_rounds<float>(B, s, [&](float last, int last_id, float& best, int& where) {
          auto offer = [&](float u, int id) {
            if ((u < last || (u == last && id > last_id)) && (u > best || (u == best && u > -INFINITY && id < where))) { best = u; where = id; }
          };
#pragma unroll 1
          for (int b = 0; b < NB; ++b) {
            load(t0 + b * E * kBmThreads, v);
#pragma unroll
            for (int i = 0; i < E; ++i) offer(v[i], id_of(t0 + b * E * kBmThreads, i));
          }
          offer(carried, carried_id);
        }, [&](int rank, float value, int id) { out[rank] = BeamCell{value, id}; });
      }
      const int had = min(B, s.n);
      if (tid >= had && tid < B) out[tid] = BeamCell{-INFINITY, 0x7fffffff};
      if (t0 + NB * E * kBmThreads < hi) {                // the best so far take part in the next tile's choice
        __syncthreads();
        carried = -INFINITY;
        if (tid < had) { carried = out[tid].value; carried_id = out[tid].id; }
        __syncthreads();
      }
    }
    // the block's sum
    float all = warp_max(m);
    if (lane == 0) s_max[warp] = all;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) all = fmaxf(all, s_max[w]);
    const double part = warp_sum_d(m > -INFINITY ? (double)(sum * __expf(m - all)) : (double)sum);
    if (lane == 0) s_sum[warp] = part;
    __syncthreads();
    if (tid == 0) {
      double l = 0.0;
      for (int w = 0; w < 8; ++w) l += s_sum[w];
      a.sums[(long)r * a.n_chunks + c] = make_float2(all, (float)l);
    }
    if (!block_last(a.tickets + r, a.n_chunks, &s_last)) return;
    // ---- the row: the best of its chunks' best, and its log-sum
    const float2* sums = a.sums + (long)r * a.n_chunks;
    const float2 first = tid < a.n_chunks ? __ldcg(sums + tid) : make_float2(-INFINITY, 0.f);
    const BeamCell* cells = a.cells + (long)r * a.n_chunks * B;
    merge_cells(cells, a.n_chunks * B, B, s, a.best + (long)r * B);
    float top = warp_max(first.x);
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_max[w]);
    auto weighed = [&](float2 q) { return q.x > -INFINITY ? (double)q.y * (double)__expf(q.x - top) : (double)q.y; };
    const double l = warp_sum_d(weighed(first));
    if (lane == 0) s_sum[warp] = l;
    __syncthreads();
    if (tid == 0) {
      double total = 0.0;
      for (int w = 0; w < 8; ++w) total += s_sum[w];
      a.lse[r] = (double)top + log(total);                // -inf where every id is masked; NaN where a logit is not finite
    }
  }
  if (!block_last(a.tickets + a.G * B + g, B, &s_last)) return;
  // ---- the search
  const int r0 = g * B;
  bool bad = false;
  if (tid < B) {
    const int q = r0 + tid;
    const bool ended = a.done && a.done[q];
    const float sc = a.scores[q];
    const double lse = __ldcg(a.lse + q);
    s_score[tid] = sc;
    s_lse[tid] = sc == -INFINITY || ended ? 0.0 : lse;
    bad = !(sc < INFINITY) || s_lse[tid] != s_lse[tid];
    s_fac[tid] = a.alpha != 0.f ? pow((double)max(1, a.lengths[q] + (ended ? 0 : 1)), -(double)a.alpha) : 1.0;
    s_pick[tid] = -1;
  }
  bad = __syncthreads_or(bad);
  auto cand = [&](int b, float value) { return (double)s_score[b] + ((double)value - s_lse[b]); };
  // within a beam the places are in order of logit and id, so that of equal ranks the lower place comes first
  auto rank_of = [&](int e) {
    const int b = e / B, j = e - b * B;
    const float value = __ldcg(&a.best[(long)(r0 + b) * B + j].value);           // read in any case: nothing waits for the tests
    double rank = -INFINITY;
    if (!bad && s_score[b] > -INFINITY) {
      if (a.done && a.done[r0 + b]) rank = j == 0 ? (double)s_score[b] * s_fac[b] : -INFINITY;
      else if (value > -INFINITY) rank = cand(b, value) * s_fac[b];
    }
    return rank;
  };
  if (B * B <= kBmThreads) pick_places<1>(B, s, s_pick, rank_of);
  else pick_places<kMaxBeams * kMaxBeams / kBmThreads>(B, s, s_pick, rank_of);
  if (tid < B) {
    const int e = s_pick[tid], b = e < 0 ? tid : e / B, q = r0 + b;
    const bool ended = a.done && a.done[q];
    BeamCell cell{0.f, max(a.eos, 0)};
    if (e >= 0 && !ended) {
      const float2 got = __ldcg(reinterpret_cast<const float2*>(a.best + (long)q * B + (e - b * B)));
      cell = BeamCell{got.x, __float_as_int(got.y)};
    }
    a.parent[r0 + tid] = b;
    a.token[r0 + tid] = cell.id;
    a.out_scores[r0 + tid] = bad ? __int_as_float(0x7fc00000) : e < 0 ? -INFINITY : ended ? s_score[b] : (float)cand(b, cell.value);
    if (a.out_done) a.out_done[r0 + tid] = e < 0 || ended || cell.id == a.eos;
    if (a.out_lengths) a.out_lengths[r0 + tid] = a.lengths[q] + (e < 0 || ended ? 0 : 1);
  }
  if (bad && tid == 0) raise_fault(a.fault, 0, FS_SAMPLER);
}

// ---- states -----------------------------------------------------------------------------------------------
struct ReorderArgs {
  uint8_t* k; uint8_t* v;
  long k_row, v_row;                                      // bytes of a position of one head; 0: no such pool
  int n_pages, n_kv, G, B, n_slots, max_pages;
  const int* table; int* table_out;
  const int* slots; const int* parent; const int* held;
  unsigned* fault;
};

constexpr int kBeamPage = 64;

// The first `n` bytes of every head's block of a page: all heads at once, eight loads of a thread in flight.
__device__ __forceinline__ void copy_heads(uint8_t* dst, const uint8_t* src, int n, int pitch, int heads) {
  constexpr int AHEAD = 8;
  const unsigned words = (unsigned)n >> 4, total = words * heads;
  for (unsigned i0 = threadIdx.x; i0 < total; i0 += AHEAD * blockDim.x) {
    uint4 v[AHEAD];
    unsigned at[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const unsigned i = i0 + u * blockDim.x, h = i / words;
      at[u] = h * pitch + (i - h * words) * 16;
      if (i < total) v[u] = *reinterpret_cast<const uint4*>(src + at[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (i0 + u * blockDim.x < total) *reinterpret_cast<uint4*>(dst + at[u]) = v[u];
  }
  const int rest = (n & 15) >> 2;                         // rows that are no multiple of 16 bytes (q8_0) may leave some words
  for (int i = threadIdx.x; i < rest * heads; i += blockDim.x) {
    const int at = i / rest * pitch + (n & ~15) + i % rest * 4;
    *reinterpret_cast<uint32_t*>(dst + at) = *reinterpret_cast<const uint32_t*>(src + at);
  }
}

// grid (G * B, layers), 256 threads: a block moves what one child takes in one layer.  All reads and writes of 8 searches of 8 (half
// of the beams moved, 302 MB): 54 us, 5.6 TB/s; with four blocks a processor instead of two and the registers that this leaves, 65.
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderArgs a) {
  __shared__ int s_parent[kMaxBeams];
  __shared__ unsigned s_more[2], s_bare[2];               // children behind their parent's first; beams without a child
  const int g = blockIdx.x / a.B, i = blockIdx.x % a.B, layer = blockIdx.y, tid = threadIdx.x, r0 = g * a.B;
  pdl_wait();
  pdl_launch();
  bool bad = false;
  if (tid < a.B) {
    const int p = a.parent[r0 + tid], s = a.slots[r0 + tid];
    s_parent[tid] = p;
    bad = p < 0 || p >= a.B || s < 0 || s >= a.n_slots;
  }
  const int held = a.held[g];
  bad = __syncthreads_or(bad) || held < 0 || held > a.max_pages * kBeamPage;
  const int col = held / kBeamPage, part = held % kBeamPage;
  if (tid < kMaxBeams) {
    bool more = false, bare = tid < a.B;
    if (tid < a.B)
      for (int j = 0; j < a.B; ++j) {
        more |= j < tid && s_parent[j] == s_parent[tid];
        bare &= s_parent[j] != tid;
      }
    const unsigned m = __ballot_sync(0xffffffffu, more), b = __ballot_sync(0xffffffffu, bare);
    if ((tid & 31) == 0) { s_more[tid >> 5] = m; s_bare[tid >> 5] = b; }
  }
  __syncthreads();
  const int slot = a.slots[r0 + i];
  if (slot < 0 || slot >= a.n_slots) { if (tid == 0) raise_fault(a.fault, layer, FS_BEAM); return; }
  const int* own = a.table + (long)slot * a.max_pages;
  const int* from = own;
  int place = -1, source = -1;                            // the page being filled, and what is copied into it
  bool copies = false, lost = false;                      // takes another page over; a page that the pools do not have
  if (bad) {                                              // nobody moves
    if (tid == 0) raise_fault(a.fault, layer, FS_BEAM);
  } else {
    from = a.table + (long)a.slots[r0 + s_parent[i]] * a.max_pages;
    if (part) {
      const unsigned long long more = s_more[0] | (unsigned long long)s_more[1] << 32;
      unsigned long long bare = s_bare[0] | (unsigned long long)s_bare[1] << 32;
      place = from[col];
      copies = more >> i & 1;
      if (copies) {
        for (int n = __popcll(more & ((1ull << i) - 1)); n > 0; --n) bare &= bare - 1;
        source = place;
        place = a.table[(long)a.slots[r0 + __ffsll((long long)bare) - 1] * a.max_pages + col];
      }
      // a beam that goes on in its own slot changes nothing here, pages or not (a place without a beam)
      lost = (copies || s_parent[i] != i) && (place < 0 || place >= a.n_pages || (copies && (source < 0 || source >= a.n_pages)));
      if (lost && tid == 0) raise_fault(a.fault, layer, FS_PAGE);
    }
  }
  if (layer == 0) {                                       // a child whose history is not there keeps its slot's row
    int* to = a.table_out + (long)slot * a.max_pages;
    for (int c = tid; c < a.max_pages; c += 256) to[c] = bad || lost || c > col ? own[c] : c < col ? from[c] : part ? place : own[c];
  }
  if (!copies || lost) return;
  const long src = ((long)layer * a.n_pages + source) * a.n_kv * kBeamPage, dst = ((long)layer * a.n_pages + place) * a.n_kv * kBeamPage;
  copy_heads(a.k + dst * a.k_row, a.k + src * a.k_row, part * (int)a.k_row, kBeamPage * (int)a.k_row, a.n_kv);
  if (a.v_row) copy_heads(a.v + dst * a.v_row, a.v + src * a.v_row, part * (int)a.v_row, kBeamPage * (int)a.v_row, a.n_kv);
}

// ---- the next pass ------------------------------------------------------------------------------------------
struct BeamAdvanceArgs {
  int* tokens; int* row_pos; int* row_seq; int* held; int* hist; int* count;
  const int* slots; const int* parent; const int* token; const int* done; const float* scores;
  int G, B, cap;
};

// One block: the rows of the next pass, and the choice written down.  A finished or missing beam is a row without a sequence.
__global__ void __launch_bounds__(256) beam_advance_kernel(const BeamAdvanceArgs a) {
  pdl_wait();
  pdl_launch();
  const int R = a.G * a.B, step = *a.count;
  for (int i = threadIdx.x; i < R; i += blockDim.x) {
    a.tokens[i] = a.token[i];
    a.row_pos[i] += 1;
    a.row_seq[i] = a.done[i] || a.scores[i] == -INFINITY ? -1 : a.slots[i];
    if (step < a.cap) {
      a.hist[(long)step * 2 * R + i] = a.parent[i];
      a.hist[((long)step * 2 + 1) * R + i] = a.token[i];
    }
  }
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) a.held[g] += 1;
  __syncthreads();
  if (threadIdx.x == 0) *a.count = step + 1;
}

}  // namespace bl

using namespace bl;

extern "C" {

// Chunks of a row: as many as one wave of four blocks a processor holds, of 4,096 values or more, and no more than a block merges
// with one cell a thread.  Device time on 148 processors at 151,936 ids that are not in L2, us: 4 rows of 4 beams, 16 chunks 13.2, 38
// (the rule) 10.9; 64 rows of 8, 4 chunks 21.8, 9 (the rule) 20.6, 10 (a second wave) 22.8, 16 25.8; 256 rows of 16, 1 chunk 48.5, 2
// (the rule) 44.2, 3 49.1; 64 rows of 64, 2 chunks 57.2, 4 (the rule, 256 cells) 50.5.
int bl_beam_chunks(int V, int rows, int B, int sms) {
  const int most = (V + 4095) / 4096, wave = 4 * sms / rows, cells = kBmMaxCells / B;
  int n = most < wave ? most : wave;
  if (n > cells) n = cells;
  return n > 1 ? n : 1;
}
static int beam_chunk(int V, int n) { return ((V + n - 1) / n + 3) / 4 * 4; }

// Bytes of scratch that bl_beam_select takes; zeroed once.
long bl_beam_work_bytes(int G, int B, int n) {
  const long R = (long)G * B;
  return R * 8 + R * n * 8 + R * n * B * 8 + R * B * 8 + (R + G) * 4;
}

// Calls as one block of memory each: a host that makes one a step hands over a pointer instead of two dozen arguments.
struct BeamSelectCall {
  const float* logits; long stride; const float* scores; const int* done; const int* lengths; void* work;
  int* parent; int* token; float* out_scores; int* out_done; int* out_lengths; unsigned* fault; cudaStream_t stream;
  int V, G, B, eos, chunks; float alpha;                    // chunks: as bl_beam_chunks says
};
struct BeamReorderCall {
  void* k; void* v; long k_row, v_row; const int* table; int* table_out; const int* slots; const int* parent; const int* held;
  unsigned* fault; cudaStream_t stream;
  int n_layer, n_pages, n_kv, n_slots, max_pages, G, B;
};

int bl_beam_select(const BeamSelectCall* call) {
  const auto [logits, stride, scores, done, lengths, work, parent, token, out_scores, out_done, out_lengths, fault, st, V, G, B, eos, chunks, alpha] = *call;
  BL_REQUIRE(V >= 1 && G >= 1 && B >= 1 && stride >= V && chunks >= 1 && chunks <= V, BL_ERR_SHAPE);
  BL_REQUIRE(B <= kMaxBeams && (long)G * B <= 65535 && (long)chunks * B <= kBmMaxCells, BL_ERR_LIMIT);
  BL_REQUIRE(alpha >= -kMaxAlpha && alpha <= kMaxAlpha, BL_ERR_SHAPE);           // ranks without an order otherwise: NaN, or all zero
  BL_REQUIRE(eos < V && (!done || eos >= 0) && (alpha == 0.f || lengths) && (!out_lengths || lengths), BL_ERR_SHAPE);
  BL_REQUIRE(((uintptr_t)logits & 3) == 0 && ((uintptr_t)work & 7) == 0, BL_ERR_ALIGN);
  // Outputs lie apart from what is read.  Blocks of a search that has been written may still be to start: one that found another
  // flag in `done` than its row had would take a ticket that nobody counts, and every later call with this scratch would be off.
  const void* const out[5] = {parent, token, out_scores, out_done, out_lengths};
  const void* const in[4] = {scores, done, lengths, logits};
  const size_t cell = (size_t)G * B * 4, rows = (((size_t)G * B - 1) * stride + V) * 4;
  auto apart = [](const void* p, size_t n, const void* q, size_t m) {
    return !p || !q || (uintptr_t)p + n <= (uintptr_t)q || (uintptr_t)q + m <= (uintptr_t)p;
  };
  for (int i = 0; i < 5; ++i) {
    for (int j = 0; j < 4; ++j) BL_REQUIRE(apart(out[i], cell, in[j], j == 3 ? rows : cell), BL_ERR_SHAPE);
    for (int j = 0; j < i; ++j) BL_REQUIRE(apart(out[i], cell, out[j], cell), BL_ERR_SHAPE);
  }
  BeamArgs a{logits, stride, V, G, B, scores, done, lengths, eos, alpha};
  a.chunk = beam_chunk(V, chunks);
  a.n_chunks = (V + a.chunk - 1) / a.chunk;
  const long R = (long)G * B;
  uint8_t* w = (uint8_t*)work;
  a.lse = (double*)w; w += R * 8;
  a.sums = (float2*)w; w += R * a.n_chunks * 8;
  a.cells = (BeamCell*)w; w += R * a.n_chunks * B * 8;
  a.best = (BeamCell*)w; w += R * B * 8;
  a.tickets = (int*)w;
  a.parent = parent; a.token = token; a.out_scores = out_scores; a.out_done = out_done; a.out_lengths = out_lengths; a.fault = fault;
  const dim3 grid(a.n_chunks, (unsigned)R);
  // A short chunk whole in registers, 4 rows of 151,936 in 38 chunks: 10.9 us, 11.8 as a part of the largest tile.  In two batches, 128
  // rows of 32,000 in 4 chunks: 16.1 us against 16.8.
  if (a.chunk <= 4096) return (int)launch(beam_select_kernel<16, 1>, grid, dim3(kBmThreads), 0, st, a);
  if (a.chunk <= 8192) return (int)launch(beam_select_kernel<16, 2>, grid, dim3(kBmThreads), 0, st, a);
  return (int)launch(beam_select_kernel<32, 4>, grid, dim3(kBmThreads), 0, st, a);
}

int bl_beam_reorder(const BeamReorderCall* call) {
  const auto [k, v, k_row, v_row, table, table_out, slots, parent, held, fault, st, n_layer, n_pages, n_kv, n_slots, max_pages, G, B] = *call;
  BL_REQUIRE(n_layer >= 1 && n_layer <= 65535 && n_pages >= 1 && n_kv >= 1 && G >= 1 && B >= 1 && n_slots >= 1 && max_pages >= 1,
             BL_ERR_SHAPE);
  BL_REQUIRE(B <= kMaxBeams, BL_ERR_LIMIT);
  BL_REQUIRE(k_row >= 4 && v_row >= 0 && table != table_out, BL_ERR_SHAPE);
  BL_REQUIRE((long)n_kv * kBeamPage * (k_row > v_row ? k_row : v_row) <= 0x7fffffffL, BL_ERR_LIMIT);
  BL_REQUIRE(k_row % 4 == 0 && v_row % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, BL_ERR_ALIGN);
  ReorderArgs a{(uint8_t*)k, (uint8_t*)v, k_row, v_row, n_pages, n_kv, G, B, n_slots, max_pages, table, table_out, slots, parent, held, fault};
  return (int)launch(beam_reorder_kernel, dim3(G * B, n_layer), dim3(256), 0, st, a);
}

// tokens, row_pos, row_seq [G * B] of a pass; held [G]; hist [cap][2][G * B] parents and tokens of each step, count its number.
int bl_beam_advance(int* tokens, int* row_pos, int* row_seq, int* held, int* hist, int cap, int* count, const int* slots, const int* parent,
                    const int* token, const int* done, const float* scores, int G, int B, cudaStream_t st) {
  BL_REQUIRE(G >= 1 && B >= 1 && cap >= 0 && (long)G * B <= 65535, BL_ERR_SHAPE);
  BeamAdvanceArgs a{tokens, row_pos, row_seq, held, hist, count, slots, parent, token, done, scores, G, B, cap};
  return (int)launch(beam_advance_kernel, dim3(1), dim3(256), 0, st, a);
}

}  // extern "C"
