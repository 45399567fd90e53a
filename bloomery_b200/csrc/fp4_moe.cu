// The routed experts of a few tokens in NVFP4 and two launches (sm_100a):
//   a[t, j] = silu(x_t Wg[e]) * (x_t Wu[e])        e = ids[t, j], x_t the token's row (behind an RMSNorm) in NVFP4
//   y[t]    = resid[t] + sum_j wts[t, j] (a[t, j] in NVFP4) Wd[e]
//
// A round of decoding hits most experts with a handful of tokens each, so what bounds it is one pass over the weights of the experts
// that are hit, and what costs beside that are the launches between: plan, gather, two quantisers, two products, combine.  Here
//   * every CTA makes the plan itself, out of the ids: at most 1,024 of them;
//   * gate and up multiply all tokens of the round with every expert that is hit: the tokens are the N side of the MMA and 32 or 64 of them
//     cost nothing beside the weights' way from memory, so nothing is sorted or gathered; the epilogue keeps the columns of the
//     expert's own tokens;
//   * the tokens' rows are quantised by the CTAs that come first, a row at a time, while the ring fills with weights;
//   * the CTA that finishes an expert's last tile quantises its rows for the second launch, which reads them as they lie,
//     expert by expert;
//   * in the second launch the CTA that finishes the last tile of 128 output columns adds up the slots of every token, in order.
// CTAs walk tiles next to each other, so that one takes part in two or three experts, or column blocks, and says so once for each.
// One token or two (FM_FEW): each CTA quantises the rows that it needs for itself, which is quicker than to wait for another one's.  Rows of
// each CTA's own / one form for all, us, eight experts a token: 30B shape 1 token 18.8 / 21.1, 2 tokens 23.3 / 23.5, 3 tokens 28.6 / 27.7; 235B
// shape 32.1 / 35.3, 57.8 / 60.3, 71.2 / 70.3; 32 experts of 2,048 x 7,168 57.5 / 61.5, 90.9 / 89.2, 140.5 / 128.9; 4 tokens on the 30B
// shape 36.5 / 32.9.
// Rows are claimed and finished by whoever is there, so no CTA waits for one that has not started; the one wait between CTAs (for the tokens'
// rows) is bounded like all others.  Sums of a slot run in one order: the same bits on every run and with every number of CTAs.
// 24 tokens on the 30B shape (258 MB of weights): 66.8 us, 3.9 TB/s, 0.59 of the copy rate; 64 tokens on the 235B shape (1.38 GB): 284 to 300 us,
// 4.6 to 4.9 TB/s under the power cap; one token 18.9 us, latency.  The plan and first rows stand in front of the weights' stream, the last tickets
// behind it.
#include <type_traits>

#include "fp4_pipe.cuh"

namespace bl {

constexpr int FM_TOKENS = 64, FM_SLOTS = 1024, FM_EXPERTS = 512, FM_WIDTH = 8192;
constexpr int FM_USED = 16;                         // experts of a token
constexpr int FM_FEW = 2, FM_FEW_SLOTS = 32;        // tokens of a round whose CTAs quantise for themselves, and slots that one warp plans
static_assert(FM_FEW * FM_USED <= FM_FEW_SLOTS, "the few-token plan has room for every slot");
constexpr int FM_THREADS = F4_EPILOGUE + 128;

struct FmArgs {
  const void* x; long ldx; int x_type;              // 0 bf16, 2 fp32
  const float* gain; double eps;
  const int* ids; const float* wts;
  int T, k, E, H, I;
  const uint8_t* wg; const uint8_t* wu; const uint8_t* wd;
  uint8_t* xq;                                      // [T] NVFP4 rows of H; few tokens: as many for each CTA
  float* act;                                       // [T * k][I], expert by expert
  uint8_t* aq;                                      // the same as NVFP4 rows; few tokens: as many for each CTA
  float* slot_out;                                  // [T * k][H]
  int* claim;                                       // rows taken, rows done, then a ticket for every expert and every block of columns
  const float* resid; long ldr;
  float* c_f32; __nv_bfloat16* c_bf16; long ldc;
  unsigned* status;
};

// Which experts are hit and by which slots: entries of one expert each, at most `most` slots in one.
template <int SLOTS, int ENTRIES>
struct FmPlan {
  int n_entries;
  struct Entry { short expert, rows; int first; } entry[ENTRIES];
  short id[SLOTS];                                  // of every slot, -1: none of ours
  short slot[SLOTS];                                // expert by expert
};
using FmFewPlan = FmPlan<FM_FEW_SLOTS, FM_FEW_SLOTS>;
using FmFullPlan = FmPlan<FM_SLOTS, FM_EXPERTS + FM_SLOTS / 32>;

// The plan is made by the warps in front of the epilogue's, which meanwhile quantise tokens and come to it later.
__device__ __forceinline__ void fm_plan_step() { asm volatile("bar.sync 2, %0;" ::"n"(F4_EPILOGUE) : "memory"); }
__device__ __forceinline__ void fm_plan_made() { asm volatile("bar.arrive 3, %0;" ::"n"(FM_THREADS) : "memory"); }
__device__ __forceinline__ void fm_plan_wait() { asm volatile("bar.sync 3, %0;" ::"n"(FM_THREADS) : "memory"); }

// Up to 32 slots, by one warp: experts in the order in which they appear.
__device__ __forceinline__ void fm_plan(FmFewPlan& p, const FmArgs& a, int, void*) {
  const int tid = threadIdx.x, n = a.T * a.k;
  if (tid < 32) {
    int e = tid < n ? a.ids[tid] : -1;
    if (e >= a.E || e < 0) e = -1;
    const unsigned same = __match_any_sync(0xffffffffu, e), below = (1u << tid) - 1;
    const bool leads = e >= 0 && (same & below) == 0;
    const unsigned leaders = __ballot_sync(0xffffffffu, leads);
    const int rows = leads ? __popc(same) : 0;
    int before = rows;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int r = __shfl_up_sync(0xffffffffu, before, d);
      if (tid >= d) before += r;
    }
    before -= rows;                                 // a leader's: slots of the experts in front of its own
    const int first = __shfl_sync(0xffffffffu, before, __ffs(same) - 1);
    if (tid < n) p.id[tid] = (short)e;
    if (leads) p.entry[__popc(leaders & below)] = FmFewPlan::Entry{(short)e, (short)rows, first};
    if (e >= 0) p.slot[first + __popc(same & below)] = (short)tid;
    if (tid == 0) p.n_entries = __popc(leaders);
  }
  fm_plan_step();
}

// Any number: a warp counts the experts of its own slots (a seventh of them, next to each other), so that a slot's place among those of its
// expert is the same in every CTA.  `scratch`: FM_EXPERTS * 9 shorts that TMA writes later.
__device__ __forceinline__ void fm_plan(FmFullPlan& p, const FmArgs& a, int most, void* scratch) {
  constexpr int W = F4_EPILOGUE / 32, PER = (FM_SLOTS + 32 * W - 1) / (32 * W);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, n = a.T * a.k;
  short* count = reinterpret_cast<short*>(scratch);                // [W][FM_EXPERTS], then what lies in front of a warp's slots
  short *all = count + W * FM_EXPERTS, *first = all + FM_EXPERTS;
  const int mine = (n + W - 1) / W, lo = min(n, w * mine), hi = min(n, lo + mine);
  int id[PER], place[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = lo + 32 * i + lane;
    id[i] = s < hi ? a.ids[s] : -1;
  }
  for (int i = tid; i < W * FM_EXPERTS / 2; i += F4_EPILOGUE) reinterpret_cast<int*>(count)[i] = 0;
  fm_plan_step();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = lo + 32 * i + lane;
    if (lo + 32 * i >= hi) break;
    if (id[i] < 0 || id[i] >= a.E) id[i] = -1;
    const unsigned same = __match_any_sync(0xffffffffu, id[i]), before = same & ((1u << lane) - 1);
    short* c = count + w * FM_EXPERTS + (id[i] >= 0 ? id[i] : 0);
    if (id[i] >= 0) place[i] = *c + __popc(before);
    __syncwarp();
    if (id[i] >= 0 && before == 0) *c += (short)__popc(same);
    __syncwarp();
    if (s < hi) p.id[s] = (short)id[i];
  }
  fm_plan_step();
  for (int e = tid; e < a.E; e += F4_EPILOGUE) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) { const int c = count[i * FM_EXPERTS + e]; count[i * FM_EXPERTS + e] = (short)sum; sum += c; }
    all[e] = (short)sum;
  }
  fm_plan_step();
  if (w == 0) {
    const int per = (a.E + 31) / 32, e0 = min(a.E, lane * per), e1 = min(a.E, e0 + per);
    int rows = 0, entries = 0;
    for (int e = e0; e < e1; ++e) { rows += all[e]; entries += (all[e] + most - 1) / most; }
    int both = rows | entries << 16, sum = both;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int r = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += r;
    }
    if (lane == 31) p.n_entries = sum >> 16;
    sum -= both;
    int ro = sum & 0xffff, en = sum >> 16;
    for (int e = e0; e < e1; ++e) {
      const int c = all[e];
      first[e] = (short)ro;
      for (int r = 0; r < c; r += most) p.entry[en++] = FmFullPlan::Entry{(short)e, (short)min(most, c - r), ro + r};
      ro += c;
    }
  }
  fm_plan_step();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lo + 32 * i + lane < hi && id[i] >= 0) p.slot[first[id[i]] + count[w * FM_EXPERTS + id[i]] + place[i]] = (short)(lo + 32 * i + lane);
  asm volatile("fence.proxy.async;" ::: "memory");                 // the scratch is a ring's from here on
  fm_plan_step();
}

// A CTA's share of n tiles: next to each other.
struct FmShare {
  int lo, hi;
  __device__ __forceinline__ explicit FmShare(int n) : lo((int)((long)n * blockIdx.x / gridDim.x)), hi((int)((long)n * (blockIdx.x + 1) / gridDim.x)) {}
  __device__ __forceinline__ int count() const { return hi - lo; }
};
template <class Plan, int AR>
struct FmUpTiles : FmShare {                        // expert by expert
  const Plan& p;
  int tiles_w, kblocks, row0, T;
  __device__ __forceinline__ FmUpTiles(const Plan& p, int I, int H, int row0, int T)
      : FmShare(p.n_entries * ((I + AR - 1) / AR)), p(p), tiles_w((I + AR - 1) / AR), kblocks((H + 255) / 256), row0(row0), T(T) {}
  __device__ __forceinline__ int entry(int i) const { return (lo + i) / tiles_w; }
  __device__ __forceinline__ F4Work at(int i) const {
    return F4Work{p.entry[entry(i)].expert, (lo + i) % tiles_w * AR, row0, T, 0, kblocks};      // all tokens
  }
};
template <class Plan, int AR>
struct FmDownTiles : FmShare {                      // columns after columns
  const Plan& p;
  int kblocks, row0;
  __device__ __forceinline__ FmDownTiles(const Plan& p, int H, int I, int row0)
      : FmShare(p.n_entries * ((H + AR - 1) / AR)), p(p), kblocks((I + 255) / 256), row0(row0) {}
  __device__ __forceinline__ typename Plan::Entry entry(int i) const { return p.entry[(lo + i) % p.n_entries]; }
  __device__ __forceinline__ F4Work at(int i) const {
    const typename Plan::Entry e = entry(i);
    return F4Work{e.expert, (lo + i) / p.n_entries * AR, row0 + e.first, e.rows, 0, kblocks};
  }
};

// A token's row in NVFP4, by the 128 threads of the epilogue warps.  It is run once or twice by a CTA: what counts is little code, which is
// fetched as it runs, so a thread walks its blocks of 16 three times instead of keeping them.  s_sum and s_max are read behind its last
// meeting: the threads meet once more before another row.
__device__ __forceinline__ void fm_token(const FmArgs& a, int t, uint8_t* row, double* s_sum, unsigned* s_max) {
  const int et = threadIdx.x - F4_EPILOGUE, lane = et & 31, w = et >> 5, blocks = a.H / 16;
  float v[16], r = 1.0f;
  auto load = [&](int b) { fp4_load16(a.x, a.x_type, (long)t * a.ldx + 16 * b, v); };
  if (a.gain) {
    auto whole = [&](double ss) {
      ss = warp_sum_d(ss);
      if (lane == 0) s_sum[w] = ss;
      f4_meet<4>();
      return s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    };
    double ss = 0.0;
#pragma unroll 1
    for (int b = et; b < blocks; b += 128) {
      load(b);
      ss += fp4_squares16(v);
    }
    double all = whole(ss);
    if (__builtin_expect(!fp4_sum_holds(all), 0)) {
      f4_meet<4>();
      ss = 0.0;
#pragma unroll 1
      for (int b = et; b < blocks; b += 128) {
        load(b);
        ss += fp4_squares16_wide(v);
      }
      all = whole(ss);
    }
    r = fp4_rsqrt(all / (double)a.H + a.eps);
  }
  unsigned top = 0;
#pragma unroll 1
  for (int b = et; b < blocks; b += 128) {
    if (blocks > 128 || !a.gain) load(b);             // else the one block is still there
    if (a.gain) fp4_scale16(v, r, a.gain + 16 * b);
    top = max(top, fp4_top<16>(v));
  }
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (lane == 0) s_max[w] = top;
  f4_meet<4>();
  const float g = fp4_row_scale(max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]))), inv6g = fp4_inv6(g);
#pragma unroll 1
  for (int b = et; b < blocks; b += 128) {
    if (blocks > 128) {
      load(b);
      if (a.gain) fp4_scale16(v, r, a.gain + 16 * b);
    }
    fp4_store_block(row, a.H, b, v, fp4_top<16>(v), g, inv6g);
  }
}
// The gain's way to this processor, before the launch in front of this one has ended.
__device__ __forceinline__ void fm_ask_gain(const FmArgs& a) {
  if (a.gain)
    for (int i = threadIdx.x * 32; i < a.H; i += FM_THREADS * 32) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.gain + i) : "memory");
}

// Rows first .. first + rows - 1 of the activations in NVFP4 in the rows of `to`: a block of 16 a thread, rows next to each other, up to
// 32 rows at a time (s_top).
__device__ __forceinline__ void fm_rows(const FmArgs& a, int first, int rows, uint8_t* to, unsigned* s_top) {
  const int et = threadIdx.x - F4_EPILOGUE, per = a.I / 16;
  for (int r0 = 0; r0 < rows; r0 += 32) {
    const int n = min(32, rows - r0) * per;
    if (et < 32) s_top[et] = 0;
    f4_meet<4>();
    const float4* x = reinterpret_cast<const float4*>(a.act + (long)(first + r0) * a.I);
    auto load = [&](int b, float* v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = x[4 * (long)b + i];
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      }
    };
#pragma unroll 1
    for (int b = et; b < n; b += 512) {
      float v[4][16];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b + 128 * j < n) load(b + 128 * j, v[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b + 128 * j < n) atomicMax(&s_top[(b + 128 * j) / per], fp4_top<16>(v[j]));
    }
    f4_meet<4>();
#pragma unroll 1
    for (int b = et; b < n; b += 128) {
      float v[16];
      load(b, v);                                     // from the first cache, mostly
      const float g = fp4_row_scale(s_top[b / per]);
      fp4_store_block(to + (first + r0 + b / per) * fp4_row_bytes(a.I), a.I, b % per, v, fp4_top<16>(v), g, fp4_inv6(g));
    }
    f4_meet<4>();
  }
}

// Rows that this CTA stores and reads by TMA itself, by an mbarrier that each of the 128 storing threads arrives at.
__device__ __forceinline__ void fm_rows_stored(uint64_t* bar) {
  asm volatile("fence.proxy.async;" ::: "memory");
  mbar_arrive(bar);
}

// The tokens' rows that other CTAs store, read by TMA: whether all are there; gives up after the limit of all waits.
__device__ __forceinline__ bool fm_tokens_ready(const FmArgs& a, volatile int* abort_flag) {
  unsigned long long t0 = 0;
  for (uint32_t it = 0;; ++it) {
    int done;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(done) : "l"(a.claim + 1) : "memory");
    if (done >= a.T) break;
    if ((it & 63) == 63) {                          // the timer takes longer than a look at the word
      const unsigned long long now = globaltimer();
      if (t0 == 0) t0 = now;
      else if (now - t0 > WAIT_LIMIT_NS) { *abort_flag = 1; return false; }
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");
  return true;
}

// Whether this CTA's `done` parts of `all` were the last; by the 128 threads, whose stores the others see then.
__device__ __forceinline__ bool fm_last(int* ticket, int done, int all, int* s_word) {
  __threadfence();
  f4_meet<4>();
  if (threadIdx.x == F4_EPILOGUE) {
    const int last = atomicAdd(ticket, done) + done == all;
    if (last) *ticket = 0;                          // ready for the next call
    __threadfence();
    *s_word = last;
  }
  f4_meet<4>();
  return *s_word != 0;
}

template <int BN, int AR, bool FEW>
struct FmShapes {
  using Up = F4Shape<true, BN, 208 * 1024, 4, AR, FEW ? 6 : BN == 32 ? 3 : 2>;
  using Down = F4Shape<false, BN, 206 * 1024, 4, AR, FEW ? 6 : 3>;
  using Plan = std::conditional_t<FEW, FmFewPlan, FmFullPlan>;
};

template <int BN, int AR, bool FEW>
__global__ void __launch_bounds__(FM_THREADS, 1) fp4_moe_up_kernel(const __grid_constant__ F4Maps map, const FmArgs a) {
  using S = typename FmShapes<BN, AR, FEW>::Up;
  using Plan = typename FmShapes<BN, AR, FEW>::Plan;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) F4Bars<S> bar;
  __shared__ __align__(8) uint64_t rows_bar;
  __shared__ Plan plan;
  __shared__ double s_sum[4];
  __shared__ unsigned s_max[4], s_top[32];
  __shared__ float s_xs[FM_TOKENS];
  __shared__ int s_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) mbar_init(&rows_bar, 128);
  f4_open<S>(bar, map);
  fm_ask_gain(a);
  pdl_wait();
  pdl_launch();
  const int row0 = FEW ? blockIdx.x * a.T : 0, et = threadIdx.x - F4_EPILOGUE;         // few tokens: rows of this CTA's own
  const long x_bytes = fp4_row_bytes(a.H), x_scale = a.H / 2 + a.H / 16;
  if (et < 0) {
    fm_plan(plan, a, FM_SLOTS, smem);
    fm_plan_made();
  } else {
    if (FEW) {
      for (int t = 0; t < a.T; ++t) {
        if (t) f4_meet<4>();                        // the row before's maxima have been read
        fm_token(a, t, a.xq + (row0 + t) * x_bytes, s_sum, s_max);
      }
      fm_rows_stored(&rows_bar);
    } else {
      for (int tries = 0; tries <= a.T; ++tries) {
        if (et == 0) s_word = atomicAdd(a.claim, 1);
        f4_meet<4>();
        const int t = s_word;
        if (t >= a.T) break;
        fm_token(a, t, a.xq + t * x_bytes, s_sum, s_max);
        __threadfence();
        asm volatile("fence.proxy.async;" ::: "memory");
        f4_meet<4>();
        if (et == 0) atomicAdd(a.claim + 1, 1);
      }
    }
    fm_plan_wait();
  }
  FmUpTiles<Plan, AR> tiles(plan, a.I, a.H, row0, a.T);

  if (warp == 0) {
    if (lane == 0) f4_weights<S>(smem, bar, map, tiles);
  } else if (warp == 6) {
    const bool go = tiles.count() > 0 && (!FEW || mbar_wait_warp(&rows_bar, 0, &bar.abort));
    if (lane == 0 && go && (FEW || fm_tokens_ready(a, &bar.abort))) f4_tokens<S>(smem, bar, map, tiles);
  } else if (warp == 1) {
    f4_issue<S>(smem, bar, tiles);
  } else if (warp < 6) {
    f4_cells<S>(smem, bar, tiles);
  } else {
    const int q = warp & 3;
    uint32_t ab = 0, aphase = 0;
    int done = 0;                                                    // tiles of the expert at hand
    const int n_tiles = tiles.count();
    auto scale_of = [&](int i, const uint8_t* m) {
      const F4Work mt = tiles.at(i);
      return *reinterpret_cast<const float*>(m + ((long)mt.group * a.I + min(mt.n0 + q * 32 + lane, a.I - 1)) * x_bytes + x_scale);
    };
    float ws_nxt = 0.0f, ws2_nxt = 0.0f;
    if (n_tiles > 0) { ws_nxt = scale_of(0, a.wg); ws2_nxt = scale_of(0, a.wu); }
    for (int i = 0; i < n_tiles; ++i) {
      const F4Work mt = tiles.at(i);
      const typename Plan::Entry e = plan.entry[tiles.entry(i)];
      const int n = mt.n0 + q * 32 + lane, end = min(a.I, mt.n0 + AR);
      const float ws = ws_nxt, ws2 = ws2_nxt;
      if (i + 1 < n_tiles) { ws_nxt = scale_of(i + 1, a.wg); ws2_nxt = scale_of(i + 1, a.wu); }
      if (!f4_all<4>(mbar_wait_warp(&bar.acc_full[ab], aphase, &bar.abort))) break;
      tc_fence_after();
      if (i == 0) {                                                  // the first products are there, and so are all rows
        if (et < a.T) s_xs[et] = __ldcg(reinterpret_cast<const float*>(a.xq + (row0 + et) * x_bytes + x_scale));
        f4_meet<4>();
      }
      const uint32_t tbase = bar.tmem + ((uint32_t)(q * 32) << 16) + ab * (2 * BN);
      for (int r0 = 0; r0 < e.rows; r0 += 4) {
        uint32_t v[4], u[4];
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = plan.slot[e.first + min(r0 + j, e.rows - 1)] / a.k;
          x[j] = s_xs[t];
          tmem_ld1(tbase + t, v[j]);
          tmem_ld1(tbase + BN + t, u[j]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float g = __uint_as_float(v[j]) * ws * x[j], up = __uint_as_float(u[j]) * ws2 * x[j];
          if (r0 + j < e.rows && n < end) a.act[(long)(e.first + r0 + j) * a.I + n] = fp4_silu(g) * up;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.acc_empty[ab]);
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
      ++done;
      if (!FEW && (i + 1 == n_tiles || tiles.entry(i + 1) != tiles.entry(i))) {
        if (fm_last(a.claim + 2 + e.expert, done, tiles.tiles_w, &s_word)) fm_rows(a, e.first, e.rows, a.aq, s_top);
        done = 0;
      }
    }
  }
  f4_close<S>(bar, a.status);
}

// AR columns of the output from column n0 on: the slots of every token, in order.  Four columns a lane, AR / 4 lanes a token, two tokens of
// a lane at once.
template <int AR>
__device__ __forceinline__ void fm_combine(const FmArgs& a, const short* id, int n0) {
  constexpr int LANES = AR / 4, AT_ONCE = 128 / LANES;
  const int et = threadIdx.x - F4_EPILOGUE, n = n0 + 4 * (et % LANES);
  if (n >= a.H) return;
  for (int t0 = et / LANES; t0 < a.T; t0 += 2 * AT_ONCE) {
    float4 s[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int t = t0 + AT_ONCE * p;
      s[p] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (a.resid && t < a.T) {
        const float* r = a.resid + (long)t * a.ldr + n;
        s[p] = make_float4(r[0], r[1], r[2], r[3]);
      }
    }
    for (int j0 = 0; j0 < a.k; j0 += 8) {
      float4 v[2][8];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = (t0 + AT_ONCE * p) * a.k + j0 + j;
          v[p][j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (t0 + AT_ONCE * p < a.T && j0 + j < a.k && id[at] >= 0) v[p][j] = __ldcg(reinterpret_cast<const float4*>(a.slot_out + (long)at * a.H + n));
        }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j) { s[p].x += v[p][j].x; s[p].y += v[p][j].y; s[p].z += v[p][j].z; s[p].w += v[p][j].w; }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int t = t0 + AT_ONCE * p;
      if (t >= a.T) break;
      const float f[4] = {s[p].x, s[p].y, s[p].z, s[p].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (a.c_f32) a.c_f32[(long)t * a.ldc + n + i] = f[i];
        else a.c_bf16[(long)t * a.ldc + n + i] = __float2bfloat16_rn(f[i]);
      }
    }
  }
}

template <int BN, int AR, bool FEW>
__global__ void __launch_bounds__(FM_THREADS, 1) fp4_moe_down_kernel(const __grid_constant__ F4Maps map, const FmArgs a) {
  using S = typename FmShapes<BN, AR, FEW>::Down;
  using Plan = typename FmShapes<BN, AR, FEW>::Plan;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) F4Bars<S> bar;
  __shared__ __align__(8) uint64_t rows_bar;
  __shared__ Plan plan;
  __shared__ float s_factor[FEW ? FM_FEW_SLOTS : FM_SLOTS];
  __shared__ unsigned s_top[32];
  __shared__ int s_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) mbar_init(&rows_bar, 128);
  f4_open<S>(bar, map);
  // The ids were there before the launch in front of this one began, and weights always are: both are read before its end is waited for.
  if (threadIdx.x < F4_EPILOGUE) {
    fm_plan(plan, a, BN, smem);
    fm_plan_made();
  } else {
    fm_plan_wait();
  }
  const int row0 = FEW ? blockIdx.x * a.T * a.k : 0;                 // few tokens: rows of this CTA's own
  FmDownTiles<Plan, AR> tiles(plan, a.H, a.I, row0);

  if (warp == 0) {
    if (lane == 0) f4_weights<S>(smem, bar, map, tiles);
  } else if (warp == 6) {
    pdl_wait();
    pdl_launch();
    const bool go = tiles.count() > 0 && (!FEW || mbar_wait_warp(&rows_bar, 0, &bar.abort));
    if (lane == 0 && go) f4_tokens<S>(smem, bar, map, tiles);
  } else if (warp == 1) {
    f4_issue<S>(smem, bar, tiles);
  } else if (warp < 6) {
    f4_cells<S>(smem, bar, tiles);
  } else {
    const int q = warp & 3, et = threadIdx.x - F4_EPILOGUE, n_tiles = tiles.count(), n_slots = a.T * a.k;
    const long a_bytes = fp4_row_bytes(a.I), a_scale = a.I / 2 + a.I / 16;
    auto scale_of = [&](int i) {
      const F4Work mt = tiles.at(i);
      return *reinterpret_cast<const float*>(a.wd + ((long)mt.group * a.H + min(mt.n0 + q * 32 + lane, a.H - 1)) * a_bytes + a_scale);
    };
    float ws_nxt = n_tiles > 0 ? scale_of(0) : 0.0f;
    pdl_wait();
    if (blockIdx.x == 0 && et < 2) a.claim[et] = 0;                  // ready for the next call
    if (FEW && n_tiles > 0) {
      for (int i = 0; i < n_tiles && i < plan.n_entries; ++i) fm_rows(a, tiles.entry(i).first, tiles.entry(i).rows, a.aq + row0 * a_bytes, s_top);
      fm_rows_stored(&rows_bar);
    }
    for (int s = et; s < n_slots && n_tiles > 0; s += 128) {         // places behind the last slot of an expert of ours are not read
      const int slot = plan.slot[s];
      if ((unsigned)slot < (unsigned)n_slots) s_factor[s] = *reinterpret_cast<const volatile float*>(a.aq + (row0 + s) * a_bytes + a_scale) * a.wts[slot];
    }
    f4_meet<4>();
    uint32_t ab = 0, aphase = 0;
    int done = 0;                                                    // tiles of the columns at hand
    for (int i = 0; i < n_tiles; ++i) {
      const F4Work mt = tiles.at(i);
      const typename Plan::Entry e = tiles.entry(i);
      const int n = mt.n0 + q * 32 + lane, end = min(a.H, mt.n0 + AR);
      const float ws = ws_nxt;
      if (i + 1 < n_tiles) ws_nxt = scale_of(i + 1);
      if (!f4_all<4>(mbar_wait_warp(&bar.acc_full[ab], aphase, &bar.abort))) break;
      tc_fence_after();
      const uint32_t tbase = bar.tmem + ((uint32_t)(q * 32) << 16) + ab * BN;
      for (int r0 = 0; r0 < e.rows; r0 += 4) {
        uint32_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) tmem_ld1(tbase + min(r0 + j, e.rows - 1), v[j]);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = e.first + min(r0 + j, e.rows - 1), slot = plan.slot[at];
          const float f = __uint_as_float(v[j]) * ws * s_factor[at];
          if (r0 + j < e.rows && n < end) a.slot_out[(long)slot * a.H + n] = f;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.acc_empty[ab]);
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
      ++done;
      if (i + 1 == n_tiles || tiles.at(i + 1).n0 != mt.n0) {
        if (fm_last(a.claim + 2 + a.E + mt.n0 / AR, done, plan.n_entries, &s_word)) fm_combine<AR>(a, plan.id, mt.n0);
        done = 0;
      }
    }
    if (plan.n_entries == 0)                                         // every slot is another tier's
      for (int j = blockIdx.x; j < (a.H + AR - 1) / AR; j += gridDim.x) fm_combine<AR>(a, plan.id, AR * j);
  }
  f4_close<S>(bar, a.status);
}

}  // namespace bl

using namespace bl;

struct Fp4MoeCall {
  const void* x; const float* gain; const int* ids; const float* wts; const void* wg; const void* wu; const void* wd; void* work;
  const float* resid; float* c_f32; void* c_bf16; unsigned* status; cudaStream_t stream;
  long ldx, ldr, ldc;
  double eps;
  int x_type, T, k, E, H, I, rows, sms;
};

namespace bl {

// The scratch of calls of up to `rows` tokens: counters, then the buffers, each at a multiple of 128 bytes.
struct FmWork {
  long xq, act, aq, slot_out, total;
  FmWork(long rows, long k, long E, long H, long I, long sms) {
    const long few = sms * (rows < FM_FEW ? rows : FM_FEW), own = few * k;
    auto up = [](long n) { return (n + 127) / 128 * 128; };
    xq = up((2 + E + (H + 31) / 32) * 4);
    act = xq + up((rows > few ? rows : few) * fp4_row_bytes((int)H));
    aq = act + up(rows * k * I * 4);
    slot_out = aq + up((rows * k > own ? rows * k : own) * fp4_row_bytes((int)I));
    total = slot_out + up(rows * k * H * 4);
  }
};

template <class S>
static void fm_limit(const void* kernel) { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM); }

// rows_x, rows_a: NVFP4 rows of tokens and of activations that the scratch holds for this call; n: tiles
template <int BN, int AR, bool FEW>
static int fm_up(const Fp4MoeCall& c, const FmArgs& a, long rows_x, long n) {
  using S = typename FmShapes<BN, AR, FEW>::Up;
  F4Maps m;
  const int rc = f4_maps<S>(&m, a.xq, rows_x, a.wg, a.wu, a.H, a.I, a.E);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) { fm_limit<S>((const void*)fp4_moe_up_kernel<BN, AR, FEW>); limit.mark(); }
  return (int)launch(fp4_moe_up_kernel<BN, AR, FEW>, dim3((unsigned)(n < c.sms ? n : c.sms)), dim3(FM_THREADS), S::SMEM, c.stream, m, a);
}
template <int BN, int AR, bool FEW>
static int fm_down(const Fp4MoeCall& c, const FmArgs& a, long rows_a, long n) {
  using S = typename FmShapes<BN, AR, FEW>::Down;
  F4Maps m;
  const int rc = f4_maps<S>(&m, a.aq, rows_a, a.wd, nullptr, a.I, a.H, a.E);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) { fm_limit<S>((const void*)fp4_moe_down_kernel<BN, AR, FEW>); limit.mark(); }
  return (int)launch(fp4_moe_down_kernel<BN, AR, FEW>, dim3((unsigned)(n < c.sms ? n : c.sms)), dim3(FM_THREADS), S::SMEM, c.stream, m, a);
}

static int fp4_moe_few(const Fp4MoeCall& c, const FmArgs& a) {
  // rows of a tile: as few as still find a processor for each tile at once
  const long hit = a.E < a.T * a.k ? a.E : a.T * a.k, rows_x = (long)c.sms * a.T, rows_a = rows_x * a.k;
  auto tiles = [&](long n, int ar) { return (n + ar - 1) / ar; };
  const int au = hit * tiles(a.I, 32) <= c.sms ? 32 : hit * tiles(a.I, 64) <= c.sms ? 64 : 128;
  int rc = au == 32 ? fm_up<32, 32, true>(c, a, rows_x, hit * tiles(a.I, 32)) : au == 64 ? fm_up<32, 64, true>(c, a, rows_x, hit * tiles(a.I, 64))
                                                                                       : fm_up<32, 128, true>(c, a, rows_x, hit * tiles(a.I, 128));
  if (rc) return rc;
  const int ad = hit * tiles(a.H, 32) <= c.sms ? 32 : hit * tiles(a.H, 64) <= c.sms ? 64 : 128;
  return ad == 32 ? fm_down<32, 32, true>(c, a, rows_a, hit * tiles(a.H, 32)) : ad == 64 ? fm_down<32, 64, true>(c, a, rows_a, hit * tiles(a.H, 64))
                                                                                        : fm_down<32, 128, true>(c, a, rows_a, hit * tiles(a.H, 128));
}
template <int BN>
static int fp4_moe_full(const Fp4MoeCall& c, const FmArgs& a) {
  const long hit = a.E < a.T * a.k ? a.E : a.T * a.k;
  const int rc = fm_up<BN, 128, false>(c, a, a.T, hit * ((a.I + 127) / 128));
  return rc ? rc : fm_down<BN, 128, false>(c, a, (long)a.T * a.k, hit * ((a.H + 127) / 128));
}

}  // namespace bl

extern "C" {

long bl_fp4_moe_work_bytes(int rows, int k, int E, int H, int I, int sms) { return FmWork(rows, k, E, H, I, sms).total; }

// y[t] = resid[t] + sum_j wts[t, j] (NVFP4 of silu(x_t Wg[e]) * (x_t Wu[e])) Wd[e], e = ids[t, j] (none where that is outside 0 .. E - 1),
// for T rows x (x_type 0 bf16, 2 fp32; gain != null: RMSNorm first), in NVFP4.  Wg, Wu [E, I] rows of H values, Wd [E, H] rows of I; work:
// bl_fp4_moe_work_bytes(rows >= T, ...) bytes, zeros before the first call; exactly one of c_f32 / c_bf16.
int bl_fp4_moe(const Fp4MoeCall* c) {
  BL_REQUIRE(c->T >= 1 && c->k >= 1 && c->E >= 1 && c->rows >= c->T && c->sms >= 1, BL_ERR_SHAPE);
  BL_REQUIRE(c->H >= 64 && c->H % 64 == 0 && c->I >= 64 && c->I % 64 == 0, BL_ERR_SHAPE);
  BL_REQUIRE(c->rows <= FM_TOKENS && c->k <= FM_USED && c->E <= FM_EXPERTS && c->H <= FM_WIDTH && c->I <= FM_WIDTH, BL_ERR_LIMIT);
  BL_REQUIRE((c->x_type == 0 || c->x_type == 2) && (!c->gain || c->x_type == 2), BL_ERR_TYPE);
  BL_REQUIRE(c->ldx >= c->H && c->ldx % (c->x_type == 2 ? 4 : 8) == 0 && ((uintptr_t)c->x & 15) == 0 && ((uintptr_t)c->gain & 15) == 0 &&
                 ((uintptr_t)c->work & 127) == 0 && ((uintptr_t)c->wg & 15) == 0 && ((uintptr_t)c->wu & 15) == 0 && ((uintptr_t)c->wd & 15) == 0,
             BL_ERR_ALIGN);
  BL_REQUIRE((c->c_f32 != nullptr) != (c->c_bf16 != nullptr), BL_ERR_SHAPE);
  const FmWork w(c->rows, c->k, c->E, c->H, c->I, c->sms);
  const int few = c->T <= FM_FEW;
  uint8_t* base = (uint8_t*)c->work;
  FmArgs a{c->x, c->ldx, c->x_type, c->gain, c->eps, c->ids, c->wts, c->T, c->k, c->E, c->H, c->I, (const uint8_t*)c->wg, (const uint8_t*)c->wu,
           (const uint8_t*)c->wd, base + w.xq, (float*)(base + w.act), base + w.aq, (float*)(base + w.slot_out), (int*)base, c->resid, c->ldr,
           c->c_f32, (__nv_bfloat16*)c->c_bf16, c->ldc, c->status};
  return few ? fp4_moe_few(*c, a) : c->T <= 32 ? fp4_moe_full<32>(*c, a) : fp4_moe_full<64>(*c, a);
}

}  // extern "C"
