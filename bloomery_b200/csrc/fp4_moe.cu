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
// Rows are claimed and finished by whoever is there, so no CTA waits for one that has not started; the one wait between CTAs (for the tokens'
// rows) is bounded like all others.  Sums of a slot run in one order: the same bits on every run and with every number of CTAs.
#include "fp4_pipe.cuh"

namespace bl {

constexpr int FM_TOKENS = 64, FM_SLOTS = 1024, FM_EXPERTS = 512, FM_WIDTH = 8192;
constexpr int FM_ROOM = 206 * 1024, FM_THREADS = 256;

struct FmArgs {
  const void* x; long ldx; int x_type;              // 0 bf16, 2 fp32
  const float* gain; double eps;
  const int* ids; const float* wts;
  int T, k, E, H, I;
  const uint8_t* wg; const uint8_t* wu; const uint8_t* wd;
  uint8_t* xq;                                      // [T] NVFP4 rows of H
  float* act;                                       // [T * k][I], expert by expert
  uint8_t* aq;                                      // the same as NVFP4 rows
  float* slot_out;                                  // [T * k][H]
  int* claim;                                       // rows taken, rows done, then a ticket for every expert and every 128 columns
  const float* resid; long ldr;
  float* c_f32; __nv_bfloat16* c_bf16; long ldc;
  unsigned* status;
};

// Which experts are hit and by which slots: entries of one expert each, at most `most` slots in one.
struct FmPlan {
  int n_entries;
  short id[FM_SLOTS];                               // of every slot, -1: none of ours
  short slot[FM_SLOTS];                             // expert by expert
  short place[FM_SLOTS];
  struct Entry { short expert, rows; int first; } entry[FM_EXPERTS + FM_SLOTS / 32];
  int count[FM_EXPERTS], first[FM_EXPERTS];
};

__device__ __forceinline__ void fm_plan(FmPlan& p, const FmArgs& a, int most) {
  const int tid = threadIdx.x, n = a.T * a.k;
  for (int e = tid; e < a.E; e += FM_THREADS) p.count[e] = 0;
  __syncthreads();
  for (int s = tid; s < n; s += FM_THREADS) {
    const int e = a.ids[s];
    p.id[s] = (short)(e >= 0 && e < a.E ? e : -1);
  }
  __syncthreads();
  // a slot's place among those of its expert: every CTA comes to the same one
  if (tid < 32)
    for (int s = tid; s - tid < n; s += 32) {
      const int e = s < n ? p.id[s] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e), before = same & ((1u << tid) - 1);
      if (e >= 0) p.place[s] = (short)(p.count[e] + __popc(before));
      __syncwarp();
      if (e >= 0 && before == 0) p.count[e] += __popc(same);
      __syncwarp();
    }
  if (tid < 32) {
    const int per = (a.E + 31) / 32, e0 = min(a.E, tid * per), e1 = min(a.E, e0 + per);
    int rows = 0, entries = 0;
    for (int e = e0; e < e1; ++e) { rows += p.count[e]; entries += (p.count[e] + most - 1) / most; }
    int ro = rows, en = entries;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int r = __shfl_up_sync(0xffffffffu, ro, d), t = __shfl_up_sync(0xffffffffu, en, d);
      if (tid >= d) { ro += r; en += t; }
    }
    if (tid == 31) p.n_entries = en;
    ro -= rows; en -= entries;
    for (int e = e0; e < e1; ++e) {
      p.first[e] = ro;
      for (int r = 0; r < p.count[e]; r += most) p.entry[en++] = FmPlan::Entry{(short)e, (short)min(most, p.count[e] - r), ro + r};
      ro += p.count[e];
    }
  }
  __syncthreads();
  for (int s = tid; s < n; s += FM_THREADS)
    if (p.id[s] >= 0) p.slot[p.first[p.id[s]] + p.place[s]] = (short)s;
  __syncthreads();
}

struct FmUpTiles {
  const FmPlan& p;
  int tiles_w, kblocks, T;
  __device__ __forceinline__ int count() const {
    const int total = p.n_entries * tiles_w;
    return total > (int)blockIdx.x ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
  }
  __device__ __forceinline__ int entry(int i) const { return ((int)blockIdx.x + i * (int)gridDim.x) / tiles_w; }
  __device__ __forceinline__ F4Work at(int i) const {
    const int t = (int)blockIdx.x + i * (int)gridDim.x;
    return F4Work{p.entry[t / tiles_w].expert, t % tiles_w * 128, 0, T, 0, kblocks};      // all tokens
  }
};
struct FmDownTiles {
  const FmPlan& p;
  int tiles_w, kblocks;
  __device__ __forceinline__ int count() const {
    const int total = p.n_entries * tiles_w;
    return total > (int)blockIdx.x ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
  }
  __device__ __forceinline__ F4Work at(int i) const {
    const int t = (int)blockIdx.x + i * (int)gridDim.x;
    const FmPlan::Entry e = p.entry[t / tiles_w];
    return F4Work{e.expert, t % tiles_w * 128, e.first, e.rows, 0, kblocks};
  }
};

// A token's row in NVFP4, by the 128 threads of the epilogue warps.
__device__ __forceinline__ void fm_token(const FmArgs& a, int t, double* s_sum, unsigned* s_max) {
  constexpr int NB = FM_WIDTH / 16 / 128;
  const int et = threadIdx.x - 128, lane = et & 31, w = et >> 5, blocks = a.H / 16;
  float v[NB][16];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (et + 128 * b < blocks) fp4_load16(a.x, a.x_type, (long)t * a.ldx + 16 * (et + 128 * b), v[b]);
  if (a.gain) {
    double ss = 0.0;
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (et + 128 * b < blocks) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fma((double)v[b][i], (double)v[b][i], ss);
      }
    ss = warp_sum_d(ss);
    if (lane == 0) s_sum[w] = ss;
    f4_meet<4>();
    const float r = (float)(1.0 / sqrt((s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]) / (double)a.H + a.eps));
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (et + 128 * b < blocks) fp4_scale16(v[b], r, a.gain + 16 * (et + 128 * b));
  }
  unsigned top = 0;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (et + 128 * b < blocks) top = max(top, fp4_top16(v[b]));
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (lane == 0) s_max[w] = top;
  f4_meet<4>();
  const float g = fp4_row_scale(max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3])));
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (et + 128 * b < blocks) fp4_store_block(a.xq + t * fp4_row_bytes(a.H), a.H, et + 128 * b, v[b], g);
}

// Rows first .. first + rows - 1 of the activations in NVFP4, a warp a row.
__device__ __forceinline__ void fm_rows(const FmArgs& a, int first, int rows) {
  const int et = threadIdx.x - 128, lane = et & 31, blocks = a.I / 16;
  for (int r = et >> 5; r < rows; r += 4) {
    const float* x = a.act + (long)(first + r) * a.I;
    uint8_t* out = a.aq + (first + r) * fp4_row_bytes(a.I);
    float v[4][16];
    unsigned top = 0;
    auto load = [&](int from) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (from + 32 * b + lane < blocks) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(x + 16 * (from + 32 * b + lane)) + i);
            v[b][4 * i] = f.x; v[b][4 * i + 1] = f.y; v[b][4 * i + 2] = f.z; v[b][4 * i + 3] = f.w;
          }
        }
    };
    for (int from = 0; from < blocks; from += 128) {               // 2,048 values at once; wider rows are read again
      load(from);
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (from + 32 * b + lane < blocks) top = max(top, fp4_top16(v[b]));
    }
    const float g = fp4_row_scale(__reduce_max_sync(0xFFFFFFFFu, top));
    for (int from = 0; from < blocks; from += 128) {
      if (blocks > 128) load(from);
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (from + 32 * b + lane < blocks) fp4_store_block(out, a.I, from + 32 * b + lane, v[b], g);
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(FM_THREADS, 1) fp4_moe_up_kernel(const __grid_constant__ F4Maps map, const FmArgs a) {
  using S = F4Shape<true, BN, FM_ROOM, 4>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) F4Bars<S> bar;
  __shared__ FmPlan plan;
  __shared__ double s_sum[4];
  __shared__ unsigned s_max[4];
  __shared__ int s_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  f4_open<S>(bar);
  pdl_wait();
  pdl_launch();
  fm_plan(plan, a, FM_SLOTS);
  FmUpTiles tiles{plan, (a.I + 127) / 128, (a.H + 255) / 256, a.T};

  if (warp == 0) {
    if (lane == 0)
      f4_produce<true, S>(smem, bar, map, tiles, [&] {
        unsigned long long t0 = 0;
        for (;;) {
          int done;
          asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(done) : "l"(a.claim + 1) : "memory");
          if (done >= a.T) break;
          const unsigned long long now = globaltimer();
          if (t0 == 0) t0 = now;
          else if (now - t0 > WAIT_LIMIT_NS) { *(volatile int*)&bar.abort = 1; return false; }
        }
        asm volatile("fence.proxy.async;" ::: "memory");             // rows that other CTAs stored, read by TMA
        return true;
      });
  } else if (warp == 1) {
    f4_issue<true, S>(smem, bar, tiles);
  } else if (warp < 4) {
    f4_turn<true, S>(smem, bar, tiles);
  } else {
    const int q = warp & 3, et = threadIdx.x - 128;
    for (;;) {
      if (et == 0) s_word = atomicAdd(a.claim, 1);
      f4_meet<4>();
      const int t = s_word;
      if (t >= a.T) break;
      fm_token(a, t, s_sum, s_max);
      __threadfence();
      asm volatile("fence.proxy.async;" ::: "memory");
      f4_meet<4>();
      if (et == 0) atomicAdd(a.claim + 1, 1);
    }
    f4_meet<4>();                                                       // s_word is read
    uint32_t ab = 0, aphase = 0;
    const int tiles_w = tiles.tiles_w;
    for (int i = 0; i < tiles.count(); ++i) {
      const F4Work mt = tiles.at(i);
      const FmPlan::Entry e = plan.entry[tiles.entry(i)];
      const int n = mt.n0 + q * 32 + lane;
      const long x_scale = a.H / 2 + a.H / 16, wrow = ((long)mt.group * a.I + min(n, a.I - 1)) * fp4_row_bytes(a.H) + x_scale;
      const float ws = *reinterpret_cast<const float*>(a.wg + wrow), ws2 = *reinterpret_cast<const float*>(a.wu + wrow);
      if (!f4_all<4>(mbar_wait_warp(&bar.acc_full[ab], aphase, &bar.abort))) break;
      tc_fence_after();
      const uint32_t tbase = bar.tmem + ((uint32_t)(q * 32) << 16) + ab * (2 * BN);
      for (int r0 = 0; r0 < e.rows; r0 += 4) {
        uint32_t v[4], u[4];
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = plan.slot[e.first + min(r0 + j, e.rows - 1)] / a.k;
          x[j] = __ldcg(reinterpret_cast<const float*>(a.xq + t * fp4_row_bytes(a.H) + x_scale));
          tmem_ld1(tbase + t, v[j]);
          tmem_ld1(tbase + BN + t, u[j]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float g = __uint_as_float(v[j]) * ws * x[j], up = __uint_as_float(u[j]) * ws2 * x[j];
          if (r0 + j < e.rows && n < a.I) a.act[(long)(e.first + r0 + j) * a.I + n] = (g / (1.0f + __expf(-g))) * up;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.acc_empty[ab]);
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
      __threadfence();
      f4_meet<4>();
      if (et == 0) {
        int* ticket = a.claim + 2 + e.expert;
        const int last = atomicAdd(ticket, 1) == tiles_w - 1;
        if (last) *ticket = 0;                                       // ready for the next call
        __threadfence();
        s_word = last;
      }
      f4_meet<4>();
      if (s_word) fm_rows(a, e.first, e.rows);
    }
  }
  f4_close<S>(bar, a.status);
}

// 128 columns of the output from column n0 on: the slots of every token, in order.
__device__ __forceinline__ void fm_combine(const FmArgs& a, const FmPlan& p, int n0) {
  const int et = threadIdx.x - 128, lane = et & 31, n = n0 + 4 * lane;
  if (n >= a.H) return;
  for (int t = et >> 5; t < a.T; t += 4) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.resid) {
      const float* r = a.resid + (long)t * a.ldr + n;
      s = make_float4(r[0], r[1], r[2], r[3]);
    }
    for (int j0 = 0; j0 < a.k; j0 += 8) {
      float4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < a.k && p.id[t * a.k + j0 + j] >= 0)
          v[j] = __ldcg(reinterpret_cast<const float4*>(a.slot_out + (long)(t * a.k + j0 + j) * a.H + n));
        else v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) { s.x += v[j].x; s.y += v[j].y; s.z += v[j].z; s.w += v[j].w; }
    }
    const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (a.c_f32) a.c_f32[(long)t * a.ldc + n + i] = f[i];
      else a.c_bf16[(long)t * a.ldc + n + i] = __float2bfloat16_rn(f[i]);
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(FM_THREADS, 1) fp4_moe_down_kernel(const __grid_constant__ F4Maps map, const FmArgs a) {
  using S = F4Shape<false, BN, FM_ROOM, 4>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) F4Bars<S> bar;
  __shared__ FmPlan plan;
  __shared__ int s_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  f4_open<S>(bar);
  // The ids were there before the launch in front of this one began, and weights always are: both are read before its end is waited for.
  fm_plan(plan, a, BN);
  FmDownTiles tiles{plan, (a.H + 127) / 128, (a.I + 255) / 256};

  if (warp == 0) {
    if (lane == 0) f4_produce<false, S>(smem, bar, map, tiles, [] { pdl_wait(); pdl_launch(); return true; });
  } else if (warp == 1) {
    f4_issue<false, S>(smem, bar, tiles);
  } else if (warp < 4) {
    f4_turn<false, S>(smem, bar, tiles);
  } else {
    const int q = warp & 3, et = threadIdx.x - 128, tiles_w = tiles.tiles_w;
    pdl_wait();
    if (blockIdx.x == 0 && et < 2) a.claim[et] = 0;                  // ready for the next call
    uint32_t ab = 0, aphase = 0;
    for (int i = 0; i < tiles.count(); ++i) {
      const F4Work mt = tiles.at(i);
      const int n = mt.n0 + q * 32 + lane;
      const long a_scale = a.I / 2 + a.I / 16;
      const float ws = *reinterpret_cast<const float*>(a.wd + ((long)mt.group * a.H + min(n, a.H - 1)) * fp4_row_bytes(a.I) + a_scale);
      if (!f4_all<4>(mbar_wait_warp(&bar.acc_full[ab], aphase, &bar.abort))) break;
      tc_fence_after();
      const uint32_t tbase = bar.tmem + ((uint32_t)(q * 32) << 16) + ab * BN;
      for (int r0 = 0; r0 < mt.rows; r0 += 4) {
        uint32_t v[4];
        float f[4];
        int slot[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = min(r0 + j, mt.rows - 1);
          slot[j] = plan.slot[mt.row0 + r];
          f[j] = *reinterpret_cast<const float*>(a.aq + (mt.row0 + r) * fp4_row_bytes(a.I) + a_scale) * a.wts[slot[j]];
          tmem_ld1(tbase + r, v[j]);
        }
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r0 + j < mt.rows && n < a.H) a.slot_out[(long)slot[j] * a.H + n] = __uint_as_float(v[j]) * ws * f[j];
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.acc_empty[ab]);
      if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
      __threadfence();
      f4_meet<4>();
      if (et == 0) {
        int* ticket = a.claim + 2 + a.E + mt.n0 / 128;
        const int last = atomicAdd(ticket, 1) == plan.n_entries - 1;
        if (last) *ticket = 0;
        __threadfence();
        s_word = last;
      }
      f4_meet<4>();
      if (s_word) fm_combine(a, plan, mt.n0);
    }
    if (plan.n_entries == 0)                                         // every slot is another tier's
      for (int j = blockIdx.x; j < tiles_w; j += gridDim.x) fm_combine(a, plan, 128 * j);
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
  FmWork(long rows, long k, long E, long H, long I) {
    auto up = [](long n) { return (n + 127) / 128 * 128; };
    xq = up((2 + E + (H + 127) / 128) * 4);
    act = xq + up(rows * fp4_row_bytes((int)H));
    aq = act + up(rows * k * I * 4);
    slot_out = aq + up(rows * k * fp4_row_bytes((int)I));
    total = slot_out + up(rows * k * H * 4);
  }
};

template <int BN>
static int fp4_moe_go(const Fp4MoeCall& c, const FmArgs& a) {
  using SU = F4Shape<true, BN, FM_ROOM, 4>;
  using SD = F4Shape<false, BN, FM_ROOM, 4>;
  F4Maps up, down;
  int rc = f4_maps<true, SU>(&up, a.xq, a.T, a.wg, a.wu, a.H, a.I, a.E);
  if (!rc) rc = f4_maps<false, SD>(&down, a.aq, (long)a.T * a.k, a.wd, nullptr, a.I, a.H, a.E);
  if (rc) return rc;
  static PerDevice limit;
  if (limit.due()) {
    cudaFuncSetAttribute(fp4_moe_up_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SU::SMEM);
    cudaFuncSetAttribute(fp4_moe_down_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SD::SMEM);
    limit.mark();
  }
  const long hit = a.E < a.T * a.k ? a.E : a.T * a.k, n_up = hit * ((a.I + 127) / 128), n_down = hit * ((a.H + 127) / 128);
  rc = (int)launch(fp4_moe_up_kernel<BN>, dim3((unsigned)(n_up < c.sms ? n_up : c.sms)), dim3(FM_THREADS), SU::SMEM, c.stream, up, a);
  if (rc) return rc;
  return (int)launch(fp4_moe_down_kernel<BN>, dim3((unsigned)(n_down < c.sms ? n_down : c.sms)), dim3(FM_THREADS), SD::SMEM, c.stream, down, a);
}

}  // namespace bl

extern "C" {

long bl_fp4_moe_work_bytes(int rows, int k, int E, int H, int I) { return FmWork(rows, k, E, H, I).total; }

// y[t] = resid[t] + sum_j wts[t, j] (NVFP4 of silu(x_t Wg[e]) * (x_t Wu[e])) Wd[e], e = ids[t, j] (none where that is outside 0 .. E - 1),
// for T rows x (x_type 0 bf16, 2 fp32; gain != null: RMSNorm first), in NVFP4.  Wg, Wu [E, I] rows of H values, Wd [E, H] rows of I; work:
// bl_fp4_moe_work_bytes(rows >= T, ...) bytes, zeros before the first call; exactly one of c_f32 / c_bf16.
int bl_fp4_moe(const Fp4MoeCall* c) {
  BL_REQUIRE(c->T >= 1 && c->k >= 1 && c->E >= 1 && c->rows >= c->T && c->sms >= 1, BL_ERR_SHAPE);
  BL_REQUIRE(c->H >= 64 && c->H % 64 == 0 && c->I >= 64 && c->I % 64 == 0, BL_ERR_SHAPE);
  BL_REQUIRE(c->rows <= FM_TOKENS && c->k <= 16 && c->E <= FM_EXPERTS && c->H <= FM_WIDTH && c->I <= FM_WIDTH, BL_ERR_LIMIT);
  BL_REQUIRE((c->x_type == 0 || c->x_type == 2) && (!c->gain || c->x_type == 2), BL_ERR_TYPE);
  BL_REQUIRE(c->ldx >= c->H && c->ldx % (c->x_type == 2 ? 4 : 8) == 0 && ((uintptr_t)c->x & 15) == 0 && ((uintptr_t)c->gain & 15) == 0 &&
                 ((uintptr_t)c->work & 127) == 0 && ((uintptr_t)c->wg & 15) == 0 && ((uintptr_t)c->wu & 15) == 0 && ((uintptr_t)c->wd & 15) == 0,
             BL_ERR_ALIGN);
  BL_REQUIRE((c->c_f32 != nullptr) != (c->c_bf16 != nullptr), BL_ERR_SHAPE);
  const FmWork w(c->rows, c->k, c->E, c->H, c->I);
  uint8_t* base = (uint8_t*)c->work;
  FmArgs a{c->x, c->ldx, c->x_type, c->gain, c->eps, c->ids, c->wts, c->T, c->k, c->E, c->H, c->I, (const uint8_t*)c->wg, (const uint8_t*)c->wu,
           (const uint8_t*)c->wd, base + w.xq, (float*)(base + w.act), base + w.aq, (float*)(base + w.slot_out), (int*)base, c->resid, c->ldr,
           c->c_f32, (__nv_bfloat16*)c->c_bf16, c->ldc, c->status};
  return c->T <= 32 ? fp4_moe_go<32>(*c, a) : fp4_moe_go<64>(*c, a);
}

}  // extern "C"
