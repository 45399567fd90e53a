// The main loop of the NVFP4 products (fp4_gemm.cu, fp4_moe.cu): two TMA threads, four warps that bring the scales to tensor memory, an
// issuing warp and the accumulators that epilogue warps read.  What a CTA works on is a list of tiles that the kernel names:
//   int count();  F4Work at(int i);      both the same for every role
#pragma once
#include "fp4_common.cuh"

namespace bl {

// Warps: 0 TMA of weights, 1 MMA and tensor memory, 2 to 5 scales, 6 TMA of tokens, 7 .. the epilogue's.
constexpr int F4_EPILOGUE = 224;            // its first thread
template <int WARPS>
__device__ __forceinline__ void f4_meet() { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); }     // the epilogue warps
// Whether all of them had what they waited for: where one gave up none goes on to a meeting.
template <int WARPS>
__device__ __forceinline__ bool f4_all(bool ok) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"((uint32_t)ok), "n"(32 * WARPS) : "memory");
  return r != 0;
}

// mbar_wait_warp, whose limit holds, with one try in front of its loop (54 clocks instead of 94 where the phase has ended, as it mostly
// has)
__device__ __forceinline__ bool f4_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xFFFFFFFFu, ok) || mbar_wait_warp(bar, parity, abort_flag);
}

struct F4Work {
  int group, n0;            // the matrix and its first row
  int row0, rows;           // token rows
  int kb0, kb1;             // blocks of 256 values
};

// What a stage holds, in bytes from its start, and what it has in tensor memory, in columns.  Scales arrive for SPAN stages at once, in a
// ring of their own: a box of 16 bytes a row costs TMA as much as one of 128.
// ROOM: bytes of shared memory for both; RAWS: slots of scales, two of which do: single matrices of 128 rows lose a stage to a third and are
// slower (queries of 4,096 tokens 114 us with two, 120.5 with three, 121 with four; gate and up of 2,000 ids 70.7, 74.1, 74.2), smaller tiles and
// rounds have room for more and are no different with them (one token 19.5 us with six or three, 20.1 with two).
// WARPS: of the epilogue, four or eight; AR: weight rows of a tile.  The instruction multiplies 128
// rows in any case; where few tokens meet few weights, tiles of fewer rows give more processors a share of the weights' way from
// memory, and what the instruction reads behind the tile's rows ends in lanes that nobody reads.
template <bool DUAL_, int BN_, int ROOM, int WARPS_, int AR_ = 128, int RAWS_ = AR_ < 128 ? 6 : 2>
struct F4Shape {
  static constexpr bool DUAL = DUAL_;
  static constexpr int RAWS = RAWS_;                               // slots of scales
  static constexpr int WARPS = WARPS_, THREADS = F4_EPILOGUE + 32 * WARPS, BN = BN_, AR = AR_;
  static constexpr int MATS = DUAL ? 2 : 1;
  static constexpr int FEW = BN > 32 ? BN / 4 : BN;                // rows of the smaller box of tokens
  static constexpr int SPAN = DUAL ? 2 : 4;
  static constexpr int A_BYTES = AR * 128, B = MATS * A_BYTES;
  static constexpr int B_CELLS = BN > 128 ? 8 : 4;                 // columns of an instruction's token scales
  static constexpr int STAGE = B + BN * 128;
  static constexpr int RAW_A = AR * 16 * SPAN, RAW_B = MATS * RAW_A, RAW = (RAW_B + BN * 16 * SPAN + 511) / 512 * 512;     // rows of 16 * SPAN bytes
  static constexpr int BEHIND = AR < 128 ? 16384 : 0;              // what the last stage's instructions may read past the rings
  static constexpr int SCALE_COLS = 16 * MATS + 4 * B_CELLS;
  static constexpr int FIT = (ROOM - RAWS * RAW - BEHIND) / STAGE, FIT2 = (512 - 2 * MATS * BN) / SCALE_COLS, FIT1 = (512 - MATS * BN) / SCALE_COLS;
  static constexpr int ACCS = FIT2 >= 3 || FIT2 >= FIT ? 2 : 1;
  static constexpr int MOST = ACCS == 2 ? FIT2 : FIT1, STAGES0 = FIT < MOST ? FIT : MOST, STAGES = STAGES0 < 12 ? STAGES0 : 12;
  static constexpr int SCALE0 = ACCS * MATS * BN;                  // first column of the scales
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + RAWS * RAW + BEHIND + 1024;
  static_assert(STAGES >= 2 && SCALE0 + STAGES * SCALE_COLS <= 512 && B % 1024 == 0 && RAW_A % 512 == 0, "tensor memory, swizzle atoms");
  static __device__ __forceinline__ uint8_t* raw(uint8_t* smem, int slot) { return smem + (size_t)STAGES * STAGE + slot * RAW; }
};

struct F4Maps { CUtensorMap x, xs, few, fews, w, ws, w2, ws2; };

template <class S>
struct F4Bars {
  uint64_t full[S::STAGES], empty[S::STAGES], raw_full[S::RAWS], raw_empty[S::RAWS], acc_full[S::ACCS], acc_empty[S::ACCS];
  uint32_t tmem;
  int abort;
};

// Barriers and tensor memory of the CTA; all threads.
template <class S>
__device__ __forceinline__ void f4_open(F4Bars<S>& b, const F4Maps& map) {
  if (threadIdx.x == 32) {
    const CUtensorMap* maps[8] = {&map.w, &map.ws, &map.x, &map.xs, &map.few, &map.fews, &map.w2, &map.ws2};
    for (int i = 0; i < 6 + 2 * (S::MATS - 1); ++i) asm volatile("prefetch.tensormap [%0];" ::"l"(maps[i]) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(&b.full[s], 6); mbar_init(&b.empty[s], 1); }
    for (int s = 0; s < S::RAWS; ++s) { mbar_init(&b.raw_full[s], 2); mbar_init(&b.raw_empty[s], 4); }
    for (int i = 0; i < S::ACCS; ++i) { mbar_init(&b.acc_full[i], 1); mbar_init(&b.acc_empty[i], S::WARPS); }
    b.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >> 5 == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
template <class S>
__device__ __forceinline__ void f4_close(F4Bars<S>& b, unsigned* status) {
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x >> 5 == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(b.tmem), "r"(512) : "memory");
  }
  if (threadIdx.x == 0 && b.abort && status) atomicMax(status, 1u);
}

// The two TMA threads; one alone was what bound the products (80 to 100 clocks a copy, up to ten of them a stage).  Weights are on their way
// before the token rows may be read.  Rows past a matrix and values past a row arrive as zeros; rows past a tile are some other tile's.
template <class S, class Tiles, class Codes, class Scales>
__device__ __forceinline__ void f4_stream(F4Bars<S>& bar, Tiles& tiles, Codes&& codes, Scales&& scales) {
  volatile int* abort_flag = &bar.abort;
  const int n = tiles.count();
  int stage = 0, slot = 0;
  uint32_t phase = 0, slot_phase = 0;
  bool ok = true;
  for (int i = 0; i < n && ok; ++i) {
    const F4Work w = tiles.at(i);
    for (int kb = w.kb0; kb < w.kb1; ++kb) {
      if ((kb - w.kb0) % S::SPAN == 0) {
        if (!(ok = mbar_wait(&bar.raw_empty[slot], slot_phase ^ 1, abort_flag))) break;
        scales(w, kb, slot);
        if (++slot == S::RAWS) { slot = 0; slot_phase ^= 1; }
      }
      if (!(ok = mbar_wait(&bar.empty[stage], phase ^ 1, abort_flag))) break;
      codes(w, kb, stage);
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
  }
  if (*abort_flag) {
    // copies of this thread may still be landing in shared memory: the CTA must not exit under them
    unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) {}
  }
}
template <class S, class Tiles>
__device__ __forceinline__ void f4_weights(uint8_t* smem, F4Bars<S>& bar, const F4Maps& map, Tiles& tiles) {
  f4_stream<S>(bar, tiles,
    [&](const F4Work& w, int kb, int stage) {
      uint8_t* s = smem + (size_t)stage * S::STAGE;
      mbar_expect_tx(&bar.full[stage], S::B);
      tma_load_3d(s, &map.w, kb * 128, w.n0, w.group, &bar.full[stage]);
      if (S::DUAL) tma_load_3d(s + S::A_BYTES, &map.w2, kb * 128, w.n0, w.group, &bar.full[stage]);
    },
    [&](const F4Work& w, int kb, int slot) {
      uint8_t* s = S::raw(smem, slot);
      mbar_expect_tx(&bar.raw_full[slot], S::RAW_B);
      tma_load_3d(s, &map.ws, kb * 16, w.n0, w.group, &bar.raw_full[slot]);
      if (S::DUAL) tma_load_3d(s + S::RAW_A, &map.ws2, kb * 16, w.n0, w.group, &bar.raw_full[slot]);
    });
}
template <class S, class Tiles>
__device__ __forceinline__ void f4_tokens(uint8_t* smem, F4Bars<S>& bar, const F4Maps& map, Tiles& tiles) {
  f4_stream<S>(bar, tiles,
    [&](const F4Work& w, int kb, int stage) {
      const bool few = w.rows <= S::FEW;
      mbar_expect_tx(&bar.full[stage], (few ? S::FEW : S::BN) * 128);
      tma_load_3d(smem + (size_t)stage * S::STAGE + S::B, few ? &map.few : &map.x, kb * 128, w.row0, 0, &bar.full[stage]);
    },
    [&](const F4Work& w, int kb, int slot) {
      const bool few = w.rows <= S::FEW;
      mbar_expect_tx(&bar.raw_full[slot], (few ? S::FEW : S::BN) * 16 * S::SPAN);
      tma_load_3d(S::raw(smem, slot) + S::RAW_B, few ? &map.fews : &map.xs, kb * 16, w.row0, 0, &bar.raw_full[slot]);
    });
}

// The issuing warp.
template <class S, class Tiles>
__device__ __forceinline__ void f4_issue(uint8_t* smem, F4Bars<S>& bar, Tiles& tiles) {
  volatile int* abort_flag = &bar.abort;
  const uint32_t tmem = bar.tmem;
  int stage = 0; uint32_t phase = 0;
  uint32_t ab = 0, aphase = 0;
  const int n = tiles.count();
  for (int i = 0; i < n; ++i) {
    const F4Work w = tiles.at(i);
    const uint32_t idesc = fp4_idesc((w.rows + 31) / 32 * 32);
    if (!mbar_wait_warp(&bar.acc_empty[ab], aphase ^ 1, abort_flag)) return;
    tc_fence_after();
    const uint32_t d0 = tmem + ab * (S::MATS * S::BN);
    for (int kb = w.kb0; kb < w.kb1; ++kb) {
      if (!f4_wait(&bar.full[stage], phase, abort_flag)) return;            // codes, and the cells of four warps
      tc_fence_after();
      const uint32_t sm = smem_u32(smem + (size_t)stage * S::STAGE), sc = tmem + S::SCALE0 + stage * S::SCALE_COLS, sb = sc + 16 * S::MATS;
      const uint64_t da = umma_desc(sm), db = umma_desc(sm + S::B);
#pragma unroll
      for (int k = 0; k < 4; ++k) {                              // 64 values are 32 bytes
#pragma unroll
        for (int m = 0; m < S::MATS; ++m)
          umma_fp4(d0 + m * S::BN, da + (uint64_t)(m * S::A_BYTES / 16 + 2 * k), db + (uint64_t)(2 * k), idesc, sc + 16 * m + 4 * k,
                   sb + S::B_CELLS * k, kb > w.kb0 || k > 0 ? 1u : 0u);
      }
      umma_commit(&bar.empty[stage]);
      if (kb == w.kb1 - 1) umma_commit(&bar.acc_full[ab]);
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
    if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
  }
}

// Warps 2 to 5: the cells of a stage, each warp its quarter of the lanes.  (Turned in shared memory by two warps and copied by the issuing one,
// 33 clocks a copy, eight of a stage's 870 clocks went with them.)  A stage is handed over while the next one's scales are read, where
// those are there already; the wait for its own stores is over by then.
template <class S, class Tiles>
__device__ __forceinline__ void f4_cells(uint8_t* smem, F4Bars<S>& bar, Tiles& tiles) {
  volatile int* abort_flag = &bar.abort;
  const int lane = threadIdx.x & 31;
  const uint32_t quarter = bar.tmem + ((threadIdx.x >> 5 & 3) << 21) + S::SCALE0;
  int stage = 0, slot = 0, pending = -1; uint32_t phase = 0, slot_phase = 0;
  auto hand_over = [&]() {
    tmem_st_wait();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.full[pending]);
    pending = -1;
  };
  const int n = tiles.count();
  for (int i = 0; i < n; ++i) {
    const F4Work w = tiles.at(i);
    const int groups = (w.rows + 31) / 32;
    for (int kb = w.kb0; kb < w.kb1; ++kb) {
      const int at = (kb - w.kb0) % S::SPAN;
      const bool last = at == S::SPAN - 1 || kb == w.kb1 - 1;      // of its slot
      if (at == 0 && !f4_wait(&bar.raw_full[slot], slot_phase, abort_flag)) return;
      const uint8_t* raw = S::raw(smem, slot);
      uint32_t ca[S::MATS][16], cb[4 * S::B_CELLS];
#pragma unroll
      for (int m = 0; m < S::MATS; ++m) fp4_cells<S::SPAN, 4>(ca[m], raw + m * S::RAW_A, at, lane, (S::AR + 31) / 32);
      fp4_cells<S::SPAN, S::B_CELLS>(cb, raw + S::RAW_B, at, lane, groups);
      if (!f4_wait(&bar.empty[stage], phase ^ 1, abort_flag)) return;       // the instructions that read the cells here have ended
      tc_fence_after();
      if (pending >= 0) hand_over();
      const uint32_t sc = quarter + stage * S::SCALE_COLS;
#pragma unroll
      for (int m = 0; m < S::MATS; ++m) fp4_st16(sc + 16 * m, ca[m]);
      if constexpr (S::B_CELLS == 8) tmem_st32(sc + 16 * S::MATS, cb);
      else fp4_st16(sc + 16 * S::MATS, cb);
      pending = stage;
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
      if (last) {
        hand_over();
        if (lane == 0) mbar_arrive(&bar.raw_empty[slot]);
        if (++slot == S::RAWS) { slot = 0; slot_phase ^= 1; }
      }
    }
  }
}

template <class S>
static int f4_maps(F4Maps* m, const void* x, long rows_x, const void* w, const void* w2, int K, int N, int groups) {
  int rc = fp4_maps(&m->x, &m->xs, x, K, rows_x, 1, S::BN, S::SPAN);
  m->few = m->x; m->fews = m->xs;
  if (!rc && S::FEW < S::BN) rc = fp4_maps(&m->few, &m->fews, x, K, rows_x, 1, S::FEW, S::SPAN);
  if (!rc) rc = fp4_maps(&m->w, &m->ws, w, K, N, groups, S::AR, S::SPAN);
  m->w2 = m->w; m->ws2 = m->ws;
  if (!rc && S::DUAL) rc = fp4_maps(&m->w2, &m->ws2, w2, K, N, groups, S::AR, S::SPAN);
  return rc;
}

}  // namespace bl
