// The main loop of the NVFP4 products (fp4_gemm.cu, fp4_moe.cu): a TMA thread, two warps that turn scales, an issuing warp and the
// accumulators that epilogue warps read.  What a CTA works on is a list of tiles that the kernel names:
//   int count();  F4Work at(int i);      both the same for every role
#pragma once
#include "fp4_common.cuh"

namespace bl {

constexpr int F4_MAX_STAGES = 8;

// Warps: 0 TMA, 1 MMA and tensor memory, 2 and 3 scales (weights, tokens), 4 .. the epilogue's.
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

struct F4Work {
  int group, n0;            // the matrix and its first row
  int row0, rows;           // token rows
  int kb0, kb1;             // blocks of 256 values
};

// What a stage holds, in bytes from its start, and what it has in tensor memory, in columns.  Scales arrive for SPAN stages at once, in a
// ring of their own: a box of 16 bytes a row costs TMA as much as one of 128.
// ROOM_: bytes of shared memory for both; WARPS_: of the epilogue, four or eight.
template <bool DUAL, int BN_, int ROOM_, int WARPS_>
struct F4Shape {
  static constexpr int WARPS = WARPS_, THREADS = 128 + 32 * WARPS, BN = BN_, MATS = DUAL ? 2 : 1;
  static constexpr int BOX = BN < 64 ? BN : 64;                    // token rows of a box
  static constexpr int SPAN = DUAL || BN > 128 ? 2 : 4;
  static constexpr int B = MATS * 16384, TA = B + BN * 128, TB = TA + MATS * 2048;
  static constexpr int B_CELLS = BN > 128 ? 8 : 4;                 // columns of an instruction's token scales
  static constexpr int STAGE = (TB + 4 * 128 * B_CELLS + 1023) / 1024 * 1024;
  static constexpr int RAW_B = MATS * 128 * 16 * SPAN, RAW = RAW_B + BN * 16 * SPAN;        // rows of 16 * SPAN bytes
  static constexpr int ROOM = ROOM_ - 2 * RAW;
  static constexpr int STAGES = ROOM / STAGE > F4_MAX_STAGES ? F4_MAX_STAGES : ROOM / STAGE;
  static constexpr int SCALE_COLS = 16 * MATS + 4 * B_CELLS;
  static constexpr int ACCS = 2 * MATS * BN + STAGES * SCALE_COLS <= 512 ? 2 : 1;
  static constexpr int SCALE0 = ACCS * MATS * BN;                  // first column of the scales
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + 2 * RAW + 1024;
  static_assert(STAGES >= 2 && SCALE0 + STAGES * SCALE_COLS <= 512, "tensor memory");
  static __device__ __forceinline__ uint8_t* raw(uint8_t* smem, int slot) { return smem + (size_t)STAGES * STAGE + slot * RAW; }
};

struct F4Maps { CUtensorMap x, xs, w, ws, w2, ws2; };

template <class S>
struct F4Bars {
  uint64_t full[S::STAGES], cells[S::STAGES], empty[S::STAGES], raw_full[2], raw_empty[2], acc_full[S::ACCS], acc_empty[S::ACCS];
  uint32_t tmem;
  int abort;
};

// Barriers and tensor memory of the CTA; all threads.
template <class S>
__device__ __forceinline__ void f4_open(F4Bars<S>& b) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(&b.full[s], 1); mbar_init(&b.cells[s], 2); mbar_init(&b.empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&b.raw_full[s], 1); mbar_init(&b.raw_empty[s], 2); }
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

// One thread.  The weights of the first stages are on their way before `ready` says that the token rows may be read.
template <bool DUAL, class S, class Tiles, class Ready>
__device__ __forceinline__ void f4_produce(uint8_t* smem, F4Bars<S>& bar, const F4Maps& map, Tiles& tiles, Ready&& ready) {
  volatile int* abort_flag = &bar.abort;
  const int n = tiles.count();
  if (n == 0) return;
  // rows past a matrix and values past a row arrive as zeros
  auto weights = [&](const F4Work& w, int kb, int stage) {
    uint8_t* s = smem + (size_t)stage * S::STAGE;
    mbar_expect_tx(&bar.full[stage], S::MATS * 16384 + (w.rows + S::BOX - 1) / S::BOX * S::BOX * 128);
    tma_load_3d(s, &map.w, kb * 128, w.n0, w.group, &bar.full[stage]);
    if (DUAL) tma_load_3d(s + 16384, &map.w2, kb * 128, w.n0, w.group, &bar.full[stage]);
  };
  auto tokens = [&](const F4Work& w, int kb, int stage) {
    uint8_t* s = smem + (size_t)stage * S::STAGE + S::B;
    for (int b = 0; b * S::BOX < w.rows; ++b) tma_load_3d(s + b * S::BOX * 128, &map.x, kb * 128, w.row0 + b * S::BOX, 0, &bar.full[stage]);
  };
  auto weight_scales = [&](const F4Work& w, int kb, int slot) {
    uint8_t* s = S::raw(smem, slot);
    mbar_expect_tx(&bar.raw_full[slot], (S::MATS * 128 + (w.rows + S::BOX - 1) / S::BOX * S::BOX) * 16 * S::SPAN);
    tma_load_3d(s, &map.ws, kb * 16, w.n0, w.group, &bar.raw_full[slot]);
    if (DUAL) tma_load_3d(s + 128 * 16 * S::SPAN, &map.ws2, kb * 16, w.n0, w.group, &bar.raw_full[slot]);
  };
  auto token_scales = [&](const F4Work& w, int kb, int slot) {
    uint8_t* s = S::raw(smem, slot) + S::RAW_B;
    for (int b = 0; b * S::BOX < w.rows; ++b)
      tma_load_3d(s + b * S::BOX * 16 * S::SPAN, &map.xs, kb * 16, w.row0 + b * S::BOX, 0, &bar.raw_full[slot]);
  };
  int i = 0;
  F4Work w = tiles.at(0);
  int kb = w.kb0;
  auto step = [&] { if (++kb == w.kb1 && ++i < n) { w = tiles.at(i); kb = w.kb0; } };
  int first = 0, slots = 0, stop = 0;                              // stages and slots filled with weights alone
  for (; first < S::STAGES && i < n; ++first, step()) {
    if ((kb - w.kb0) % S::SPAN == 0) {
      if (slots == 2) break;
      weight_scales(w, kb, slots++);
    }
    weights(w, kb, first);
  }
  stop = first;
  const bool go = ready();
  if (go) {
    i = 0; w = tiles.at(0); kb = w.kb0;
    int stage = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0;
    for (int done = 0; i < n; ++done, step()) {
      if ((kb - w.kb0) % S::SPAN == 0) {
        if (slots > 0) {
          --slots;
        } else {
          if (!mbar_wait(&bar.raw_empty[slot], slot_phase ^ 1, abort_flag)) break;
          weight_scales(w, kb, slot);
        }
        token_scales(w, kb, slot);
        if (++slot == 2) { slot = 0; slot_phase ^= 1; }
      }
      if (done >= stop) {
        if (!mbar_wait(&bar.empty[stage], phase ^ 1, abort_flag)) break;
        weights(w, kb, stage);
      }
      tokens(w, kb, stage);
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
  }
  if (*abort_flag) {
    // copies of this thread may still be landing in shared memory: the CTA must not exit under them
    unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) {}
  }
}

// The issuing warp.
template <bool DUAL, class S, class Tiles>
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
      if (!mbar_wait_warp(&bar.full[stage], phase, abort_flag) || !mbar_wait_warp(&bar.cells[stage], phase, abort_flag)) return;
      tc_fence_after();
      const uint32_t sm = smem_u32(smem + (size_t)stage * S::STAGE), sc = tmem + S::SCALE0 + stage * S::SCALE_COLS;
      const uint32_t sb = sc + 16 * S::MATS;
      // a stage's cells are its own: the instructions that read them ended before the stage was filled again
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int m = 0; m < S::MATS; ++m) fp4_scales_to_tmem(sc + 16 * m + 4 * k, sm + S::TA + 2048 * m + 512 * k);
#pragma unroll
        for (int h = 0; h < S::B_CELLS / 4; ++h) fp4_scales_to_tmem(sb + S::B_CELLS * k + 4 * h, sm + S::TB + 2048 * h + 512 * k);
      }
      const uint64_t da = umma_desc(sm), db = umma_desc(sm + S::B);
#pragma unroll
      for (int k = 0; k < 4; ++k) {                              // 64 values are 32 bytes
#pragma unroll
        for (int m = 0; m < S::MATS; ++m)
          umma_fp4(d0 + m * S::BN, da + (uint64_t)(m * 16384 / 16 + 2 * k), db + (uint64_t)(2 * k), idesc, sc + 16 * m + 4 * k,
                   sb + S::B_CELLS * k, kb > w.kb0 || k > 0 ? 1u : 0u);
      }
      umma_commit(&bar.empty[stage]);
      if (kb == w.kb1 - 1) umma_commit(&bar.acc_full[ab]);
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
    if (++ab == S::ACCS) { ab = 0; aphase ^= 1; }
  }
}

// Warps 2 (weights) and 3 (tokens).
template <bool DUAL, class S, class Tiles>
__device__ __forceinline__ void f4_turn(uint8_t* smem, F4Bars<S>& bar, Tiles& tiles) {
  volatile int* abort_flag = &bar.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int stage = 0, slot = 0; uint32_t phase = 0, slot_phase = 0;
  const int n = tiles.count();
  for (int i = 0; i < n; ++i) {
    const F4Work w = tiles.at(i);
    const int groups = (w.rows + 31) / 32;
    for (int kb = w.kb0; kb < w.kb1; ++kb) {
      const int at = (kb - w.kb0) % S::SPAN;
      if (at == 0 && !mbar_wait_warp(&bar.raw_full[slot], slot_phase, abort_flag)) return;
      if (!mbar_wait_warp(&bar.empty[stage], phase ^ 1, abort_flag)) return;       // the cells that were here have been read
      uint8_t* s = smem + (size_t)stage * S::STAGE;
      const uint4* raw = reinterpret_cast<const uint4*>(S::raw(smem, slot)) + at;
      if (warp == 2) {
#pragma unroll
        for (int m = 0; m < S::MATS; ++m) fp4_turn_scales<S::SPAN>(raw + 128 * S::SPAN * m, reinterpret_cast<uint4*>(s + S::TA + 2048 * m), lane, 4);
      } else {
#pragma unroll
        for (int h = 0; h < S::B_CELLS / 4; ++h)
          fp4_turn_scales<S::SPAN>(raw + S::RAW_B / 16 + 128 * S::SPAN * h, reinterpret_cast<uint4*>(s + S::TB + 2048 * h), lane, groups - 4 * h);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.cells[stage]);
      if (at == S::SPAN - 1 || kb == w.kb1 - 1) {
        if (lane == 0) mbar_arrive(&bar.raw_empty[slot]);
        if (++slot == 2) { slot = 0; slot_phase ^= 1; }
      }
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
  }
}

template <bool DUAL, class S>
static int f4_maps(F4Maps* m, const void* x, long rows_x, const void* w, const void* w2, int K, int N, int groups) {
  int rc = fp4_maps(&m->x, &m->xs, x, K, rows_x, 1, S::BOX, S::SPAN);
  if (!rc) rc = fp4_maps(&m->w, &m->ws, w, K, N, groups, 128, S::SPAN);
  m->w2 = m->w; m->ws2 = m->ws;
  if (!rc && DUAL) rc = fp4_maps(&m->w2, &m->ws2, w2, K, N, groups, 128, S::SPAN);
  return rc;
}

}  // namespace bl
