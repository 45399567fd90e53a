// The main loop of the NVFP4 products (fp4_gemm.cu, fp4_moe.cu): a TMA thread, two warps that turn scales, an issuing warp and the
// accumulators that epilogue warps read.  What a CTA works on is a list of tiles that the kernel names:
//   int count();  F4Work at(int i);      both the same for every role
#pragma once
#include "fp4_common.cuh"

namespace bl {

constexpr int F4_THREADS = 256;             // warp 0 TMA, 1 MMA + TMEM, 2..5 epilogue, 6 and 7 scales
constexpr int F4_MAX_STAGES = 8;

struct F4Work {
  int group, n0;            // the matrix and its first row
  int row0, rows;           // token rows
  int kb0, kb1;             // blocks of 256 values
};

// What a stage holds, in bytes from its start, and what it has in tensor memory, in columns
template <bool DUAL, int BN_>
struct F4Shape {
  static constexpr int BN = BN_, MATS = DUAL ? 2 : 1;
  static constexpr int BOX = BN < 64 ? BN : 64;                    // token rows of a box
  static constexpr int B = MATS * 16384, RA = B + BN * 128, RB = RA + MATS * 2048, TA = RB + BN * 16, TB = TA + MATS * 2048;
  static constexpr int B_CELLS = BN > 128 ? 8 : 4;                 // columns of an instruction's token scales
  static constexpr int STAGE = (TB + 4 * 128 * B_CELLS + 1023) / 1024 * 1024;
  static constexpr int STAGES = 208 * 1024 / STAGE > F4_MAX_STAGES ? F4_MAX_STAGES : 208 * 1024 / STAGE;
  static constexpr int SCALE_COLS = 16 * MATS + 4 * B_CELLS;
  static constexpr int ACCS = 2 * MATS * BN + STAGES * SCALE_COLS <= 512 ? 2 : 1;
  static constexpr int SCALE0 = ACCS * MATS * BN;                  // first column of the scales
  static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024;
  static_assert(STAGES >= 2 && SCALE0 + STAGES * SCALE_COLS <= 512, "tensor memory");
};

struct F4Maps { CUtensorMap x, xs, w, ws, w2, ws2; };

template <class S>
struct F4Bars {
  uint64_t full[S::STAGES], cells[S::STAGES], empty[S::STAGES], acc_full[S::ACCS], acc_empty[S::ACCS];
  uint32_t tmem;
  int abort;
};

// Barriers and tensor memory of the CTA; all threads.
template <class S>
__device__ __forceinline__ void f4_open(F4Bars<S>& b) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) { mbar_init(&b.full[s], 1); mbar_init(&b.cells[s], 2); mbar_init(&b.empty[s], 1); }
    for (int i = 0; i < S::ACCS; ++i) { mbar_init(&b.acc_full[i], 1); mbar_init(&b.acc_empty[i], 4); }
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
  auto weights = [&](const F4Work& w, int kb, int stage) {
    uint8_t* s = smem + (size_t)stage * S::STAGE;
    const int boxes = (w.rows + S::BOX - 1) / S::BOX;
    mbar_expect_tx(&bar.full[stage], S::MATS * (16384 + 2048) + boxes * S::BOX * (128 + 16));
    // rows past a matrix and values past a row arrive as zeros
    tma_load_3d(s, &map.w, kb * 128, w.n0, w.group, &bar.full[stage]);
    tma_load_3d(s + S::RA, &map.ws, kb * 16, w.n0, w.group, &bar.full[stage]);
    if (DUAL) {
      tma_load_3d(s + 16384, &map.w2, kb * 128, w.n0, w.group, &bar.full[stage]);
      tma_load_3d(s + S::RA + 2048, &map.ws2, kb * 16, w.n0, w.group, &bar.full[stage]);
    }
  };
  auto tokens = [&](const F4Work& w, int kb, int stage) {
    uint8_t* s = smem + (size_t)stage * S::STAGE;
    for (int b = 0; b * S::BOX < w.rows; ++b) {
      tma_load_3d(s + S::B + b * S::BOX * 128, &map.x, kb * 128, w.row0 + b * S::BOX, 0, &bar.full[stage]);
      tma_load_3d(s + S::RB + b * S::BOX * 16, &map.xs, kb * 16, w.row0 + b * S::BOX, 0, &bar.full[stage]);
    }
  };
  const int n = tiles.count();
  int issued = 0, i = 0, kb = 0;
  F4Work w{};
  if (n > 0) { w = tiles.at(0); kb = w.kb0; }
  auto step = [&] { if (++kb == w.kb1 && ++i < n) { w = tiles.at(i); kb = w.kb0; } };
  for (; issued < S::STAGES && i < n; ++issued, step()) weights(w, kb, issued);
  if (n > 0 && ready()) {
    const int first = issued;
    i = 0; w = tiles.at(0); kb = w.kb0;
    for (int s = 0; s < first; ++s, step()) tokens(w, kb, s);
    int stage = first == S::STAGES ? 0 : first;
    uint32_t phase = first == S::STAGES;
    for (; i < n; ++issued, step()) {
      if (!mbar_wait(&bar.empty[stage], phase ^ 1, abort_flag)) break;
      weights(w, kb, stage);
      tokens(w, kb, stage);
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
  }
  if (*abort_flag) {
    // copies of this thread may still be landing in shared memory: the CTA must not exit under them
    unsigned long long t0 = globaltimer();
    while (issued > 0 && globaltimer() - t0 < 2000000ull) {}
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

// Warps 6 (weights) and 7 (tokens).
template <bool DUAL, class S, class Tiles>
__device__ __forceinline__ void f4_turn(uint8_t* smem, F4Bars<S>& bar, Tiles& tiles) {
  volatile int* abort_flag = &bar.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int stage = 0; uint32_t phase = 0;
  const int n = tiles.count();
  for (int i = 0; i < n; ++i) {
    const F4Work w = tiles.at(i);
    const int groups = (w.rows + 31) / 32;
    for (int kb = w.kb0; kb < w.kb1; ++kb) {
      if (!mbar_wait_warp(&bar.full[stage], phase, abort_flag)) return;
      uint8_t* s = smem + (size_t)stage * S::STAGE;
      if (warp == 6) {
#pragma unroll
        for (int m = 0; m < S::MATS; ++m)
          fp4_turn_scales(reinterpret_cast<const uint4*>(s + S::RA + 2048 * m), reinterpret_cast<uint4*>(s + S::TA + 2048 * m), lane, 4);
      } else {
#pragma unroll
        for (int h = 0; h < S::B_CELLS / 4; ++h)
          fp4_turn_scales(reinterpret_cast<const uint4*>(s + S::RB + 2048 * h), reinterpret_cast<uint4*>(s + S::TB + 2048 * h), lane, groups - 4 * h);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.cells[stage]);
      if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
  }
}

template <bool DUAL, class S>
static int f4_maps(F4Maps* m, const void* x, long rows_x, const void* w, const void* w2, int K, int N, int groups) {
  int rc = fp4_maps(&m->x, &m->xs, x, K, rows_x, 1, S::BOX);
  if (!rc) rc = fp4_maps(&m->w, &m->ws, w, K, N, groups, 128);
  m->w2 = m->w; m->ws2 = m->ws;
  if (!rc && DUAL) rc = fp4_maps(&m->w2, &m->ws2, w2, K, N, groups, 128);
  return rc;
}

}  // namespace bl
