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
#include "common.cuh"

namespace bl {

constexpr int kMaxBeams = 64;

struct BeamArgs {
  const float* logits; long stride; int V, G, B;
  const float* scores;                                    // [G][B], -inf: no beam
  const int* done; const int* lengths;                    // optional [G][B]
  int eos; float alpha;
  double* lse;                                            // [G * B]
  int* parent; int* token; float* out_scores; int* out_done; int* out_lengths;
  unsigned* fault;
};

// grid (G * B), 512 threads: lse of a row; NaN where a logit is NaN or +inf
__global__ void __launch_bounds__(512) beam_lse_kernel(const BeamArgs a) {
  __shared__ float s_m[16];
  __shared__ double s_l[16];
  const int r = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  pdl_launch();
  const float* x = a.logits + (long)r * a.stride;
  if ((a.done && a.done[r]) || a.scores[r] == -INFINITY) return;
  float m = -INFINITY;
  bool bad = false;
  for (int t = tid; t < a.V; t += 512) { bad |= !(x[t] < INFINITY); m = fmaxf(m, x[t]); }
  m = warp_max(m);
  if ((tid & 31) == 0) s_m[tid >> 5] = m;
  bad = __syncthreads_or(bad);
  for (int w = 0; w < 16; ++w) m = fmaxf(m, s_m[w]);
  float l = 0.f;
  if (m > -INFINITY) for (int t = tid; t < a.V; t += 512) l += expf(x[t] - m);
  const double d = warp_sum_d((double)l);
  if ((tid & 31) == 0) s_l[tid >> 5] = d;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int w = 0; w < 16; ++w) all += s_l[w];
    a.lse[r] = bad ? (double)NAN : (double)m + log(all);
  }
}

// grid (G), 1024 threads: B rounds, each finds the best candidate behind the last one
__global__ void __launch_bounds__(1024) beam_pick_kernel(const BeamArgs a) {
  __shared__ double s_fac[kMaxBeams], s_key[32];
  __shared__ long s_at[32];
  const int g = blockIdx.x, tid = threadIdx.x, B = a.B, V = a.V, r0 = g * B;
  pdl_wait();
  pdl_launch();
  bool bad = false;
  if (tid < B) {
    const int r = r0 + tid;
    const bool over = a.done && a.done[r];
    const float sc = a.scores[r];
    bad = !(sc < INFINITY) || (!over && sc > -INFINITY && a.lse[r] != a.lse[r]);
    s_fac[tid] = a.alpha != 0.f ? pow((double)max(1, a.lengths[r] + (over ? 0 : 1)), -(double)a.alpha) : 1.0;
  }
  bad = __syncthreads_or(bad);
  double last = INFINITY;
  long last_at = -1;
  for (int i = 0; i < B; ++i) {
    double best = -INFINITY;
    long at = -1;
    auto offer = [&](double key, long where) {
      if (key > -INFINITY && (key < last || (key == last && where > last_at)) && (key > best || (key == best && where < at))) { best = key; at = where; }
    };
    for (int b = 0; !bad && b < B; ++b) {
      const int r = r0 + b;
      const double sc = a.scores[r];
      if (sc == -INFINITY) continue;
      if (a.done && a.done[r]) {
        if (tid == 0) offer(sc * s_fac[b], (long)b * V + a.eos);
        continue;
      }
      for (int t = tid; t < V; t += 1024) offer((sc + ((double)a.logits[(long)r * a.stride + t] - a.lse[r])) * s_fac[b], (long)b * V + t);
    }
    for (int o = 16; o > 0; o >>= 1) {
      const double k = __shfl_xor_sync(0xffffffffu, best, o);
      const long w = __shfl_xor_sync(0xffffffffu, at, o);
      if (w >= 0 && (at < 0 || k > best || (k == best && w < at))) { best = k; at = w; }
    }
    __syncthreads();
    if ((tid & 31) == 0) { s_key[tid >> 5] = best; s_at[tid >> 5] = at; }
    __syncthreads();
    for (int w = 0; w < 32; ++w)
      if (s_at[w] >= 0 && (at < 0 || s_key[w] > best || (s_key[w] == best && s_at[w] < at))) { best = s_key[w]; at = s_at[w]; }
    if (tid == 0) {
      const int p = at < 0 ? i : (int)(at / V), t = at < 0 ? max(a.eos, 0) : (int)(at % V), r = r0 + p;
      const bool over = a.done && a.done[r];
      a.parent[r0 + i] = p;
      a.token[r0 + i] = t;
      a.out_scores[r0 + i] = bad ? __int_as_float(0x7fc00000) : at < 0 ? -INFINITY : over ? a.scores[r]
                             : (float)((double)a.scores[r] + ((double)a.logits[(long)r * a.stride + t] - a.lse[r]));
      if (a.out_done) a.out_done[r0 + i] = at < 0 || over || t == a.eos;
      if (a.out_lengths) a.out_lengths[r0 + i] = a.lengths[r] + (at < 0 || over ? 0 : 1);
      if (bad && i == 0) raise_fault(a.fault, 0, FS_SAMPLER);
    }
    last = best;
    last_at = at;
    if (at < 0) last = -INFINITY;
  }
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

__device__ __forceinline__ void copy_bytes(uint8_t* dst, const uint8_t* src, int n) {
  const int n16 = n >> 4;
  for (int i = threadIdx.x; i < n16; i += blockDim.x) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
  const int rest = (n & 15) >> 2;
  if (threadIdx.x < rest) reinterpret_cast<uint32_t*>(dst + 16 * n16)[threadIdx.x] = reinterpret_cast<const uint32_t*>(src + 16 * n16)[threadIdx.x];
}

// grid (G * B, layers), 256 threads
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
  if (bad) {                                              // nobody moves
    if (tid == 0) raise_fault(a.fault, layer, FS_BEAM);
  } else {
    from = a.table + (long)a.slots[r0 + s_parent[i]] * a.max_pages;
    if (part) {
      const unsigned long long more = s_more[0] | (unsigned long long)s_more[1] << 32;
      unsigned long long bare = s_bare[0] | (unsigned long long)s_bare[1] << 32;
      place = from[col];
      if (more >> i & 1) {
        for (int n = __popcll(more & ((1ull << i) - 1)); n > 0; --n) bare &= bare - 1;
        source = place;
        place = a.table[(long)a.slots[r0 + __ffsll((long long)bare) - 1] * a.max_pages + col];
      }
    }
  }
  if (layer == 0) {
    int* to = a.table_out + (long)slot * a.max_pages;
    for (int c = tid; c < a.max_pages; c += 256) to[c] = !bad && c < col ? from[c] : place >= 0 && c == col ? place : own[c];
  }
  if (source < 0) return;
  if (source >= a.n_pages || place < 0 || place >= a.n_pages) { if (tid == 0) raise_fault(a.fault, layer, FS_PAGE); return; }
  for (int h = 0; h < a.n_kv; ++h) {
    const long src = ((long)layer * a.n_pages + source) * a.n_kv + h, dst = ((long)layer * a.n_pages + place) * a.n_kv + h;
    copy_bytes(a.k + dst * kBeamPage * a.k_row, a.k + src * kBeamPage * a.k_row, part * (int)a.k_row);
    if (a.v_row) copy_bytes(a.v + dst * kBeamPage * a.v_row, a.v + src * kBeamPage * a.v_row, part * (int)a.v_row);
  }
}

}  // namespace bl

using namespace bl;

extern "C" {

int bl_beam_select(const float* logits, long stride, int V, int G, int B, const float* scores, const int* done, const int* lengths,
                   int eos, float alpha, void* work, int* parent, int* token, float* out_scores, int* out_done, int* out_lengths,
                   unsigned* fault, cudaStream_t st) {
  BL_REQUIRE(V >= 1 && G >= 1 && B >= 1 && stride >= V, BL_ERR_SHAPE);
  BL_REQUIRE(B <= kMaxBeams && (long)G * B <= 65535, BL_ERR_LIMIT);
  BL_REQUIRE(eos < V && (!done || eos >= 0) && (alpha == 0.f || lengths) && (!out_lengths || lengths), BL_ERR_SHAPE);
  BeamArgs a{logits, stride, V, G, B, scores, done, lengths, eos, alpha, (double*)work, parent, token, out_scores, out_done,
             out_lengths, fault};
  cudaError_t e = launch(beam_lse_kernel, dim3(G * B), dim3(512), 0, st, a);
  if (e != cudaSuccess) return (int)e;
  return (int)launch(beam_pick_kernel, dim3(G), dim3(1024), 0, st, a);
}

int bl_beam_reorder(void* k, void* v, long k_row, long v_row, int n_layer, int n_pages, int n_kv, const int* table, int* table_out,
                    int n_slots, int max_pages, const int* slots, const int* parent, const int* held, int G, int B, unsigned* fault,
                    cudaStream_t st) {
  BL_REQUIRE(n_layer >= 1 && n_layer <= 65535 && n_pages >= 1 && n_kv >= 1 && G >= 1 && B >= 1 && n_slots >= 1 && max_pages >= 1,
             BL_ERR_SHAPE);
  BL_REQUIRE(B <= kMaxBeams, BL_ERR_LIMIT);
  BL_REQUIRE(k_row >= 4 && v_row >= 0 && table != table_out, BL_ERR_SHAPE);
  BL_REQUIRE(k_row % 4 == 0 && v_row % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, BL_ERR_ALIGN);
  ReorderArgs a{(uint8_t*)k, (uint8_t*)v, k_row, v_row, n_pages, n_kv, G, B, n_slots, max_pages, table, table_out, slots, parent, held, fault};
  return (int)launch(beam_reorder_kernel, dim3(G * B, n_layer), dim3(256), 0, st, a);
}

}  // extern "C"
