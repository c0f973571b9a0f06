// kf_attention_chunk.h -- a chunk of tokens of linear attention: its decays, and how the time axis is split over workgroups.
#pragma once
#include "kf_frag.h"

constexpr int KF_CHUNK = 64;

// Decays of one chunk, G_i = sum of the log decays up to and with token i (summed in 64 bits; each exponent is rounded once).
// No exponent is positive: pairs (i, j) in different 16-token tiles take exp(G_i - G_j) as the product of two factors <= 1 that meet
// at the end of j's tile, so that only the tiles on the diagonal need an exponential for each pair.
template <int C>
struct KfChunkDecay {
  float from_start[C];            // exp(G_i): from the chunk's start through token i
  float to_end[C];                // exp(G_(C-1) - G_j): from behind token j to the chunk's end
  float to_tile_end[C];           // exp(G_e - G_j), e the last token of j's tile
  float from_tile[C / 16 - 1][C]; // exp(G_i - G_e), e the last token of an earlier tile
  float hi[C], lo[C];             // G in two floats, for the diagonal

  // by one whole wave, lane l with token l; tokens that are not `live` (lanes from C on are not) neither decay nor write
  __device__ __forceinline__ void fill(float log_decay, bool live) {
    const int l = threadIdx.x & 63;
    double G = live ? (double)kf_clamp_log_decay(log_decay) : 0.0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double x = __shfl_up(G, d);
      if (l >= d) G += x;
    }
    const double end = __shfl(G, 63), tile_end = __shfl(G, l | 15);
    float d[C / 16 - 1];
#pragma unroll
    for (int t = 0; t < C / 16 - 1; ++t) d[t] = (float)(G - __shfl(G, 16 * t + 15));
    if (l < C) {
      from_start[l] = expf((float)G);
      to_end[l] = expf((float)(end - G));
      to_tile_end[l] = expf((float)(tile_end - G));
#pragma unroll
      for (int t = 0; t < C / 16 - 1; ++t) from_tile[t][l] = expf(d[t] > 0.f ? 0.f : d[t]);  // (a NaN stays one)
      hi[l] = (float)G;
      lo[l] = (float)(G - (double)hi[l]);
    }
  }
  __device__ __forceinline__ float pair(int i, int j) const { return __expf((hi[i] - hi[j]) + (lo[i] - lo[j])); }
};

struct KfAttnSplit {
  long works;      // workgroups that have work
  int segments;    // of the time axis
  int seg_chunks;  // chunks of each
  int v_tiles;
  int vec_q, vec_k, vec_v, vec_g;  // rows may be read 16 bytes at a time
};

// Workgroup -> work, neighbours (the tiles of V and the heads that read the same q and k) on the same one of the 8 dies, whose
// L2 they share: workgroups go round the dies, so each die takes a run of consecutive works.
static __device__ __forceinline__ long kf_xcd_work(long works) {
  const long per = (works + 7) >> 3;
  return (blockIdx.x & 7) * per + (blockIdx.x >> 3);
}
static inline unsigned kf_xcd_grid(long works) { return (unsigned)(8 * ((works + 7) >> 3)); }

// A fragment of A stays aligned: base and every stride a multiple of 16 bytes.
static inline int kf_rows_aligned(const void* p, const long* strides, int n, int dim, int elem) {
  if (((uintptr_t)p & 15) || dim % 8) return 0;
  for (int i = 0; i < n; ++i)
    if ((strides[i] * elem) % 16) return 0;
  return 1;
}
