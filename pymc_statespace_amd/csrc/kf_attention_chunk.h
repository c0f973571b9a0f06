// kf_attention_chunk.h -- a chunk of tokens of linear attention: its decays, and how the time axis is split over workgroups.
#pragma once
#include "kf_frag.h"

constexpr int KF_CHUNK = 64;

template <int N> static __device__ __forceinline__ double kf_row_shr(double x) {  // from N lanes below in the row of 16, 0 from outside
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), 0x110 + N, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), 0x110 + N, 0xf, 0xf, true);
  return __hiloint2double(hi, lo);
}
static __device__ __forceinline__ double kf_readlane(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane), __builtin_amdgcn_readlane(__double2loint(x), lane));
}

// A segment's decay is handed on as its square root, and a state multiplied by that twice: positive log decays may come to more over a
// segment than fp32 holds while every state stays inside (a zero one, for instance, which must not meet an infinity).  The root of what
// does not fit either is the largest number: it takes any state that is not zero out of range, as the growth itself would.
static __device__ __forceinline__ bool kf_too_large(float x) { return x > 3.402823466e38f; }
static __device__ __forceinline__ float kf_root_decay(float x) { return kf_too_large(x) ? 3.402823466e38f : x; }

// Decays of one chunk, G_i = sum of the log decays up to and with token i (summed in 64 bits; each exponent is rounded once).
// No exponent is positive: pairs (i, j) in different 16-token tiles take exp(G_i - G_j) as the product of two factors <= 1 that meet
// at the end of j's tile, so that only the tiles on the diagonal need an exponential for each pair.
template <int C>
struct alignas(16) KfChunkDecay {  // (its rows are read 16 bytes at a time)
  float from_start[C];            // exp(G_i): from the chunk's start through token i
  float to_end[C];                // exp(G_(C-1) - G_j): from behind token j to the chunk's end
  float to_tile_end[C];           // exp(G_e - G_j), e the last token of j's tile
  float from_tile[C / 16 - 1][C]; // exp(G_i - G_e), e the last token of an earlier tile
  float hi[C], lo[C];             // G in two floats, for the diagonal
  float root;                     // exp(G_(C-1) / 2), see kf_root_decay

  // by one whole wave, lane l with token l; tokens that are not `live` (lanes from C on are not) neither decay nor write
  // (ROOT: `root` too, for what sums up segments)
  template <bool ROOT> __device__ __forceinline__ void fill(float log_decay, bool live) {
    const int l = threadIdx.x & 63, row = l >> 4;
    double G = live ? (double)kf_clamp_log_decay(log_decay) : 0.0;
    // running sums inside each row of 16 lanes, then over the rows
    G += kf_row_shr<1>(G);
    G += kf_row_shr<2>(G);
    G += kf_row_shr<4>(G);
    G += kf_row_shr<8>(G);
    double end[4];  // G at the end of each tile
    end[0] = kf_readlane(G, 15);
    end[1] = end[0] + kf_readlane(G, 31);
    end[2] = end[1] + kf_readlane(G, 47);
    end[3] = end[2] + kf_readlane(G, 63);
    G += row == 0 ? 0.0 : row == 1 ? end[0] : row == 2 ? end[1] : end[2];
    if (l < C) {
      from_start[l] = __expf((float)G);
      to_end[l] = __expf((float)(end[C / 16 - 1] - G));
      to_tile_end[l] = __expf((float)((row == 0 ? end[0] : row == 1 ? end[1] : row == 2 ? end[2] : end[3]) - G));
#pragma unroll
      for (int t = 0; t < C / 16 - 1; ++t) {
        from_tile[t][l] = row > t ? __expf((float)(G - end[t])) : 0.f;
      }
      if (ROOT && l == 0) root = kf_root_decay(__expf((float)(0.5 * end[C / 16 - 1])));
      hi[l] = (float)G;
      lo[l] = (float)(G - (double)hi[l]);
    }
  }
  // exp(G_i - G_j) for j .. j + 3 (of the same tile; where j is behind i the value means nothing, and may be infinite)
  __device__ __forceinline__ kf_f32x4 pairs(int i, int j) const {
    const float h = hi[i], s = lo[i];
    const kf_f32x4 hj = *reinterpret_cast<const kf_f32x4*>(&hi[j]), sj = *reinterpret_cast<const kf_f32x4*>(&lo[j]);
    kf_f32x4 e;
#pragma unroll
    for (int r = 0; r < 4; ++r) e[r] = __expf((h - hj[r]) + (s - sj[r]));
    return e;
  }
};

// What each segment adds to a state (slots 0 .. n - 1 of `cells` 16-byte pieces for each head) into the state that the next segment
// starts from, in place; products[s]: what becomes of a state from before all of them (its square root, like the factors).  `back`: from
// the last slot to the first, with the decay of the segment behind each slot.  Up to KF_FUSED_SEGMENTS segments each workgroup sums up what is before it by itself
// (about 0.4 us for each 64 KB); beyond, this kernel (4 to 6 us) is the shorter way and keeps the sum linear in their number.
constexpr int KF_FUSED_SEGMENTS = 8;
static __global__ __launch_bounds__(256) void kf_attention_scan_kernel(kf_f32x4* adds_s, kf_f32x4* adds_r, const float* factors, float* products_s,
                                                                       float* products_r, long heads, int n, long cells, int factor_stride,
                                                                       int threads, int V, int K) {
  const long x = (long)blockIdx.x * 256 + threadIdx.x;
  if (x >= heads * cells) return;
  const bool back = blockIdx.y;  // (the gradient's second state)
  kf_f32x4* adds = back ? adds_r : adds_s;
  float* products = back ? products_r : products_s;
  const long head = x / cells, e = x - head * cells;
  if (threads) {  // (the gradient's states: tile e / threads of V, tile of K by wave; those of nothing but padding are not kept)
    const int t = (int)(e / threads), w = (int)(e - (long)t * threads) >> 6;
    if (16 * t >= V || 16 * w >= K) return;
  }
  kf_f32x4* a = adds + head * n * cells + e;
  const float* f = factors + head * factor_stride + (back ? 1 : 0);
  kf_f32x4 sum = {0, 0, 0, 0};
  float product = 1.f;
  for (int s0 = 0; s0 < n; s0 += 8) {
    kf_f32x4 in[8];
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int s = s0 + j < n ? s0 + j : n - 1, slot = back ? n - 1 - s : s;
      in[j] = a[slot * cells];
      d[j] = f[slot];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s0 + j < n) {
        const int slot = back ? n - 1 - s0 - j : s0 + j;
        sum = sum * d[j] * d[j] + in[j];
        product = kf_root_decay(product * d[j]);
        a[slot * cells] = sum;
        if (e == 0) products[head * n + slot] = product;
      }
  }
}
static inline void kf_attention_scan(float* adds_s, float* adds_r, const float* factors, float* products_s, float* products_r, long heads, int n,
                                     long floats, int factor_stride, int threads, int V, int K, hipStream_t stream) {
  hipLaunchKernelGGL(kf_attention_scan_kernel, dim3((unsigned)((heads * (floats / 4) + 255) / 256), adds_r ? 2 : 1), dim3(256), 0, stream,
                     (kf_f32x4*)adds_s, (kf_f32x4*)adds_r, factors, products_s, products_r, heads, n, floats / 4, factor_stride, threads, V, K);
}

struct KfAttnSplit {
  long works;      // workgroups that have work
  int segments;    // of the time axis
  int seg_chunks;  // chunks of each
  int v_tiles;
};

// Workgroup -> work, neighbours (the tiles of V and the heads that read the same q and k) on the same one of the 8 dies, whose
// L2 they share: workgroups go round the dies, so each die takes a run of consecutive works.
static __device__ __forceinline__ long kf_xcd_work(long works) {
  const long per = (works + 7) >> 3;
  return (blockIdx.x & 7) * per + (blockIdx.x >> 3);
}
// (the last workgroup has the highest work: none where the division leaves a rest, and then it is not launched.  A launch has fewer than
// 2^32 threads, and 4 tiles of V of 2^22 - 1 heads, 256 threads each, would come to 2^32 with it)
static inline unsigned kf_xcd_grid(long works) { return (unsigned)(8 * ((works + 7) >> 3) - (works % 8 != 0)); }
