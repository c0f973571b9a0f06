// kf_attention_backward.hip -- the gradient of linear attention with a decay for each head, in chunks of C tokens.
//
// With S_0 the state at a chunk's start, R = dL/dS behind its last token, G_i the log decays summed through token i, E the chunk's
// whole decay, D_ij = e^{G_i - G_j} for j <= i, A_ij = q_i . k_j, B_ij = do_i . v_j:
//     dq_i = s [ e^{G_i} S_0 do_i + sum_j D_ij B_ij k_j ]
//     dk_j = e^{G_C - G_j} R v_j + s sum_i D_ij B_ij q_i
//     dv_j = e^{G_C - G_j} R' k_j + s sum_i D_ij A_ij do_i
//     dL/d log a_t = sum_{i >= t} (sum_j W_ij + q_i . dq_i|state) - sum_{j >= t} sum_i W_ij + sum_{j < t} k_j . dk_j|state + E <R, S_0>
// with W_ij = s D_ij A_ij B_ij: what passes through the decay of token t.  All of it from this chunk's own numbers (the shorter form,
// a running sum of q.dq - k.dk over the whole sequence, loses what those sums share).  Then R <- E R + sum_i s e^{G_i} q_i do_i'.
//
// Roundings (bf16 data): scores times their decays, and R where the keys meet it for dv, 2^-9 each, like the gradients themselves.  What
// enters fp32 results -- dq and dk through the states, whose products with q and k are part of the decays' gradient, and the sums of S
// and R -- is multiplied in three exact parts.  fp32 and fp16 data: fp32 throughout.
//
// Measured: 4 x 2048 tokens, 16 heads of 128 x 128, bf16: 41 + 40 + 117 us (187 without a profiler) for 236 MB (50 us at the 4.7 TB/s of a large copy); 134 MB of
// starts are written and read on top.  16 x 128 tokens, 8 heads of 64 x 64, fp16: 9 + 18 us.  3 x 333 ragged tokens, 6 heads of 40 x 72
// on 2 groups, fp32: 12 + 7 + 24 + 4 us.  The gradient kernel has one workgroup on a compute unit (148 KB of LDS, 256 registers), whose
// 8 waves go through the chunk's phases together: 1590 vector instructions a wave and chunk (split operands: 440) are 41 % of its time,
// LDS 20 %, the matrix pipe 19 %, waits 40 %.  Without the fences between depths the compiler holds all of them at once and spills: 325 us.
// The same batch in fp16 393 us, in fp32 410 (eight fp32 instructions for one of bf16).  K or V below 8 takes the 128-wide kernel with loads
// of single elements, whose bf16 instance spills 29 registers: 16 heads of 4 x 4 196 us.
//
// Launches: (1) where the time axis is cut into segments, what each segment adds to S and to R; (2) where segments have several chunks,
// S at every chunk's start, kept as the accumulators that hold it; (3) the chunks of each segment from its last to its first, R in registers; (4) sums over
// the heads that share queries and keys, and over tokens for fixed decays.
#include "kf_attention_chunk.h"

namespace {

// K and V are padded to one size D; a workgroup has D / 16 waves, wave w has columns 16 w .. of K (in dv: of V).
template <typename A> constexpr int chunk_of() { return sizeof(typename A::elem) == 2 ? 64 : 32; }  // fp32 tiles are twice as wide: half as many tokens

struct Split {
  long works;
  int segments, seg_chunks;
  long chunks;
  float *adds_s, *adds_r, *factors;  // [B H][segments - 1][D D], [B H][segments] (the root of each segment's whole decay)
  float *products_s, *products_r;    // [B H][segments - 1]: see kf_attention_scan_kernel
  kf_f32x4* starts;                  // S_0 of every chunk: [B H][chunks][D / 16][threads]
  float *part_q, *part_k;            // [B][T][H][K], where heads share q and k
  double* part_decay;                // [B H][segments], where decays are fixed
};

template <int C, typename A, typename T, int D, int MODE>
struct Stage {  // C rows of a tensor through registers into LDS
  typedef KfRow<A, T, MODE> Row;
  typedef KfTile<A, D> Tile;
  static constexpr int N = C * D / 8 / (4 * D);
  typename Row::Raw r[N];
  static __device__ __forceinline__ int last_row(long t0, long n) { return (int)(n - t0 < C ? n - t0 : C) - 1; }
  __device__ __forceinline__ void load(const T* p, long stride, long t0, long n, int dim) {  // t0 < n
    const int last = last_row(t0, n), row0 = threadIdx.x / (D / 8), col = 8 * (threadIdx.x % (D / 8));
    const T* base = p + t0 * stride;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int row = row0 + 32 * u;
      r[u] = Row::raw(base, (unsigned)__umul24((unsigned)(row < last ? row : last), (unsigned)stride), col, dim);
    }
  }
  __device__ __forceinline__ void put(typename A::elem* s, long t0, long n, int dim) const {  // the chunk that was loaded
    const int last = last_row(t0, n), row0 = threadIdx.x / (D / 8), col = 8 * (threadIdx.x % (D / 8));
#pragma unroll
    for (int u = 0; u < N; ++u) Tile::put8(s, row0 + 32 * u, col, Row::finish(r[u], col, dim, row0 + 32 * u <= last));
  }
};

// One sweep over a segment's chunks of acc[v][k] <- E acc + sum_t weight_t y_t x_t': S (x = k, y = v, forward in time) or R (x = q,
// y = do, backward).  STARTS: S, started from the segments before, kept at every chunk's start; else what the segment adds.
template <typename A, typename T, int D, int MODE, bool STARTS>
__global__ __launch_bounds__(4 * D) void attention_sweep_kernel(KfAttnArgs a, Split sp) {
  constexpr int C = chunk_of<A>(), NT = D / 16, TH = 4 * D;
  typedef typename A::elem E;
  typedef KfTile<A, D> TD;
  __shared__ __attribute__((aligned(16))) E sX[C * D];
  __shared__ __attribute__((aligned(16))) E sY[C * D];
  __shared__ KfChunkDecay<C> dec[2];
  const long work = kf_xcd_work(sp.works);
  if (work >= sp.works) return;
  const int segs = STARTS ? sp.segments : sp.segments - 1;
  long rest = work;
  bool back = false;
  if (!STARTS) {
    back = rest & 1;
    rest >>= 1;
  }
  const int h = (int)(rest % a.H);
  rest /= a.H;
  const int s0 = (int)(rest % segs);
  const long b = rest / segs;
  const int seg = back ? s0 + 1 : s0;  // (nothing is behind the last segment, nothing before the first)
  const long bh = b * a.H + h;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 15, g = l >> 4;
  const KfLanes lt = TD::lanes(i, g);
  const long n = kf_row_length(a.lengths, b, a.T);
  const int grp = h / (a.H / a.G);
  const T* x = back ? (const T*)a.q + b * a.qs[0] + grp * a.qs[2] : (const T*)a.k + b * a.ks[0] + grp * a.ks[2];
  const T* y = back ? (const T*)a.g_o + b * a.gs[0] + h * a.gs[2] : (const T*)a.v + b * a.vs[0] + h * a.vs[2];
  const long xs = back ? a.qs[1] : a.ks[1], ys = back ? a.gs[1] : a.vs[1];
  const float* ld = a.log_decay + (a.per_token ? b * a.T * a.H + h : (long)h);
  const long c0 = (long)seg * sp.seg_chunks, c1 = c0 + sp.seg_chunks < sp.chunks ? c0 + sp.seg_chunks : sp.chunks;
  const long live = (n + C - 1) / C, last = c1 < live ? c1 : live;  // chunks that hold tokens: c0 .. last - 1

  // tiles of nothing but padding are not kept; where one would be read, the first one is, which is there already, and left out
  auto real = [&](int t) { return 16 * t < a.V && 16 * w < a.K; };
  auto add = [&](kf_f32x4& x, float f, const kf_f32x4* u, int t) {
    const kf_f32x4 y = u[real(t) ? t * TH : 0];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = real(t) ? x[r] * f * f + y[r] : x[r];
  };
  kf_f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    acc[t] = kf_f32x4{0, 0, 0, 0};
    const int kk = 16 * w + i;
    if (STARTS && a.s0 && kk < a.K) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * t + 4 * g + r < a.V) acc[t][r] = a.s0[(bh * a.K + kk) * a.V + 16 * t + 4 * g + r];
    }
  }
  if (STARTS) {
    const bool summed = sp.segments > KF_FUSED_SEGMENTS;
    for (int s = summed && seg ? seg - 1 : 0; s < seg; ++s) {
      const float f = summed ? sp.products_s[bh * (sp.segments - 1) + s] : sp.factors[bh * sp.segments + s];
      const kf_f32x4* u = reinterpret_cast<const kf_f32x4*>(sp.adds_s) + (bh * (sp.segments - 1) + s) * (D * D / 4) + tid;
#pragma unroll
      for (int t = 0; t < NT; ++t) add(acc[t], f, u, t);
    }
  }
  float through = 1.f;  // the root of the segment's decay
  Stage<C, A, T, D, MODE> rx, ry;
  float rg = 0.f;
  const long steps = last > c0 ? last - c0 : 0;
  auto at = [&](long s) { return back ? last - 1 - s : c0 + s; };
  const long ld_step = a.per_token ? a.H : 0;
  auto decay_of = [&](long c) { return ld[(c * C + l < 0 ? 0 : c * C + l < n ? c * C + l : n - 1) * ld_step]; };  // (in bounds for any c)
  if (steps) {
    rx.load(x, xs, at(0) * C, n, a.K);
    ry.load(y, ys, at(0) * C, n, a.V);
    rg = decay_of(at(1));
    if (w == 0) dec[0].template fill<!STARTS>(decay_of(at(0)), l < C && at(0) * C + l < n);
  }
  for (long s = 0; s < steps; ++s) {
    if (STARTS) {
      kf_f32x4* out = sp.starts + (bh * sp.chunks + at(s)) * (D / 32 * 2 * TH) + tid;
#pragma unroll
      for (int u = 0; u < D / 32; ++u) {
        out[(2 * u) * TH] = acc[2 * u];
        out[(2 * u + 1) * TH] = acc[2 * u + 1];
      }
      if (s + 1 == steps) break;  // (the next segment starts from what was summed up for it)
    }
    rx.put(sX, at(s) * C, n, a.K);
    ry.put(sY, at(s) * C, n, a.V);
    __syncthreads();
    // (loads that no branch surrounds, so that each wait is for its own: behind the last chunk the same one again)
    const long next = s + 1 < steps ? s + 1 : s;
    const float g1 = rg;
    rg = decay_of(at(s + 2));
    rx.load(x, xs, at(next) * C, n, a.K);
    ry.load(y, ys, at(next) * C, n, a.V);
    if (w == (int)(s % NT)) dec[(s + 1) & 1].template fill<!STARTS>(g1, l < C && at(s + 1) >= 0 && at(s + 1) * C + l < n);
    const KfChunkDecay<C>& d = dec[s & 1];
    const float fe = d.from_start[C - 1];
    if (!STARTS) through = kf_root_decay(through * d.root);
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] *= fe;
#pragma unroll
    for (int u = 0; u < C / 32; ++u) {
      float wt[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int tok = 32 * u + 16 * (e >> 2) + 4 * g + (e & 3);
        wt[e] = back ? d.from_start[tok] * a.scale : d.to_end[tok];
      }
      KfSplit<A> xw;
      xw.set(TD::col(sX, lt, 32 * u, 16 * w), wt);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = xw.mma_right(TD::col(sY, lt, 32 * u, 16 * t), acc[t]);
    }
    __syncthreads();
  }
  if (!STARTS) {
    kf_f32x4* u = reinterpret_cast<kf_f32x4*>(back ? sp.adds_r : sp.adds_s) + (bh * (sp.segments - 1) + s0) * (D * D / 4) + tid;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (real(t)) u[t * TH] = acc[t];
    // (each segment's decay from one of the sweeps that pass through it: the first from S, the others from R)
    if (tid == 0 && (back || s0 == 0)) sp.factors[bh * sp.segments + seg] = through;
  }
}

template <typename A, typename T, int D, int MODE>
__global__ __launch_bounds__(4 * D, 2) void attention_gradient_kernel(KfAttnArgs a, Split sp) {
  constexpr int C = chunk_of<A>(), NT = D / 16, CT = C / 16, TH = 4 * D;
  typedef KfTile<A, D> TD;  // rows of q, k, v, do, R
  typedef KfTile<A, C> TC;  // rows of scores
  typedef typename A::elem E;
  typedef typename A::frag F;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  E* sQ = (E*)smem;
  E* sK = sQ + C * D;
  E* sV = sK + C * D;
  E* sG = sV + C * D;
  E* sR = sG + C * D;   // R as an operand, [k][v]
  E* sP = sR + D * D;   // s D A, [i][j]
  E* sB = sP + C * C;   // s D B
  KfChunkDecay<C>* dec = (KfChunkDecay<C>*)(sB + C * C);
  float* rs = (float*)(dec + 2);  // [CT][C]: sums of W over the columns of one tile
  float* cs = rs + CT * C;        // [CT][C]: over the rows
  float* xs = cs + CT * C;        // [NT][C]: q . dq|state, this wave's columns of K
  float* ys = xs + NT * C;        // [NT][C]: k . dk|state
  float* cr = ys + NT * C;        // [NT]: <R, S_0>

  const long work = kf_xcd_work(sp.works);
  if (work >= sp.works) return;
  long rest = work;
  const int h = (int)(rest % a.H);
  rest /= a.H;
  const int seg = (int)(rest % sp.segments);
  const long b = rest / sp.segments;
  const long bh = b * a.H + h;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 15, g = l >> 4;
  const KfLanes lt0 = TD::lanes(i, g), lc0 = TC::lanes(i, g);
  KfLanes lt = lt0, lc = lc0;
  // each part of the loop builds its LDS addresses from these six anew: held across it they would not fit the registers
  auto fresh = [&]() {
    lt = kf_fresh(lt0);
    lc = kf_fresh(lc0);
  };
  const long n = kf_row_length(a.lengths, b, a.T);
  const int grp = h / (a.H / a.G);
  const T* q = (const T*)a.q + b * a.qs[0] + grp * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + grp * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[2];
  const T* go = (const T*)a.g_o + b * a.gs[0] + h * a.gs[2];
  const float* ld = a.log_decay + (a.per_token ? b * a.T * a.H + h : (long)h);
  const long c0 = (long)seg * sp.seg_chunks, c1 = c0 + sp.seg_chunks < sp.chunks ? c0 + sp.seg_chunks : sp.chunks;
  const long live = (n + C - 1) / C, last = c1 < live ? c1 : live;
  const bool shared_heads = a.G != a.H;

  auto real = [&](int t) { return 16 * t < a.V && 16 * w < a.K; };
  auto add = [&](kf_f32x4& x, float f, const kf_f32x4* u, int t) {  // as in the sweeps
    const kf_f32x4 y = u[real(t) ? t * TH : 0];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = real(t) ? x[r] * f * f + y[r] : x[r];
  };
  kf_f32x4 R[NT];  // rows v, columns k
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    R[t] = kf_f32x4{0, 0, 0, 0};
    const int kk = 16 * w + i;
    if (a.g_sT && kk < a.K) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * t + 4 * g + r < a.V) R[t][r] = a.g_sT[(bh * a.K + kk) * a.V + 16 * t + 4 * g + r];
    }
  }
  const bool summed = sp.segments > KF_FUSED_SEGMENTS;
  for (int s = summed && seg + 1 < sp.segments ? seg + 1 : sp.segments - 1; s > seg; --s) {
    const float f = summed ? sp.products_r[bh * (sp.segments - 1) + s - 1] : sp.factors[bh * sp.segments + s];
    const kf_f32x4* u = reinterpret_cast<const kf_f32x4*>(sp.adds_r) + (bh * (sp.segments - 1) + s - 1) * (D * D / 4) + tid;
#pragma unroll
    for (int t = 0; t < NT; ++t) add(R[t], f, u, t);
  }

  // gradients of rows behind the sequence's end
  {
    const long lo = (last > c0 ? last : c0) * C, hi = c1 * C < a.T ? c1 * C : a.T;
    for (long t = lo + tid / D; t < hi; t += 4) {
      const int c = tid % D;
      const long row = (b * a.T + t) * a.H + h;
      if (c < a.V) ((T*)a.g_v)[row * a.V + c] = kf_from_float<T>(0.f);
      if (c < a.K) {
        if (shared_heads) {
          sp.part_q[row * a.K + c] = 0.f;
          sp.part_k[row * a.K + c] = 0.f;
        } else {
          ((T*)a.g_q)[row * a.K + c] = kf_from_float<T>(0.f);
          ((T*)a.g_k)[row * a.K + c] = kf_from_float<T>(0.f);
        }
      }
      if (a.per_token && c == 0) a.g_decay[row] = 0.f;
    }
  }
  for (int x = tid; x < 2 * C * C; x += TH) sP[x] = E(0);  // tiles above the diagonal stay zero

  Stage<C, A, T, D, MODE> rq, rk, rv, rd;
  float rg = 0.f;
  kf_f32x4 S0[NT];
  auto load = [&](long c) {
    rq.load(q, a.qs[1], c * C, n, a.K);
    rk.load(k, a.ks[1], c * C, n, a.K);
    rv.load(v, a.vs[1], c * C, n, a.V);
    rd.load(go, a.gs[1], c * C, n, a.V);
  };
  const bool single = sp.seg_chunks == 1;
  auto load_start = [&](long c) {  // (a segment of one chunk: not asked for, but loaded without a branch, the same line each time)
    const kf_f32x4* in = sp.starts + (single ? 0 : (bh * sp.chunks + c) * (D / 32 * 2 * TH)) + tid;
    const int step = single ? 0 : TH;
#pragma unroll
    for (int u = 0; u < NT; ++u) S0[u] = in[u * step];
  };
  const long ld_step = a.per_token ? a.H : 0;
  auto decay_of = [&](long c) { return ld[(c * C + l < 0 ? 0 : c * C + l < n ? c * C + l : n - 1) * ld_step]; };  // (in bounds for any c)
  if (last > c0) {
    load(last - 1);
    if (single) {
      // the state at the segment's start, as the sweep over starts has it
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        S0[t] = kf_f32x4{0, 0, 0, 0};
        const int kk = 16 * w + i;
        if (a.s0 && kk < a.K) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * t + 4 * g + r < a.V) S0[t][r] = a.s0[(bh * a.K + kk) * a.V + 16 * t + 4 * g + r];
        }
      }
      for (int s = summed && seg ? seg - 1 : 0; s < seg; ++s) {
        const float f = summed ? sp.products_s[bh * (sp.segments - 1) + s] : sp.factors[bh * sp.segments + s];
        const kf_f32x4* u = reinterpret_cast<const kf_f32x4*>(sp.adds_s) + (bh * (sp.segments - 1) + s) * (D * D / 4) + tid;
#pragma unroll
        for (int t = 0; t < NT; ++t) add(S0[t], f, u, t);
      }
    } else {
      load_start(last - 1);
    }
    rg = decay_of(last - 2);
    if (w == 0) dec[0].template fill<false>(decay_of(last - 1), l < C && (last - 1) * C + l < n);
  }
  double decay_sum = 0.;
  int turn = 0;
  for (long c = last - 1; c >= c0; --c, turn ^= 1) {
    const long t0 = c * C;
    fresh();
    rq.put(sQ, t0, n, a.K);
    rk.put(sK, t0, n, a.K);
    rv.put(sV, t0, n, a.V);
    rd.put(sG, t0, n, a.V);
#pragma unroll
    for (int t = 0; t < NT; ++t) TD::put4(sR, lt, 16 * w, 16 * t, R[t]);
    __syncthreads();
    // (loads that no branch surrounds, so that each wait is for its own: before the first chunk the same one again)
    const long next = c > c0 ? c - 1 : c;
    const float g1 = rg;
    rg = decay_of(c - 2);
    load(next);
    if (w == NT - 1) dec[turn ^ 1].template fill<false>(g1, l < C && c > 0 && t0 - C + l < n);
    const KfChunkDecay<C>& d = dec[turn];

    // scores: tile (it, jt) of A and B, rows j, columns i
    fresh();
    for (int x = w; x < CT * (CT + 1) / 2; x += NT) {
      int it = 0;
      while ((it + 1) * (it + 2) / 2 <= x) ++it;
      const int jt = x - it * (it + 1) / 2, i1 = kf_fresh(i), gs = kf_fresh(g), row = 16 * it + i1;
      kf_f32x4 sa = {0, 0, 0, 0}, sb = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < D / 32; ++u) {
        sa = A::mma(TD::row(sK, lt, 16 * jt, 32 * u), TD::row(sQ, lt, 16 * it, 32 * u), sa);
        sb = A::mma(TD::row(sV, lt, 16 * jt, 32 * u), TD::row(sG, lt, 16 * it, 32 * u), sb);
      }
      kf_f32x4 p, pb, wj;
      float wi = 0.f;
      kf_f32x4 fac;
      if (it == jt) fac = d.pairs(row, 16 * jt + 4 * gs) * a.scale;
      else fac = *reinterpret_cast<const kf_f32x4*>(&d.to_tile_end[16 * jt + 4 * gs]) * (d.from_tile[jt][row] * a.scale);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * gs + r;
        const bool in = j <= row;
        const float f = fac[r];
        p[r] = in ? sa[r] * f : 0.f;
        pb[r] = in ? sb[r] * f : 0.f;
        wj[r] = in ? sa[r] * pb[r] : 0.f;
        wi += wj[r];
      }
      TC::put4(sP, lc, 16 * it, 16 * jt, p);
      TC::put4(sB, lc, 16 * it, 16 * jt, pb);
      wi += __shfl_xor(wi, 16);
      wi += __shfl_xor(wi, 32);
      if (gs == 0) rs[jt * C + row] = wi;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        wj[r] = kf_row_sum(wj[r]);
        if (i1 == 0) cs[it * C + 16 * jt + 4 * gs + r] = wj[r];
      }
    }

    // through the states; rows k (dv: rows v), columns tokens
    fresh();
    kf_f32x4 dq[CT], dk[CT], dv[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) dq[t] = dk[t] = dv[t] = kf_f32x4{0, 0, 0, 0};
    float cross = 0.f;
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
      __builtin_amdgcn_sched_barrier(0);  // (one depth at a time: all of them at once would not fit the registers)
      KfSplit<A> fs, fr;
      fs.set(S0[2 * u], S0[2 * u + 1]);
      fr.set(R[2 * u], R[2 * u + 1]);
#pragma unroll
      for (int e = 0; e < 8; ++e) cross += S0[2 * u + (e >> 2)][e & 3] * R[2 * u + (e >> 2)][e & 3];
      const F fc = TD::col(sR, lt, 32 * u, 16 * w);  // rows v of this wave, depth k
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        if (t && t % 2 == 0) __builtin_amdgcn_sched_barrier(0);
        dq[t] = fs.mma(TD::row_t(sG, lt, 16 * t, 32 * u), dq[t]);
        dk[t] = fr.mma(TD::row_t(sV, lt, 16 * t, 32 * u), dk[t]);
        dv[t] = A::mma(fc, TD::row_t(sK, lt, 16 * t, 32 * u), dv[t]);
      }
    }
    load_start(next);
    cross = kf_row_sum(cross);
    cross += __shfl_xor(cross, 16);
    cross += __shfl_xor(cross, 32);
    if (l == 0) cr[w] = cross;
    const int i1 = kf_fresh(i);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const int tok = 16 * t + i1;
      const float fi = a.scale * d.from_start[tok], fj = d.to_end[tok];
      dq[t] *= fi;
      dk[t] *= fj;
      dv[t] *= fj;
      const kf_f32x4 qv = TD::get4(sQ, lt, 16 * t, 16 * w), kv = TD::get4(sK, lt, 16 * t, 16 * w);
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x += qv[r] * dq[t][r];
        y += kv[r] * dk[t][r];
      }
      x += __shfl_xor(x, 16);
      x += __shfl_xor(x, 32);
      y += __shfl_xor(y, 16);
      y += __shfl_xor(y, 32);
      if (g == 0) {
        xs[w * C + tok] = x;
        ys[w * C + tok] = y;
      }
    }
    __syncthreads();

    // inside the chunk, and R at its start
    fresh();
    const float fe = d.from_start[C - 1];
#pragma unroll
    for (int t = 0; t < NT; ++t) R[t] *= fe;
#pragma unroll
    for (int u = 0; u < C / 32; ++u) {
      __builtin_amdgcn_sched_barrier(0);
      const F ck = TD::col(sK, lt, 32 * u, 16 * w), cq = TD::col(sQ, lt, 32 * u, 16 * w),
              cg = TD::col(sG, lt, 32 * u, 16 * w);
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        if (2 * u <= t) dq[t] = A::mma(ck, TC::row_t(sB, lc, 16 * t, 32 * u), dq[t]);
        if (2 * u + 1 >= t) {
          dk[t] = A::mma(cq, TC::col(sB, lc, 32 * u, 16 * t), dk[t]);
          dv[t] = A::mma(cg, TC::col(sP, lc, 32 * u, 16 * t), dv[t]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      float wt[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) wt[e] = a.scale * d.from_start[32 * u + 16 * (e >> 2) + 4 * g + (e & 3)];
      KfSplit<A> qw;
      qw.set(cq, wt);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t && t % 4 == 0) __builtin_amdgcn_sched_barrier(0);
        R[t] = qw.mma_right(TD::col(sG, lt, 32 * u, 16 * t), R[t]);
      }
    }
    const int c4 = 16 * w + 4 * kf_fresh(g);
    long row = (b * a.T + t0 + kf_fresh(i)) * a.H + h;
#pragma unroll
    for (int t = 0; t < CT; ++t, row += 16 * a.H) {
      const long tok = t0 + 16 * t + i;
      if (tok < a.T) {
        if (tok >= n) dq[t] = dk[t] = dv[t] = kf_f32x4{0, 0, 0, 0};
        kf_store4((T*)a.g_v + row * a.V + c4, dv[t], a.V - c4);
        if (shared_heads) {
          kf_store4(sp.part_q + row * a.K + c4, dq[t], a.K - c4);
          kf_store4(sp.part_k + row * a.K + c4, dk[t], a.K - c4);
        } else {
          kf_store4((T*)a.g_q + row * a.K + c4, dq[t], a.K - c4);
          kf_store4((T*)a.g_k + row * a.K + c4, dk[t], a.K - c4);
        }
      }
    }
    if (w == 0) {
      // d log a: token t0 + l (its sums are complete since the barrier above)
      const bool tok = l < C;
      double up = 0., down = 0., all = 0.;
      if (tok) {
        for (int x = 0; x < CT; ++x) up += (x <= (l >> 4) ? (double)rs[x * C + l] : 0.) - (x >= (l >> 4) ? (double)cs[x * C + l] : 0.);
        for (int x = 0; x < NT; ++x) {
          up += (double)xs[x * C + l];
          down += (double)ys[x * C + l];
        }
      }
      for (int x = 0; x < NT; ++x) all += (double)cr[x];
      const double own = down;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const double su = __shfl_down(up, m), sd = __shfl_up(down, m);
        if (l + m < 64) up += su;
        if (l >= m) down += sd;
      }
      const double dg = up + (down - own) + all * (double)fe;
      const long t = t0 + l;
      const bool valid = tok && t < n;
      if (a.per_token) {
        if (tok && t < a.T) a.g_decay[(b * a.T + t) * a.H + h] = valid ? (float)dg : 0.f;
      } else {
        decay_sum += valid ? dg : 0.;
      }
    }
    __syncthreads();
  }
  if (!a.per_token && w == 0) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) decay_sum += __shfl_xor(decay_sum, m);
    if (l == 0) sp.part_decay[bh * sp.segments + seg] = decay_sum;
  }
  if (a.g_s0 && seg == 0) {
    const int kk = 16 * w + i;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (kk < a.K && 16 * t + 4 * g + r < a.V) a.g_s0[(bh * a.K + kk) * a.V + 16 * t + 4 * g + r] = R[t][r];
  }
}

// What is summed over workgroups: a group's heads, into the type of q and k (the first 2 `blocks` workgroups, if heads share them), and,
// for fixed decays, sequences and segments, one wave for each head (the rest).
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(KfAttnArgs a, const float* part_q, const float* part_k, const double* part_decay, unsigned blocks, int segments) {
  if (blockIdx.x < 2 * blocks) {
    const long total = a.B * a.T * a.G * a.K;
    const bool second = blockIdx.x >= blocks;
    const float* part = second ? part_k : part_q;
    const int per = a.H / a.G;
    for (long i = (long)(blockIdx.x - (second ? blocks : 0)) * 256 + threadIdx.x; i < total; i += blocks * 256l) {
      const int c = (int)(i % a.K);
      const long row = i / a.K, bt = row / a.G;
      const int g = (int)(row - bt * a.G);
      float s = 0.f;
      for (int j = 0; j < per; ++j) s += part[(bt * a.H + g * per + j) * a.K + c];
      ((T*)(second ? a.g_k : a.g_q))[i] = kf_from_float<T>(s);
    }
  } else if (threadIdx.x < 64) {
    const int h = (int)(blockIdx.x - 2 * blocks);
    double s = 0.;
    for (long x = threadIdx.x; x < a.B * segments; x += 64) s += part_decay[((x / segments) * a.H + h) * segments + x % segments];
#pragma unroll
    for (int m = 1; m < 64; m *= 2) s += __shfl_xor(s, m);
    if (threadIdx.x == 0) a.g_decay[h] = (float)s;
  }
}

struct Plan {
  int D;
  int mode;
  Split sp;
  size_t adds, factors, products, starts, part, decay;
  size_t bytes() const { return 2 * adds + factors + 2 * products + starts + 2 * part + decay; }
};

Plan plan(const kf_handle* h, const KfAttnArgs& a) {
  Plan p;
  const int most = a.K > a.V ? a.K : a.V, C = a.dtype == KF_DTYPE_BF16 ? chunk_of<KfBf16>() : chunk_of<KfF32>();
  p.mode = kf_rows_mode(a.K, a.V);
  p.D = p.mode == KF_ROWS_NARROW ? 128 : most <= 32 ? 32 : most <= 64 ? 64 : 128;
  Split& s = p.sp;
  s.chunks = (a.T + C - 1) / C;
  const long rows = a.B * a.H, cu = h->n_cu > 0 ? h->n_cu : 256;
  // as many workgroups as the card holds at once (by LDS: one on each compute unit for D = 128, more for smaller ones), where there are
  // chunks for them (18 heads of 333 tokens in fp32: with at least 4 chunks in a segment 150 us, 2: 93, 1: 65)
  const long room = cu * (p.D == 128 ? 1 : p.D == 64 ? 2 : 4);
  long segs = (room + rows - 1) / rows;
  segs = segs > s.chunks ? s.chunks : segs;
  segs = segs < 1 ? 1 : segs;
  s.seg_chunks = (int)((s.chunks + segs - 1) / segs);
  s.segments = (int)((s.chunks + s.seg_chunks - 1) / s.seg_chunks);
  s.works = rows * s.segments;
  const size_t state = (size_t)p.D * p.D * 4;
  p.adds = kf_seq_round(rows * (s.segments - 1) * state);
  p.factors = kf_seq_round((size_t)rows * s.segments * 4);
  p.products = kf_seq_round((size_t)rows * (s.segments - 1) * 4);
  p.starts = kf_seq_round(s.seg_chunks > 1 ? (size_t)rows * s.chunks * state : (size_t)4 * p.D * 16);
  p.part = a.G != a.H ? kf_seq_round((size_t)a.B * a.T * a.H * a.K * 4) : 0;
  p.decay = a.per_token ? 0 : kf_seq_round((size_t)rows * s.segments * 8);
  return p;
}

template <typename A, typename T, int D, int MODE>
int launch(kf_handle* h, const KfAttnArgs& a, const Plan& p, hipStream_t stream) {
  constexpr int C = chunk_of<A>();
  constexpr size_t lds = sizeof(typename A::elem) * ((4 * C + D) * D + 2 * C * C) + 2 * sizeof(KfChunkDecay<C>) +
                         sizeof(float) * (2 * (C / 16) * C + 2 * (D / 16) * C + D / 16);
  static_assert(lds <= 160 * 1024, "LDS of one workgroup");
  const Split& s = p.sp;
  if (s.segments > 1) {
    Split two = s;
    two.works = 2 * (s.works / s.segments) * (s.segments - 1);
    hipLaunchKernelGGL((attention_sweep_kernel<A, T, D, MODE, false>), dim3(kf_xcd_grid(two.works)), dim3(4 * D), 0, stream, a, two);
    if (s.segments > KF_FUSED_SEGMENTS)
      kf_attention_scan(s.adds_s, s.adds_r, s.factors, s.products_s, s.products_r, a.B * a.H, s.segments - 1, (long)D * D, s.segments, 4 * D, a.V, a.K, stream);
  }
  // (segments of one chunk start from what the first launch left: 16 x 128 tokens, 8 heads of 64 x 64, fp16, 31 us with this launch,
  // 26 without; 3 x 333 tokens, fp32, 58 and 52)
  if (s.seg_chunks > 1) hipLaunchKernelGGL((attention_sweep_kernel<A, T, D, MODE, true>), dim3(kf_xcd_grid(s.works)), dim3(4 * D), 0, stream, a, s);
  KF_HIP_CHECK(h, hipFuncSetAttribute(reinterpret_cast<const void*>(attention_gradient_kernel<A, T, D, MODE>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL((attention_gradient_kernel<A, T, D, MODE>), dim3(kf_xcd_grid(s.works)), dim3(4 * D), lds, stream, a, s);
  const long cells = (a.B * a.T * a.G * a.K + 255) / 256;
  const unsigned blocks = a.G == a.H ? 0 : (unsigned)(cells < 1 << 20 ? cells : 1 << 20), heads = a.per_token ? 0 : (unsigned)a.H;
  if (blocks || heads)
    hipLaunchKernelGGL(attention_join_kernel<T>, dim3(2 * blocks + heads), dim3(256), 0, stream, a, s.part_q, s.part_k, s.part_decay, blocks, s.segments);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

template <typename A, typename T, int MODE>
int launch_m(kf_handle* h, const KfAttnArgs& a, const Plan& p, hipStream_t stream) {
  switch (p.D) {
    case 32: return launch<A, T, 32, MODE>(h, a, p, stream);
    case 64: return launch<A, T, 64, MODE>(h, a, p, stream);
    default: return launch<A, T, 128, MODE>(h, a, p, stream);
  }
}

template <typename A, typename T>
int launch_d(kf_handle* h, const KfAttnArgs& a, const Plan& p, hipStream_t stream) {
  if (p.mode == KF_ROWS_NARROW) return launch<A, T, 128, KF_ROWS_NARROW>(h, a, p, stream);
  if (p.mode == KF_ROWS_CUT) return launch_m<A, T, KF_ROWS_CUT>(h, a, p, stream);
  return launch_m<A, T, KF_ROWS_WHOLE>(h, a, p, stream);
}

}  // namespace

size_t kf_attention_backward_workspace(const kf_handle* h, const KfAttnArgs& a) { return plan(h, a).bytes(); }

int kf_launch_attention_backward(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream) {
  Plan p = plan(h, a);
  Split& s = p.sp;
  char* w = (char*)ws;
  s.adds_s = (float*)w; w += p.adds;
  s.adds_r = (float*)w; w += p.adds;
  s.factors = (float*)w; w += p.factors;
  s.products_s = (float*)w; w += p.products;
  s.products_r = (float*)w; w += p.products;
  s.starts = (kf_f32x4*)w; w += p.starts;
  s.part_q = (float*)w; w += p.part;
  s.part_k = (float*)w; w += p.part;
  s.part_decay = (double*)w;
  switch (a.dtype) {
    case KF_DTYPE_F32: return launch_d<KfF32, float>(h, a, p, stream);
    case KF_DTYPE_F16: return launch_d<KfF32, __half>(h, a, p, stream);
    default: return launch_d<KfBf16, __hip_bfloat16>(h, a, p, stream);
  }
}
