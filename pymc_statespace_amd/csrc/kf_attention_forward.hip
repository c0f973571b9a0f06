// kf_attention_forward.hip -- linear attention with a decay for each head over whole sequences, in chunks of 64 tokens:
//     o_i = s [ e^{G_i} S' q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j ],   S <- e^{G_63} S + sum_j e^{G_63 - G_j} k_j v_j'
// (S the state at the chunk's start).  One workgroup of four waves walks the chunks of one segment of one head with its K x VT part
// of the state in accumulator registers.  Where sequences and heads are too few to fill the card the time axis is cut into segments: a
// first launch computes what each segment adds to the state, and the second starts each segment from the sum of what came before it
// (k and v are then read twice; one segment reads every input once).
//
// Roundings (bf16 data; fp32 and fp16 data are multiplied in fp32): the state's copy that the queries meet and the scores times their
// decays, 2^-9 each, like o itself -- together 2.3e-3 of o where o's own rounding is 1.7e-3.  The state is exact to fp32's sums:
// weighted keys enter it in three parts (KfSplit).
//
// Measured: 4 x 2048 tokens, 16 heads of 128 x 128, bf16: 25 + 46 us for 139 MB (30 us at the 4.7 TB/s of a large copy).  32768 tokens, 32
// heads of 128 x 64: 88 + 7 + 153 us for 408 MB (87 us).  5 x 1000 ragged tokens, 6 heads of 72 x 56, fp32: 12 + 32 us.  The first case in
// fp16 205 us, in fp32 208 (eight fp32 instructions for one of bf16); its 16 heads as 4 x 4, by the 128-wide kernel with loads of single
// elements, 48 in bf16.  The first case's second launch takes 33 us of its 46 with its loads, stores and barriers alone; what the rest adds
// is issue: two waves on a SIMD (220 registers) spend 46 % of its cycles on vector instructions -- 290 of 670 for each chunk cut the
// weighted keys --, the matrix pipe is busy 23 %, LDS 18 %.  A third wave (168 registers) spills and gains nothing.
#include "kf_attention_chunk.h"

namespace {

// A: arithmetic (KfBf16, KfF32).  T: type of q, k, v, o.  KP, VT: K and this workgroup's columns of V, padded.  MODE: KF_ROWS_*.
// OUT false: only what the segment adds to the state.
//
// What a chunk needs from memory is asked for one chunk ahead, by loads that no branch surrounds (a load that may or may not have been
// issued makes every later wait one for all of them): at a segment's end they ask for the last chunk again.
template <typename A, typename T, int KP, int VT, int MODE, bool OUT>
__global__ __launch_bounds__(256, 2) void attention_chunk_kernel(KfAttnArgs a, KfAttnSplit sp, float* adds, float* factors, const float* products) {
  typedef typename A::elem E;
  typedef typename A::frag F;
  typedef KfRow<A, T, MODE> Row;
  typedef KfTile<A, KP> TK;  // k, and the state's transpose
  typedef KfTile<A, VT> TV;  // v, columns paired (kf_paired): so are the state's columns all through this kernel
  constexpr int NT = VT / 16, KK = KP / 32;
  constexpr int WK = KP / 16 < 4 ? KP / 16 : 4, WN = 4 / WK;  // the state's tiles: WK waves along K, WN along V
  constexpr int SM = KP / 16 / WK, SN = NT / WN;
  constexpr int RK = 2048 / KP, RV = 2048 / VT;
  constexpr int AT = sizeof(typename A::elem) == 2 ? 2 : 1;  // tiles at a time
  __shared__ __attribute__((aligned(16))) E sK[KF_CHUNK * KP];
  __shared__ __attribute__((aligned(16))) E sV[KF_CHUNK * VT];
  __shared__ __attribute__((aligned(16))) E sS[OUT ? VT * KP : 8];  // the state's transpose as an operand
  __shared__ __attribute__((aligned(16))) KfChunkDecay<KF_CHUNK> dec[2];

  const long work = kf_xcd_work(sp.works);
  if (work >= sp.works) return;
  const int segs = OUT ? sp.segments : sp.segments - 1;
  const int vt = (int)(work % sp.v_tiles);
  long rest = work / sp.v_tiles;
  const int h = (int)(rest % a.H);
  rest /= a.H;
  const int seg = (int)(rest % segs);
  const long b = rest / segs;
  const long bh = b * a.H + h;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 15, g = l >> 4;
  const KfLanes lk = TK::lanes(i, g), lv = TV::lanes(i, g);
  const int mt0 = (w % WK) * SM, nt0 = (w / WK) * SN;
  const int v0 = vt * VT, nv = a.V - v0;
  const long n = kf_row_length(a.lengths, b, a.T);
  const int grp = h / (a.H / a.G);
  const T* q = (const T*)a.q + b * a.qs[0] + grp * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + grp * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[2];
  const float* ld = a.log_decay + (a.per_token ? b * a.T * a.H + h : (long)h);
  const long ld_step = a.per_token ? a.H : 0;
  const long chunks = (a.T + KF_CHUNK - 1) / KF_CHUNK;
  const long c0 = (long)seg * sp.seg_chunks, c1 = c0 + sp.seg_chunks < chunks ? c0 + sp.seg_chunks : chunks;
  const long live = (n + KF_CHUNK - 1) / KF_CHUNK, end = c1 < live ? c1 : live;  // chunks with tokens: c0 .. end - 1

  kf_f32x4 S[SM][SN];
#pragma unroll
  for (int m = 0; m < SM; ++m)
#pragma unroll
    for (int t = 0; t < SN; ++t) {
      S[m][t] = kf_f32x4{0, 0, 0, 0};
      const int c = kf_paired((nt0 + t) * 16 + i);
      if (OUT && a.s0 && c < nv) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kk = (mt0 + m) * 16 + 4 * g + r;
          if (kk < a.K) S[m][t][r] = a.s0[(bh * a.K + kk) * a.V + v0 + c];
        }
      }
    }
  // what the segments before this one add, each decayed through those behind it
  const long cell = (bh * (sp.segments - 1)) * sp.v_tiles;
  if (OUT) {
    // (many segments: already summed up, with the products of the decays)
    const bool summed = sp.segments > KF_FUSED_SEGMENTS;
    for (int s = summed && seg ? seg - 1 : 0; s < seg; ++s) {
      const float root = (summed ? products : factors)[bh * (sp.segments - 1) + s];
      float f = root * root;  // (5 x 1000 tokens: 42.5 us, 43.3 with both multiplications each time)
      if (kf_too_large(f)) {
#pragma unroll
        for (int m = 0; m < SM; ++m)
#pragma unroll
          for (int t = 0; t < SN; ++t) S[m][t] *= root;
        f = root;
      }
      const kf_f32x4* u = reinterpret_cast<const kf_f32x4*>(adds) + (cell + (long)s * sp.v_tiles + vt) * (KP * VT / 4) + tid;
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int t = 0; t < SN; ++t) S[m][t] = S[m][t] * f + u[(m * SN + t) * 256];
    }
  }
  float through = 1.f;  // the root of the segment's decay

  typename Row::Raw rk[KK], rv[VT / 32], rq[KK];  // the next chunk's, as loaded
  float rg = 0.f;                                  // and the log decay of one token of the chunk behind it
  // this lane's part of a chunk: rows kr + u RK of k, vr + u RV of v, row 16 w + i of q
  const int kr = tid / (KP / 8), kc = 8 * (tid % (KP / 8)), vr = tid / (VT / 8), vc = 8 * (tid % (VT / 8));
  auto last_row = [&](long c) { return (int)(n - c * KF_CHUNK < KF_CHUNK ? n - c * KF_CHUNK : KF_CHUNK) - 1; };
  const unsigned kst = (unsigned)a.ks[1], vst = (unsigned)a.vs[1], qst = (unsigned)a.qs[1];
  auto off = [](int r, int last, unsigned stride) { return (unsigned)__umul24((unsigned)(r < last ? r : last), stride); };
  auto load = [&](long c) {
    const int last = last_row(c);
    const T *pk = k + c * KF_CHUNK * a.ks[1], *pv = v + c * KF_CHUNK * a.vs[1];
#pragma unroll
    for (int u = 0; u < KK; ++u) rk[u] = Row::raw(pk, off(kr + u * RK, last, kst), kc, a.K);
#pragma unroll
    for (int u = 0; u < VT / 32; ++u) rv[u] = Row::raw(pv, off(vr + u * RV, last, vst), v0 + vc, a.V);
  };
  auto load_q = [&](long c) {
    const T* pq = q + c * KF_CHUNK * a.qs[1];
    const unsigned r = off(16 * w + i, last_row(c), qst);
#pragma unroll
    for (int u = 0; u < KK; ++u) rq[u] = Row::raw(pq, r, 32 * u + 8 * g, a.K);
  };
  // full chunks without padded columns need no zeros
  const bool whole = MODE == KF_ROWS_WHOLE && a.K == KP && nv >= VT;
  auto put = [&](int last, auto plain) {
    constexpr bool P = decltype(plain)::value;
#pragma unroll
    for (int u = 0; u < KK; ++u) TK::put8(sK, kr + u * RK, kc, Row::template finish<P>(rk[u], kc, a.K, kr + u * RK <= last));
#pragma unroll
    for (int u = 0; u < VT / 32; ++u) TV::put8_paired(sV, vr + u * RV, vc, Row::template finish<P>(rv[u], v0 + vc, a.V, vr + u * RV <= last));
  };
  auto log_decay = [&](long c) { return ld[(c * KF_CHUNK + l < n ? c * KF_CHUNK + l : n - 1) * ld_step]; };
  auto put_state = [&]() {
#pragma unroll
    for (int m = 0; m < SM; ++m)
#pragma unroll
      for (int t = 0; t < SN; ++t) TK::put4(sS, lk, (nt0 + t) * 16, (mt0 + m) * 16, S[m][t]);
  };

  if (c0 < end) {
    const float first = log_decay(c0);
    rg = log_decay(c0 + 1);
    load(c0);
    if (OUT) load_q(c0);
    if (w == 0) dec[c0 & 1].template fill<!OUT>(first, c0 * KF_CHUNK + l < n);
    if (OUT) put_state();
  }
  for (long c = c0; c < end; ++c) {
    const long t0 = c * KF_CHUNK, next = c + 1 < end ? c + 1 : c;
    const int last = last_row(c);  // rows behind it are zero
    const bool plain = whole && last == KF_CHUNK - 1;
    if (plain) put(last, std::true_type{});
    else put(last, std::false_type{});
    __syncthreads();
    const float g1 = rg;
    rg = log_decay(c + 2);
    load(next);
    if (w == (int)(c & 3)) dec[(c + 1) & 1].template fill<!OUT>(g1, (c + 1) * KF_CHUNK + l < n);
    const KfChunkDecay<KF_CHUNK>& D = dec[c & 1];

    if (OUT) {
      const int row = 16 * w + i;
      F fq[KK];
      if (plain) {
#pragma unroll
        for (int u = 0; u < KK; ++u) fq[u] = Row::template finish<true>(rq[u], 0, 0, true);
      } else {
#pragma unroll
        for (int u = 0; u < KK; ++u) fq[u] = Row::finish(rq[u], 32 * u + 8 * g, a.K, row <= last);
      }
      // scores, transposed: rows j, columns i; as operands, two tiles each.  (w is the same for a whole wave.)  Here and below all of a
      // tile's (bf16: two tiles') operands are asked for before its first product: by itself the compiler asks for one at a time.
      F p[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        kf_f32x4 two[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int y0 = 0; y0 < 2; y0 += AT)
          if (2 * x + y0 <= w) {
            F fk[AT][KK];
#pragma unroll
            for (int y = 0; y < AT; ++y)
#pragma unroll
              for (int u = 0; u < KK; ++u) fk[y][u] = TK::row(sK, lk, 16 * (2 * x + y0 + y), 32 * u);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < KK; ++u)
#pragma unroll
              for (int y = 0; y < AT; ++y) two[y0 + y] = A::mma(fk[y][u], fq[u], two[y0 + y]);
          }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int jt = 2 * x + y;
          kf_f32x4 s = {0, 0, 0, 0};
          if (jt <= w) {
            s = two[y];
            if (jt < w) {
              s *= D.from_tile[jt < 3 ? jt : 2][row] * a.scale;
              s *= *reinterpret_cast<const kf_f32x4*>(&D.to_tile_end[16 * jt + 4 * g]);
            } else {
              s *= D.pairs(row, 16 * jt + 4 * g) * a.scale;
#pragma unroll
              for (int r = 0; r < 4; ++r) s[r] = 4 * g + r <= i ? s[r] : 0.f;
            }
          }
          two[y] = s;
        }
        p[x] = A::from(two[0], two[1]);
      }
      const float fs = D.from_start[row] * a.scale;
      const long t = t0 + row;
      T* out = (T*)a.o + ((b * a.T + t) * a.H + h) * (long)a.V + v0;
      // columns 16 u .. 16 u + 31 of V as two tiles, of which a lane has 8 neighbours: 16 u + 8 g .. + 7
      KfOut8<T> ready[NT / 2];
      float check = 0.f;
#pragma unroll
      for (int u = 0; u < NT; u += 2) {
        kf_f32x4 o[2];
#pragma unroll
        for (int y0 = 0; y0 < 2; y0 += AT) {
          F fS[AT][KK], fv[AT][2];
          kf_f32x4 before[AT] = {}, inside[AT] = {};
#pragma unroll
          for (int y = 0; y < AT; ++y) {
#pragma unroll
            for (int x = 0; x < KK; ++x) fS[y][x] = TK::row(sS, lk, 16 * (u + y0 + y), 32 * x);
#pragma unroll
            for (int x = 0; x < 2; ++x) fv[y][x] = TV::col(sV, lv, 32 * x, 16 * (u + y0 + y));
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int x = 0; x < KK; ++x)
#pragma unroll
            for (int y = 0; y < AT; ++y) before[y] = A::mma(fS[y][x], fq[x], before[y]);
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < AT; ++y) inside[y] = A::mma(fv[y][x], p[x], inside[y]);
#pragma unroll
          for (int y = 0; y < AT; ++y) o[y0 + y] = before[y] * fs + inside[y];
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) check = fmaf(o[y][r], 0.f, check);
        if (!plain) {  // (a row behind the end has a query of zeros; the state may be infinite all the same)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            o[0][r] = t < n ? o[0][r] : 0.f;
            o[1][r] = t < n ? o[1][r] : 0.f;
          }
        }
        ready[u / 2].set(o[0], o[1]);
      }
      const bool strange = __any(check != 0.f);  // something is not finite
      if (strange) {
        // A token's infinity or NaN in v would reach the rows before it as 0 x inf: the products once more without such values, and
        // these added only to the rows from their token on.  (The same operations as above: rows that no such value reaches keep their bits.)
#pragma unroll 1
        for (int v1 = 0; v1 < VT; v1 += 16) {
          kf_f32x4 before = {0, 0, 0, 0}, inside = {0, 0, 0, 0};
#pragma unroll
          for (int x = 0; x < KK; ++x) before = A::mma(TK::row(sS, lk, v1, 32 * x), fq[x], before);
#pragma unroll
          for (int x = 0; x < 2; ++x) inside = A::mma(A::finite(TV::col(sV, lv, 32 * x, v1)), p[x], inside);
          kf_f32x4 o = before * fs + inside;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll 1
            for (int j = 0; j < 32; ++j) {  // token 32 x + j: value e = 4 (j / 16) + j % 4 of lane group (j % 16) / 4
              float pj = 0.f;
#pragma unroll
              for (int e = 0; e < 8; ++e) pj = e == 4 * (j >> 4) + (j & 3) ? A::value(p[x], e) : pj;
              pj = __shfl(pj, ((j & 15) >> 2) * 16 + i);
              if (32 * x + j <= row)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float z = A::get(sV + TV::at(32 * x + j, v1 + 4 * g + r));
                  if (!kf_finite(z)) o[r] += pj * z;
                }
            }
          }
          const int cv = kf_paired(v1 + 4 * g);
          if (t < n) kf_store4(out + cv, o, nv - cv);
        }
      }
      // (loads and stores are waited for in the order they were issued in: the next chunk's loads first)
      load_q(next);
      if (t < a.T && (!strange || t >= n)) {
#pragma unroll
        for (int u = 0; u < NT; u += 2) ready[u / 2].store(out + 16 * u + 8 * g, nv - 16 * u - 8 * g);
      }
    }

    // the state at the chunk's end
    const float fe = D.from_start[KF_CHUNK - 1];
    if (!OUT) through = kf_root_decay(through * D.root);
#pragma unroll
    for (int m = 0; m < SM; ++m)
#pragma unroll
      for (int t = 0; t < SN; ++t) S[m][t] *= fe;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const kf_f32x4 w0 = *reinterpret_cast<const kf_f32x4*>(&D.to_end[32 * x + 4 * g]), w1 = *reinterpret_cast<const kf_f32x4*>(&D.to_end[32 * x + 16 + 4 * g]);
      const float wt[8] = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]};
      F fv[SN];
#pragma unroll
      for (int t = 0; t < SN; ++t) fv[t] = TV::col(sV, lv, 32 * x, 16 * (nt0 + t));
#pragma unroll
      for (int m = 0; m < SM; ++m) {
        KfSplit<A> kw;
        kw.set(TK::col(sK, lk, 32 * x, 16 * (mt0 + m)), wt);
#pragma unroll
        for (int t = 0; t < SN; ++t) S[m][t] = kw.mma(fv[t], S[m][t]);
      }
    }
    __syncthreads();
    if (OUT) put_state();
  }
  if (OUT) {
    // rows behind the sequence's end, in chunks that hold none of it
    const int cols = nv < VT ? nv : VT;
    for (long x = (end > c0 ? end : c0) * KF_CHUNK + tid / VT; x < c1 * KF_CHUNK && x < a.T; x += 256 / VT)
      if (tid % VT < cols) ((T*)a.o)[((b * a.T + x) * a.H + h) * (long)a.V + v0 + tid % VT] = kf_from_float<T>(0.f);
    if (a.sT && seg == sp.segments - 1) {
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int t = 0; t < SN; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int kk = (mt0 + m) * 16 + 4 * g + r, cc = kf_paired((nt0 + t) * 16 + i);
            if (kk < a.K && cc < nv) a.sT[(bh * a.K + kk) * a.V + v0 + cc] = S[m][t][r];
          }
    }
  } else {
    kf_f32x4* u = reinterpret_cast<kf_f32x4*>(adds) + (cell + (long)seg * sp.v_tiles + vt) * (KP * VT / 4) + tid;
#pragma unroll
    for (int m = 0; m < SM; ++m)
#pragma unroll
      for (int t = 0; t < SN; ++t) u[(m * SN + t) * 256] = S[m][t];
    if (tid == 0 && vt == 0) factors[bh * (sp.segments - 1) + seg] = through;
  }
}

struct Plan {
  int KP, VT;
  int mode;
  KfAttnSplit sp;
  size_t adds, factors, bytes;
};

Plan plan(const kf_handle* h, const KfAttnArgs& a) {
  Plan p;
  p.mode = kf_rows_mode(a.K, a.V);
  const bool narrow = p.mode == KF_ROWS_NARROW;  // one kernel, of the largest K
  p.KP = narrow ? 128 : a.K <= 32 ? 32 : a.K <= 64 ? 64 : 128;
  // (128 columns at a time would take scores and weighted keys once for each head, but need all 256 registers and twice as many
  // segments: 4 x 2048 tokens, V = 128, 52 us instead of 48)
  p.VT = a.dtype == KF_DTYPE_BF16 && a.V > 32 && !narrow ? 64 : 32;
  KfAttnSplit& s = p.sp;
  s.v_tiles = (a.V + p.VT - 1) / p.VT;
  const long chunks = (a.T + KF_CHUNK - 1) / KF_CHUNK, rows = a.B * a.H * s.v_tiles;
  const long cu = h->n_cu > 0 ? h->n_cu : 256;
  // two workgroups for each compute unit, where there are chunks for them (5 x 1000 tokens in fp32, 60 tiles of heads: with at least 4
  // chunks in a segment 53 us, 2: 46 us)
  long segs = (2 * cu + rows - 1) / rows;
  segs = segs > chunks / 2 ? chunks / 2 : segs;
  segs = segs < 1 ? 1 : segs;
  s.seg_chunks = (int)((chunks + segs - 1) / segs);
  s.segments = (int)((chunks + s.seg_chunks - 1) / s.seg_chunks);
  s.works = rows * s.segments;
  p.adds = kf_seq_round((size_t)rows * (s.segments - 1) * p.KP * p.VT * 4);
  p.factors = kf_seq_round((size_t)a.B * a.H * (s.segments - 1) * 4);
  p.bytes = p.adds + 2 * p.factors;
  return p;
}

template <typename A, typename T, int KP, int VT, int MODE>
int launch(kf_handle* h, const KfAttnArgs& a, const Plan& p, void* ws, hipStream_t stream) {
  float* adds = (float*)ws;
  float* factors = (float*)((char*)ws + p.adds);
  float* products = (float*)((char*)factors + p.factors);
  if (p.sp.segments > 1) {
    KfAttnSplit s = p.sp;
    s.works = p.sp.works / p.sp.segments * (p.sp.segments - 1);
    hipLaunchKernelGGL((attention_chunk_kernel<A, T, KP, VT, MODE, false>), dim3(kf_xcd_grid(s.works)), dim3(256), 0, stream, a, s, adds, factors, products);
    if (s.segments > KF_FUSED_SEGMENTS)
      kf_attention_scan(adds, nullptr, factors, products, nullptr, a.B * a.H, s.segments - 1, (long)s.v_tiles * KP * VT, s.segments - 1, 0, 0, 0, stream);
  }
  hipLaunchKernelGGL((attention_chunk_kernel<A, T, KP, VT, MODE, true>), dim3(kf_xcd_grid(p.sp.works)), dim3(256), 0, stream, a, p.sp, adds, factors, products);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

template <typename A, typename T, int VT, int MODE>
int launch_k(kf_handle* h, const KfAttnArgs& a, const Plan& p, void* ws, hipStream_t stream) {
  switch (p.KP) {
    case 32: return launch<A, T, 32, VT, MODE>(h, a, p, ws, stream);
    case 64: return launch<A, T, 64, VT, MODE>(h, a, p, ws, stream);
    default: return launch<A, T, 128, VT, MODE>(h, a, p, ws, stream);
  }
}

template <typename A, typename T>
int launch_t(kf_handle* h, const KfAttnArgs& a, const Plan& p, void* ws, hipStream_t stream) {
  if (p.mode == KF_ROWS_NARROW) return launch<A, T, 128, 32, KF_ROWS_NARROW>(h, a, p, ws, stream);
  if constexpr (std::is_same<A, KfBf16>::value)
    if (p.VT == 64) return p.mode == KF_ROWS_CUT ? launch_k<A, T, 64, KF_ROWS_CUT>(h, a, p, ws, stream) : launch_k<A, T, 64, KF_ROWS_WHOLE>(h, a, p, ws, stream);
  return p.mode == KF_ROWS_CUT ? launch_k<A, T, 32, KF_ROWS_CUT>(h, a, p, ws, stream) : launch_k<A, T, 32, KF_ROWS_WHOLE>(h, a, p, ws, stream);
}

}  // namespace

size_t kf_attention_forward_workspace(const kf_handle* h, const KfAttnArgs& a) {
  const Plan p = plan(h, a);
  return p.sp.segments > 1 ? p.bytes : 0;
}

int kf_launch_attention(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream) {
  const Plan p = plan(h, a);
  switch (a.dtype) {
    case KF_DTYPE_F32: return launch_t<KfF32, float>(h, a, p, ws, stream);
    case KF_DTYPE_F16: return launch_t<KfF32, __half>(h, a, p, ws, stream);
    default: return launch_t<KfBf16, __hip_bfloat16>(h, a, p, ws, stream);
  }
}
