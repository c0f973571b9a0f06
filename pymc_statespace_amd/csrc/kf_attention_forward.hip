// kf_attention_forward.hip -- linear attention with a decay for each head over whole sequences, in chunks of 64 tokens:
//     o_i = s [ e^{G_i} S' q_i + sum_{j <= i} e^{G_i - G_j} (q_i . k_j) v_j ],   S <- e^{G_63} S + sum_j e^{G_63 - G_j} k_j v_j'
// (S the state at the chunk's start).  One workgroup of four waves walks the chunks of one segment of one head with its K x VT part
// of the state in accumulator registers; every input is read once, o written once.  Where sequences and heads are too few to fill
// the card the time axis is cut into segments: a first launch computes what each segment adds to the state, and the second starts
// each segment from the sum of what came before it.
#include "kf_attention_chunk.h"

namespace {

// A: arithmetic (KfBf16, KfF32).  T: type of q, k, v, o.  KP, VT: K and this workgroup's columns of V, padded.
// OUT false: only what the segment adds to the state.
template <typename A, typename T, int KP, int VT, bool OUT>
__global__ __launch_bounds__(256, 2) void attention_chunk_kernel(KfAttnArgs a, KfAttnSplit sp, float* adds, float* factors) {
  typedef typename A::elem E;
  typedef typename A::frag F;
  constexpr int LK = KP + A::PAD, LV = VT + A::PAD, NT = VT / 16, KK = KP / 32;
  constexpr int WK = KP / 16 < 4 ? KP / 16 : 4, WN = 4 / WK;  // the state's tiles: WK waves along K, WN along V
  constexpr int SM = KP / 16 / WK, SN = NT / WN;
  __shared__ __attribute__((aligned(16))) E sK[KF_CHUNK * LK];
  __shared__ __attribute__((aligned(16))) E sV[KF_CHUNK * LV];
  __shared__ __attribute__((aligned(16))) E sS[OUT ? VT * LK : 8];  // the state's transpose as an operand
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
  const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, i = l & 15, g = l >> 4;
  const int mt0 = (w % WK) * SM, nt0 = (w / WK) * SN;
  const int v0 = vt * VT, nv = a.V - v0;
  const long n = kf_row_length(a.lengths, b, a.T);
  const int grp = h / (a.H / a.G);
  const T* q = (const T*)a.q + b * a.qs[0] + grp * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + grp * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[2] + v0;
  const float* ld = a.log_decay + (a.per_token ? b * a.T * a.H + h : (long)h);
  const long chunks = (a.T + KF_CHUNK - 1) / KF_CHUNK;
  const long c0 = (long)seg * sp.seg_chunks, c1 = c0 + sp.seg_chunks < chunks ? c0 + sp.seg_chunks : chunks;

  kf_f32x4 S[SM][SN];
#pragma unroll
  for (int m = 0; m < SM; ++m)
#pragma unroll
    for (int t = 0; t < SN; ++t) {
      S[m][t] = kf_f32x4{0, 0, 0, 0};
      const int c = (nt0 + t) * 16 + i;
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
    for (int s = 0; s < seg; ++s) {
      const float f = factors[bh * (sp.segments - 1) + s];
      const kf_f32x4* u = reinterpret_cast<const kf_f32x4*>(adds) + (cell + (long)s * sp.v_tiles + vt) * (KP * VT / 4) + tid;
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int t = 0; t < SN; ++t) S[m][t] = S[m][t] * f + u[(m * SN + t) * 256];
    }
  }
  bool have = OUT && (a.s0 || seg);  // the state may not be zero
  float through = 1.f;

  F rk[KK], rv[VT / 32], rq[KK];
  float rg = 0.f;
  auto load = [&](long c) {
    const long t0 = c * KF_CHUNK;
#pragma unroll
    for (int u = 0; u < KK; ++u) {
      const int x = tid + 256 * u, row = x / (KP / 8), col = 8 * (x % (KP / 8));
      rk[u] = KfLoad8<A, T>::load(k + (t0 + row) * a.ks[1] + col, t0 + row < n ? a.K - col : 0, sp.vec_k);
    }
#pragma unroll
    for (int u = 0; u < VT / 32; ++u) {
      const int x = tid + 256 * u, row = x / (VT / 8), col = 8 * (x % (VT / 8));
      rv[u] = KfLoad8<A, T>::load(v + (t0 + row) * a.vs[1] + col, t0 + row < n ? nv - col : 0, sp.vec_v);
    }
    if (OUT) {
      const long t = t0 + 16 * w + i;
#pragma unroll
      for (int u = 0; u < KK; ++u) rq[u] = KfLoad8<A, T>::load(q + t * a.qs[1] + 32 * u + 8 * g, t < n ? a.K - 32 * u - 8 * g : 0, sp.vec_q);
    }
  };
  auto load_decay = [&](long c) { return c * KF_CHUNK + l < n ? (a.per_token ? ld[(c * KF_CHUNK + l) * a.H] : ld[0]) : 0.f; };

  if (c0 * KF_CHUNK < n) {
    load(c0);
    if (w == (int)(c0 & 3)) dec[c0 & 1].fill(load_decay(c0), c0 * KF_CHUNK + l < n);
  }
  if (OUT && have) {
#pragma unroll
    for (int m = 0; m < SM; ++m)
#pragma unroll
      for (int t = 0; t < SN; ++t) A::put4(sS + ((nt0 + t) * 16 + i) * LK + (mt0 + m) * 16 + 4 * g, S[m][t]);
  }
  long c = c0;
  for (; c < c1 && c * KF_CHUNK < n; ++c) {
    const long t0 = c * KF_CHUNK;
#pragma unroll
    for (int u = 0; u < KK; ++u) {
      const int x = tid + 256 * u;
      A::put8(sK + (x / (KP / 8)) * LK + 8 * (x % (KP / 8)), rk[u]);
    }
#pragma unroll
    for (int u = 0; u < VT / 32; ++u) {
      const int x = tid + 256 * u;
      A::put8(sV + (x / (VT / 8)) * LV + 8 * (x % (VT / 8)), rv[u]);
    }
    F fq[KK];
#pragma unroll
    for (int u = 0; u < KK; ++u) fq[u] = rq[u];
    __syncthreads();
    const bool more = c + 1 < c1 && (c + 1) * KF_CHUNK < n;
    if (more) {
      load(c + 1);
      if (w == (int)((c + 1) & 3)) rg = load_decay(c + 1);
    }
    const KfChunkDecay<KF_CHUNK>& D = dec[c & 1];

    if (OUT) {
      const int row = 16 * w + i;
      // scores, transposed: rows j, columns i
      kf_f32x4 p[4];
#pragma unroll
      for (int jt = 0; jt < 4; ++jt) {
        p[jt] = kf_f32x4{0, 0, 0, 0};
        if (jt <= w) {
          kf_f32x4 s = {0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < KK; ++u) s = A::mma(A::row(sK + (16 * jt + i) * LK + 32 * u + 8 * g), fq[u], s);
          if (jt < w) {
            const float f = D.from_tile[jt < 3 ? jt : 2][row] * a.scale;
            const kf_f32x4 e = *reinterpret_cast<const kf_f32x4*>(&D.to_tile_end[16 * jt + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) p[jt][r] = s[r] * (f * e[r]);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) p[jt][r] = 4 * g + r <= i ? s[r] * (D.pair(row, 16 * jt + 4 * g + r) * a.scale) : 0.f;
          }
        }
      }
      const float fs = D.from_start[row] * a.scale;
      auto from_state = [&](int t) {
        kf_f32x4 o = {0, 0, 0, 0};
        if (have) {
#pragma unroll
          for (int u = 0; u < KK; ++u) o = A::mma(A::row(sS + (16 * t + i) * LK + 32 * u + 8 * g), fq[u], o);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] *= fs;
        }
        return o;
      };
      kf_f32x4 o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] = from_state(t);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (2 * x <= w) {
          const F fp = A::from(p[2 * x], p[2 * x + 1]);
#pragma unroll
          for (int t = 0; t < NT; ++t) o[t] = A::mma(A::col(sV + 32 * x * LV + 16 * t, LV, i, g), fp, o[t]);
        }
      // A token's infinity or NaN in v would reach the rows before it as 0 x inf.  Where anything is not finite, the products are
      // taken again without such values, and these added only to the rows from their token on.
      float check = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) check = fmaf(o[t][r], 0.f, check);
      if (__any(check != 0.f)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          o[t] = from_state(t);
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (2 * x <= w) o[t] = A::mma(A::finite(A::col(sV + 32 * x * LV + 16 * t, LV, i, g)), A::from(p[2 * x], p[2 * x + 1]), o[t]);
#pragma unroll
          for (int jt = 0; jt < 4; ++jt)
            if (jt <= w)
#pragma unroll 1
              for (int j = 0; j < 16; ++j) {
                const float pj = __shfl((j & 3) == 0 ? p[jt][0] : (j & 3) == 1 ? p[jt][1] : (j & 3) == 2 ? p[jt][2] : p[jt][3], (j >> 2) * 16 + i);
                if (16 * jt + j <= row)
#pragma unroll
                  for (int r = 0; r < 4; ++r) {
                    const float x = A::get(sV + (16 * jt + j) * LV + 16 * t + 4 * g + r);
                    if (!(fabsf(x) <= 3.4e38f)) o[t][r] += pj * x;
                  }
              }
        }
      }
      const long t = t0 + row;
      if (t < a.T) {
        T* out = (T*)a.o + ((b * a.T + t) * a.H + h) * (long)a.V + v0;
#pragma unroll
        for (int u = 0; u < NT; ++u) kf_store4(out + 16 * u + 4 * g, t < n ? o[u] : kf_f32x4{0, 0, 0, 0}, nv - 16 * u - 4 * g, a.V % 4 == 0);
      }
    }

    // the state at the chunk's end (nobody needs the last one of a call that does not ask for it)
    const float fe = D.from_start[KF_CHUNK - 1];
    through *= fe;
#pragma unroll
    for (int m = 0; m < SM; ++m)
#pragma unroll
      for (int t = 0; t < SN; ++t) S[m][t] *= fe;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float wt[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) wt[e] = D.to_end[32 * x + 16 * (e >> 2) + 4 * g + (e & 3)];
      F fv[SN];
#pragma unroll
      for (int t = 0; t < SN; ++t) fv[t] = A::col(sV + 32 * x * LV + 16 * (nt0 + t), LV, i, g);
#pragma unroll
      for (int m = 0; m < SM; ++m) {
        KfWeighted<A> kw;
        kw.set(A::col(sK + 32 * x * LK + 16 * (mt0 + m), LK, i, g), wt);
#pragma unroll
        for (int t = 0; t < SN; ++t) S[m][t] = kw.mma(fv[t], S[m][t]);
      }
    }
    have = true;
    if (more && w == (int)((c + 1) & 3)) dec[(c + 1) & 1].fill(rg, (c + 1) * KF_CHUNK + l < n);
    __syncthreads();
    if (OUT && more) {
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int t = 0; t < SN; ++t) A::put4(sS + ((nt0 + t) * 16 + i) * LK + (mt0 + m) * 16 + 4 * g, S[m][t]);
    }
  }
  if (OUT) {
    // rows behind the sequence's end, in chunks that hold none of it
    const int cols = nv < VT ? nv : VT;
    for (long x = c * KF_CHUNK + tid / VT; x < c1 * KF_CHUNK && x < a.T; x += 256 / VT)
      if (tid % VT < cols) ((T*)a.o)[((b * a.T + x) * a.H + h) * (long)a.V + v0 + tid % VT] = kf_from_float<T>(0.f);
    if (a.sT && seg == sp.segments - 1) {
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int t = 0; t < SN; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int kk = (mt0 + m) * 16 + 4 * g + r, cc = (nt0 + t) * 16 + i;
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
  KfAttnSplit sp;
  size_t adds, bytes;
};

Plan plan(const kf_handle* h, const KfAttnArgs& a) {
  Plan p;
  p.KP = a.K <= 32 ? 32 : a.K <= 64 ? 64 : 128;
  p.VT = a.dtype == KF_DTYPE_BF16 && a.V > 32 ? 64 : 32;
  KfAttnSplit& s = p.sp;
  s.v_tiles = (a.V + p.VT - 1) / p.VT;
  const long chunks = (a.T + KF_CHUNK - 1) / KF_CHUNK, rows = a.B * a.H * s.v_tiles;
  const long cu = h->n_cu > 0 ? h->n_cu : 256;
  // two workgroups for each compute unit; no segment under 4 chunks, of which a segment costs the card about one more to combine
  long segs = (2 * cu + rows - 1) / rows;
  segs = segs > 32 ? 32 : segs;
  segs = segs > chunks / 4 ? chunks / 4 : segs;
  segs = segs < 1 ? 1 : segs;
  s.seg_chunks = (int)((chunks + segs - 1) / segs);
  s.segments = (int)((chunks + s.seg_chunks - 1) / s.seg_chunks);
  s.works = rows * s.segments;
  p.adds = kf_seq_round((size_t)rows * (s.segments - 1) * p.KP * p.VT * 4);
  p.bytes = p.adds + kf_seq_round((size_t)a.B * a.H * (s.segments - 1) * 4);
  return p;
}

template <typename A, typename T, int KP, int VT>
int launch(kf_handle* h, const KfAttnArgs& a, const Plan& p, void* ws, hipStream_t stream) {
  float* adds = (float*)ws;
  float* factors = (float*)((char*)ws + p.adds);
  if (p.sp.segments > 1) {
    KfAttnSplit s = p.sp;
    s.works = p.sp.works / p.sp.segments * (p.sp.segments - 1);
    hipLaunchKernelGGL((attention_chunk_kernel<A, T, KP, VT, false>), dim3(kf_xcd_grid(s.works)), dim3(256), 0, stream, a, s, adds, factors);
  }
  hipLaunchKernelGGL((attention_chunk_kernel<A, T, KP, VT, true>), dim3(kf_xcd_grid(p.sp.works)), dim3(256), 0, stream, a, p.sp, adds, factors);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

template <typename A, typename T, int VT>
int launch_k(kf_handle* h, const KfAttnArgs& a, const Plan& p, void* ws, hipStream_t stream) {
  switch (p.KP) {
    case 32: return launch<A, T, 32, VT>(h, a, p, ws, stream);
    case 64: return launch<A, T, 64, VT>(h, a, p, ws, stream);
    default: return launch<A, T, 128, VT>(h, a, p, ws, stream);
  }
}

}  // namespace

size_t kf_attention_forward_workspace(const kf_handle* h, const KfAttnArgs& a) {
  const Plan p = plan(h, a);
  return p.sp.segments > 1 ? p.bytes : 0;
}

int kf_launch_attention(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream) {
  Plan p = plan(h, a);
  const int e = a.dtype == KF_DTYPE_F32 ? 4 : 2;
  p.sp.vec_q = kf_rows_aligned(a.q, a.qs, 3, a.K, e);
  p.sp.vec_k = kf_rows_aligned(a.k, a.ks, 3, a.K, e);
  p.sp.vec_v = kf_rows_aligned(a.v, a.vs, 3, a.V, e);
  switch (a.dtype) {
    case KF_DTYPE_F32: return launch_k<KfF32, float, 32>(h, a, p, ws, stream);
    case KF_DTYPE_F16: return launch_k<KfF32, __half, 32>(h, a, p, ws, stream);
    default: return p.VT == 64 ? launch_k<KfBf16, __hip_bfloat16, 64>(h, a, p, ws, stream) : launch_k<KfBf16, __hip_bfloat16, 32>(h, a, p, ws, stream);
  }
}
