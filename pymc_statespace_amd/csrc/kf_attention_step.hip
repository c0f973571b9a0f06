// kf_attention_step.hip -- linear attention with a decay for each head, one token of each sequence:
//     S <- exp(log_decay) S + k v',   o = s S' q
// Bound by reading and writing S.  One workgroup for each (row, head): a thread holds VEC neighbouring columns of every RP-th row of
// S, all of them loaded before the first is used, and the sums over the rows meet in LDS.  96 rows (10 % of them empty), 32 heads of
// 128 x 128: 78 us for 362 MB, 4.6 TB/s, the rate of a large copy.  One row, 8 heads of 64 x 64: 5 us, the latency of a launch and of the
// loads.  A row of S after the other, 4 bytes a lane: 178 us.  V that is no multiple of 4, or a state off its 16 bytes, takes 4 bytes a lane:
// V = 126 72 us, V = 128 62 (96 rows, none empty, the state in the caches), V = 33 48 us, V = 32 18.  All in fp32; only o is rounded.
#include "kf_sequence.h"

namespace {

constexpr int TH = 256, MAXD = 128;

template <int VEC> struct Vec { typedef float type __attribute__((ext_vector_type(VEC))); };
template <> struct Vec<1> { typedef float type; };

// LV: threads along a row of S, a power of two, LV VEC >= V.
template <typename T, int VEC, int LV>
__global__ __launch_bounds__(TH) void attention_step_kernel(KfAttnStepArgs a) {
  typedef typename Vec<VEC>::type W;
  constexpr int RP = TH / LV, PASSES = MAXD / RP > 0 ? MAXD / RP : 1;
  __shared__ float sq[MAXD], sk[MAXD];
  __shared__ __attribute__((aligned(16))) float red[TH / 64][LV * VEC];
  const long b0 = blockIdx.x / a.H;
  const int h = (int)(blockIdx.x - b0 * a.H), g = h / (a.H / a.G);
  const int tid = threadIdx.x, c = (tid % LV) * VEC, r0 = tid / LV;
  const bool on = c < a.V;
  const long slot = a.slots ? a.slots[b0] : b0;
  T* o = (T*)a.o;
  if (slot < 0 || slot >= a.n_slots) {
    for (int x = tid; x < a.V; x += TH) o[(b0 * a.H + h) * a.V + x] = kf_from_float<T>(0.f);
    if (a.info && h == 0 && tid == 0) a.info[b0] = slot < 0 ? 0 : 1;
    return;
  }
  const long at = ((slot * a.H + h) * a.K + r0) * (long)a.V + c;
  W S[PASSES];
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    S[u] = W(0.f);
    if (on && r0 + u * RP < a.K) S[u] = *reinterpret_cast<const W*>(a.state + at + (long)u * RP * a.V);
  }
  // Rows that name the same slot are one chain of tokens in the order of the rows: the first of them carries the state through all
  // of them, the others have nothing to do.
  bool chain = false;
  if (a.slots) {
    int seen = 0;
    for (long b = tid; b < a.B; b += TH)
      if (b != b0 && a.slots[b] == slot) seen |= b < b0 ? 1 : 2;
    if (__syncthreads_or(seen & 1)) return;
    chain = __syncthreads_or(seen & 2) != 0;
  }
  for (long b = b0; b < (chain ? a.B : b0 + 1); ++b) {
    if (b != b0 && a.slots[b] != slot) continue;
    __syncthreads();  // (the last token's sums are read)
    if (tid < 2 * MAXD) {
      const int x = tid & (MAXD - 1);
      const T* p = tid < MAXD ? (const T*)a.q + b * a.qs[0] + g * a.qs[1] : (const T*)a.k + b * a.ks[0] + g * a.ks[1];
      (tid < MAXD ? sq : sk)[x] = x < a.K ? kf_to_float(p[x]) : 0.f;
    }
    W vt = W(0.f);
    if (on) {
      const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[1] + c;
      if constexpr (VEC == 1) vt = kf_to_float(v[0]);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) vt[e] = kf_to_float(v[e]);
    }
    const float d = expf(kf_clamp_log_decay(a.log_decay[a.per_row ? b * a.H + h : h]));
    __syncthreads();
    W r = W(0.f);
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
      const int k = r0 + u * RP;
      if (k < a.K) {
        S[u] = S[u] * d + vt * sk[k];
        r += S[u] * sq[k];
      }
    }
    // rows of this wave, then of the workgroup's four
#pragma unroll
    for (int m = LV; m < 64; m *= 2) {
      if constexpr (VEC == 1) r += __shfl_xor(r, m);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[e] += __shfl_xor(r[e], m);
    }
    constexpr int SPAN = LV < 64 ? LV : 64;  // threads of a wave that hold different columns
    if ((tid & 63) < SPAN) *reinterpret_cast<W*>(&red[tid >> 6][c]) = r;
    __syncthreads();
    for (int x = tid; x < a.V; x += TH) {
      float s = 0.f;
      if constexpr (LV <= 64) {
#pragma unroll
        for (int w = 0; w < TH / 64; ++w) s += red[w][x];
      } else {  // a row of S spans several waves
        for (int w = x / VEC / 64; w < TH / 64; w += LV / 64) s += red[w][x];
      }
      o[(b * a.H + h) * a.V + x] = kf_from_float<T>(a.scale * s);
    }
    if (a.info && h == 0 && tid == 0) a.info[b] = 0;
  }
#pragma unroll
  for (int u = 0; u < PASSES; ++u)
    if (on && r0 + u * RP < a.K) *reinterpret_cast<W*>(a.state_out + at + (long)u * RP * a.V) = S[u];
}

template <typename T>
int launch(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.B * a.H));
  const bool vec = a.V % 4 == 0 && !((uintptr_t)a.state & 15) && !((uintptr_t)a.state_out & 15);
  const int n = vec ? a.V / 4 : a.V;
  if (vec) {
    if (n <= 8) hipLaunchKernelGGL((attention_step_kernel<T, 4, 8>), grid, dim3(TH), 0, stream, a);
    else if (n <= 16) hipLaunchKernelGGL((attention_step_kernel<T, 4, 16>), grid, dim3(TH), 0, stream, a);
    else hipLaunchKernelGGL((attention_step_kernel<T, 4, 32>), grid, dim3(TH), 0, stream, a);
  } else {
    if (n <= 32) hipLaunchKernelGGL((attention_step_kernel<T, 1, 32>), grid, dim3(TH), 0, stream, a);
    else hipLaunchKernelGGL((attention_step_kernel<T, 1, 128>), grid, dim3(TH), 0, stream, a);
  }
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

}  // namespace

int kf_launch_attention_step(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case KF_DTYPE_F32: return launch<float>(h, a, stream);
    case KF_DTYPE_BF16: return launch<__hip_bfloat16>(h, a, stream);
    default: return launch<__half>(h, a, stream);
  }
}
