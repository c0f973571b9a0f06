// kf_attention.hip -- linear attention with a decay for each head, one token at a time:
//     S_t = a_t S_{t-1} + k_t v_t',   o_t = s S_t' q_t,   a_t = exp(log_decay_t)
// and its gradient.  With R_t = dL/dS_t:  R_t = s q_t do_t' + a_{t+1} R_{t+1},  dq_t = s S_t do_t,  dk_t = R_t v_t,
// dv_t = R_t' k_t,  d log a_t = <R_t, a_t S_{t-1}> = (sum over later tokens of q.dq - k.dk, this token included) + <dS_T, S_T>.
#include "kf_sequence.h"

namespace {

constexpr int MAXD = 128;  // the largest K and V

// MODE 0: dq, forward in time, a thread per row of S.  MODE 1: dk and dS_0, backward, a thread per row of R.
// MODE 2: dv, backward, a thread per column of R.  dq, dk per head in 32 bits (summed over a group's heads afterwards).
template <typename T, int MODE>
__global__ __launch_bounds__(MAXD) void attention_backward_kernel(KfAttnArgs a, float* part, float* tail) {
  __shared__ float s1[MAXD], s2[MAXD];
  __shared__ float red[MAXD];
  const long bh = blockIdx.x;
  const long b = bh / a.H;
  const int h = (int)(bh - b * a.H), g = h / (a.H / a.G);
  const int c = threadIdx.x;
  const int D = MODE == 2 ? a.V : a.K, E = MODE == 2 ? a.K : a.V;  // rows of threads, registers of each
  const long n = kf_row_length(a.lengths, b, a.T);
  const T* q = (const T*)a.q + b * a.qs[0] + g * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + g * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + h * a.vs[2];
  const T* go = (const T*)a.g_o + b * a.gs[0] + h * a.gs[2];
  const float* init = MODE == 0 ? a.s0 : a.g_sT;
  float S[MAXD];
#pragma unroll
  for (int i = 0; i < MAXD; ++i) {
    const long at = MODE == 2 ? (bh * a.K + i) * a.V + c : (bh * a.K + c) * a.V + i;
    S[i] = (init && c < D && i < E) ? init[at] : 0.f;
  }
  if (MODE == 0) {
    // <dS_T, S_T> needs the last state: added below, after the loop
  }
  for (long step = 0; step < a.T; ++step) {
    const long t = MODE == 0 ? step : a.T - 1 - step;
    const long row = (b * a.T + t) * a.H + h;
    if (t >= n) {
      if (c < D) {
        if (MODE == 2) ((T*)a.g_v)[row * a.V + c] = kf_from_float<T>(0.f);
        else part[row * a.K + c] = 0.f;
      }
      continue;
    }
    const float d = expf(kf_clamp_log_decay(a.per_token ? a.log_decay[row] : a.log_decay[h]));
    __syncthreads();
    // what a thread multiplies its own scalar with: v / do over V (modes 0, 1), q / k over K (mode 2)
    if (MODE == 2) {
      s1[c] = c < a.K ? kf_to_float(q[t * a.qs[1] + c]) : 0.f;
      s2[c] = c < a.K ? kf_to_float(k[t * a.ks[1] + c]) : 0.f;
    } else {
      s1[c] = c < a.V ? kf_to_float(v[t * a.vs[1] + c]) : 0.f;
      s2[c] = c < a.V ? kf_to_float(go[t * a.gs[1] + c]) : 0.f;
    }
    __syncthreads();
    float own, r = 0.f;
    if (MODE == 0) {
      own = c < D ? kf_to_float(k[t * a.ks[1] + c]) : 0.f;
#pragma unroll
      for (int i = 0; i < MAXD; ++i) {
        S[i] = d * S[i] + own * s1[i];
        r += S[i] * s2[i];
      }
      if (c < D) part[row * a.K + c] = a.scale * r;
    } else if (MODE == 1) {
      own = a.scale * (c < D ? kf_to_float(q[t * a.qs[1] + c]) : 0.f);
#pragma unroll
      for (int i = 0; i < MAXD; ++i) {
        S[i] += own * s2[i];
        r += S[i] * s1[i];
        S[i] *= d;
      }
      if (c < D) part[row * a.K + c] = r;
    } else {
      own = a.scale * (c < D ? kf_to_float(go[t * a.gs[1] + c]) : 0.f);
#pragma unroll
      for (int i = 0; i < MAXD; ++i) {
        S[i] += own * s1[i];
        r += S[i] * s2[i];
        S[i] *= d;
      }
      if (c < D) ((T*)a.g_v)[row * a.V + c] = kf_from_float<T>(r);
    }
  }
  if (MODE == 1 && a.g_s0 && c < D) {
#pragma unroll
    for (int i = 0; i < MAXD; ++i)
      if (i < E) a.g_s0[(bh * a.K + c) * a.V + i] = S[i];
  }
  if (MODE == 0) {
    float r = 0.f;
    if (a.g_sT && c < D) {
#pragma unroll
      for (int i = 0; i < MAXD; ++i)
        if (i < E) r += S[i] * a.g_sT[(bh * a.K + c) * a.V + i];
    }
    red[c] = r;
    __syncthreads();
    if (c == 0) {
      double s = 0.;
      for (int i = 0; i < MAXD; ++i) s += red[i];
      tail[bh] = (float)s;
    }
  }
}

// sums a group's heads into the type of q / k
template <typename T>
__global__ __launch_bounds__(256) void attention_group_kernel(KfAttnArgs a, const float* part, T* out) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long total = a.B * a.T * a.G * a.K;
  if (i >= total) return;
  const int c = (int)(i % a.K);
  const long row = i / a.K, bt = row / a.G;
  const int g = (int)(row - bt * a.G), per = a.H / a.G;
  float s = 0.f;
  for (int j = 0; j < per; ++j) s += part[(bt * a.H + g * per + j) * a.K + c];
  out[i] = kf_from_float<T>(s);
}

template <typename T>
__global__ __launch_bounds__(64) void attention_decay_kernel(KfAttnArgs a, const float* pq, const float* pk, const float* tail, float* out) {
  const long bh = blockIdx.x;
  const long b = bh / a.H;
  const int h = (int)(bh - b * a.H), g = h / (a.H / a.G);
  const long n = kf_row_length(a.lengths, b, a.T);
  const T* q = (const T*)a.q + b * a.qs[0] + g * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + g * a.ks[2];
  double run = tail[bh], sum = 0.;
  for (long t = a.T - 1; t >= 0; --t) {
    const long row = (b * a.T + t) * a.H + h;
    if (t >= n) {
      if (a.per_token && threadIdx.x == 0) out[row] = 0.f;
      continue;
    }
    double r = 0.;
    for (int i = threadIdx.x; i < a.K; i += 64)
      r += (double)kf_to_float(q[t * a.qs[1] + i]) * pq[row * a.K + i] - (double)kf_to_float(k[t * a.ks[1] + i]) * pk[row * a.K + i];
    for (int m = 32; m; m >>= 1) r += __shfl_xor(r, m);
    run += r;
    sum += run;
    if (a.per_token && threadIdx.x == 0) out[row] = (float)run;
  }
  if (!a.per_token && threadIdx.x == 0) out[bh] = (float)sum;
}

__global__ __launch_bounds__(64) void attention_decay_sum_kernel(KfAttnArgs a, const float* part) {
  const int h = blockIdx.x;
  double s = 0.;
  for (long b = threadIdx.x; b < a.B; b += 64) s += part[b * a.H + h];
  for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m);
  if (threadIdx.x == 0) a.g_decay[h] = (float)s;
}

// one workgroup per (row, head, 64 columns of V).  Rows that name the same slot are one chain of tokens in the order of the
// rows: the first of them carries the state through all of them, the others have nothing to do.
template <typename T>
__global__ __launch_bounds__(64) void attention_step_kernel(KfAttnStepArgs a) {
  __shared__ float sq[MAXD], sk[MAXD];
  const long b0 = blockIdx.x / a.H;
  const int h = (int)(blockIdx.x - b0 * a.H), g = h / (a.H / a.G);
  const int c = blockIdx.y * 64 + threadIdx.x;
  const bool on = c < a.V;
  const long slot = a.slots ? a.slots[b0] : b0;
  T* o = (T*)a.o;
  if (slot < 0 || slot >= a.n_slots) {
    if (on) o[(b0 * a.H + h) * a.V + c] = kf_from_float<T>(0.f);
    if (a.info && h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.info[b0] = slot < 0 ? 0 : 1;
    return;
  }
  if (a.slots) {
    int before = 0;
    for (long b = threadIdx.x; b < b0; b += 64) before |= a.slots[b] == slot;
    if (__any(before)) return;
  }
  float S[MAXD];
  const long at = (slot * a.H + h) * (long)a.K * a.V;
#pragma unroll
  for (int i = 0; i < MAXD; ++i) S[i] = on && i < a.K ? a.state[at + (long)i * a.V + c] : 0.f;
  for (long b = b0; b < (a.slots ? a.B : b0 + 1); ++b) {
    if (b != b0 && a.slots[b] != slot) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < MAXD; i += 64) {
      sq[i] = i < a.K ? kf_to_float(((const T*)a.q)[b * a.qs[0] + g * a.qs[1] + i]) : 0.f;
      sk[i] = i < a.K ? kf_to_float(((const T*)a.k)[b * a.ks[0] + g * a.ks[1] + i]) : 0.f;
    }
    __syncthreads();
    const float d = expf(kf_clamp_log_decay(a.log_decay[a.per_row ? b * a.H + h : h]));
    const float vt = on ? kf_to_float(((const T*)a.v)[b * a.vs[0] + h * a.vs[1] + c]) : 0.f;
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < MAXD; ++i) {
      S[i] = d * S[i] + sk[i] * vt;
      r += sq[i] * S[i];
    }
    if (on) o[(b * a.H + h) * a.V + c] = kf_from_float<T>(a.scale * r);
    if (a.info && h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.info[b] = 0;
  }
#pragma unroll
  for (int i = 0; i < MAXD; ++i)
    if (on && i < a.K) a.state_out[at + (long)i * a.V + c] = S[i];
}

template <typename T>
int backward_t(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream) {
  const size_t rows = (size_t)a.B * a.T * a.H;
  char* w = (char*)ws;
  float* pq = (float*)w; w += kf_seq_round(rows * a.K * 4);
  float* pk = (float*)w; w += kf_seq_round(rows * a.K * 4);
  float* tail = (float*)w; w += kf_seq_round((size_t)a.B * a.H * 4);
  float* dsum = (float*)w;
  const unsigned bh = (unsigned)(a.B * a.H);
  hipLaunchKernelGGL((attention_backward_kernel<T, 0>), dim3(bh), dim3(MAXD), 0, stream, a, pq, tail);
  hipLaunchKernelGGL((attention_backward_kernel<T, 1>), dim3(bh), dim3(MAXD), 0, stream, a, pk, tail);
  hipLaunchKernelGGL((attention_backward_kernel<T, 2>), dim3(bh), dim3(MAXD), 0, stream, a, pk, tail);
  hipLaunchKernelGGL(attention_decay_kernel<T>, dim3(bh), dim3(64), 0, stream, a, pq, pk, tail, a.per_token ? a.g_decay : dsum);
  if (!a.per_token) hipLaunchKernelGGL(attention_decay_sum_kernel, dim3(a.H), dim3(64), 0, stream, a, dsum);
  const unsigned blocks = (unsigned)((a.B * a.T * a.G * a.K + 255) / 256);
  hipLaunchKernelGGL(attention_group_kernel<T>, dim3(blocks), dim3(256), 0, stream, a, pq, (T*)a.g_q);
  hipLaunchKernelGGL(attention_group_kernel<T>, dim3(blocks), dim3(256), 0, stream, a, pk, (T*)a.g_k);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

template <typename T>
int step_t(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(attention_step_kernel<T>, dim3((unsigned)(a.B * a.H), (a.V + 63) / 64), dim3(64), 0, stream, a);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

}  // namespace

size_t kf_attention_workspace(const kf_handle* h, const KfAttnArgs& a, bool backward) {
  if (!backward) return kf_attention_forward_workspace(h, a);
  const size_t rows = (size_t)a.B * a.T * a.H;
  return 2 * kf_seq_round(rows * a.K * 4) + 2 * kf_seq_round((size_t)a.B * a.H * 4);
}

int kf_launch_attention_backward(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream) {
  switch (a.dtype) {
    case KF_DTYPE_F32: return backward_t<float>(h, a, ws, stream);
    case KF_DTYPE_BF16: return backward_t<__hip_bfloat16>(h, a, ws, stream);
    default: return backward_t<__half>(h, a, ws, stream);
  }
}

int kf_launch_attention_step(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case KF_DTYPE_F32: return step_t<float>(h, a, stream);
    case KF_DTYPE_BF16: return step_t<__hip_bfloat16>(h, a, stream);
    default: return step_t<__half>(h, a, stream);
  }
}
