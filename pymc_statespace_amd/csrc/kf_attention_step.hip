// kf_attention_step.hip -- linear attention with a decay for each head, one token of each sequence:
//     S <- exp(log_decay) S + k v',   o = s S' q
#include "kf_sequence.h"

namespace {

constexpr int MAXD = 128;  // the largest K and V

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
int step_t(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(attention_step_kernel<T>, dim3((unsigned)(a.B * a.H), (a.V + 63) / 64), dim3(64), 0, stream, a);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

}  // namespace

int kf_launch_attention_step(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case KF_DTYPE_F32: return step_t<float>(h, a, stream);
    case KF_DTYPE_BF16: return step_t<__hip_bfloat16>(h, a, stream);
    default: return step_t<__half>(h, a, stream);
  }
}
