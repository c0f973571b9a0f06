// kf_sequence.h -- what the sequence operators (linear attention with decays, orthogonalised updates) share.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "kf_internal.h"

struct KfAttnArgs {
  long B, T;
  int G, H, K, V;
  int dtype, per_token;
  float scale;
  const void *q, *k, *v, *g_o;           // last axis contiguous, strides below (elements): batch, token (below 2^24), head
  long qs[3], ks[3], vs[3], gs[3];
  const float* log_decay;                // [B][T][H] (per_token) or [H]
  const float* s0;                       // [B][H][K][V] or NULL
  const int32_t* lengths;                // [B] or NULL
  void* o;                               // [B][T][H][V]
  float* sT;                             // [B][H][K][V] or NULL
  const float* g_sT;                     // [B][H][K][V] or NULL
  void *g_q, *g_k, *g_v;                 // contiguous, types of q, k, v
  float *g_decay, *g_s0;                 // shapes of log_decay, s0; NULL = not wanted
};

struct KfAttnStepArgs {
  long B, n_slots;
  int G, H, K, V;
  int dtype, per_row;                    // per_row: log_decay is [B][H], else [H]
  float scale;
  const void *q, *k, *v;
  long qs[2], ks[2], vs[2];              // batch, head
  const float* log_decay;
  const int32_t* slots;                  // [B] or NULL (row b has slot b)
  const float* state;                    // [n_slots][H][K][V]
  float* state_out;                      // the same shape; may be `state`
  void* o;                               // [B][H][V]
  int32_t* info;                         // [B] or NULL
};

size_t kf_attention_forward_workspace(const kf_handle* h, const KfAttnArgs& a);
int kf_launch_attention(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream);
size_t kf_attention_backward_workspace(const kf_handle* h, const KfAttnArgs& a);
int kf_launch_attention_backward(kf_handle* h, const KfAttnArgs& a, void* ws, hipStream_t stream);
int kf_launch_attention_step(kf_handle* h, const KfAttnStepArgs& a, hipStream_t stream);

struct KfOrthArgs {
  long n;
  int rows, cols, dtype, steps;
  double coef[KF_ORTHOGONALISE_STEPS_MAX][3];
  double top[KF_ORTHOGONALISE_STEPS_MAX];  // no singular value is above this before step s
  double eps;
  const void* M;
  void* X;
};
bool kf_orthogonalise_on_chip(const KfOrthArgs& a);
size_t kf_orthogonalise_ws(const kf_handle* h, const KfOrthArgs& a);
int kf_launch_orthogonalise(kf_handle* h, const KfOrthArgs& a, void* ws, hipStream_t stream);

// A log decay below this is taken as this: exp(-1e4) is zero in every precision used, and sums over a chunk stay finite
// where -infinity (a reset of the state) would leave inf - inf.  A NaN passes through.
static __device__ __forceinline__ float kf_clamp_log_decay(float g) { return g < -1.0e4f ? -1.0e4f : g; }

static __device__ __forceinline__ float kf_to_float(float x) { return x; }
static __device__ __forceinline__ float kf_to_float(__half x) { return __half2float(x); }
static __device__ __forceinline__ float kf_to_float(__hip_bfloat16 x) { return __bfloat162float(x); }
template <typename T> static __device__ __forceinline__ T kf_from_float(float x);
template <> __device__ __forceinline__ float kf_from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half kf_from_float<__half>(float x) { return __float2half(x); }
template <> __device__ __forceinline__ __hip_bfloat16 kf_from_float<__hip_bfloat16>(float x) { return __float2bfloat16(x); }

static inline size_t kf_seq_round(size_t n) { return (n + 255) & ~(size_t)255; }

static __device__ __forceinline__ long kf_row_length(const int32_t* lengths, long b, long T) {
  if (!lengths) return T;
  const long n = lengths[b];
  return n < 0 ? 0 : n > T ? T : n;
}
