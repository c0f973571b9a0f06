// kf_orthogonalise.hip -- a batch of matrices moved towards their orthogonal factors by Newton-Schulz products:
//     X = M / (|M|_F + eps);   per step   A = X X',   X <- a X + (b A + c A A) X
// on the transpose where there are more rows than columns, so that A has the smaller side.
#include "kf_sequence.h"

namespace {

template <typename T> struct Acc { typedef float type; };
template <> struct Acc<double> { typedef double type; };
static __device__ __forceinline__ double to_acc(double x) { return x; }
static __device__ __forceinline__ float to_acc(float x) { return x; }
static __device__ __forceinline__ float to_acc(__half x) { return __half2float(x); }
static __device__ __forceinline__ float to_acc(__hip_bfloat16 x) { return __bfloat162float(x); }
template <typename T> static __device__ __forceinline__ T from_acc(typename Acc<T>::type x) { return kf_from_float<T>(x); }
template <> __device__ __forceinline__ double from_acc<double>(double x) { return x; }

// |M|_F^2 in 64 bits: one workgroup per matrix, the same order on every run
template <typename T>
__global__ __launch_bounds__(256) void orth_norm_kernel(const T* M, long size, double* sum) {
  __shared__ double red[256];
  const T* m = M + (long)blockIdx.x * size;
  double s = 0.;
  for (long i = threadIdx.x; i < size; i += 256) {
    const double x = (double)to_acc(m[i]);
    s += x * x;
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = 128; w; w >>= 1) {
    if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) sum[blockIdx.x] = red[0];
}

template <typename T>
__global__ __launch_bounds__(256) void orth_scale_kernel(const T* M, long n, int rows, int cols, double eps, const double* sum,
                                                         typename Acc<T>::type* X) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, size = (long)rows * cols;
  if (i >= n * size) return;
  const long z = i / size, e = i - z * size;
  const double f = 1.0 / (sqrt(sum[z]) + eps);
  const long to = rows > cols ? z * size + (e % cols) * rows + e / cols : i;
  X[to] = (typename Acc<T>::type)((double)to_acc(M[i]) * f);
}

template <typename T>
__global__ __launch_bounds__(256) void orth_store_kernel(const typename Acc<T>::type* X, long n, int rows, int cols, T* out) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, size = (long)rows * cols;
  if (i >= n * size) return;
  const long z = i / size, e = i - z * size;
  out[i] = from_acc<T>(X[rows > cols ? z * size + (e % cols) * rows + e / cols : i]);
}

// C (m x n) = alpha op(A B) + beta D, A (m x k) row-major, B (k x n) row-major or (NT) given as (n x k)
template <typename C, bool NT>
__global__ __launch_bounds__(256) void orth_product_kernel(int m, int n, int k, const C* A, const C* B, const C* D, C* out, C alpha, C beta) {
  __shared__ C sa[16][65], sb[16][65];
  const long z = blockIdx.z;
  A += z * m * (long)k;
  B += z * n * (long)k;
  D += z * m * (long)n;
  out += z * m * (long)n;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  C acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int kk = i & 15, r = i >> 4;
      sa[kk][r] = r0 + r < m && k0 + kk < k ? A[(long)(r0 + r) * k + k0 + kk] : C(0);
      if (NT) {
        sb[kk][r] = c0 + r < n && k0 + kk < k ? B[(long)(c0 + r) * k + k0 + kk] : C(0);
      } else {
        const int cc = i & 63, k2 = i >> 6;
        sb[k2][cc] = c0 + cc < n && k0 + k2 < k ? B[(long)(k0 + k2) * n + c0 + cc] : C(0);
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[kk][ty + 16 * i] * sb[kk][tx + 16 * j];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + ty + 16 * i, c = c0 + tx + 16 * j;
      if (r < m && c < n) out[(long)r * n + c] = alpha * acc[i][j] + (beta != C(0) ? beta * D[(long)r * n + c] : C(0));
    }
}

template <typename T>
int orth_t(kf_handle* h, const KfOrthArgs& a, void* ws, hipStream_t stream) {
  typedef typename Acc<T>::type C;
  const int d = a.rows < a.cols ? a.rows : a.cols, L = a.rows < a.cols ? a.cols : a.rows;
  const size_t big = kf_seq_round((size_t)a.n * d * L * sizeof(C)), small = kf_seq_round((size_t)a.n * d * d * sizeof(C));
  char* w = (char*)ws;
  double* sum = (double*)w; w += kf_seq_round((size_t)a.n * 8);
  C* X = (C*)w; w += big;
  C* Y = (C*)w; w += big;
  C* A = (C*)w; w += small;
  C* B = (C*)w;
  const long total = a.n * (long)d * L;
  const unsigned blocks = (unsigned)((total + 255) / 256);
  hipLaunchKernelGGL(orth_norm_kernel<T>, dim3((unsigned)a.n), dim3(256), 0, stream, (const T*)a.M, (long)d * L, sum);
  hipLaunchKernelGGL(orth_scale_kernel<T>, dim3(blocks), dim3(256), 0, stream, (const T*)a.M, a.n, a.rows, a.cols, a.eps, sum, X);
  const unsigned td = (d + 63) / 64, tl = (L + 63) / 64, z = (unsigned)a.n;
  for (int s = 0; s < a.steps; ++s) {
    const C ca = (C)a.coef[s][0], cb = (C)a.coef[s][1], cc = (C)a.coef[s][2];
    hipLaunchKernelGGL((orth_product_kernel<C, true>), dim3(td, td, z), dim3(256), 0, stream, d, d, L, X, X, A, A, C(1), C(0));
    hipLaunchKernelGGL((orth_product_kernel<C, true>), dim3(td, td, z), dim3(256), 0, stream, d, d, d, A, A, A, B, cc, cb);
    hipLaunchKernelGGL((orth_product_kernel<C, false>), dim3(tl, td, z), dim3(256), 0, stream, d, L, d, B, X, X, Y, C(1), ca);
    C* t = X; X = Y; Y = t;
  }
  hipLaunchKernelGGL(orth_store_kernel<T>, dim3(blocks), dim3(256), 0, stream, X, a.n, a.rows, a.cols, (T*)a.X);
  KF_HIP_CHECK(h, hipGetLastError());
  return KF_OK;
}

}  // namespace

size_t kf_orthogonalise_ws(const kf_handle*, const KfOrthArgs& a) {
  const size_t e = a.dtype == KF_DTYPE_F64 ? 8 : 4;
  const size_t d = a.rows < a.cols ? a.rows : a.cols, L = a.rows < a.cols ? a.cols : a.rows;
  return kf_seq_round((size_t)a.n * 8) + 2 * kf_seq_round((size_t)a.n * d * L * e) + 2 * kf_seq_round((size_t)a.n * d * d * e);
}

int kf_launch_orthogonalise(kf_handle* h, const KfOrthArgs& a, void* ws, hipStream_t stream) {
  switch (a.dtype) {
    case KF_DTYPE_F64: return orth_t<double>(h, a, ws, stream);
    case KF_DTYPE_F32: return orth_t<float>(h, a, ws, stream);
    case KF_DTYPE_BF16: return orth_t<__hip_bfloat16>(h, a, ws, stream);
    default: return orth_t<__half>(h, a, ws, stream);
  }
}
